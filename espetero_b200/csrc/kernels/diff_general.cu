// Differential attention for every shape: any head dim the library has, any page size, tile height, group size, mask and pool type.
// The kernel the dispatcher falls back to, and the plain second implementation the tests hold the fast kernels against.
//
// One warp owns one (row, head): 32 keys per step, lane = key for the two scores (q1 . k1 and q2 . k2, halves of one K row, read
// once), two online softmaxes in the exp2 domain by warp shuffles, lane = HD / 32 dims for P_1 V and P_2 V, which share every V
// row they read. Sums are fp32 and the weights are not rounded. Bound by the CUDA cores' fp32 rate and by K rows read lane by lane:
// 2048 causal rows of 16 heads take 6.2 ms with 128 dims (diff_umma: 49 us) and 3.7 ms with 64; 32 tokens behind 4096 keys 3.3 ms (diff_decode:
// 85 us). Even for 16 rows without a cache (10.2 us against 10.1) or one key (10.4 against 10.2) it wins nothing, so it takes only what the
// others do not.
#include "diff.cuh"

namespace esp {
namespace {

constexpr int kWarps = 4;

template <int QDT>
__device__ __forceinline__ float dot8(const uint4& v, const float* q, float acc) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem16<QDT>::unpack2(w[i]);
    acc = fmaf(q[2 * i], f.x, acc);
    acc = fmaf(q[2 * i + 1], f.y, acc);
  }
  return acc;
}

template <int HD, int QDT, int KVDT>
__global__ void __launch_bounds__(kWarps * 32) diff_general_kernel(const DiffArgs a) {
  constexpr int DPL = HD / 32, MAP = HD / 2;
  using Q16 = Elem16<QDT>;
  __shared__ float qs[kWarps][HD];
  const KernelArgs& k = a.k;
  const esp_attn_params& p = k.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int kvh = blockIdx.x % p.Hkv;
  const esp_attn_tile tile = k.tiles[blockIdx.x / p.Hkv];
  const esp_attn_tree tree = k.trees[tile.tree];
  const int G = k.G;
  const int rows_live = min(k.tile_rows, tree.base + tree.M - tile.r0);
  const size_t blk = size_t(p.bt) * p.kv_ld;
  const float sl2 = k.scale * kLog2e;

  for (int pair = blockIdx.y * kWarps + warp; pair < rows_live * G; pair += kWarps * gridDim.y) {
    const int fm = pair / G, hg = pair % G, row = tile.r0 + fm, rr = row - tree.base, h = kvh * G + hg;
    __syncwarp();
    for (int d = lane; d < HD; d += 32) qs[warp][d] = Q16::to_f32(static_cast<const typename Q16::T*>(k.Q)[size_t(row) * p.q_ld + size_t(h) * HD + d]);
    __syncwarp();
    const float* q = qs[warp];

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, acc[2][DPL];
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[0][i] = acc[1][i] = 0.0f;

    // One step of 32 keys: s = this lane's two scores in exp2 units (-inf: not visible); v(jj, p1, p2) adds key jj's row.
    auto step = [&](const float (&s)[2], auto&& v) {
      float pr[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = s[c];
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float mn = fmaxf(m[c], top);
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float keep = fast_exp2(m[c] - ref);
        pr[c] = fast_exp2(s[c] - ref);
        float sum = pr[c];
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[c] = fmaf(l[c], keep, sum);
        m[c] = mn;
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[c][i] *= keep;
      }
      for (int jj = 0; jj < 32; ++jj) {
        const float p1 = __shfl_sync(0xffffffffu, pr[0], jj), p2 = __shfl_sync(0xffffffffu, pr[1], jj);
        if (p1 == 0.0f && p2 == 0.0f) continue;  // warp-uniform; keys that are not visible are never read
        v(jj, p1, p2);
      }
    };

    // Cached keys. The table's contents live on the device: an id outside the region is recorded and its keys are skipped.
    auto block_of = [&](int j, bool& ok) {
      const int b = k.blocks[tree.table + j / p.bt];
      ok = b >= 0 && b < k.n_blocks;
      if (!ok) atomicExch(k.status, kStatusBadBlock);
      return size_t(ok ? b : 0);
    };
    for (int j0 = tile.k0; j0 < tile.k1; j0 += 32) {
      const int j = j0 + lane;
      float s[2] = {-INFINITY, -INFINITY};
      bool ok = false;
      const size_t b = j < tile.k1 ? block_of(j, ok) : 0;
      if (ok) {
        const size_t at = p.kv_base + b * 2 * blk + size_t(j % p.bt) * p.kv_ld + size_t(kvh) * HD;
        float unit = sl2;
        if constexpr (KVDT == ESP_E4M3) unit *= k.kv_scales[b * 2 * p.Hkv + kvh];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float dot = 0.0f;
          if constexpr (KVDT == ESP_E4M3) {
            const uint8_t* src = static_cast<const uint8_t*>(k.kv) + at + c * MAP;
#pragma unroll 4
            for (int d = 0; d < MAP; d += 4) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(src + d);
              const uint32_t lo = e4m3x2_to_f16x2(uint16_t(w & 0xFFFFu)), hi = e4m3x2_to_f16x2(uint16_t(w >> 16));
              const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&lo)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              const float* qd = q + c * MAP + d;
              dot = fmaf(qd[0], f0.x, dot), dot = fmaf(qd[1], f0.y, dot), dot = fmaf(qd[2], f1.x, dot), dot = fmaf(qd[3], f1.y, dot);
            }
          } else {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(k.kv) + at + c * MAP);
#pragma unroll 4
            for (int d = 0; d < MAP / 8; ++d) dot = dot8<KVDT>(src[d], q + c * MAP + 8 * d, dot);
          }
          s[c] = dot * unit;
        }
      }
      step(s, [&](int jj, float p1, float p2) {
        bool v_ok;
        const size_t bv = block_of(j0 + jj, v_ok);
        const size_t at = p.kv_base + (bv * 2 + 1) * blk + size_t((j0 + jj) % p.bt) * p.kv_ld + size_t(kvh) * HD + lane * DPL;
        float unit = 1.0f;
        if constexpr (KVDT == ESP_E4M3) unit = k.kv_scales[(bv * 2 + 1) * p.Hkv + kvh];
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
          float x;
          if constexpr (KVDT == ESP_E4M3) x = e4m3_to_f32(static_cast<const uint8_t*>(k.kv)[at + i]) * unit;
          else x = Elem16<KVDT>::to_f32(static_cast<const typename Elem16<KVDT>::T*>(k.kv)[at + i]);
          acc[0][i] = fmaf(p1, x, acc[0][i]);
          acc[1][i] = fmaf(p2, x, acc[1][i]);
        }
      });
    }

    // The tree's own rows, under its mask.
    if (tile.last) {
      int4 d = make_int4(0, 0, 0, 0);
      uint64_t am = 0;
      int k_last;
      if (k.anc_mask) {
        am = k.anc_mask[row];
        k_last = min(tree.M, 64) - 1;
      } else {
        d = row_record(k, row, tree.M);
        k_last = min(tree.M - 1, max(rr, d.z - 1));
      }
      for (int j0 = 0; j0 <= k_last; j0 += 32) {
        const int j = j0 + lane;
        bool vis = j <= k_last;
        if (k.anc_mask) vis = vis && ((am >> j) & 1ull);
        else vis = vis && (j < d.z || (j >= d.x && j <= rr));
        float s[2] = {-INFINITY, -INFINITY};
        if (vis) {
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(k.Kb) + size_t(tree.base + j) * p.kv_ld + size_t(kvh) * HD);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float dot = 0.0f;
#pragma unroll 4
            for (int i = 0; i < MAP / 8; ++i) dot = dot8<QDT>(src[c * (MAP / 8) + i], q + c * MAP + 8 * i, dot);
            s[c] = dot * sl2;
          }
        }
        step(s, [&](int jj, float p1, float p2) {
          const typename Q16::T* src = static_cast<const typename Q16::T*>(k.Vb) + size_t(tree.base + j0 + jj) * p.kv_ld + size_t(kvh) * HD + lane * DPL;
#pragma unroll
          for (int i = 0; i < DPL; ++i) {
            const float x = Q16::to_f32(src[i]);
            acc[0][i] = fmaf(p1, x, acc[0][i]);
            acc[1][i] = fmaf(p2, x, acc[1][i]);
          }
        });
      }
    }

    if (tile.part >= 0) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* rec = k.parts + diff_record(k, tile.part, kvh, fm, hg, c);
#pragma unroll
        for (int i = 0; i < DPL; ++i) rec[lane * DPL + i] = acc[c][i];
        if (lane == 0) rec[HD] = m[c] * kLn2, rec[HD + 1] = l[c];
      }
      continue;
    }
    const float inv1 = l[0] > 0.0f ? 1.0f / l[0] : 0.0f, inv2 = l[1] > 0.0f ? diff_lam(a, row, h) / l[1] : 0.0f;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      acc[0][i] = acc[0][i] * inv1 - acc[1][i] * inv2;
      ss = fmaf(acc[0][i], acc[0][i], ss);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float f = diff_row_factor(a, ss, HD);
    typename Q16::T* op = static_cast<typename Q16::T*>(k.O) + size_t(row) * p.q_ld + size_t(h) * HD + lane * DPL;
#pragma unroll
    for (int i = 0; i < DPL; ++i) op[i] = Q16::from_f32(acc[0][i] * f * (a.norm_w ? a.norm_w[lane * DPL + i] : 1.0f));
  }
}

template <int HD, int QDT>
cudaError_t launch_typed(const DiffArgs& a, cudaStream_t stream) {
  // a tile's (row, head) pairs over several CTAs while the grid is small
  const int64_t ctas = int64_t(a.k.n_tiles) * a.k.p.Hkv;
  const int pairs = a.k.tile_rows * a.k.G;
  const dim3 grid(unsigned(ctas), unsigned(std::clamp<int64_t>(148 * 8 / ctas, 1, (pairs + kWarps - 1) / kWarps)));
  if (a.k.kv_dtype == ESP_E4M3) return launch_pdl(diff_general_kernel<HD, QDT, ESP_E4M3>, grid, dim3(kWarps * 32), 0, stream, a);
  return launch_pdl(diff_general_kernel<HD, QDT, QDT>, grid, dim3(kWarps * 32), 0, stream, a);
}

}  // namespace

cudaError_t launch_diff_general(const DiffArgs& a, cudaStream_t stream, uint64_t* launches) {
  if (a.k.n_tiles <= 0) return cudaSuccess;
  const bool f16 = a.k.q_dtype == ESP_F16;
  cudaError_t e = cudaErrorInvalidValue;
  switch (a.k.HD) {
    case 64: e = f16 ? launch_typed<64, ESP_F16>(a, stream) : launch_typed<64, ESP_BF16>(a, stream); break;
    case 128: e = f16 ? launch_typed<128, ESP_F16>(a, stream) : launch_typed<128, ESP_BF16>(a, stream); break;
    case 256: e = f16 ? launch_typed<256, ESP_F16>(a, stream) : launch_typed<256, ESP_BF16>(a, stream); break;
    case 512: e = f16 ? launch_typed<512, ESP_F16>(a, stream) : launch_typed<512, ESP_BF16>(a, stream); break;
  }
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
