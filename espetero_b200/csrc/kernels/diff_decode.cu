// Differential attention of single new tokens over the paged cache (sm_100a).
//
// One CTA per (kv head, tile): the tile's cached keys [k0, k1) of one sequence, plus the token's own key when tile.last.
// HBM-bound: every cached byte is read once, 2 Hkv HD elements per key, for 6 HD flops per query head.
//
// How the two maps share one stream of keys. A head's query is [q1 | q2], a key [k1 | k2]. With the block of 16 keys as the rows of
// S^T[16 keys x 8] = K . Q^T (mma.sync m16n8k16), the 8 columns are
//   G <= 4 (NT = 1): column c = map c / 4 of head c % 4, its query zero in the other map's dims: both maps of four heads for the
//                    instructions that eight plain heads cost, in the scores as in O^T[HD x 8] += V^T . P^T;
//   G <= 8 (NT = 2): one score tile per map, each over its own half of the dims (no more instructions than NT = 1), and two
//                    O^T tiles, which share every V fragment.
// V and K arrive by TMA (two bulk tensor loads per block, 128-byte swizzle, rows through the page table) in rings that belong to
// single warps, so nothing in the loop waits for another warp. Softmax in the exp2 domain over the key lanes; P^T re-enters as the
// B operand (movmatrix), rounded to 16 bits: what the MMA takes; sums and the rows' totals stay fp32 and unrounded. E4M3 codes
// are widened to fp16 in registers (exact), and bf16 queries scaled into its range, the K scale goes on the score, the power of
// two in the V scale on the weight and the rest on the block's P . V: the largest weight, 1, is exact.
// 32 sequences of 512 .. 32768 keys, H32 / Hkv4 / HD128, bf16: 92 us with the join = 5.7 TB/s, 0.87 of the copy peak; 131072 keys, Hkv8 / HD256, E4M3:
// 94 us = 5.7 TB/s. 16 x 8192 E4M3 keys of 128 dims: 72 us = 3.7 TB/s, bound by the widening's instructions.
// All waits are bounded; a CTA that gives up writes empty records and says so in the status word.
#include "diff.cuh"

namespace esp {
namespace {

template <int HD_, int KVDT_, int QDT_, int NT_, int NW_, int STAGES_, int CTAS_>
struct Cfg {
  static constexpr int HD = HD_, QDT = QDT_, NT = NT_, NW = NW_, STAGES = STAGES_, CTAS = CTAS_;
  static constexpr bool FP8 = KVDT_ == ESP_E4M3;
  static constexpr int CDT = FP8 ? ESP_F16 : KVDT_;   // MMA operand type
  static constexpr bool SCALED_Q = FP8 && QDT == ESP_BF16;  // queries beyond the operand type's range
  static constexpr int ROW_BYTES = HD * (FP8 ? 1 : 2);
  static constexpr int NCH = ROW_BYTES / 128;         // 128-byte lines per key
  static constexpr int TILE = 16 * ROW_BYTES;         // K or V of a block
  static constexpr int STAGE = 2 * TILE;
  static constexpr int WARP_BYTES = STAGES * STAGE;
  static constexpr int OLD = HD + 4;                  // row stride of the warps' results
  static constexpr int SMEM = NW * WARP_BYTES + 1024;
  static constexpr int NMT = HD / 16;
  static_assert((8 * NT * OLD + 16 * NT) * 4 <= WARP_BYTES, "a warp's result must fit its ring");
};

// Byte offset of (key, byte of the head's row) in a K or V tile: [line][16 keys][128 B], each group swizzled by TMA.
__device__ __forceinline__ uint32_t tile_off(uint32_t r, uint32_t b) { return (b >> 7) * 2048u + swz128(r, b & 127u); }

template <class C>
__global__ void __launch_bounds__(C::NW * 32, C::CTAS) diff_decode_kernel(const __grid_constant__ CUtensorMap pool_map, const DiffArgs d) {
  constexpr int HD = C::HD, NW = C::NW, STAGES = C::STAGES, NMT = C::NMT, OLD = C::OLD, NT = C::NT;
  using QE = Elem16<C::QDT>;
  using CE = Elem16<C::CDT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[NW][STAGES];
  __shared__ int gave_up;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const KernelArgs& a = d.k;
  const esp_attn_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.x % p.Hkv;
  // While the kernel before this one drains: L2 hints for each warp's first blocks, every index checked. A stale table costs a
  // wasted hint, never a result.
  if (lane < STAGES - 1 && a.n_trees > 0 && a.n_block_entries > 0 && a.blocks != nullptr) {
    const int4 t0 = __ldcg(reinterpret_cast<const int4*>(a.tiles + blockIdx.x / p.Hkv));  // tree, r0, k0, k1
    if (t0.x >= 0 && t0.x < a.n_trees) {
      const int4 tr = __ldcg(reinterpret_cast<const int4*>(a.trees + t0.x));  // base, P, table, M
      const int j0 = (t0.z & ~15) + 16 * (warp + lane * NW);
      const long long idx = (long long)tr.z + j0 / p.bt;
      if (t0.z >= 0 && j0 < t0.w && tr.z >= 0 && idx < a.n_block_entries) {
        const int b = __ldcg(a.blocks + idx);
        if (b >= 0 && b < a.n_blocks) {
          const int y = b * 2 * p.bt + j0 % p.bt;
          tma_prefetch_3d(&pool_map, 0, y, kvh * C::NCH);
          tma_prefetch_3d(&pool_map, 0, y + p.bt, kvh * C::NCH);
        }
      }
    }
  }
  pdl_wait();
  const esp_attn_tile tile = a.tiles[blockIdx.x / p.Hkv];
  const esp_attn_tree tree = a.trees[tile.tree];
  const int G = a.G, row = tile.r0;
  const float sl2 = a.scale * kLog2e;
  uint8_t* wsm = smem + size_t(warp) * C::WARP_BYTES;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&pool_map);
    gave_up = 0;
  }
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(&full_bar[warp][s], 1);
    mbar_fence_init();
  }
  __syncthreads();

  // ---- this warp's 16-key blocks: warp, warp + NW, ... of the tile (cut from the 16-aligned key below k0)
  const int kbase = tile.k0 & ~15;
  const int nblk = tile.k1 > tile.k0 ? (tile.k1 - kbase + 15) >> 4 : 0;
  const int n_it = nblk > warp ? (nblk - warp + NW - 1) / NW : 0;
  int iss_win = -32, iss_y = 0, use_win = -32;  // lane L of a window holds the table entry of iteration win + L
  float use_ks = 1.0f, use_vs = 1.0f;
  auto block_of_it = [&](int it, int& j0) {
    j0 = kbase + 16 * (warp + it * NW);
    int b = a.blocks[tree.table + j0 / p.bt];
    if (b < 0 || b >= a.n_blocks) {  // the table's contents live on the device: recorded, and a block that exists is read
      atomicExch(a.status, kStatusBadBlock);
      b = 0;
    }
    return b;
  };
  auto issue = [&](int it) {
    if (it - iss_win >= 32) {
      iss_win = it;
      if (it + lane < n_it) {
        int j0;
        const int b = block_of_it(it + lane, j0);
        iss_y = b * 2 * p.bt + j0 % p.bt;
      }
    }
    const int y = __shfl_sync(0xffffffffu, iss_y, it - iss_win);
    if (lane == 0) {
      const int slot = it % STAGES;
      uint8_t* dst = wsm + slot * C::STAGE;
      mbar_arrive_expect_tx(&full_bar[warp][slot], C::STAGE);
      tma_load_3d(dst, &pool_map, &full_bar[warp][slot], 0, y, kvh * C::NCH);
      tma_load_3d(dst + C::TILE, &pool_map, &full_bar[warp][slot], 0, y + p.bt, kvh * C::NCH);
    }
  };
  for (int s = 0; s < STAGES - 1 && s < n_it; ++s) issue(s);

  // ---- Q fragments (B operand: k = dim, n = column g), in registers for the whole tile
  uint32_t qf[HD / 16][2];
  {
    const int head = min(NT == 1 ? (g & 3) : g, G - 1);
    const typename QE::T* q = static_cast<const typename QE::T*>(a.Q) + size_t(row) * p.q_ld + size_t(kvh * G + head) * HD;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const bool mine = NT == 2 || (ks >= HD / 32) == (g >= 4);  // NT = 1: a column's query is zero in the other map's dims
      if constexpr (!C::FP8) {
        qf[ks][0] = mine ? *reinterpret_cast<const uint32_t*>(q + 16 * ks + 2 * t) : 0u;
        qf[ks][1] = mine ? *reinterpret_cast<const uint32_t*>(q + 16 * ks + 8 + 2 * t) : 0u;
      } else {
        // K fragments of an E4M3 tile hold dims 4t .. 4t + 3 of each 16: fragment columns (2t, 2t + 1) and (2t + 8, 2t + 9)
        // stand for dims (4t, 4t + 1) and (4t + 2, 4t + 3)
        const uint2 w = *reinterpret_cast<const uint2*>(q + 16 * ks + 4 * t);
        qf[ks][0] = mine ? w.x : 0u;
        qf[ks][1] = mine ? w.y : 0u;
      }
    }
  }
  // bf16 queries become fp16 operands: exactly, after each (head, map) has been brought to a largest magnitude of 2^14 .. 2^15 by a power of two,
  // which the scores take back. What lies more than 2^31 below a query's largest element is rounded.
  float q_back[NT][2];  // columns 2t, 2t + 1
  if constexpr (C::SCALED_Q) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int k0 = n * (HD / 32), k1 = NT == 1 ? HD / 16 : k0 + HD / 32;
      uint32_t top = 0;  // of |q|, as bits: bf16 pairs
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        if (ks >= k0 && ks < k1) top = __vmaxu2(__vmaxu2(top, qf[ks][0] & 0x7FFF7FFFu), qf[ks][1] & 0x7FFF7FFFu);
      top = max(top & 0xFFFFu, top >> 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int up = min(14 + 127 - int(top >> 7), 126);  // log2 of the factor
      const float f = __uint_as_float(uint32_t(127 + up) << 23), back = __uint_as_float(uint32_t(127 - up) << 23);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        if (ks >= k0 && ks < k1) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 x = QE::unpack2(qf[ks][i]);
            qf[ks][i] = CE::pack2(x.x * f, x.y * f);
          }
        }
      q_back[n][0] = __shfl_sync(0xffffffffu, back, 8 * t), q_back[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
    }
  }

  float o[NT][NMT][4];
  float m[NT][2], l[NT][2];  // columns 2t, 2t + 1 (l: this lane's keys only)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < NMT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
  }
  const int mi = lane >> 3, rj = lane & 7;
  const uint32_t key_k = rj + 8 * (mi & 1), sel_k = mi >> 1;  // K: ldmatrix
  const uint32_t key_v = rj + 8 * (mi >> 1), sel_v = mi & 1;  // V: ldmatrix.trans

  for (int it = 0; it < n_it; ++it) {
    if (it + STAGES - 1 < n_it) issue(it + STAGES - 1);
    const int slot = it % STAGES;
    float kscale = 1.0f, vscale = 1.0f;
    if constexpr (C::FP8) {
      if (it - use_win >= 32) {
        use_win = it;
        if (it + lane < n_it) {
          int j0;
          const int b = block_of_it(it + lane, j0);
          use_ks = a.kv_scales[size_t(b) * 2 * p.Hkv + kvh];
          use_vs = a.kv_scales[(size_t(b) * 2 + 1) * p.Hkv + kvh];
        }
      }
      kscale = __shfl_sync(0xffffffffu, use_ks, it - use_win);
      vscale = __shfl_sync(0xffffffffu, use_vs, it - use_win);
    }
    if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[warp][slot], (it / STAGES) & 1))) {  // one verdict for the warp
      if (lane == 0) {
        atomicExch(a.status, kStatusTmaTimeout);
        gave_up = 1;
      }
      break;
    }
    uint8_t* vt = wsm + slot * C::STAGE + C::TILE;
    const int jb = kbase + 16 * (warp + it * NW);
    const int n_valid = min(16, tile.k1 - jb), n_skip = tile.k0 - jb;
    if (n_valid < 16) {
      // rows past the range hold other keys or stale bytes: V must be zero there (0 * NaN), K is masked by selection
      const int n = (16 - n_valid) * C::NCH * 8;
      for (int i = lane; i < n; i += 32) {
        const int r = n_valid + i / (C::NCH * 8), rem = i % (C::NCH * 8);
        *reinterpret_cast<uint4*>(vt + (rem >> 3) * 2048 + r * 128 + (rem & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
    }
    const uint32_t kt_u = smem_u32(wsm + slot * C::STAGE), vt_u = smem_u32(vt);

    // ---- S^T: two accumulators per tile shorten the dependent chains
    float s[NT][2][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][0][i] = s[n][1][i] = 0.0f;
    if constexpr (!C::FP8) {
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t af[4];
        ldmatrix_x4(af, kt_u + (ks >> 2) * 2048 + key_k * 128 + (((((ks & 3) << 1) + sel_k) ^ (key_k & 7)) << 4));
        mma_16816<C::CDT>(s[NT == 1 ? 0 : ks / (HD / 32)][ks & 1], af, qf[ks][0], qf[ks][1]);
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < HD / 32; ++kk) {
        uint32_t r[4];
        ldmatrix_x4(r, kt_u + (kk >> 2) * 2048 + key_k * 128 + (((((kk & 3) << 1) + sel_k) ^ (key_k & 7)) << 4));
        const uint32_t a0[4] = {e4m3x2_to_f16x2(uint16_t(r[0] & 0xFFFFu)), e4m3x2_to_f16x2(uint16_t(r[1] & 0xFFFFu)),
                                e4m3x2_to_f16x2(uint16_t(r[0] >> 16)), e4m3x2_to_f16x2(uint16_t(r[1] >> 16))};
        const uint32_t a1[4] = {e4m3x2_to_f16x2(uint16_t(r[2] & 0xFFFFu)), e4m3x2_to_f16x2(uint16_t(r[3] & 0xFFFFu)),
                                e4m3x2_to_f16x2(uint16_t(r[2] >> 16)), e4m3x2_to_f16x2(uint16_t(r[3] >> 16))};
        const int n = NT == 1 ? 0 : kk / (HD / 64);
        mma_16816<C::CDT>(s[n][0], a0, qf[2 * kk][0], qf[2 * kk][1]);
        mma_16816<C::CDT>(s[n][1], a1, qf[2 * kk + 1][0], qf[2 * kk + 1][1]);
      }
    }
    const float sc = sl2 * kscale;
    // What is rounded to 16 bits is the weight times the power of two in the V scale, and the reference the largest of these: neither a page of
    // small values that is well attended nor one of large values that is hardly attended loses its weights. The rest of the scale,
    // 1 .. 2, goes on the product.
    const float v_log2 = C::FP8 ? log2_floor(vscale) : 0.0f, v_inv = C::FP8 ? __uint_as_float(uint32_t(127 - int(v_log2)) << 23) : 1.0f;
    const bool out_lo = g >= n_valid || g < n_skip, out_hi = g + 8 >= n_valid || g + 8 < n_skip;
    uint32_t pb[NT][2];
    float corr[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // lane: (key g, columns 2t, 2t + 1), (key g + 8, the same)
      const float sc0 = C::SCALED_Q ? sc * q_back[n][0] : sc, sc1 = C::SCALED_Q ? sc * q_back[n][1] : sc;
      float s0 = s[n][0][0] + s[n][1][0], s1 = s[n][0][1] + s[n][1][1], s2 = s[n][0][2] + s[n][1][2], s3 = s[n][0][3] + s[n][1][3];
      if constexpr (C::FP8) s0 = fmaf(s0, sc0, v_log2), s1 = fmaf(s1, sc1, v_log2), s2 = fmaf(s2, sc0, v_log2), s3 = fmaf(s3, sc1, v_log2);
      else s0 *= sc0, s1 *= sc1, s2 *= sc0, s3 *= sc1;
      if (out_lo) s0 = s1 = -INFINITY;
      if (out_hi) s2 = s3 = -INFINITY;
      float x0 = fmaxf(s0, s2), x1 = fmaxf(s1, s3);
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
      }
      const float n0 = fmaxf(m[n][0], x0), n1 = fmaxf(m[n][1], x1);  // a block has a live key
      corr[n][0] = fast_exp2(m[n][0] - n0), corr[n][1] = fast_exp2(m[n][1] - n1);
      const float p0 = fast_exp2(s0 - n0), p1 = fast_exp2(s1 - n1), p2 = fast_exp2(s2 - n0), p3 = fast_exp2(s3 - n1);
      l[n][0] = fmaf(l[n][0], corr[n][0], C::FP8 ? (p0 + p2) * v_inv : p0 + p2);
      l[n][1] = fmaf(l[n][1], corr[n][1], C::FP8 ? (p1 + p3) * v_inv : p1 + p3);
      m[n][0] = n0, m[n][1] = n1;
      pb[n][0] = movmatrix_trans(CE::pack2(p0, p1));
      pb[n][1] = movmatrix_trans(CE::pack2(p2, p3));
    }

    // ---- O^T = O^T * corr + V^T . P^T
    if constexpr (!C::FP8) {
#pragma unroll
      for (int i = 0; i < NMT; ++i) {
        uint32_t af[4];
        ldmatrix_x4_trans(af, vt_u + (i >> 2) * 2048 + key_v * 128 + (((((i & 3) << 1) + sel_v) ^ (key_v & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float(&x)[4] = o[n][i];
          x[0] *= corr[n][0], x[1] *= corr[n][1], x[2] *= corr[n][0], x[3] *= corr[n][1];
          mma_16816<C::CDT>(x, af, pb[n][0], pb[n][1]);
        }
      }
    } else {
      const float v_rest = vscale * v_inv;
      // A maximum grows less and less often: the sums are only moved when one of the warp's has.
      bool grown = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) grown = grown || corr[n][0] != 1.0f || corr[n][1] != 1.0f;
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < NMT; ++i) o[n][i][0] *= corr[n][0], o[n][i][1] *= corr[n][1], o[n][i][2] *= corr[n][0], o[n][i][3] *= corr[n][1];
      }
      // per 32 dims: dims 32u + 4g .. + 3 of keys 2t, 2t + 1, 2t + 8, 2t + 9, paired by key: m-tile 2u has rows
      // g <-> dim 32u + 4g, g + 8 <-> 32u + 4g + 1, m-tile 2u + 1 the two dims after them
#pragma unroll
      for (int u = 0; u < HD / 32; ++u) {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = *reinterpret_cast<const uint32_t*>(vt + tile_off(uint32_t(2 * t + (q & 1) + 8 * (q >> 1)), uint32_t(32 * u + 4 * g)));
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) lo[q] = e4m3x2_to_f16x2(uint16_t(w[q] & 0xFFFFu)), hi[q] = e4m3x2_to_f16x2(uint16_t(w[q] >> 16));
        const uint32_t fa[4] = {__byte_perm(lo[0], lo[1], 0x5410), __byte_perm(lo[0], lo[1], 0x7632), __byte_perm(lo[2], lo[3], 0x5410), __byte_perm(lo[2], lo[3], 0x7632)};
        const uint32_t fb[4] = {__byte_perm(hi[0], hi[1], 0x5410), __byte_perm(hi[0], hi[1], 0x7632), __byte_perm(hi[2], hi[3], 0x5410), __byte_perm(hi[2], hi[3], 0x7632)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float(&x)[4] = o[n][2 * u];
          float(&y)[4] = o[n][2 * u + 1];
          float dx[4] = {0.f, 0.f, 0.f, 0.f}, dy[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816<C::CDT>(dx, fa, pb[n][0], pb[n][1]);
          mma_16816<C::CDT>(dy, fb, pb[n][0], pb[n][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = fmaf(dx[i], v_rest, x[i]), y[i] = fmaf(dy[i], v_rest, y[i]);
        }
      }
    }
    __syncwarp();  // every lane is done with the slot before lane 0 refills it
  }
  pdl_launch_dependents();  // the join may be scheduled while this grid drains

  // ---- the warps' results through shared memory (their rings are idle now)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], off);
      l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], off);
    }
  __syncthreads();
  if (gave_up) {
    // loads may still be in flight into the rings: they are not reused. Empty records, or a zero row.
    for (int hg = warp; hg < G; hg += NW) {
      if (tile.part >= 0) {
        for (int c = 0; c < 2; ++c) {
          float* rec = a.parts + diff_record(a, tile.part, kvh, 0, hg, c);
          for (int i = lane; i < HD; i += 32) rec[i] = 0.0f;
          if (lane == 0) rec[HD] = -INFINITY, rec[HD + 1] = 0.0f;
        }
      } else {
        typename QE::T* op = static_cast<typename QE::T*>(a.O) + size_t(row) * p.q_ld + size_t(kvh * G + hg) * HD;
        for (int i = lane; i < HD; i += 32) op[i] = QE::from_f32(0.0f);
      }
    }
    return;
  }
  {
    float* osm = reinterpret_cast<float*>(wsm);
    float* msm = osm + 8 * NT * OLD;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* on = osm + (8 * n + 2 * t) * OLD;
#pragma unroll
      for (int i = 0; i < NMT; ++i) {
        const int lo = C::FP8 ? 32 * (i >> 1) + 4 * g + 2 * (i & 1) : 16 * i + g, hi = C::FP8 ? lo + 1 : lo + 8;
        on[lo] = o[n][i][0], on[OLD + lo] = o[n][i][1], on[hi] = o[n][i][2], on[OLD + hi] = o[n][i][3];
      }
      if (g == 0) {
        msm[8 * n + 2 * t] = m[n][0], msm[8 * n + 2 * t + 1] = m[n][1];
        msm[8 * NT + 8 * n + 2 * t] = l[n][0], msm[8 * NT + 8 * n + 2 * t + 1] = l[n][1];
      }
    }
  }
  __syncthreads();

  constexpr int DPL = HD / 32;
  for (int hg = warp; hg < G; hg += NW) {
    const int h = kvh * G + hg;
    float M[2], L[2], acc[2][DPL];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = (NT == 1 ? 4 : 8) * c + hg;
      M[c] = -INFINITY, L[c] = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) M[c] = fmaxf(M[c], reinterpret_cast<const float*>(smem + size_t(w) * C::WARP_BYTES)[8 * NT * OLD + col]);
#pragma unroll
      for (int i = 0; i < DPL; ++i) acc[c][i] = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float* ow = reinterpret_cast<const float*>(smem + size_t(w) * C::WARP_BYTES);
        const float mw = ow[8 * NT * OLD + col];
        const float wg = (mw == -INFINITY) ? 0.0f : fast_exp2(mw - M[c]);
        L[c] = fmaf(wg, ow[8 * NT * OLD + 8 * NT + col], L[c]);
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[c][i] = fmaf(wg, ow[col * OLD + lane + 32 * i], acc[c][i]);
      }
    }
    if (tile.last) {
      // the token's own key and value (batch row tree.base); lane holds dims lane + 32 i, map 1's in the lower half of i
      const typename QE::T* q = static_cast<const typename QE::T*>(a.Q) + size_t(row) * p.q_ld + size_t(h) * HD;
      const typename QE::T* kr = static_cast<const typename QE::T*>(a.Kb) + size_t(tree.base) * p.kv_ld + size_t(kvh) * HD;
      const typename QE::T* vr = static_cast<const typename QE::T*>(a.Vb) + size_t(tree.base) * p.kv_ld + size_t(kvh) * HD;
      float dot[2] = {0.0f, 0.0f}, v[DPL];
      // a mask may hide the row from itself
      const int4 seg = a.anc_mask ? make_int4(0, 0, 0, 0) : reinterpret_cast<const int4*>(a.desc)[row];
      const bool self = a.anc_mask ? (a.anc_mask[row] & 1ull) : (seg.z > 0 || seg.x <= 0);
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        dot[i / (DPL / 2)] = fmaf(QE::to_f32(q[lane + 32 * i]), QE::to_f32(kr[lane + 32 * i]), dot[i / (DPL / 2)]);
        v[i] = QE::to_f32(vr[lane + 32 * i]);
      }
#pragma unroll
      for (int off = 16; off; off >>= 1) {
        dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], off);
        dot[1] += __shfl_xor_sync(0xffffffffu, dot[1], off);
      }
      if (self) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float sx = dot[c] * sl2, M2 = fmaxf(M[c], sx);
          const float keep = (M[c] == -INFINITY) ? 0.0f : fast_exp2(M[c] - M2), pw = fast_exp2(sx - M2);
          L[c] = fmaf(L[c], keep, pw);
#pragma unroll
          for (int i = 0; i < DPL; ++i) acc[c][i] = fmaf(pw, v[i], acc[c][i] * keep);
          M[c] = M2;
        }
      }
    }
    if (tile.part >= 0) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* rec = a.parts + diff_record(a, tile.part, kvh, 0, hg, c);
#pragma unroll
        for (int i = 0; i < DPL; ++i) rec[lane + 32 * i] = acc[c][i];
        if (lane == 0) rec[HD] = M[c] * kLn2, rec[HD + 1] = L[c];
      }
      continue;
    }
    const float inv1 = L[0] > 0.0f ? 1.0f / L[0] : 0.0f, inv2 = L[1] > 0.0f ? diff_lam(d, row, h) / L[1] : 0.0f;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      acc[0][i] = acc[0][i] * inv1 - acc[1][i] * inv2;
      ss = fmaf(acc[0][i], acc[0][i], ss);
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    const float f = diff_row_factor(d, ss, HD);
    typename QE::T* op = static_cast<typename QE::T*>(a.O) + size_t(row) * p.q_ld + size_t(h) * HD;
#pragma unroll
    for (int i = 0; i < DPL; ++i) op[lane + 32 * i] = QE::from_f32(acc[0][i] * f * (d.norm_w ? d.norm_w[lane + 32 * i] : 1.0f));
  }
}

// Warps and stages as in the plain decode kernel: rings for two CTAs per SM (one drains while the other streams); 4 KB blocks
// (128-dim E4M3) do as much work per block for half the bytes, so more CTAs with short rings share an SM.
template <int HD, int KVDT, int QDT, int NT>
using CfgOf = Cfg<HD, KVDT, QDT, NT, 4, 3, (HD == 128 && KVDT == ESP_E4M3) ? (NT == 1 ? 4 : 3) : 2>;

template <class C>
cudaError_t setup_one() {
  return cudaFuncSetAttribute(diff_decode_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
}
template <int HD, int QDT>
cudaError_t setup_types(int32_t G, int32_t kv_dtype) {
  if (kv_dtype == ESP_E4M3) return G <= 4 ? setup_one<CfgOf<HD, ESP_E4M3, QDT, 1>>() : setup_one<CfgOf<HD, ESP_E4M3, QDT, 2>>();
  return G <= 4 ? setup_one<CfgOf<HD, QDT, QDT, 1>>() : setup_one<CfgOf<HD, QDT, QDT, 2>>();
}
template <class C>
cudaError_t launch_one(const DiffArgs& a, const CUtensorMap& m, cudaStream_t stream) {
  return launch_pdl(diff_decode_kernel<C>, dim3(unsigned(a.k.n_tiles) * unsigned(a.k.p.Hkv)), dim3(C::NW * 32), C::SMEM, stream, m, a);
}
template <int HD, int QDT>
cudaError_t launch_types(const DiffArgs& a, const CUtensorMap& m, cudaStream_t stream) {
  const bool packed = a.k.G <= 4;
  if (a.k.kv_dtype == ESP_E4M3) return packed ? launch_one<CfgOf<HD, ESP_E4M3, QDT, 1>>(a, m, stream) : launch_one<CfgOf<HD, ESP_E4M3, QDT, 2>>(a, m, stream);
  return packed ? launch_one<CfgOf<HD, QDT, QDT, 1>>(a, m, stream) : launch_one<CfgOf<HD, QDT, QDT, 2>>(a, m, stream);
}

}  // namespace

bool diff_decode_supports(int32_t HD, int32_t G, int32_t bt) { return (HD == 128 || HD == 256) && G >= 1 && G <= 8 && bt % 16 == 0; }

cudaError_t diff_decode_setup(int32_t HD, int32_t G, int32_t q_dtype, int32_t kv_dtype, int32_t bt) {
  if (!diff_decode_supports(HD, G, bt)) return cudaSuccess;
  if (HD == 128) return q_dtype == ESP_F16 ? setup_types<128, ESP_F16>(G, kv_dtype) : setup_types<128, ESP_BF16>(G, kv_dtype);
  return q_dtype == ESP_F16 ? setup_types<256, ESP_F16>(G, kv_dtype) : setup_types<256, ESP_BF16>(G, kv_dtype);
}

cudaError_t launch_diff_decode(const DiffArgs& a, const CUtensorMap& pool_map, cudaStream_t stream, uint64_t* launches) {
  if (a.k.n_tiles <= 0) return cudaSuccess;
  const bool f16 = a.k.q_dtype == ESP_F16;
  const cudaError_t e = a.k.HD == 128 ? (f16 ? launch_types<128, ESP_F16>(a, pool_map, stream) : launch_types<128, ESP_BF16>(a, pool_map, stream))
                                      : (f16 ? launch_types<256, ESP_F16>(a, pool_map, stream) : launch_types<256, ESP_BF16>(a, pool_map, stream));
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
