// kv_append for sm_100a: the new tokens' queries, keys and values on their way into the paged cache.
//
// Per row, head and map (maps = 1, or 2 for differential heads; D = HD / maps dims each), pairs (x, y) of a query or key turn by
// the row's angle a_f = pos * inv_freq_f:
//   x' = x cos a_f - y sin a_f,   y' = y cos a_f + x sin a_f,
// everything is rounded once to 16 bits, and keys and values go to (block, position) of the pool as well (E4M3 pools: the code of
// the rounded value over the block's scale).
//
// The angle: an fp32 product loses 2^-25 of up to 10^5 radians at far positions, more than a bf16 step. pos * inv_freq / 2 pi is
// formed in double (the product of an int32 and an fp32 number is exact there), whole turns are taken off, and the rest, at most
// half a turn, is good to fp32: rot_half values per row, formed once per CTA in shared memory.
//
// HBM-bound for prompts (every byte is read and written once), latency-bound for single tokens. A thread's item is one rotating
// pair of 8-dim chunks, (d, d + rot_half), or one chunk that needs no partner: 16-byte loads and stores, and since an item's
// reads precede its own writes and no other item touches them, outputs may lie over the sources. Rows whose addresses or sizes do
// not allow 16-byte accesses take the same kernel with one-dim items.
#include "common.cuh"
#include "../launch.h"

namespace esp {
namespace {

constexpr int kThreads = 256;

template <int QDT, bool SRC32, bool FP8_POOL, int VEC>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendArgs args, const int HD, const int rows_per_cta) {
  using QE = Elem16<QDT>;
  using T = typename QE::T;
  const esp_kv_append_args& a = args.a;
  const esp_attn_params& p = a.p;
  extern __shared__ float2 turn[];  // [row of the CTA][rot_half]: cos, sin
  const int D = HD / a.maps, half = a.rot_half;
  const int row0 = blockIdx.x * rows_per_cta;
  const int n_rows = min(rows_per_cta, a.rows - row0);
  pdl_wait();  // the projection, and what a pass before this one may still read of the pool

  for (int i = threadIdx.x; i < n_rows * half; i += kThreads) {
    const int r = i / half, f = i - r * half;
    const double turns = double(a.pos[row0 + r]) * double(a.inv_freq[f]) * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * float(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c, s);
  }
  __syncthreads();
  pdl_launch_dependents();

  // items of one map: rotating chunk pairs first, then the chunks that pass through; adjacent pairs lie within a chunk
  const int n_pair = a.adjacent ? 0 : half / VEC;
  const int per_map = a.adjacent ? D / VEC : n_pair + (D - 2 * half) / VEC;
  const int per_head = per_map * a.maps, v_head = HD / VEC;
  const int n_q = a.Q ? p.H * per_head : 0, n_k = p.Hkv * per_head, n_v = p.Hkv * v_head;
  const int per_row = n_q + n_k + n_v;

  auto load = [&](const void* base, int64_t at, float (&x)[VEC]) {
    if constexpr (SRC32) {
      const float* src = static_cast<const float*>(base) + at;
      if constexpr (VEC == 8) {
        const float4 u = reinterpret_cast<const float4*>(src)[0], w = reinterpret_cast<const float4*>(src)[1];
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
      } else {
        x[0] = src[0];
      }
    } else {
      const T* src = static_cast<const T*>(base) + at;
      if constexpr (VEC == 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(src);
        const float2 f0 = QE::unpack2(u.x), f1 = QE::unpack2(u.y), f2 = QE::unpack2(u.z), f3 = QE::unpack2(u.w);
        x[0] = f0.x, x[1] = f0.y, x[2] = f1.x, x[3] = f1.y, x[4] = f2.x, x[5] = f2.y, x[6] = f3.x, x[7] = f3.y;
      } else {
        x[0] = QE::to_f32(src[0]);
      }
    }
  };
  // 16-bit values of x at `dst`; x becomes those values again (what an E4M3 pool encodes)
  auto round16 = [&](float (&x)[VEC], uint32_t (&w)[VEC == 8 ? 4 : 1]) {
    if constexpr (VEC == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = QE::pack2(x[2 * i], x[2 * i + 1]);
    } else {
      w[0] = QE::pack2(x[0], 0.0f);
    }
  };
  auto store16 = [&](void* base, size_t at, const uint32_t (&w)[VEC == 8 ? 4 : 1]) {
    T* dst = static_cast<T*>(base) + at;
    if constexpr (VEC == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint16_t*>(dst) = uint16_t(w[0]);
  };
  auto store_pool = [&](size_t at, const uint32_t (&w)[VEC == 8 ? 4 : 1], float scale) {
    if constexpr (!FP8_POOL) {
      store16(a.kv, at, w);
    } else {
      // division, as esp_kv_save does, so that both give the same codes
      uint8_t* dst = static_cast<uint8_t*>(a.kv) + at;
      if constexpr (VEC == 8) {
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = QE::unpack2(w[i]);
          const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f.x, scale), __fdiv_rn(f.y, scale)), __NV_SATFINITE, __NV_E4M3);
          o[i >> 1] |= two << (16 * (i & 1));
        }
        *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
      } else {
        *dst = f32_to_e4m3(__fdiv_rn(QE::unpack2(w[0]).x, scale));
      }
    }
  };

  const int total = n_rows * per_row;
  for (int idx = blockIdx.y * kThreads + threadIdx.x; idx < total; idx += kThreads * gridDim.y) {
    const int r = idx / per_row, item = idx - r * per_row;
    const int row = row0 + r;
    const float2* tr = turn + r * half;
    const bool is_v = item >= n_q + n_k, is_q = item < n_q;
    const int rel = is_q ? item : (is_v ? item - n_q - n_k : item - n_q);
    const int head = rel / (is_v ? v_head : per_head);
    int in_head = rel - head * (is_v ? v_head : per_head);
    int d0 = in_head * VEC, d1 = -1, f0 = -1;  // first dim of the item, of its partner chunk, and the frequency of its first pair
    if (!is_v) {
      const int map = in_head / per_map, in_map = in_head - map * per_map;
      if (a.adjacent) {
        d0 = in_map * VEC;
        f0 = d0 < 2 * half ? d0 / 2 : -1;
      } else if (in_map < n_pair) {
        d0 = f0 = in_map * VEC, d1 = d0 + half;
      } else {
        d0 = 2 * half + (in_map - n_pair) * VEC;
      }
      d0 += map * D;
      if (d1 >= 0) d1 += map * D;
    }
    const void* src = is_q ? a.Q : (is_v ? a.V : a.K);
    const int64_t at = int64_t(row) * (is_q ? a.q_src_ld : (is_v ? a.v_src_ld : a.k_src_ld)) + int64_t(head) * HD;

    float x[VEC], y[VEC];
    load(src, at + d0, x);
    if (d1 >= 0) load(src, at + d1, y);
    if (d1 >= 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 cs = tr[f0 + i];
        const float u = x[i];
        x[i] = u * cs.x - y[i] * cs.y;
        y[i] = y[i] * cs.x + u * cs.y;
      }
    } else if (f0 >= 0) {
      if constexpr (VEC == 8) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const float2 cs = tr[f0 + i / 2];
          const float u = x[i];
          x[i] = u * cs.x - x[i + 1] * cs.y;
          x[i + 1] = x[i + 1] * cs.x + u * cs.y;
        }
      }
    }
    uint32_t wx[VEC == 8 ? 4 : 1], wy[VEC == 8 ? 4 : 1];
    if (is_q) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] *= a.qscale;
      round16(x, wx);
      const size_t to = size_t(row) * p.q_ld + size_t(head) * HD;
      store16(a.Qo, to + d0, wx);
      if (d1 >= 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[i] *= a.qscale;
        round16(y, wy);
        store16(a.Qo, to + d1, wy);
      }
      continue;
    }
    round16(x, wx);
    if (d1 >= 0) round16(y, wy);
    void* batch = is_v ? a.Vb : a.Kb;
    if (batch) {
      const size_t to = size_t(row) * p.kv_ld + size_t(head) * HD;
      store16(batch, to + d0, wx);
      if (d1 >= 0) store16(batch, to + d1, wy);
    }
    if (a.kv) {
      const int2 slot = reinterpret_cast<const int2*>(a.slots)[row];
      if (slot.x < 0) continue;
      if (slot.x >= a.n_blocks || slot.y < 0 || slot.y >= p.bt) {  // the table lives on the device: no host check sees it
        atomicExch(args.status, kStatusBadBlock);
        continue;
      }
      const size_t blk = size_t(p.bt) * p.kv_ld;
      const size_t to = p.kv_base + (size_t(slot.x) * 2 + (is_v ? 1 : 0)) * blk + size_t(slot.y) * p.kv_ld + size_t(head) * HD;
      float scale = 1.0f;
      if constexpr (FP8_POOL) scale = a.kv_scales[(size_t(slot.x) * 2 + (is_v ? 1 : 0)) * p.Hkv + head];
      store_pool(to + d0, wx, scale);
      if (d1 >= 0) store_pool(to + d1, wy, scale);
    }
  }
}

// Adjacent pairs without 16-byte accesses: one item = one pair (or, past the rotating dims, two dims that pass through). The same
// arithmetic; kept apart because its item holds two neighbouring dims.
template <int QDT, bool SRC32, bool FP8_POOL>
__global__ void __launch_bounds__(kThreads) kv_append_adjacent_kernel(const AppendArgs args, const int HD) {
  using QE = Elem16<QDT>;
  using T = typename QE::T;
  const esp_kv_append_args& a = args.a;
  const esp_attn_params& p = a.p;
  extern __shared__ float2 turn[];
  const int D = HD / a.maps, half = a.rot_half, row = blockIdx.x;
  pdl_wait();
  for (int f = threadIdx.x; f < half; f += kThreads) {
    const double turns = double(a.pos[row]) * double(a.inv_freq[f]) * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * float(turns - rint(turns)), &s, &c);
    turn[f] = make_float2(c, s);
  }
  __syncthreads();
  pdl_launch_dependents();
  const int n_q = a.Q ? p.H * HD / 2 : 0, n_k = p.Hkv * HD / 2;
  for (int item = blockIdx.y * kThreads + threadIdx.x; item < n_q + 2 * n_k; item += kThreads * gridDim.y) {
    const bool is_q = item < n_q, is_v = item >= n_q + n_k;
    const int rel = is_q ? item : (is_v ? item - n_q - n_k : item - n_q);
    const int head = rel / (HD / 2), d = 2 * (rel - head * (HD / 2));
    const void* src = is_q ? a.Q : (is_v ? a.V : a.K);
    const int64_t at = int64_t(row) * (is_q ? a.q_src_ld : (is_v ? a.v_src_ld : a.k_src_ld)) + int64_t(head) * HD + d;
    float x, y;
    if constexpr (SRC32) x = static_cast<const float*>(src)[at], y = static_cast<const float*>(src)[at + 1];
    else x = QE::to_f32(static_cast<const T*>(src)[at]), y = QE::to_f32(static_cast<const T*>(src)[at + 1]);
    const int f = (d % D) / 2;
    if (!is_v && f < half) {
      const float2 cs = turn[f];
      const float u = x;
      x = u * cs.x - y * cs.y;
      y = y * cs.x + u * cs.y;
    }
    if (is_q) {
      T* dst = static_cast<T*>(a.Qo) + size_t(row) * p.q_ld + size_t(head) * HD + d;
      dst[0] = QE::from_f32(x * a.qscale), dst[1] = QE::from_f32(y * a.qscale);
      continue;
    }
    const T rx = QE::from_f32(x), ry = QE::from_f32(y);
    if (void* batch = is_v ? a.Vb : a.Kb) {
      T* dst = static_cast<T*>(batch) + size_t(row) * p.kv_ld + size_t(head) * HD + d;
      dst[0] = rx, dst[1] = ry;
    }
    if (!a.kv) continue;
    const int2 slot = reinterpret_cast<const int2*>(a.slots)[row];
    if (slot.x < 0) continue;
    if (slot.x >= a.n_blocks || slot.y < 0 || slot.y >= p.bt) {
      atomicExch(args.status, kStatusBadBlock);
      continue;
    }
    const size_t blk = size_t(p.bt) * p.kv_ld;
    const size_t to = p.kv_base + (size_t(slot.x) * 2 + (is_v ? 1 : 0)) * blk + size_t(slot.y) * p.kv_ld + size_t(head) * HD + d;
    if constexpr (FP8_POOL) {
      const float scale = a.kv_scales[(size_t(slot.x) * 2 + (is_v ? 1 : 0)) * p.Hkv + head];
      uint8_t* dst = static_cast<uint8_t*>(a.kv) + to;
      dst[0] = f32_to_e4m3(__fdiv_rn(QE::to_f32(rx), scale)), dst[1] = f32_to_e4m3(__fdiv_rn(QE::to_f32(ry), scale));
    } else {
      T* dst = static_cast<T*>(a.kv) + to;
      dst[0] = rx, dst[1] = ry;
    }
  }
}

template <int QDT, bool SRC32, bool FP8_POOL>
cudaError_t launch_typed(const AppendArgs& args, int32_t HD, cudaStream_t stream) {
  const esp_kv_append_args& a = args.a;
  const size_t ssz = SRC32 ? 4 : 2;
  auto ok16 = [](const void* q, int64_t row_bytes) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && row_bytes % 16 == 0; };
  const bool wide = (a.adjacent ? a.rot_half % 4 : a.rot_half % 8) == 0 && ok16(a.Q, a.q_src_ld * int64_t(ssz)) && ok16(a.K, a.k_src_ld * int64_t(ssz)) &&
                    ok16(a.V, a.v_src_ld * int64_t(ssz)) && ok16(a.Qo, 0) && ok16(a.Kb, 0) && ok16(a.Vb, 0) && ok16(a.kv, 0);
  const int vec = wide ? 8 : 1;
  const int heads = (a.Q ? a.p.H : 0) + 2 * a.p.Hkv;
  const int per_row = heads * HD / vec;  // items of a row, at most
  // A row with fewer chunks than a CTA has threads shares its CTA with others; a batch with fewer rows than SMs spreads each row
  // over several CTAs.
  const int rpc = wide ? int(std::max<int64_t>(1, std::min<int64_t>(2 * kThreads / per_row, a.rows / 148))) : 1;
  const unsigned gx = unsigned((a.rows + rpc - 1) / rpc);
  const int most_y = (rpc * per_row + kThreads - 1) / kThreads;
  const unsigned gy = unsigned(std::max(1, std::min(most_y, int(4 * 148 / gx))));
  const size_t smem = size_t(rpc) * a.rot_half * sizeof(float2);
  if (wide) return launch_pdl(kv_append_kernel<QDT, SRC32, FP8_POOL, 8>, dim3(gx, gy), dim3(kThreads), smem, stream, args, HD, rpc);
  if (a.adjacent) return launch_pdl(kv_append_adjacent_kernel<QDT, SRC32, FP8_POOL>, dim3(gx, gy), dim3(kThreads), smem, stream, args, HD);
  return launch_pdl(kv_append_kernel<QDT, SRC32, FP8_POOL, 1>, dim3(gx, gy), dim3(kThreads), smem, stream, args, HD, rpc);
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& a, int32_t HD, int32_t q_dtype, bool fp8_pool, cudaStream_t stream, uint64_t* launches) {
  if (a.a.rows <= 0) return cudaSuccess;
  const bool f16 = q_dtype == ESP_F16, s32 = a.a.src_f32 != 0;
  cudaError_t e;
  if (f16) {
    if (s32) e = fp8_pool ? launch_typed<ESP_F16, true, true>(a, HD, stream) : launch_typed<ESP_F16, true, false>(a, HD, stream);
    else e = fp8_pool ? launch_typed<ESP_F16, false, true>(a, HD, stream) : launch_typed<ESP_F16, false, false>(a, HD, stream);
  } else {
    if (s32) e = fp8_pool ? launch_typed<ESP_BF16, true, true>(a, HD, stream) : launch_typed<ESP_BF16, true, false>(a, HD, stream);
    else e = fp8_pool ? launch_typed<ESP_BF16, false, true>(a, HD, stream) : launch_typed<ESP_BF16, false, false>(a, HD, stream);
  }
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
