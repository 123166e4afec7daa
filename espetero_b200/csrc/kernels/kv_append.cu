// kv_append for sm_100a: the new tokens' queries, keys and values on their way into the paged cache.
//
// Per row, head and map (maps = 1, or 2 for differential heads; D = HD / maps dims each), pairs (x, y) of a query or key turn by
// the row's angle a_f = pos * inv_freq_f:
//   x' = x cos a_f - y sin a_f,   y' = y cos a_f + x sin a_f,
// everything is rounded once to 16 bits, and keys and values go to (block, position) of the pool as well (E4M3 pools: the code of
// the rounded value over the block's scale).
//
// The angle: an fp32 product loses 2^-25 of up to 10^5 radians at far positions, more than a bf16 step. pos * inv_freq / 2 pi is
// formed in double (the product is exact for |pos| < 2^29: 29 bits by 24), whole turns are taken off, and the rest, at most half a turn, is good to
// fp32 for angles up to 2^29 radians: two roundings of 2^-53 leave 2^-25 of a turn there.
//
// HBM-bound for prompts (every byte is read and written once), latency-bound for single tokens. A warp owns one row, or a part of it when
// rows are few. A lane's item is a rotating pair of 8-dim chunks, (d, d + rot_half), or one chunk that needs no partner; 32 lanes
// cover 32 / P2 maps, P2 = the items of a map rounded up to a power of two, so a lane's place within a map is the same in every step:
// it forms its 4 or 8 sines and cosines once, in registers, addresses advance by a constant, and nothing is shared between warps.
// 8192 rows of H32 / Hkv4 / HD128, fp16: 34.4 us = 5.37 TB/s = 0.82 of the copy peak (71.7 us with a table of sines per CTA and items
// dealt out by division, which left the instruction issue and the CTAs' trips to memory in charge); 5001 fp32 rows of H16 / Hkv2 / HD256:
// 33.1 us = 4.95 TB/s. kBatch items are asked for before the first is turned: 2 at 24 warps per SM; 4 and 8 measured 36.6 and 41.2 us, 1
// 43.0.
// An item's reads precede its own writes and no other item touches its bytes, so outputs may lie over the sources.
#include <type_traits>

#include "common.cuh"
#include "../launch.h"

namespace esp {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;  // small CTAs: their slots free up one by one (with 8 warps 3 to 5 % slower past one wave)
constexpr int kBatch = 2;  // items a lane asks for at once

__device__ __forceinline__ float2 turn_of(int pos, float inv_freq) {
  const double turns = double(pos) * double(inv_freq) * 0.15915494309189533577;
  float s, c;
  sincospif(2.0f * float(turns - rint(turns)), &s, &c);
  return make_float2(c, s);
}

// Where a row's keys (which = 0) or values go in the pool; false: nowhere. The table lives on the device, no host check sees it.
__device__ __forceinline__ bool pool_row(const AppendArgs& args, int row, int2& slot) {
  const esp_kv_append_args& a = args.a;
  slot = reinterpret_cast<const int2*>(a.slots)[row];
  if (slot.x < 0) return false;
  if (slot.x >= a.n_blocks || slot.y < 0 || slot.y >= a.p.bt) {
    atomicExch(args.status, kStatusBadBlock);
    return false;
  }
  return true;
}
__device__ __forceinline__ size_t pool_at(const esp_attn_params& p, const int2& slot, int which) {
  return p.kv_base + (size_t(slot.x) * 2 + which) * (size_t(p.bt) * p.kv_ld) + size_t(slot.y) * p.kv_ld;
}

// How a row falls into steps of 32 lanes.
struct Steps {
  int32_t q, k, v;      // steps of the queries, keys and values
  int32_t log_p2;       // lanes per map: 1 << log_p2
  int32_t n_pair;       // chunk pairs of a map (0 for adjacent pairs, which lie within a chunk)
  int32_t per_map;      // items of a map
  int32_t per_part;     // steps a warp takes
  int32_t parts;        // warps per row
};

template <bool SRC32>
struct Raw {  // 8 dims as they were loaded
  uint4 a;
  uint4 b;
};
template <>
struct Raw<false> {
  uint4 a;
};

template <int QDT, bool SRC32, bool FP8_POOL, bool ADJ>
__global__ void __launch_bounds__(kThreads, 6) kv_append_kernel(const AppendArgs args, const Steps st, const int HD) {
  using QE = Elem16<QDT>;
  using T = typename QE::T;
  using S = std::conditional_t<SRC32, float, T>;
  const esp_kv_append_args& a = args.a;
  const esp_attn_params& p = a.p;
  const int lane = threadIdx.x & 31;
  const int64_t task = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int row = int(task / st.parts), part = int(task - int64_t(row) * st.parts);
  pdl_wait();  // the projection, and what a pass before this one may still read of the pool
  pdl_launch_dependents();
  if (row >= a.rows) return;
  const int D = HD / a.maps, half = a.rot_half;
  const int s0 = part * st.per_part, s1 = min(s0 + st.per_part, st.q + st.k + st.v);

  // this lane's place within a map: its chunk, the distance to the chunk's partner (0: none), the frequency of its first pair
  const int in_map = lane & ((1 << st.log_p2) - 1), maps_per_step = 32 >> st.log_p2, map_in_step = lane >> st.log_p2;
  const bool in_use = in_map < st.per_map, paired = !ADJ && in_map < st.n_pair;
  const int c0 = (paired || ADJ) ? in_map * 8 : 2 * half + (in_map - st.n_pair) * 8;
  const bool turns = ADJ ? c0 < 2 * half : paired;
  float2 cs[ADJ ? 4 : 8];
  if (turns && s0 < st.q + st.k) {
    const int pos = a.pos[row], f0 = ADJ ? c0 / 2 : c0;
    float fr[ADJ ? 4 : 8];
#pragma unroll
    for (int i = 0; i < (ADJ ? 4 : 8); ++i) fr[i] = a.inv_freq[f0 + i];
#pragma unroll
    for (int i = 0; i < (ADJ ? 4 : 8); ++i) cs[i] = turn_of(pos, fr[i]);
  }
  int2 slot = make_int2(-1, 0);
  const bool kept = a.kv && s1 > st.q && pool_row(args, row, slot);

  auto load = [](const S* src) {
    Raw<SRC32> w;
    w.a = reinterpret_cast<const uint4*>(src)[0];
    if constexpr (SRC32) w.b = reinterpret_cast<const uint4*>(src)[1];
    return w;
  };
  auto values = [](const Raw<SRC32>& w, float (&x)[8]) {
    const uint32_t u[4] = {w.a.x, w.a.y, w.a.z, w.a.w};
    if constexpr (SRC32) {
      const uint32_t v[4] = {w.b.x, w.b.y, w.b.z, w.b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u[i]), x[4 + i] = __uint_as_float(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = QE::unpack2(u[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  };
  auto round16 = [](const float (&x)[8]) { return make_uint4(QE::pack2(x[0], x[1]), QE::pack2(x[2], x[3]), QE::pack2(x[4], x[5]), QE::pack2(x[6], x[7])); };
  auto store_pool = [&](size_t at, const uint4& w, float scale) {
    if constexpr (!FP8_POOL) {
      *reinterpret_cast<uint4*>(static_cast<T*>(a.kv) + at) = w;
    } else {
      // division, as esp_kv_save does, so that both give the same codes
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
      uint32_t o[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = QE::unpack2(u[i]);
        const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f.x, scale), __fdiv_rn(f.y, scale)), __NV_SATFINITE, __NV_E4M3);
        o[i >> 1] |= two << (16 * (i & 1));
      }
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.kv) + at) = make_uint2(o[0], o[1]);
    }
  };

  // One kind (0 queries, 1 keys, 2 values): steps [t0, t1) of its own; consecutive steps lie `stride` dims apart in source and outputs.
  auto walk = [&](auto kind_c, int t0, int t1) {
    constexpr int kind = decltype(kind_c)::value;
    if (t0 >= t1) return;
    const int stride = kind == 2 ? 256 : maps_per_step * D;                    // dims of a step
    const int first = kind == 2 ? lane * 8 : map_in_step * D + c0;              // this lane's dims in step 0
    const int width = (kind == 0 ? p.H : p.Hkv) * HD;                           // dims of the row
    const bool mine = kind == 2 || in_use;
    const S* src = static_cast<const S*>(kind == 0 ? a.Q : (kind == 1 ? a.K : a.V)) + int64_t(row) * (kind == 0 ? a.q_src_ld : (kind == 1 ? a.k_src_ld : a.v_src_ld));
    T* out = kind == 0 ? static_cast<T*>(a.Qo) + size_t(row) * p.q_ld : static_cast<T*>(kind == 1 ? a.Kb : a.Vb);
    if (kind != 0 && out) out += size_t(row) * p.kv_ld;
    const size_t pool = kind != 0 && kept ? pool_at(p, slot, kind == 2) : 0;
#pragma unroll 1
    for (int t = t0; t < t1; t += kBatch) {
      Raw<SRC32> rx[kBatch], ry[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int at = first + (t + u) * stride;
        if (mine && t + u < t1 && at < width) {
          rx[u] = load(src + at);
          if (!ADJ && kind != 2 && paired) ry[u] = load(src + at + half);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int at = first + (t + u) * stride;
        if (!(mine && t + u < t1 && at < width)) continue;
        float v0[8], v1[8] = {};
        values(rx[u], v0);
        if (!ADJ && kind != 2 && paired) {
          values(ry[u], v1);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 c = cs[ADJ ? 0 : i];
            const float e = v0[i];
            v0[i] = e * c.x - v1[i] * c.y;
            v1[i] = v1[i] * c.x + e * c.y;
          }
        } else if (ADJ && kind != 2 && turns) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = v0[2 * i];
            v0[2 * i] = e * cs[i].x - v0[2 * i + 1] * cs[i].y;
            v0[2 * i + 1] = v0[2 * i + 1] * cs[i].x + e * cs[i].y;
          }
        }
        if (kind == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v0[i] *= a.qscale, v1[i] *= a.qscale;
        }
        const uint4 w0 = round16(v0), w1 = round16(v1);
        const bool two = !ADJ && kind != 2 && paired;
        if (kind == 0 || out) {
          *reinterpret_cast<uint4*>(out + at) = w0;
          if (two) *reinterpret_cast<uint4*>(out + at + half) = w1;
        }
        if (kind != 0 && kept) {
          float scale = 1.0f;
          if constexpr (FP8_POOL) scale = a.kv_scales[(size_t(slot.x) * 2 + size_t(kind == 2)) * p.Hkv + at / HD];
          store_pool(pool + at, w0, scale);
          if (two) store_pool(pool + at + half, w1, scale);
        }
      }
    }
  };
  walk(std::integral_constant<int, 0>{}, min(s0, st.q), min(s1, st.q));
  walk(std::integral_constant<int, 1>{}, max(s0 - st.q, 0), min(s1 - st.q, st.k));
  walk(std::integral_constant<int, 2>{}, max(s0 - st.q - st.k, 0), s1 - st.q - st.k);
}

// Rows whose addresses, strides or rotary widths do not allow 16-byte accesses, and maps of more than 256 dims: the same arithmetic, an item is
// two dims - a rotating pair, or past the rotating dims two neighbours.
template <int QDT, bool SRC32, bool FP8_POOL>
__global__ void __launch_bounds__(kThreads) kv_append_narrow_kernel(const AppendArgs args, const int HD) {
  using QE = Elem16<QDT>;
  using T = typename QE::T;
  const esp_kv_append_args& a = args.a;
  const esp_attn_params& p = a.p;
  extern __shared__ float2 turn[];
  const int D = HD / a.maps, half = a.rot_half, row = blockIdx.x;
  pdl_wait();
  for (int f = threadIdx.x; f < half; f += kThreads) turn[f] = turn_of(a.pos[row], a.inv_freq[f]);
  __syncthreads();
  pdl_launch_dependents();
  int2 slot = make_int2(-1, 0);
  const bool kept = a.kv && pool_row(args, row, slot);
  const int n_q = a.Q ? p.H * HD / 2 : 0, n_k = p.Hkv * HD / 2;
  for (int item = blockIdx.y * kThreads + threadIdx.x; item < n_q + 2 * n_k; item += kThreads * gridDim.y) {
    const bool is_q = item < n_q, is_v = item >= n_q + n_k;
    const int rel = is_q ? item : (is_v ? item - n_q - n_k : item - n_q);
    const int head = rel / (HD / 2), in_head = rel - head * (HD / 2), map = in_head / (D / 2), i = in_head - map * (D / 2);
    const bool turns = !is_v && i < half;
    const int d0 = map * D + (turns && !a.adjacent ? i : 2 * i), d1 = d0 + (turns && !a.adjacent ? half : 1);
    const void* src = is_q ? a.Q : (is_v ? a.V : a.K);
    const int64_t at = int64_t(row) * (is_q ? a.q_src_ld : (is_v ? a.v_src_ld : a.k_src_ld)) + int64_t(head) * HD;
    float x, y;
    if constexpr (SRC32) x = static_cast<const float*>(src)[at + d0], y = static_cast<const float*>(src)[at + d1];
    else x = QE::to_f32(static_cast<const T*>(src)[at + d0]), y = QE::to_f32(static_cast<const T*>(src)[at + d1]);
    if (turns) {
      const float2 cs = turn[i];
      const float e = x;
      x = e * cs.x - y * cs.y;
      y = y * cs.x + e * cs.y;
    }
    if (is_q) {
      T* dst = static_cast<T*>(a.Qo) + size_t(row) * p.q_ld + size_t(head) * HD;
      dst[d0] = QE::from_f32(x * a.qscale), dst[d1] = QE::from_f32(y * a.qscale);
      continue;
    }
    const T rx = QE::from_f32(x), ry = QE::from_f32(y);
    if (void* batch = is_v ? a.Vb : a.Kb) {
      T* dst = static_cast<T*>(batch) + size_t(row) * p.kv_ld + size_t(head) * HD;
      dst[d0] = rx, dst[d1] = ry;
    }
    if (!kept) continue;
    const size_t to = pool_at(p, slot, is_v) + size_t(head) * HD;
    if constexpr (FP8_POOL) {
      const float scale = a.kv_scales[(size_t(slot.x) * 2 + is_v) * p.Hkv + head];
      uint8_t* dst = static_cast<uint8_t*>(a.kv) + to;
      dst[d0] = f32_to_e4m3(__fdiv_rn(QE::to_f32(rx), scale)), dst[d1] = f32_to_e4m3(__fdiv_rn(QE::to_f32(ry), scale));
    } else {
      T* dst = static_cast<T*>(a.kv) + to;
      dst[d0] = rx, dst[d1] = ry;
    }
  }
}

template <int QDT, bool SRC32, bool FP8_POOL>
cudaError_t launch_typed(const AppendArgs& args, int32_t HD, cudaStream_t stream) {
  const esp_kv_append_args& a = args.a;
  const size_t ssz = SRC32 ? 4 : 2;
  auto ok16 = [](const void* q, int64_t row_bytes) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && row_bytes % 16 == 0; };
  const int D = HD / a.maps, n_pair = a.adjacent ? 0 : a.rot_half / 8, per_map = a.adjacent ? D / 8 : n_pair + (D - 2 * a.rot_half) / 8;
  const bool wide = (a.adjacent ? a.rot_half % 4 : a.rot_half % 8) == 0 && per_map <= 32 && ok16(a.Q, a.q_src_ld * int64_t(ssz)) &&
                    ok16(a.K, a.k_src_ld * int64_t(ssz)) && ok16(a.V, a.v_src_ld * int64_t(ssz)) && ok16(a.Qo, 0) && ok16(a.Kb, 0) && ok16(a.Vb, 0) && ok16(a.kv, 0);
  if (!wide) {
    const int items = ((a.Q ? a.p.H : 0) + 2 * a.p.Hkv) * HD / 2;
    const unsigned gy = unsigned(std::clamp(4 * 148 / a.rows, 1, (items + kThreads - 1) / kThreads));
    return launch_pdl(kv_append_narrow_kernel<QDT, SRC32, FP8_POOL>, dim3(unsigned(a.rows), gy), dim3(kThreads), size_t(a.rot_half) * sizeof(float2), stream, args, HD);
  }
  Steps st{};
  while ((1 << st.log_p2) < per_map) ++st.log_p2;
  const int maps_per_step = 32 >> st.log_p2;
  st.q = a.Q ? (a.p.H * a.maps + maps_per_step - 1) / maps_per_step : 0;
  st.k = (a.p.Hkv * a.maps + maps_per_step - 1) / maps_per_step;
  st.v = (a.p.Hkv * HD / 8 + 31) / 32;
  st.n_pair = n_pair, st.per_map = per_map;
  // Rows that do not fill the SMs' warps (about 16 an SM) are cut into parts of at least one batch, single tokens down to one step.
  const int steps = st.q + st.k + st.v;
  const int64_t want = 148 * 16;
  const int least = a.rows * int64_t(steps) <= want ? 1 : kBatch;
  st.parts = int(std::clamp<int64_t>((want + a.rows - 1) / a.rows, 1, (steps + least - 1) / least));
  // One and a bit times the warps that the SMs hold would leave them half empty the second time: such rows are halved. (5001 fp32 rows of
  // H16 / Hkv2 / HD256: 36.8 -> 34.4 us. Elsewhere the sines formed twice cost more: 3000 rows 13.9 -> 15.0 us, 6000 67.1 -> 72.2, 8192 34.5 ->
  // 35.9.)
  const int64_t wave = 148 * 6 * kWarps;
  if (a.rows > wave && 2 * int64_t(a.rows) <= 3 * wave) st.parts = std::min(2, steps);
  st.per_part = (steps + st.parts - 1) / st.parts;
  st.parts = (steps + st.per_part - 1) / st.per_part;
  const int64_t tasks = int64_t(a.rows) * st.parts;
  return launch_pdl(a.adjacent ? kv_append_kernel<QDT, SRC32, FP8_POOL, true> : kv_append_kernel<QDT, SRC32, FP8_POOL, false>, dim3(unsigned((tasks + kWarps - 1) / kWarps)), dim3(kThreads), 0, stream, args, st, HD);
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
