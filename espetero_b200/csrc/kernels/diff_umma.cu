// Differential attention on the 5th-generation tensor cores (sm_100a), 128-dim heads: prefill, chunks behind a prefix, draft trees.
//
// A CTA owns 128 (row, head) pairs - tile_rows rows x 128 / tile_rows heads of one kv head - and both softmax maps of each:
//   S_c[128 x 64] = Q_c . K_c^T    c = 1, 2: 4 tcgen05.mma each over map c's 64 dims, which are one 64-dim chunk of the Q and K tiles
//   P_c = exp2(scale (S_c - m_c))  one softmax warpgroup per map, thread i = row i
//   O_c[128 x 128] += P_c . V      4 tcgen05.mma, A = P_c from tensor memory, B = V from shared memory: one V tile for both maps
// P_c is written over S_c as 16-bit pairs (the MMA takes A and B in one 16-bit type; the row sums stay fp32 and unrounded).
//
// Tensor memory: O_1, O_2 (128 fp32 columns each) and two buffers of 64 columns for each S_c: all 512. Tiles of 128 keys are worked on
// in halves of 64: while a warpgroup is on one half of its map, the other's scores are being made or wait, so it never sits through
// P . V and the next Q . K^T. With one buffer of 128 columns per map it did: 2 x 8192 causal rows (H16) took 1068 us instead of
// 932. (An instruction of 64 columns takes about as long as one of 128, so Q . K^T costs twice its share; the pipe has room.)
// (P . V has a barrier per buffer too: a warpgroup that hands over its last unit may still have two of them in flight.)
// O is rescaled only when a row's maximum grows by more than 2^8; its owner then waits for the P . V in flight.
// After the last unit the maps meet: each warpgroup hands half of its normalised O to the other through shared memory, and both
// finish 64 columns of D = O_1 / l_1 - lam O_2 / l_2 and its norm.
//
// Bound: per 128 keys the exponentials of two maps (2 * 128 * 128 at 16 a clock: 2048 clocks of the special-function unit), 1800
// clocks of MMA, 1800 clocks of the shared-memory port (224 KB of operands and tiles).
// One CTA per SM. Warps 0-3 softmax of map 1, 4-7 of map 2, 8 MMA issue (owns tensor memory), 9 / 10 K / V producers (TMA, one load
// per 16-key page and 64-dim chunk). Hand-offs by mbarrier; every wait is bounded: after a timeout the CTA records a code, stops
// waiting, finishes its loop, frees its tensor memory and returns.
// E4M3 pools (F8): the pages are 16-bit codes (diff_widen.cu); the K producer leaves each block's page scales in shared memory, the
// K scale goes on the score and the V scale on the weight.
#include "diff_tile.cuh"

namespace esp {
namespace {

using namespace difft;

constexpr int HD = 128;
constexpr int CHUNK = 128 * 128;                 // bytes of a 64-dim chunk of a tile: [128 rows][128 B]
constexpr int TILE = 2 * CHUNK;                  // Q, K or V tile
constexpr int KS = 3, VS = 3;                    // ring depths: 192 KB in flight for prefixes streamed from HBM
constexpr int TILES_BYTES = (1 + KS + VS) * TILE;
constexpr int BU = 64;                           // keys per half block
constexpr uint32_t COL_S = 0, COL_O = 256;       // S_c, buffer i at COL_S + 128 c + 64 i (P_c over its first 32 columns), O_c at COL_O + 128 c
constexpr float kGrow = 8.0f;                    // log2 units a row's maximum may grow before O is rescaled
constexpr int kSoftmax = 256, kMmaWarp = 8, kWarpK = 9, kWarpV = 10, kThreads = 352;

struct Shared {
  uint64_t k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full[2][2], p_full[2][2], o_done[2][2], sc_full[kScaleSlots];
  uint32_t tmem;
  volatile int dead;
  float k_scale[kScaleSlots][kPages], v_scale[kScaleSlots][kPages];
};
constexpr int SMEM = TILES_BYTES + 1024;
static_assert(sizeof(Shared) <= 1024, "bookkeeping behind the tiles");
static_assert(kScaleSlots > KS + 2, "page scales must outlive their readers");

template <int QDT, bool F8>
__global__ void __launch_bounds__(kThreads, 1)
    diff_umma_kernel(const __grid_constant__ CUtensorMap pool_map, const __grid_constant__ CUtensorMap kb_map, const __grid_constant__ CUtensorMap vb_map,
                     const DiffArgs args) {
  using QE = Elem16<QDT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem + TILES_BYTES);
  const KernelArgs& a = args.k;
  const esp_attn_params& p = a.p;
  uint8_t* q_sm = smem;
  uint8_t* k_sm = smem + TILE;
  uint8_t* v_sm = smem + (1 + KS) * TILE;
  if ((smem_u32(smem) & 1023u) != 0) {  // never expected; the swizzle would be wrong
    if (threadIdx.x == 0) atomicExch(a.status, kStatusBadBlock);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < KS; ++s) mbar_init(&sh.k_full[s], kPages), mbar_init(&sh.k_empty[s], 1);
    for (int s = 0; s < VS; ++s) mbar_init(&sh.v_full[s], kPages), mbar_init(&sh.v_empty[s], 1);
    for (int c = 0; c < 2; ++c)
      for (int i = 0; i < 2; ++i) mbar_init(&sh.s_full[c][i], 1), mbar_init(&sh.p_full[c][i], BM), mbar_init(&sh.o_done[c][i], 1);
    for (int s = 0; s < kScaleSlots; ++s) mbar_init(&sh.sc_full[s], 1);
    mbar_fence_init();
    sh.dead = 0;
  }
  __syncthreads();
  pdl_wait();  // the plan, Q and the mask records belong to the stream's order

  const esp_attn_tile tile = a.tiles[int(gridDim.x) - 1 - int(blockIdx.x)];  // long (late) tiles first
  const esp_attn_tree tree = a.trees[tile.tree];
  const int G = a.G, TR = a.tile_rows, HPC = BM / TR;
  const int kvh = (int(blockIdx.y) * HPC) / G;
  const int end = tree.base + tree.M, rows_live = min(TR, end - tile.r0);
  const BlockList L = block_list(a, tile, tree, rows_live, lane);
  const int nb = L.n();

  auto wait_bar = [&](uint64_t* bar, uint32_t parity, int code) {
    if (mbar_try_wait(bar, parity) || sh.dead) return;
    if (!mbar_wait(bar, parity)) {
      sh.dead = 1;
      atomicExch(a.status, code);
    }
  };

  if (warp == kWarpK || warp == kWarpV) {
    const bool is_v = warp == kWarpV;
    if (lane == 0) tma_prefetch_desc(is_v ? &vb_map : &kb_map), tma_prefetch_desc(&pool_map);
    const int depth = is_v ? VS : KS;
    uint64_t* full = is_v ? sh.v_full : sh.k_full;
    uint64_t* empty = is_v ? sh.v_empty : sh.k_empty;
    uint8_t* ring = is_v ? v_sm : k_sm;
    int stage = 0;
    uint32_t par = 1;  // the first use of a slot finds it empty
    walk_pages<F8>(a, tree, L, is_v ? 1 : 0, lane, [&](int b, int kind, int y, int blk) {
      uint8_t* dst = ring + stage * TILE + lane * 2048;
      float ks = 1.0f, vs = kind < 0 ? 0.0f : 1.0f;
      if (F8 && !is_v && kind == 0) {
        ks = a.kv_scales[size_t(blk) * 2 * p.Hkv + kvh];
        vs = a.kv_scales[(size_t(blk) * 2 + 1) * p.Hkv + kvh];
      }
      wait_bar(&empty[stage], par, kStatusMmaTimeout);
      if (kind < 0) {
        mbar_arrive(&full[stage]);
      } else {
        const CUtensorMap* m = kind ? (is_v ? &vb_map : &kb_map) : &pool_map;
        mbar_arrive_expect_tx(&full[stage], 4096);
        tma_load_3d(dst, m, &full[stage], 0, y, kvh * 2);
        tma_load_3d(dst + CHUNK, m, &full[stage], 0, y, kvh * 2 + 1);
      }
      if (F8 && !is_v) {
        // The slot's last readers are done: a K slot is released once Q . K^T of its block is, two units ahead of the softmax at
        // most, so the producer is at most KS + 2 blocks ahead of it, and there are more slots than that.
        const int slot = b % kScaleSlots;
        sh.k_scale[slot][lane] = ks, sh.v_scale[slot][lane] = vs;
        __syncwarp(0xFFu);
        if (lane == 0) mbar_arrive(&sh.sc_full[slot]);
      }
      if (++stage == depth) stage = 0, par ^= 1;
    });
  } else if (warp == kMmaWarp) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
    tc_fence_before_sync();
    named_barrier(1, kSoftmax + 32);  // Q is staged, tensor memory allocated
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    if (nb > 0) {
      const uint32_t one = elect_one();
      constexpr uint32_t idesc_qk = umma_idesc<QDT>(BM, BU, 0, 0), idesc_pv = umma_idesc<QDT>(BM, HD, 0, 1);
      const uint64_t q_desc = umma_smem_desc(smem_u32(q_sm), 16, 1024), k_desc = umma_smem_desc(smem_u32(k_sm), 16, 1024);
      const uint64_t v_desc = umma_smem_desc(smem_u32(v_sm), CHUNK, 1024);
      const uint32_t q_lo = uint32_t(q_desc), k_lo0 = uint32_t(k_desc), v_lo0 = uint32_t(v_desc);
      const uint32_t hi_qk = uint32_t(q_desc >> 32), hi_v = uint32_t(v_desc >> 32);
      int kst = 0, vst = 0;
      uint32_t kpar = 0, vpar = 0;
      // S_c of the half h of the block in K slot kst
      auto issue_qk = [&](int c, int h) {
        if (c == 0 && h == 0) {
          wait_bar(&sh.k_full[kst], kpar, kStatusTmaTimeout);
          tc_fence_after_sync();
        }
        const uint32_t k_lo = k_lo0 + uint32_t(kst) * (TILE >> 4);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma_ss(one, tmem + COL_S + c * 128 + h * BU, q_lo + ((c * CHUNK + ks * 32) >> 4), hi_qk, k_lo + ((c * CHUNK + h * (BU * 128) + ks * 32) >> 4), hi_qk, idesc_qk, ks > 0);
        mma_commit(one, &sh.s_full[c][h]);
        if (c == 1 && h == 1) {
          mma_commit(one, &sh.k_empty[kst]);
          if (++kst == KS) kst = 0, kpar ^= 1;
        }
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) issue_qk(0, h), issue_qk(1, h);
#pragma unroll 1
      for (int b = 0; b < nb; ++b) {
        const uint32_t v_lo = v_lo0 + uint32_t(vst) * (TILE >> 4), more = b > 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            wait_bar(&sh.p_full[c][h], b & 1, kStatusMmaTimeout);
            if (c == 0 && h == 0) wait_bar(&sh.v_full[vst], vpar, kStatusTmaTimeout);
            tc_fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < BU / 16; ++ks)
              mma_ts(one, tmem + COL_O + c * HD, tmem + COL_S + c * 128 + h * BU + ks * 8, v_lo + ((h * (BU * 128) + ks * 16 * 128) >> 4), hi_v, idesc_pv, (h > 0 || ks > 0) ? 1u : more);
            mma_commit(one, &sh.o_done[c][h]);
            if (c == 1 && h == 1) mma_commit(one, &sh.v_empty[vst]);
            if (b + 1 < nb) issue_qk(c, h);  // the next block's half, over P_c: behind the P_c . V that reads it
          }
        }
        if (++vst == VS) vst = 0, vpar ^= 1;
      }
    }
  } else if (warp < kMmaWarp) {
    const int map = tid >> 7, srow = tid & (BM - 1), fm = srow / HPC, head = int(blockIdx.y) * HPC + srow % HPC;
    const bool row_ok = fm < rows_live;
    const int row = row_ok ? tile.r0 + fm : end - 1, rr = row - tree.base;
    int4 dsc = make_int4(0, 0, 0, 0);
    uint64_t am = 0;
    const bool use_anc = a.anc_mask != nullptr;
    {
      // this thread's half of its Q row - its map's 64 dims - into the map's chunk (K-major, 128-byte swizzle)
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const typename QE::T*>(a.Q) + size_t(row) * p.q_ld + size_t(head) * HD + map * 64);
      uint8_t* qd = q_sm + map * CHUNK + srow * 128;
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(qd + ((i ^ (srow & 7)) << 4)) = src[i];
      fence_proxy_async_smem();
      if (tile.last) {
        if (use_anc) am = a.anc_mask[row];
        else dsc = reinterpret_cast<const int4*>(a.desc)[row];
      }
    }
    tc_fence_before_sync();
    named_barrier(1, kSoftmax + 32);
    tc_fence_after_sync();
    const uint32_t t_lane = sh.tmem + (uint32_t((warp & 3) * 32) << 16);  // this warp's quarter of the lanes
    const uint32_t t_s = t_lane + COL_S + map * 128, t_o = t_lane + COL_O + map * HD;
    const float sl2 = a.scale * kLog2e;
    float m_ref = -INFINITY, l_run = 0.0f, v_ref = F8 ? 0.0f : 1.0f;
    int vst = 0;
    uint32_t vpar = 0;
    const uint64_t sl2x2 = f32x2_pack(sl2, sl2);
    for (int b = 0; b < nb; ++b) {
      const bool whole = L.whole(b);
      const uint32_t par = b & 1;
      if constexpr (F8) wait_bar(&sh.sc_full[b % kScaleSlots], uint32_t(b / kScaleSlots) & 1u, kStatusTmaTimeout);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t buf = t_s + h * BU;
        wait_bar(&sh.s_full[map][h], par, kStatusMmaTimeout);
        tc_fence_after_sync();
        uint32_t s0[32], s1[32];
        tmem_ld32(buf, s0);
        tmem_ld32(buf + 32, s1);
        tmem_wait_ld_of(s0);
        tmem_wait_ld_of(s1);
        float vfac = 1.0f, vs[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (F8) {
          float ks[4], largest = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ks[i] = sh.k_scale[b % kScaleSlots][4 * h + i], vs[i] = sh.v_scale[b % kScaleSlots][4 * h + i];
            largest = fmaxf(largest, vs[i]);
          }
          vfac = follow_scale(v_ref, largest);
          const float inv = pow2_inverse(v_ref);
#pragma unroll
          for (int i = 0; i < 4; ++i) vs[i] *= inv;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            s0[i] = __float_as_uint(__uint_as_float(s0[i]) * ks[i >> 4]);
            s1[i] = __float_as_uint(__uint_as_float(s1[i]) * ks[2 + (i >> 4)]);
          }
        }
        if (!whole) {
          hide_columns(L, b, h * BU, dsc, am, use_anc, rr, s0, s1);
          const int first = max(L.n_valid(b), h * BU), n = (h + 1) * BU - first;
          if (map == 0 && n > 0) {
            // V rows past the range are stale or foreign: 0 * NaN must not happen. Map 1's warpgroup clears the half's before it hands
            // over P_1; P_2 . V is issued after P_1 . V.
            wait_bar(&sh.v_full[vst], vpar, kStatusTmaTimeout);
            for (int i = srow; i < n * 16; i += BM) {
              const int r = first + i / 16, c = i % 16;
              *reinterpret_cast<uint4*>(v_sm + vst * TILE + (c >> 3) * CHUNK + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        const float mx = sl2 * fmaxf(chunk_max(s0), chunk_max(s1));  // scale > 0
        float factor = vfac;
        const bool grow = mx > m_ref + kGrow;  // also the first finite maximum
        if (grow) {
          const float f = fast_exp2(m_ref - mx);
          factor *= f, l_run *= f;
          m_ref = mx;
        }
        if ((b > 0 || h > 0) && __any_sync(0xffffffffu, grow || vfac != 1.0f)) {
          wait_bar(&sh.o_done[map][h ^ 1], h ? par : par ^ 1, kStatusMmaTimeout);  // every half before this one is in O_c
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * c, o);
            tmem_wait_ld_of(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
            tmem_st32(t_o + 32 * c, o);
          }
        }
        const float neg_m = m_ref == -INFINITY ? 0.0f : -m_ref;
        const uint64_t neg_m2 = f32x2_pack(neg_m, neg_m);
        uint64_t sum[2] = {f32x2_pack(0.0f, 0.0f), f32x2_pack(0.0f, 0.0f)};
        uint32_t pk[32];
        chunk_weights<QDT, F8>(s0, pk, sl2x2, neg_m2, sum, vs[0], vs[1]);
        chunk_weights<QDT, F8>(s1, pk + 16, sl2x2, neg_m2, sum, vs[2], vs[3]);
        tmem_st32(buf, pk);
        float a0, a1;
        f32x2_unpack(f32x2_add(sum[0], sum[1]), a0, a1);
        l_run += a0 + a1;
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(&sh.p_full[map][h]);
      }
      if (++vst == VS) vst = 0, vpar ^= 1;
    }

    // ---- epilogue
    pdl_launch_dependents();
    if (nb > 0) {
      wait_bar(&sh.o_done[map][1], (nb - 1) & 1, kStatusMmaTimeout);
      tc_fence_after_sync();
    }
    auto load_o = [&](int col, float (&v)[32]) {
      if (nb > 0) {
        uint32_t o[32];
        tmem_ld32(t_o + col, o);
        tmem_wait_ld_of(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.0f;
      }
    };
    if (tile.part >= 0) {
      float* rec = a.parts + diff_record(a, tile.part, kvh, fm, head % G, map);
      const float unit = F8 && nb > 0 ? v_ref : 1.0f;
#pragma unroll 1
      for (int col = 0; col < HD; col += 32) {
        float v[32];
        load_o(col, v);
        if (row_ok) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) *reinterpret_cast<float2*>(rec + col + i) = make_float2(v[i] * unit, v[i + 1] * unit);
        }
      }
      if (row_ok) *reinterpret_cast<float2*>(rec + HD) = make_float2(m_ref * kLn2, l_run);
    } else {
      // map 1 takes columns [0, 64), map 2 [64, 128): each hands the other's half over in shared memory ([column][row]: lanes side
      // by side), already divided by its sum (and times lam). The K tiles are spent: every Q . K^T came before the last P . V.
      float* give = reinterpret_cast<float*>(k_sm) + (map ^ 1) * 64 * BM;
      const float* take = reinterpret_cast<const float*>(k_sm) + map * 64 * BM;
      float* sq = reinterpret_cast<float*>(v_sm);  // both warpgroups have seen their last P . V at the barrier below
      const float inv = l_run > 0.0f ? (map ? -diff_lam(args, row, head) : 1.0f) * (F8 ? v_ref : 1.0f) / l_run : 0.0f;
#pragma unroll 1
      for (int q = 0; q < 2; ++q) {
        float v[32];
        load_o(64 * (map ^ 1) + 32 * q, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) give[(32 * q + i) * BM + srow] = v[i] * inv;
      }
      float dv[64];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float v[32];
        load_o(64 * map + 32 * q, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) dv[32 * q + i] = v[i] * inv;
      }
      named_barrier(2, kSoftmax);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        dv[i] += take[i * BM + srow];
        ss = fmaf(dv[i], dv[i], ss);
      }
      sq[map * BM + srow] = ss;
      named_barrier(2, kSoftmax);
      const float f = diff_row_factor(args, ss + sq[(map ^ 1) * BM + srow], HD);
      if (row_ok) {
        typename QE::T* op = static_cast<typename QE::T*>(a.O) + size_t(row) * p.q_ld + size_t(head) * HD + map * 64;
        const float* w = args.norm_w ? args.norm_w + map * 64 : nullptr;
#pragma unroll
        for (int i = 0; i < 64; i += 8) {
          float x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = dv[i + k] * f * (w ? w[i + k] : 1.0f);
          *reinterpret_cast<uint4*>(op + i) = make_uint4(QE::pack2(x[0], x[1]), QE::pack2(x[2], x[3]), QE::pack2(x[4], x[5]), QE::pack2(x[6], x[7]));
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(sh.tmem, 512);
}

}  // namespace

// 128 / tile_rows heads of a tile must belong to one kv head.
bool diff_umma_supports(int32_t HDim, int32_t G, int32_t tile_rows, int32_t bt) {
  if (HDim != HD || bt <= 0 || bt % 16 != 0) return false;
  if (tile_rows != 16 && tile_rows != 32 && tile_rows != 64 && tile_rows != 128) return false;
  const int hpc = BM / tile_rows;
  return hpc <= G && G % hpc == 0;
}

cudaError_t diff_umma_setup() {
  cudaError_t e = cudaFuncSetAttribute(diff_umma_kernel<ESP_F16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(diff_umma_kernel<ESP_BF16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(diff_umma_kernel<ESP_F16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(diff_umma_kernel<ESP_BF16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  return e;
}

cudaError_t launch_diff_umma(const DiffArgs& a, bool f8, const CUtensorMap& pool_map, const CUtensorMap& kb_map, const CUtensorMap& vb_map, cudaStream_t stream,
                             uint64_t* launches) {
  if (a.k.n_tiles <= 0) return cudaSuccess;
  const dim3 grid(unsigned(a.k.n_tiles), unsigned(a.k.p.H / (BM / a.k.tile_rows)));
  const bool f16 = a.k.q_dtype == ESP_F16;
  auto kernel = f8 ? (f16 ? diff_umma_kernel<ESP_F16, true> : diff_umma_kernel<ESP_BF16, true>) : (f16 ? diff_umma_kernel<ESP_F16, false> : diff_umma_kernel<ESP_BF16, false>);
  const cudaError_t e = launch_pdl(kernel, grid, dim3(kThreads), SMEM, stream, pool_map, kb_map, vb_map, a);
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
