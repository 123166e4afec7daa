// Differential attention on the 5th-generation tensor cores (sm_100a), 128- and 256-dim heads: prefill, chunks behind a prefix, draft
// trees.
//
// A tile is 128 (row, head) pairs - tile_rows rows x 128 / tile_rows heads of one kv head. Two CTAs, a cluster, work on it, one per
// softmax map c:
//   S_c[128 x BU] = Q_c . K_c^T   tcgen05.mma over the map's HD / 2 dims: its own half of the Q and K tiles, so nothing is computed twice
//   P_c = exp2(scale (S_c - m_c)) thread = row
//   O_c[128 x HD] += P_c . V      A = P_c from tensor memory (16-bit pairs over S_c: the MMA takes A and B in one 16-bit type; the row
//                                 sums stay fp32 and unrounded), B = V from shared memory
// and the maps meet at the end: each CTA sends half of the columns of its O_c / l_c (map 2's times -lam) into the other's shared memory,
// both add, exchange the rows' sums of squares and write HD / 2 columns of the normalised difference.
//
// Tensor memory holds O_c and two buffers of S_c: with 256-dim heads 256 + 2 x 128 columns, one CTA per SM; with 128-dim heads 128 +
// 2 x 64 (tiles of 128 keys in two units), two CTAs per SM. Two softmax warpgroups take the units in turn, so that one's loads, maxima
// and hand-overs run under the other's exponentials. They share O, hence the rows' reference maxima: a warp reads them from its
// partner (the warp of the other group with the same rows) after its own maximum, and passes them on before its exponentials.
// The reference only moves when a maximum exceeds it by 2^8; the warp that moves it rescales its rows of O, after the P . V of the unit
// before.
//
// Bound per 128 keys of a tile: 256-dim heads 1536 clocks of MMA per map (8 instructions of N = 128 and 8 of N = 256, 64 and 128
// clocks each) on an SM, 1024 of exponentials; 128-dim heads 1024 of exponentials per map, two maps per SM, against 1600 of MMA.
// Measured, causal rows of 16 heads: 128 dims, 4096 rows 129 us (797 TFLOP/s), 8192 rows 421 us (979); 256 dims 199 us (1035) and 655 us
// (1260). 256-dim heads run at 1800 clocks a unit, 85 % of the MMA bound, but one CTA per SM hides nothing of a CTA's start and end:
// 6 k clocks until the first scores (plan, masks and page table, one dependent load after another), 14 k for the last P . V, the
// exchange of halves (64 KB each way at 21 bytes a clock) and the output. 128-dim heads hide that under the SM's other CTA; there the
// exponentials' pipe is 54 % busy and the issue slots 53 %: a warp's chain of load, maximum, exponentials and store is what four
// warps per scheduler do not cover. Dropped: both maps in one CTA, a warpgroup each, K and V loaded once (2 x 8192 rows, H16: 953 us
// against 880; with the next scores fetched ahead 1009), turns between the maps by barrier (970), exponentials by polynomial on the FMA
// pipe (equal or slower).
// Warps 0-7 softmax, 8 MMA issue (owns tensor memory), 9 / 10 K / V producers (TMA, one load per 16-key page and 64-dim chunk of the pool,
// one per 64 or 128 rows of the batch; the Q tile, too, where it is 128 rows of one head), 11 idle (it
// completes the warpgroup that hands registers over). Hand-offs by mbarrier; every wait is bounded: after a timeout the CTA records a
// code, stops waiting, asks for no more copies, finishes its loop, gives copies and MMAs under way a millisecond, frees its tensor memory and
// returns. (A flag on the MMA warp's issue cost 4 % of every pass; its queue holds few MMAs at a time.)
// E4M3 pools (F8): the pages are 16-bit codes (diff_widen.cu); the K producer leaves each block's page scales in shared memory, the
// K scale goes on the score and the V scale on the weight, whose reference is the largest product of the two.
#include "diff_tile.cuh"

namespace esp {
namespace {

using namespace difft;

constexpr float kGrow = 8.0f;  // log2 units a row's maximum may grow before O is rescaled
constexpr int kSoftmax = 256, kMmaWarp = 8, kWarpK = 9, kWarpV = 10, kThreads = 384;
constexpr int KS = 2;          // K ring, in tiles of 128 keys

template <int HD_>
struct Geo {
  static constexpr int HD = HD_, MAP = HD / 2;
  static constexpr int CHUNK = 128 * 128;          // bytes of a 64-dim chunk of a tile: [128 rows][128 B]
  static constexpr int QC = MAP / 64, VC = HD / 64;  // chunks of a Q or K tile (one map), of a V tile
  // V ring, two blocks deep. 256-dim heads: slots of 64 keys, refilled while the other half of their block is still read (8192 causal
  // rows, H16: 677 -> 652 us); 128-dim heads: whole blocks (halves cost the producers more than they gave: 700 rows behind 20001
  // E4M3 keys 592 us against 647).
  static constexpr int VK = HD == 256 ? 64 : 128, SPB = BN / VK, VS = 2 * SPB;
  static constexpr int V_CHUNK = VK * 128;         // bytes of a 64-dim chunk of a V slot: [VK rows][128 B]
  static constexpr int K_TILE = QC * CHUNK, V_SLOT = VC * V_CHUNK;
  static constexpr int TILES = (1 + KS) * K_TILE + VS * V_SLOT;
  static constexpr int BU = HD == 256 ? 128 : 64;  // keys per unit
  static constexpr int UPB = BN / BU;              // units per block
  static constexpr int SMEM = TILES + (HD == 256 ? 2048 : 1024);  // two CTAs of 113 KB (and the 1 KB each that is taken for them) fill an SM
  static constexpr int PART = BU / 2;              // keys whose weights are handed over together
  static constexpr uint32_t COL_O = 0, COL_S = HD; // S buffer i at COL_S + BU i (P over its first BU / 2 columns)
  static constexpr uint32_t COLS = HD + 2 * BU;    // 512 or 256
  static constexpr int CTAS = HD == 256 ? 1 : 2;   // per SM
  // 256-dim heads: a softmax thread holds its 128 scores; the last warpgroup hands registers over (128 x 96 + 256 x 200 <= 384 x 168).
  // 128-dim heads: two CTAs leave 80 registers a thread, so a unit's 64 scores are read twice, 32 at a time: for the maximum, then for
  // the weights. (Held at once, with 96 registers for the softmax threads, they spilled: 2 x 8192 rows, H16, took 2255 us instead of 944.)
  static constexpr bool HOLD = HD == 256;
};

constexpr int kRegsAux = 96, kRegsSoftmax = 200;  // 256-dim heads
// Blocks whose page scales are kept. The producer writes those of block b + 4 once
// K tile b + 2 is released, that is once its last unit's Q . K^T is through, which is issued behind the P . V of two units before: of a
// unit of block b + 1, or with one unit per block of block b. The readers of block b are then done.
constexpr int kSlots = 4;
static_assert(kSlots >= KS + 2, "page scales must outlive their readers");
template <int VS>
struct Shared {
  uint64_t q_full, k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full[2], p_full[2][2], o_done[2], sc_full[kSlots], m_ready[2], take_full;
  uint32_t tmem;
  volatile int dead;
  float k_scale[kSlots][kPages], v_scale[kSlots][kPages];
  float m_ref[BM];
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_store(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
// Asynchronous copy into the peer's shared memory; its barrier counts the bytes.
__device__ __forceinline__ void peer_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(smem_u32(src)), "r"(bytes), "r"(bar) : "memory");
}

template <int HD, int QDT, bool F8>
__global__ void __launch_bounds__(kThreads, Geo<HD>::CTAS)
    diff_umma_kernel(const __grid_constant__ CUtensorMap pool_map, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kb_map,
                     const __grid_constant__ CUtensorMap vb_map, const DiffArgs args) {
  using C = Geo<HD>;
  using QE = Elem16<QDT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  using Sh = Shared<C::VS>;
  constexpr int VS = C::VS;
  static_assert(C::TILES + int(sizeof(Sh)) <= C::SMEM, "bookkeeping behind the tiles");
  Sh& sh = *reinterpret_cast<Sh*>(smem + C::TILES);
  const KernelArgs& a = args.k;
  const esp_attn_params& p = a.p;
  uint8_t* q_sm = smem;
  uint8_t* k_sm = smem + C::K_TILE;
  uint8_t* v_sm = smem + (1 + KS) * C::K_TILE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int map = int(blockIdx.z);  // = rank in the cluster
  if (tid == 0) {
    if ((smem_u32(smem) & 1023u) != 0) atomicExch(a.status, kStatusBadBlock);  // never expected; the swizzle would be wrong
    mbar_init(&sh.q_full, 1);
    for (int s = 0; s < KS; ++s) mbar_init(&sh.k_full[s], kPages), mbar_init(&sh.k_empty[s], 1);
    for (int s = 0; s < VS; ++s) mbar_init(&sh.v_full[s], kPages / C::SPB), mbar_init(&sh.v_empty[s], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1), mbar_init(&sh.p_full[i][0], BM), mbar_init(&sh.p_full[i][1], BM), mbar_init(&sh.o_done[i], 1);
      mbar_init(&sh.m_ready[i], 4);
    }
    for (int s = 0; s < kSlots; ++s) mbar_init(&sh.sc_full[s], 1);
    mbar_init(&sh.take_full, 1);
    mbar_fence_init();
    sh.dead = 0;
  }
  // While the kernel before this one drains: the lines that the first steps read, one address after another, are brought into L2, every
  // index checked. A stale plan costs a wasted hint, never a result.
  const int groups = p.H / (BM / a.tile_rows);
  const esp_attn_tile* my_tile = a.tiles + (a.n_tiles - 1 - int(blockIdx.x) / groups);
  if (warp == kWarpK) {
    const int4 t0 = __ldcg(reinterpret_cast<const int4*>(my_tile));  // tree, r0, k0, k1
    if (t0.x >= 0 && t0.x < a.n_trees) {
      const int4 tr = __ldcg(reinterpret_cast<const int4*>(a.trees + t0.x));  // base, P, table, M
      const long long row = (long long)t0.y + lane * 8;  // eight records to a line
      if (a.desc && t0.y >= 0 && lane * 8 < a.tile_rows && row < args.n_rows) prefetch_l2(a.desc + 4 * row);
      const long long at = (long long)tr.z + t0.z / p.bt + lane * 32;
      if (a.blocks && tr.z >= 0 && t0.z >= 0 && t0.z + lane * 32 * p.bt < t0.w && at < a.n_block_entries) prefetch_l2(a.blocks + at);
    }
  }
  __syncthreads();
  pdl_wait();  // the plan, Q and the mask records belong to the stream's order

  // Long (late) tiles first, a tile's heads side by side: what runs last is short.
  const int G = a.G, TR = a.tile_rows, HPC = BM / TR;
  const esp_attn_tile tile = *my_tile;
  const esp_attn_tree tree = a.trees[tile.tree];
  const int head0 = (int(blockIdx.x) % groups) * HPC;  // the tile's heads, all of one kv head
  const int kvh = head0 / G;
  const int end = tree.base + tree.M, rows_live = min(TR, end - tile.r0);
  const BlockList L = block_list(a, tile, tree, rows_live, lane);
  const int nb = L.n(), N = nb * C::UPB;
  const bool whole_rows = tile.part < 0;

  auto wait_bar = [&](uint64_t* bar, uint32_t parity, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    if (sh.dead) return false;
    if (mbar_wait(bar, parity)) return true;
    sh.dead = 1;
    atomicExch(a.status, code);
    return false;
  };

  if (warp >= kMmaWarp) {
    if constexpr (C::HOLD) regs_dec<kRegsAux>();
    if (warp == kWarpK || warp == kWarpV) {
      const bool is_v = warp == kWarpV;
      if (lane == 0) tma_prefetch_desc(is_v ? &vb_map : &kb_map), tma_prefetch_desc(&pool_map);
      // One code for both: two copies of the walk cost 4 to 5 % of a pass over cached pages.
      const int depth = is_v ? VS : KS, step = is_v ? C::SPB : 1, lanes = is_v ? kPages / C::SPB : kPages;  // slots, slots per block, lanes per slot
      uint64_t* full0 = is_v ? sh.v_full : sh.k_full;
      uint64_t* empty0 = is_v ? sh.v_empty : sh.k_empty;
      const int part = C::SPB > 1 && is_v && lane >= lanes ? 1 : 0, l = lane - part * lanes;  // this lane's slot of the block, its place there
      int stage = 0;
      uint32_t par = 1;  // the first use of a slot finds it empty
      auto advance = [&]() {
        if ((stage += step) == depth) stage = 0, par ^= 1;
      };
      auto scales = [&](int b, float ks, float vs) {  // this lane's page of block b
        if (!F8 || is_v) return;
        const int slot = b % kSlots;
        sh.k_scale[slot][lane] = ks, sh.v_scale[slot][lane] = vs;
        __syncwarp(0xFFu);
        if (lane == 0) mbar_arrive(&sh.sc_full[slot]);
      };
      if (!is_v && TR == BM && N > 0 && lane == 0) {  // a tile of one head: its Q rows are contiguous, too
        mbar_arrive_expect_tx(&sh.q_full, C::K_TILE);
#pragma unroll
        for (int i = 0; i < C::QC; ++i) tma_load_3d(q_sm + i * C::CHUNK, &q_map, &sh.q_full, 0, tile.r0, head0 * C::VC + map * C::QC + i);
      }
      __syncwarp();
      walk_pages<F8>(
          a, tree, L, is_v ? 1 : 0, lane,
          [&](int b, int kind, int y, int blk) {
            float ks = 1.0f, vs = kind < 0 ? 0.0f : 1.0f;
            if (F8 && !is_v && kind == 0) {
              ks = a.kv_scales[size_t(blk) * 2 * p.Hkv + kvh];
              vs = a.kv_scales[(size_t(blk) * 2 + 1) * p.Hkv + kvh];
            }
            uint64_t* full = full0 + stage + part;
            if (!wait_bar(empty0 + stage + part, par, kStatusMmaTimeout)) {
              // nothing is asked for any more
            } else if (kind < 0) {
              mbar_arrive(full);
            } else if (is_v) {
              uint8_t* dst = v_sm + (stage + part) * C::V_SLOT + l * 2048;
              mbar_arrive_expect_tx(full, 2048 * C::VC);
#pragma unroll
              for (int i = 0; i < C::VC; ++i) tma_load_3d(dst + i * C::V_CHUNK, &pool_map, full, 0, y, kvh * C::VC + i);
            } else {
              uint8_t* dst = k_sm + stage * C::K_TILE + l * 2048;
              mbar_arrive_expect_tx(full, 2048 * C::QC);
#pragma unroll
              for (int i = 0; i < C::QC; ++i) tma_load_3d(dst + i * C::CHUNK, &pool_map, full, 0, y, kvh * C::VC + map * C::QC + i);
            }
            scales(b, ks, vs);
            advance();
          },
          // Batch rows are contiguous: one load per slot and chunk, by as many lanes. (Rows behind the tree's last one come along:
          // other trees' or none, zero past the tensor. Their scores are hidden and their V rows cleared.)
          [&](int b, int y) {
            uint64_t* full = full0 + stage + part;
            if (!wait_bar(empty0 + stage + part, par, kStatusMmaTimeout)) {
            } else if (l < (is_v ? C::VC : C::QC)) {
              mbar_arrive_expect_tx(full, is_v ? C::V_CHUNK : C::CHUNK);
              if (is_v) tma_load_3d(v_sm + (stage + part) * C::V_SLOT + l * C::V_CHUNK, &vb_map, full, 0, y + C::VK * part, kvh * C::VC + l);
              else tma_load_3d(k_sm + stage * C::K_TILE + l * C::CHUNK, &kb_map, full, 0, y, kvh * C::VC + map * C::QC + l);
            } else {
              mbar_arrive(full);
            }
            scales(b, 1.0f, 1.0f);
            advance();
          });
      __syncwarp();
    } else if (warp == kMmaWarp) {
      tmem_alloc(&sh.tmem, C::COLS);
      tmem_relinquish();
      tc_fence_before_sync();
      named_barrier(1, kSoftmax + 32);  // Q is staged, tensor memory allocated
      tc_fence_after_sync();
      const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
      if (N > 0) {
        const uint32_t one = elect_one();
        constexpr uint32_t idesc_qk = umma_idesc<QDT>(BM, C::BU, 0, 0), idesc_pv = umma_idesc<QDT>(BM, HD, 0, 1);
        const uint64_t q_desc = umma_smem_desc(smem_u32(q_sm), 16, 1024), k_desc = umma_smem_desc(smem_u32(k_sm), 16, 1024);
        const uint64_t v_desc = umma_smem_desc(smem_u32(v_sm), C::V_CHUNK, 1024);
        const uint32_t q_lo = uint32_t(q_desc), k_lo0 = uint32_t(k_desc), v_lo0 = uint32_t(v_desc);
        const uint32_t hi_qk = uint32_t(q_desc >> 32), hi_v = uint32_t(v_desc >> 32);
        int kst = 0, vst = 0;
        uint32_t kpar = 0, vpar = 0;
        // S of unit n = (block of K slot kst, half h), into buffer i = n & 1
        auto issue_qk = [&](int h, int i) {
          if (h == 0) {
            wait_bar(&sh.k_full[kst], kpar, kStatusTmaTimeout);
            tc_fence_after_sync();
          }
          const uint32_t k_lo = k_lo0 + uint32_t(kst) * (C::K_TILE >> 4) + uint32_t((h * C::BU * 128) >> 4);
#pragma unroll
          for (int ks = 0; ks < C::MAP / 16; ++ks)
            mma_ss(one, tmem + C::COL_S + i * C::BU, q_lo + (((ks >> 2) * C::CHUNK + (ks & 3) * 32) >> 4), hi_qk, k_lo + (((ks >> 2) * C::CHUNK + (ks & 3) * 32) >> 4), hi_qk,
                   idesc_qk, ks > 0);
          mma_commit(one, &sh.s_full[i]);
          if (h == C::UPB - 1) {
            mma_commit(one, &sh.k_empty[kst]);
            if (++kst == KS) kst = 0, kpar ^= 1;
          }
        };
        if (TR == BM) wait_bar(&sh.q_full, 0, kStatusTmaTimeout);
        issue_qk(0, 0);
        if (N > 1) issue_qk(1 % C::UPB, 1);
#pragma unroll 1
        for (int n0 = 0; n0 < N; n0 += 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = n0 + i, h = i % C::UPB;
            if (n >= N) break;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              constexpr int KSTEPS = C::PART / 16;
              const int key0 = h * C::BU + part * C::PART;  // of the block
              const bool opens = key0 % C::VK == 0, closes = (key0 + C::PART) % C::VK == 0;  // a V slot
              wait_bar(&sh.p_full[i][part], uint32_t(n >> 1) & 1u, kStatusMmaTimeout);
              if (opens) wait_bar(&sh.v_full[vst], vpar, kStatusTmaTimeout);
              tc_fence_after_sync();
              const uint32_t v_lo = v_lo0 + uint32_t(vst) * (C::V_SLOT >> 4) + uint32_t((key0 % C::VK) * 128 >> 4);
#pragma unroll
              for (int ks = 0; ks < KSTEPS; ++ks)
                mma_ts(one, tmem + C::COL_O, tmem + C::COL_S + i * C::BU + (part * KSTEPS + ks) * 8, v_lo + ((ks * 16 * 128) >> 4), hi_v, idesc_pv,
                       part > 0 || ks > 0 ? 1u : uint32_t(n > 0));
              if (closes) {
                mma_commit(one, &sh.v_empty[vst]);
                if (++vst == VS) vst = 0, vpar ^= 1;
              }
            }
            mma_commit(one, &sh.o_done[i]);
            if (n + 2 < N) issue_qk(h, i);  // over P of unit n: behind the P . V that reads it
          }
        }
      }
    }
    if (whole_rows) cluster_sync(), cluster_sync();  // the softmax warps' epilogue
  } else {
    if constexpr (C::HOLD) regs_inc<kRegsSoftmax>();
    const int wg = tid >> 7, srow = tid & (BM - 1), fm = srow / HPC, head = head0 + srow % HPC, wq = warp & 3;
    const bool row_ok = fm < rows_live;
    const int row = row_ok ? tile.r0 + fm : end - 1, rr = row - tree.base;
    int4 dsc = make_int4(0, 0, 0, 0);
    uint64_t am = 0;
    const bool use_anc = a.anc_mask != nullptr;
    if (TR != BM) {
      // the map's dims of this Q row, half of them per warpgroup (K-major, 128-byte swizzle)
      constexpr int LINES = C::MAP / 16;  // 16-byte pieces per thread
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const typename QE::T*>(a.Q) + size_t(row) * p.q_ld + size_t(head) * HD + map * C::MAP);
#pragma unroll
      for (int k = 0; k < LINES; ++k) {
        const int i = wg * LINES + k;
        *reinterpret_cast<uint4*>(q_sm + (i >> 3) * C::CHUNK + srow * 128 + (((i & 7) ^ (srow & 7)) << 4)) = src[i];
      }
      fence_proxy_async_smem();
    }
    if (tile.last) {
      if (use_anc) am = a.anc_mask[row];
      else dsc = row_record(a, row, tree.M);
    }
    tc_fence_before_sync();
    named_barrier(1, kSoftmax + 32);
    tc_fence_after_sync();
    const uint32_t t_lane = sh.tmem + (uint32_t(wq * 32) << 16);  // this warp's quarter of the lanes
    const uint32_t t_o = t_lane + C::COL_O, buf = t_lane + C::COL_S + wg * C::BU;
    const float sl2 = a.scale * kLog2e;
    const uint64_t sl2x2 = f32x2_pack(sl2, sl2);
    float m_seen = -INFINITY, l_run = 0.0f;  // this group's sum, against the reference it last saw
    constexpr int NS = C::BU / 32;
    for (int n = wg; n < N; n += 2) {
      const int b = n / C::UPB, c0 = (n % C::UPB) * C::BU;
      const uint32_t par = uint32_t(n >> 1) & 1u;
      const bool whole = L.whole(b);
      // the reference, from the partner warp that had the unit before: its maximum has long been known when these scores arrive
      float m_old = -INFINITY;
      if (n > 0) {
        wait_bar(&sh.m_ready[wg ^ 1], uint32_t((n - 1) >> 1) & 1u, kStatusMmaTimeout);
        m_old = *const_cast<volatile float*>(&sh.m_ref[srow]);
      }
      float ks[2 * NS] = {}, vs[2 * NS] = {};  // the pages' K scales, times the softmax's, and V scales
      if constexpr (F8) {
        wait_bar(&sh.sc_full[b % kSlots], uint32_t(b / kSlots) & 1u, kStatusTmaTimeout);
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) {
          ks[i] = fmaxf(sl2 * sh.k_scale[b % kSlots][c0 / 16 + i], 1.17549435e-38f), vs[i] = sh.v_scale[b % kSlots][c0 / 16 + i];  // -inf * 0 must not happen
        }
      }
      wait_bar(&sh.s_full[wg], par, kStatusMmaTimeout);
      tc_fence_after_sync();
      // 32 scores, hidden where the row does not see the key; and their maximum in log2 units
      auto shape = [&](uint32_t (&x)[32], int i) {
        if (!whole) hide(x, visible32(L, b, c0 + 32 * i, dsc, am, use_anc, rr));
      };
      auto top = [&](const uint32_t (&x)[32], int i) { return F8 ? chunk_max(x, ks[2 * i], ks[2 * i + 1], log2_floor(vs[2 * i]), log2_floor(vs[2 * i + 1])) : sl2 * chunk_max(x); };  // scale > 0
      constexpr int HELD = C::HOLD ? NS : 1;
      uint32_t s[HELD][32];
      float mx = -INFINITY;
      if constexpr (C::HOLD) {
#pragma unroll
        for (int i = 0; i < NS; ++i) tmem_ld32(buf + 32 * i, s[i]);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          tmem_wait_ld_of(s[i]);
          shape(s[i], i);
          mx = fmaxf(mx, top(s[i], i));
        }
      } else {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          tmem_ld32(buf + 32 * i, s[0]);
          tmem_wait_ld_of(s[0]);
          shape(s[0], i);
          mx = fmaxf(mx, top(s[0], i));
        }
      }
      if (!whole) {
        // V rows that no row of the tile sees - past the range: stale or foreign; tree nodes in nobody's mask - may hold anything, and 0 * NaN must
        // not happen. Cleared before P is handed over.
#pragma unroll 1
        for (int k0 = c0; k0 < c0 + C::BU; k0 += 64) {
          const uint64_t seen = L.seen64(b, k0);
          if (seen == ~0ull) continue;
          const int first = __ffsll((long long)~seen) - 1, q = b * C::SPB + k0 / C::VK;  // the q-th slot use
          wait_bar(&sh.v_full[q % VS], uint32_t(q / VS) & 1u, kStatusTmaTimeout);
          for (int i = srow; i < (64 - first) * 8 * C::VC; i += BM) {
            const int r = first + i / (8 * C::VC), c = i % (8 * C::VC);
            if (!((seen >> r) & 1ull))
              *reinterpret_cast<uint4*>(v_sm + (q % VS) * C::V_SLOT + (c >> 3) * C::V_CHUNK + (k0 % C::VK + r) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
      }
      const bool grow = mx > m_old + kGrow;  // also the first finite maximum
      const float m_new = grow ? mx : m_old;
      *const_cast<volatile float*>(&sh.m_ref[srow]) = m_new;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.m_ready[wg]);
      if (m_new > m_seen) {
        l_run *= fast_exp2(m_seen - m_new);
        m_seen = m_new;
      }
      if (n > 0 && __any_sync(0xffffffffu, grow)) {
        wait_bar(&sh.o_done[wg ^ 1], uint32_t((n - 1) >> 1) & 1u, kStatusMmaTimeout);  // every unit before this one is in O
        tc_fence_after_sync();
        const float factor = grow ? fast_exp2(m_old - m_new) : 1.0f;
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
      const float neg_m = m_new == -INFINITY ? 0.0f : -m_new;
      const uint64_t neg_m2 = f32x2_pack(neg_m, neg_m);
      uint64_t sum[2] = {f32x2_pack(0.0f, 0.0f), f32x2_pack(0.0f, 0.0f)};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if constexpr (!C::HOLD) {  // P of chunk i lies in columns the chunks to come do not use
          tmem_ld32(buf + 32 * i, s[0]);
          tmem_wait_ld_of(s[0]);
          shape(s[0], i);
        }
        uint32_t pk[16];
        chunk_weights<QDT, F8>(s[C::HOLD ? i : 0], pk, F8 ? f32x2_pack(ks[2 * i], ks[2 * i]) : sl2x2, F8 ? f32x2_pack(ks[2 * i + 1], ks[2 * i + 1]) : sl2x2, neg_m2, sum, vs[2 * i], vs[2 * i + 1]);
        tmem_st16(buf + 16 * i, pk);
        if ((i + 1) % (C::PART / 32) == 0) {  // a part is ready: its P . V starts under the rest
          tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(&sh.p_full[wg][i / (C::PART / 32)]);
        }
      }
      float a0, a1;
      f32x2_unpack(f32x2_add(sum[0], sum[1]), a0, a1);
      l_run += a0 + a1;
    }

    // ---- epilogue
    pdl_launch_dependents();
    // what the finish needs of memory, asked for before the waits
    const float lam = whole_rows && map ? diff_lam(args, row, head) : 0.0f;
    float4 w4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (whole_rows && args.norm_w && tid < HD / 4) w4 = reinterpret_cast<const float4*>(args.norm_w)[tid];
    named_barrier(2, kSoftmax);  // both groups are through: the reference is final, and all but the last two P . V are known to be done
    float m_fin = -INFINITY;
    if (N > 0) {
      wait_bar(&sh.o_done[(N - 1) & 1], uint32_t((N - 1) >> 1) & 1u, kStatusMmaTimeout);
      tc_fence_after_sync();
      m_fin = *const_cast<volatile float*>(&sh.m_ref[srow]);
    }
    // the groups' sums (the rings are idle: every load has been waited for and every MMA that reads them is done)
    float* lsum = reinterpret_cast<float*>(k_sm);
    lsum[tid] = m_seen == -INFINITY ? 0.0f : l_run * fast_exp2(m_seen - m_fin);
    named_barrier(2, kSoftmax);
    const float l = lsum[srow] + lsum[BM + srow];
    auto load_o = [&](int col, float (&v)[32]) {
      if (N > 0) {
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
    if (!whole_rows) {
      float* rec = a.parts + diff_record(a, tile.part, kvh, fm, head % G, map);
#pragma unroll 1
      for (int col = wg * C::MAP; col < (wg + 1) * C::MAP; col += 32) {
        float v[32];
        load_o(col, v);
        if (row_ok) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) *reinterpret_cast<float2*>(rec + col + i) = make_float2(v[i], v[i + 1]);
        }
      }
      if (row_ok && wg == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(m_fin * kLn2, l);
    } else {
      constexpr int MINE = HD / 4;               // columns a thread finishes: CTA `map` has [map HD / 2, ..), group wg half of those
      constexpr int HALF = C::MAP * BM * 4;      // bytes that change sides
      static_assert(2 * HALF <= VS * C::V_SLOT, "give and take lie in the V ring");
      uint8_t* give = v_sm;                                 // [HD / 8][128 rows][4 columns], lanes side by side
      float* take = reinterpret_cast<float*>(v_sm + HALF);  // the same, written by the peer
      float* sq = reinterpret_cast<float*>(q_sm);           // [CTA * 2 + group][128 rows]: the rows' sums of squares; written by both
      const float inv = l > 0.0f ? (map ? -lam : 1.0f) / l : 0.0f;
      float* w_sm = reinterpret_cast<float*>(k_sm) + 2 * BM;  // the norm's weights
      if (args.norm_w && tid < HD / 4) reinterpret_cast<float4*>(w_sm)[tid] = w4;
      if (tid == 0) mbar_arrive_expect_tx(&sh.take_full, HALF);
#pragma unroll 1
      for (int q = 0; q < MINE / 32; ++q) {
        float v[32];
        load_o((map ^ 1) * C::MAP + wg * MINE + 32 * q, v);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          reinterpret_cast<float4*>(give)[(wg * (MINE / 4) + 8 * q + i / 4) * BM + srow] = make_float4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv);
      }
      fence_proxy_async_smem();
      cluster_sync();  // both halves lie ready, neither CTA uses its tiles any more
      if (tid == 0) peer_copy(peer_addr(take, uint32_t(map ^ 1)), give, HALF, peer_addr(&sh.take_full, uint32_t(map ^ 1)));
      float dv[MINE];
#pragma unroll
      for (int q = 0; q < MINE / 32; ++q) {
        float v[32];
        load_o(map * C::MAP + wg * MINE + 32 * q, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) dv[32 * q + i] = v[i] * inv;
      }
      wait_bar(&sh.take_full, 0, kStatusMmaTimeout);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < MINE; i += 4) {
        const float4 o = reinterpret_cast<const float4*>(take)[(wg * (MINE / 4) + i / 4) * BM + srow];
        dv[i] += o.x, dv[i + 1] += o.y, dv[i + 2] += o.z, dv[i + 3] += o.w;
#pragma unroll
        for (int k = 0; k < 4; ++k) ss = fmaf(dv[i + k], dv[i + k], ss);
      }
      sq[(map * 2 + wg) * BM + srow] = ss;
      peer_store(peer_addr(sq, uint32_t(map ^ 1)) + uint32_t(((map * 2 + wg) * BM + srow) * 4), ss);
      cluster_sync();  // and both copies have been received
      ss = sq[srow] + sq[BM + srow] + sq[2 * BM + srow] + sq[3 * BM + srow];  // the same order in both CTAs
      const float f = diff_row_factor(args, ss, HD);
      // The rows leave through shared memory, HD / 2 columns of a row side by side.
      constexpr int PIECES = C::MAP / 8;  // of 16 bytes in a row, swizzled by row
      uint4* rows = reinterpret_cast<uint4*>(k_sm + C::K_TILE);
      const float* w = w_sm + map * C::MAP + wg * MINE;  // every lane reads the same word
#pragma unroll
      for (int i = 0; i < MINE; i += 8) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = dv[i + k] * f;
        if (args.norm_w) {
          const float4 w0 = *reinterpret_cast<const float4*>(w + i), w1 = *reinterpret_cast<const float4*>(w + i + 4);
          x[0] *= w0.x, x[1] *= w0.y, x[2] *= w0.z, x[3] *= w0.w, x[4] *= w1.x, x[5] *= w1.y, x[6] *= w1.z, x[7] *= w1.w;
        }
        rows[srow * PIECES + ((wg * (MINE / 8) + i / 8) ^ (srow & 7))] = make_uint4(QE::pack2(x[0], x[1]), QE::pack2(x[2], x[3]), QE::pack2(x[4], x[5]), QE::pack2(x[6], x[7]));
      }
      named_barrier(2, kSoftmax);
      typename QE::T* out = static_cast<typename QE::T*>(a.O) + size_t(tile.r0) * p.q_ld + size_t(head0) * HD + map * C::MAP;
#pragma unroll 4
      for (int i = tid; i < BM * PIECES; i += kSoftmax) {
        const int r = i / PIECES, c = i % PIECES;
        if (r / HPC < rows_live) *reinterpret_cast<uint4*>(out + size_t(r / HPC) * p.q_ld + size_t(r % HPC) * HD + 8 * c) = rows[r * PIECES + (c ^ (r & 7))];
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (sh.dead) {  // copies and MMAs still under way (the peer's half among them) land before their memory is given back
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 1000000ull) {}
  }
  if (warp == kMmaWarp) tmem_dealloc(sh.tmem, C::COLS);
}

template <int HD, int QDT, bool F8>
cudaError_t setup_one() {
  return cudaFuncSetAttribute(diff_umma_kernel<HD, QDT, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<HD>::SMEM);
}
// A pass over an E4M3 pool that reads no cached key runs without F8.
template <int HD, int QDT>
cudaError_t setup_types(int32_t kv_dtype) {
  const cudaError_t e = setup_one<HD, QDT, false>();
  return e == cudaSuccess && kv_dtype == ESP_E4M3 ? setup_one<HD, QDT, true>() : e;
}
template <int HD>
cudaError_t launch_hd(const DiffArgs& a, bool f8, const CUtensorMap& pool_map, const CUtensorMap& q_map, const CUtensorMap& kb_map, const CUtensorMap& vb_map, cudaStream_t stream) {
  const bool f16 = a.k.q_dtype == ESP_F16;
  auto kernel = f8 ? (f16 ? diff_umma_kernel<HD, ESP_F16, true> : diff_umma_kernel<HD, ESP_BF16, true>)
                   : (f16 ? diff_umma_kernel<HD, ESP_F16, false> : diff_umma_kernel<HD, ESP_BF16, false>);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.k.n_tiles) * unsigned(a.k.p.H / (BM / a.k.tile_rows)), 1, 2), cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Geo<HD>::SMEM, cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 2;
  cfg.attrs = attr, cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, pool_map, q_map, kb_map, vb_map, a);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace

// 128 / tile_rows heads of a tile must belong to one kv head.
bool diff_umma_supports(int32_t HD, int32_t G, int32_t tile_rows, int32_t bt) {
  if ((HD != 128 && HD != 256) || bt <= 0 || bt % 16 != 0) return false;
  if (tile_rows != 16 && tile_rows != 32 && tile_rows != 64 && tile_rows != 128) return false;
  const int hpc = BM / tile_rows;
  return hpc <= G && G % hpc == 0;
}

cudaError_t diff_umma_setup(int32_t HD, int32_t G, int32_t q_dtype, int32_t kv_dtype, int32_t tile_rows, int32_t bt) {
  if (!diff_umma_supports(HD, G, tile_rows, bt)) return cudaSuccess;
  if (HD == 128) return q_dtype == ESP_F16 ? setup_types<128, ESP_F16>(kv_dtype) : setup_types<128, ESP_BF16>(kv_dtype);
  return q_dtype == ESP_F16 ? setup_types<256, ESP_F16>(kv_dtype) : setup_types<256, ESP_BF16>(kv_dtype);
}

cudaError_t launch_diff_umma(const DiffArgs& a, bool f8, const CUtensorMap& pool_map, const CUtensorMap& q_map, const CUtensorMap& kb_map, const CUtensorMap& vb_map,
                             cudaStream_t stream, uint64_t* launches) {
  if (a.k.n_tiles <= 0) return cudaSuccess;
  const cudaError_t e = a.k.HD == 128 ? launch_hd<128>(a, f8, pool_map, q_map, kb_map, vb_map, stream) : launch_hd<256>(a, f8, pool_map, q_map, kb_map, vb_map, stream);
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
