// What the two tcgen05 kernels of differential attention share: which key blocks a tile visits and what its rows see of them, the
// pages of a block, and a few instruction wrappers.
#pragma once

#include <climits>

#include "diff.cuh"
#include "umma.cuh"

namespace esp {
namespace difft {

constexpr int BM = 128;          // (row, head) pairs of a tile: the lanes of tensor memory
constexpr int BN = 128;          // keys per block
constexpr int kPages = BN / 16;  // TMA pages per K or V tile

__device__ __forceinline__ uint64_t low_bits64(int n) { return n <= 0 ? 0ull : (n >= 64 ? ~0ull : ((1ull << n) - 1ull)); }

__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 32 lanes x 32 bit, 16 consecutive columns.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(taddr)
      : "memory");
}
// tcgen05.wait::ld that names the registers of an earlier load, so that no use of them moves above it.
__device__ __forceinline__ void tmem_wait_ld_of(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// The key blocks of a tile: its cached range in blocks of 128, then the batch blocks some row of the tile can see - those below
// the rows' ancestor ranges (desc.z) and those of their own segments (desc.x .. row) -, as bounds over the tile's rows.
struct BlockList {
  int k0, k1, nbc;      // cached keys and their blocks
  int nbb;              // batch blocks
  int k_last;           // last batch key any row can see
  int a_hi, b_lo;       // batch blocks [0, a_hi) and from b_lo on
  int anc_min, seg_max; // keys below anc_min are seen by every row; segments start at seg_max at the latest
  int r_first;          // the tile's first row, relative to its tree
  __device__ __forceinline__ int n() const { return nbc + nbb; }
  __device__ __forceinline__ int j0(int b) const {
    if (b < nbc) return k0 + BN * b;
    const int i = b - nbc;
    return BN * (i < a_hi ? i : b_lo + (i - a_hi));
  }
  __device__ __forceinline__ int n_valid(int b) const { return min(BN, (b < nbc ? k1 : k_last + 1) - j0(b)); }
};

// Whole-warp call; every warp forms the list for itself from the rows' records.
__device__ __forceinline__ BlockList block_list(const KernelArgs& a, const esp_attn_tile& tile, const esp_attn_tree& tree, int rows_live, int lane) {
  BlockList L;
  L.k0 = tile.k0, L.k1 = tile.k1, L.nbc = (tile.k1 - tile.k0 + BN - 1) / BN;
  L.nbb = 0, L.k_last = -1, L.a_hi = L.b_lo = 0, L.anc_min = 0, L.seg_max = 0, L.r_first = tile.r0 - tree.base;
  if (!tile.last) return L;
  if (a.anc_mask) {
    L.k_last = min(tree.M, 64) - 1;
    L.nbb = L.a_hi = (L.k_last + BN) / BN;
    return L;
  }
  int anc_max = 0, seg_min = 1 << 30, anc_min = 1 << 30, seg_max = 0;
  for (int r = lane; r < rows_live; r += 32) {
    const int4 d = reinterpret_cast<const int4*>(a.desc)[tile.r0 + r];
    anc_max = max(anc_max, d.z), anc_min = min(anc_min, d.z), seg_min = min(seg_min, d.x), seg_max = max(seg_max, d.x);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    anc_max = max(anc_max, __shfl_xor_sync(0xffffffffu, anc_max, o)), anc_min = min(anc_min, __shfl_xor_sync(0xffffffffu, anc_min, o));
    seg_min = min(seg_min, __shfl_xor_sync(0xffffffffu, seg_min, o)), seg_max = max(seg_max, __shfl_xor_sync(0xffffffffu, seg_max, o));
  }
  const int r_last = L.r_first + rows_live - 1;
  L.anc_min = anc_min, L.seg_max = seg_max;
  L.k_last = min(tree.M - 1, max(r_last, anc_max - 1));
  const int n_all = (L.k_last + BN) / BN;
  L.a_hi = min((max(anc_max, 0) + BN - 1) / BN, n_all);
  L.b_lo = max(L.a_hi, max(seg_min, 0) / BN);
  L.nbb = L.a_hi + max(0, min(r_last / BN, n_all - 1) - L.b_lo + 1);
  return L;
}

// What one row sees of block b: 128 bits. Returns false when every column is visible (the words are then not set).
__device__ __forceinline__ bool row_visibility(const BlockList& L, int b, const int4& d, uint64_t am, bool use_anc, int rr, uint32_t (&vw)[4]) {
  const bool cached = b < L.nbc;
  const int j0 = L.j0(b), n_valid = L.n_valid(b);
  bool need = n_valid < BN;
  if (!cached) need = need || use_anc || !((j0 + BN - 1 < L.anc_min) || (j0 >= L.seg_max && j0 + BN - 1 <= L.r_first));
  if (!need) return false;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int jb = j0 + 64 * hf;
    uint64_t vm = low_bits64(n_valid - 64 * hf);
    if (!cached) {
      if (use_anc) vm &= hf == 0 ? am : 0ull;  // one block, j0 = 0
      else vm &= low_bits64(d.z - jb) | (low_bits64(rr + 1 - jb) & ~low_bits64(d.x - jb));  // j < d.z || d.x <= j <= rr
    }
    vw[2 * hf] = uint32_t(vm), vw[2 * hf + 1] = uint32_t(vm >> 32);
  }
  return true;
}

// A TMA producer warp's walk over the pages of its tile's blocks: lane w < 8 handles the w-th 16-key page of every block. `load(kind, y)`
// is called by those lanes, block after block: kind -1 nothing to load (past the range), 0 row y of the pool, 1 row y of Kb / Vb.
// `which`: 0 keys, 1 values. Table entries are fetched four blocks per load, two groups ahead of their use; an entry outside the
// region is recorded and block 0 is read in its place.
template <class Load>
__device__ __forceinline__ void walk_pages(const KernelArgs& a, const esp_attn_tree& tree, const BlockList& L, int which, int lane, Load&& load) {
  const int bt = a.p.bt;
  auto group = [&](int g) {
    const int b = 4 * g + (lane >> 3), j = L.k0 + BN * b + 16 * (lane & 7);
    if (!(b < L.nbc && j < L.k1)) return -1;
    int blk = a.blocks[tree.table + j / bt];
    if (blk < 0 || blk >= a.n_blocks) {
      atomicExch(a.status, kStatusBadBlock);
      blk = 0;
    }
    return blk;
  };
  int cur = group(0), nxt = group(1);
  for (int b = 0; b < L.nbc; ++b) {
    if (b && (b & 3) == 0) {
      cur = nxt;
      nxt = group((b >> 2) + 1);
    }
    const int blk = __shfl_sync(0xffffffffu, cur, ((b & 3) << 3) | (lane & 7));
    if (lane < kPages) load(blk >= 0 ? 0 : -1, (blk * 2 + which) * bt + (L.k0 + BN * b + 16 * lane) % bt);
  }
  for (int b = L.nbc; b < L.n(); ++b) {
    const int j = L.j0(b) + 16 * lane;
    if (lane < kPages) load(j <= L.k_last ? 1 : -1, tree.base + j);
  }
}

// One row's 128 scores s (raw products) -> 128 weights as 16-bit pairs, in the exp2 domain against m_ref, lazily rescaled: the reference
// maximum only moves when a block exceeds it by 2^8. The caller moves O when `grow` says so.
struct RowState {
  float m_ref = -INFINITY, l = 0.0f;
};

__device__ __forceinline__ float chunk_max(uint32_t (&s)[32], bool mask, uint32_t w) {
  float m0 = -INFINITY, m1 = -INFINITY;
  if (mask) {
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      const float x = ((w >> c) & 1u) ? __uint_as_float(s[c]) : -INFINITY;
      s[c] = __float_as_uint(x);
      m0 = fmaxf(m0, x);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      m0 = fmax3(m0, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
      m1 = fmax3(m1, __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
    }
  }
  return fmaxf(m0, m1);
}

// 32 scores -> 16 packed pairs of weights; `sum` (two partial sums) gains the unrounded weights.
template <int QDT>
__device__ __forceinline__ void chunk_weights(const uint32_t (&s)[32], uint32_t (&pk)[16], uint64_t sl2x2, uint64_t neg_m2, uint64_t (&sum)[2]) {
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint64_t x2 = f32x2_fma(f32x2_pack(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sl2x2, neg_m2);
    float x0, x1;
    f32x2_unpack(x2, x0, x1);
    const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
    sum[c & 1] = f32x2_add(sum[c & 1], f32x2_pack(p0, p1));
    pk[c] = Elem16<QDT>::pack2(p0, p1);
  }
}

}  // namespace difft
}  // namespace esp
