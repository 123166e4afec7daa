// Parts of the tcgen05 kernel of differential attention: which key blocks a tile visits and what its rows see of them, the pages of a block,
// maxima and weights of a chunk of scores, and a few instruction wrappers.
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

// MMA issue by a whole converged warp, of which one lane (`one` = 1) issues. The warp's loop counters and descriptors then stay in
// uniform registers; a loop that only one lane runs spends about 100 clocks per instruction group on moving them there: a tenth of
// diff_umma's loop when it was measured.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(one));
  return one;
}
// Descriptors as their low words (the high word of this file's tiles never changes).
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %2};\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
      "}\n" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t"
      "}\n" ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "}\n" ::"r"(smem_u32(bar)), "r"(one)
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
  uint64_t nodes;       // ancestor masks: the tree's rows that some row of the tile sees; else all ones
  int full_c, full_a, seg_0, seg_n;  // blocks every row sees whole: [0, full_c), nbc + [0, full_a), seg_0 + [0, seg_n)
  __device__ __forceinline__ bool whole(int b) const { return b < full_c || uint32_t(b - nbc) < uint32_t(full_a) || uint32_t(b - seg_0) < uint32_t(seg_n); }
  __device__ __forceinline__ int n() const { return nbc + nbb; }
  __device__ __forceinline__ int j0(int b) const {
    if (b < nbc) return k0 + BN * b;
    const int i = b - nbc;
    return BN * (i < a_hi ? i : b_lo + (i - a_hi));
  }
  __device__ __forceinline__ int n_valid(int b) const { return min(BN, (b < nbc ? k1 : k_last + 1) - j0(b)); }
  // Which of 64 keys of block b from column c on (a multiple of 64) any row of the tile may see.
  __device__ __forceinline__ uint64_t seen64(int b, int c) const { return low_bits64(n_valid(b) - c) & (b < nbc || c > 0 ? ~0ull : nodes); }
};

// Whole-warp call; every warp forms the list for itself from the rows' records.
__device__ __forceinline__ BlockList block_list(const KernelArgs& a, const esp_attn_tile& tile, const esp_attn_tree& tree, int rows_live, int lane) {
  BlockList L;
  L.k0 = tile.k0, L.k1 = tile.k1, L.nbc = (tile.k1 - tile.k0 + BN - 1) / BN;
  L.nbb = 0, L.k_last = -1, L.a_hi = L.b_lo = 0, L.anc_min = 0, L.seg_max = 0, L.r_first = tile.r0 - tree.base;
  L.full_c = (tile.k1 - tile.k0) / BN, L.full_a = L.seg_n = 0, L.seg_0 = 0;
  L.nodes = ~0ull;
  if (!tile.last) return L;
  if (a.anc_mask) {
    L.k_last = min(tree.M, 64) - 1;
    L.nbb = L.a_hi = (L.k_last + BN) / BN;
    uint64_t any = 0;
    for (int r = lane; r < rows_live; r += 32) any |= a.anc_mask[tile.r0 + r];
    L.nodes = uint64_t(__reduce_or_sync(0xffffffffu, uint32_t(any))) | uint64_t(__reduce_or_sync(0xffffffffu, uint32_t(any >> 32))) << 32;
    return L;
  }
  int anc_max = 0, seg_min = tree.M, anc_min = tree.M, seg_max = 0;
  for (int r = lane; r < rows_live; r += 32) {
    const int4 d = row_record(a, tile.r0 + r, tree.M);
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
  L.a_hi = min((anc_max + BN - 1) / BN, n_all);
  L.b_lo = max(L.a_hi, seg_min / BN);
  L.nbb = L.a_hi + max(0, min(r_last / BN, n_all - 1) - L.b_lo + 1);
  // whole blocks: those that end below every row's ancestors, and - batch blocks [lo, hi) of the rows' segments - those that start
  // at or after every segment's start and end at or before the first row
  L.full_a = min(L.a_hi, anc_min / BN);
  const int lo = max(L.b_lo, (seg_max + BN - 1) / BN), hi = (L.r_first + 1) / BN;
  L.seg_0 = L.nbc + L.a_hi + (lo - L.b_lo), L.seg_n = max(0, hi - lo);
  return L;
}

// What a row sees of 32 columns of block b from column c on (a multiple of 32): one bit per column.
__device__ __forceinline__ uint32_t visible32(const BlockList& L, int b, int c, const int4& d, uint64_t am, bool use_anc, int rr) {
  const int jb = L.j0(b) + c;
  uint64_t vm = low_bits64(L.n_valid(b) - c);
  if (b >= L.nbc) {
    if (use_anc) vm &= jb < 64 ? am >> jb : 0ull;  // an ancestor mask covers the tree's first 64 rows, which are all it may have
    else vm &= low_bits64(d.z - jb) | (low_bits64(rr + 1 - jb) & ~low_bits64(d.x - jb));  // j < d.z || d.x <= j <= rr
  }
  return uint32_t(vm);
}
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t visible) {
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (!((visible >> c) & 1u)) s[c] = 0xFF800000u;  // -inf
}

// A TMA producer warp's walk over its tile's blocks. `page(b, kind, y, blk)` is called by lanes 0 .. 7 for the lane's 16-key page of cached
// block b: kind -1 nothing to load (past the range), 0 row y of the pool (its page is `blk` of the region). `rows(b, y)` is called by
// the same lanes for batch block b, which begins at row y of Kb / Vb. `which`: 0 keys, 1 values. F8: the pool map covers the widened
// pages, which lie in the order of the block list. Table entries are fetched four blocks per load, two groups ahead of their use; an
// entry outside the region is recorded and block 0 stands in for it.
template <bool F8, class Page, class Rows>
__device__ __forceinline__ void walk_pages(const KernelArgs& a, const esp_attn_tree& tree, const BlockList& L, int which, int lane, Page&& page, Rows&& rows) {
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
    const int j = L.k0 + BN * b + 16 * lane;
    const int at = F8 ? tree.table + j / bt : blk;
    if (lane < kPages) page(b, blk >= 0 ? 0 : -1, (at * 2 + which) * bt + j % bt, blk);
  }
  for (int b = L.nbc; b < L.n(); ++b)
    if (lane < kPages) rows(b, tree.base + L.j0(b));
}

__device__ __forceinline__ float chunk_max(const uint32_t (&s)[32]) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 32; c += 2) m[(c >> 1) & 3] = fmax3(m[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
  return fmax3(fmaxf(m[0], m[1]), m[2], m[3]);
}

// Over an E4M3 pool a row's reference is the largest scaled score + log2 of the page's V scale: the scale of a page goes on the weights before
// they are rounded to 16 bits, and what has to stay in fp16's range is their product. (Against the scores' maximum alone, a page of large values
// that a row hardly attends would push the weights of the others under fp16's.) k0, k1 = scale of the softmax, in log2 units, times the
// (positive) K scales of the chunk's two pages, v0, v1 their log2_floor.
__device__ __forceinline__ float chunk_max(const uint32_t (&s)[32], float k0, float k1, float v0, float v1) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 32; c += 2) m[(c >> 4) * 2 + ((c >> 1) & 1)] = fmax3(m[(c >> 4) * 2 + ((c >> 1) & 1)], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
  return fmaxf(fmaf(fmaxf(m[0], m[1]), k0, v0), fmaf(fmaxf(m[2], m[3]), k1, v1));
}

// 32 scores -> 16 packed pairs of weights exp2(sl s - m), sl = sl_a for the chunk's first 16 columns and sl_b for the others (a page each);
// `sum` (two partial sums) gains the unrounded weights. F8: v0, v1 = the V scales of the two pages, on the weights that are handed on.
template <int QDT, bool F8>
__device__ __forceinline__ void chunk_weights(const uint32_t (&s)[32], uint32_t* pk, uint64_t sl_a, uint64_t sl_b, uint64_t neg_m2, uint64_t (&sum)[2], float v0, float v1) {
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint64_t x2 = f32x2_fma(f32x2_pack(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), c < 8 ? sl_a : sl_b, neg_m2);
    float x0, x1;
    f32x2_unpack(x2, x0, x1);
    const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
    sum[c & 1] = f32x2_add(sum[c & 1], f32x2_pack(p0, p1));
    const float v = c < 8 ? v0 : v1;
    pk[c] = F8 ? Elem16<QDT>::pack2(p0 * v, p1 * v) : Elem16<QDT>::pack2(p0, p1);
  }
}

}  // namespace difft
}  // namespace esp
