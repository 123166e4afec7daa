// E4M3 pages as 16-bit pages, for the tcgen05 kernels of differential attention, whose operands come by TMA in one 16-bit type.
//
// The codes are widened, not the values: an e4m3 number is exact in fp16 and in bf16, code * scale is not. The page scales stay fp32
// and meet the scores and the weights inside the attention kernel. Entry e of the block list becomes page e of `out`, for the
// entries that a tree with rows reads, ceil(P / bt) from its table: room in a padded table costs nothing (16 rows behind 20001 keys, a table for 64
// times as many: 30 us; 1200 with every entry widened). The trees are read on the device, so a replayed graph follows lengths that changed
// there; of trees with one table the longest has its pages.
// HBM-bound: one byte read, two written per element; a thread takes 16 codes at a time, two at once. A warp sums up the pages of 32 trees and
// finds its page's by a ballot. 20001 keys of 8 kv heads, 128 dims: 123 MB in 28 us = 4.4 TB/s (the same without the trees; 300 keys 6.2 us
// against 5.6: one more load that the next waits for).
#include "diff.cuh"

namespace esp {
namespace {

constexpr int kThreads = 256;
constexpr int kCtas = 64;  // CTAs per SM of a long pass; a CTA that has several pages takes them one after another
constexpr int kPiece = 512;  // 16-code chunks of a page that a CTA takes at a time

template <int QDT>
__device__ __forceinline__ void widen16(const uint4& v, uint4* out) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    o[k] = e4m3x2_to_f16x2(uint16_t((w[k >> 1] >> (16 * (k & 1))) & 0xFFFFu));
    if constexpr (QDT == ESP_BF16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[k]));
      o[k] = Elem16<QDT>::pack2(f.x, f.y);
    }
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

template <int QDT>
__global__ void __launch_bounds__(kThreads) diff_widen_kernel(const KernelArgs a, uint4* out, const uint32_t chunks, const bool shared) {
  const int lane = threadIdx.x & 31;
  const uint32_t c0 = blockIdx.y * kPiece + threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  for (int t0 = 0; t0 < a.n_trees; t0 += 32) {
    // lane = tree: its pages, and those of the trees up to it
    int first = -1 - lane, count = 0;
    if (t0 + lane < a.n_trees) {
      const esp_attn_tree t = a.trees[t0 + lane];
      if (t.M > 0 && t.P > 0 && t.table >= 0 && t.table < a.n_block_entries) first = t.table, count = min((t.P - 1) / a.p.bt + 1, a.n_block_entries - first);
    }
    if (shared) {  // of the trees with one table the longest has its pages
      int mine = count;
      for (int u = 0; u < 32; ++u) {
        const int f = __shfl_sync(0xffffffffu, first, u), c = __shfl_sync(0xffffffffu, count, u);
        if (f == first && (c > count || (c == count && u < lane))) mine = 0;
      }
      count = mine;
    }
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int pages = __shfl_sync(0xffffffffu, upto, 31);
    for (int page = blockIdx.x; page < pages; page += gridDim.x) {
      const int tree = __popc(__ballot_sync(0xffffffffu, upto <= page)), e = page + __shfl_sync(0xffffffffu, first - (upto - count), tree), b = a.blocks[e];
      uint4 v[kPiece / kThreads];
#pragma unroll
      for (int i = 0; i < kPiece / kThreads; ++i) {
        v[i] = make_uint4(0, 0, 0, 0);  // zeros for an entry outside the region, which the attention kernel reports when it needs it
        const uint32_t c = c0 + i * kThreads;
        if (c < chunks && b >= 0 && b < a.n_blocks) v[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.kv) + a.p.kv_base + (size_t(b) * chunks + c) * 16);
      }
#pragma unroll
      for (int i = 0; i < kPiece / kThreads; ++i) {
        const uint32_t c = c0 + i * kThreads;
        if (c < chunks) widen16<QDT>(v[i], out + 2 * (size_t(e) * chunks + c));
      }
    }
  }
}

}  // namespace

cudaError_t launch_diff_widen(const KernelArgs& a, void* out, int64_t n_pages, bool shared, cudaStream_t stream, uint64_t* launches) {
  if (n_pages <= 0) return cudaSuccess;
  const uint32_t chunks = uint32_t(2 * size_t(a.p.bt) * size_t(a.p.kv_ld) / 16);
  const unsigned pieces = (chunks + kPiece - 1) / kPiece;
  const dim3 grid(unsigned(std::clamp<int64_t>(148 * kCtas / pieces, 1, n_pages)), pieces);
  const cudaError_t e = a.q_dtype == ESP_F16 ? launch_pdl(diff_widen_kernel<ESP_F16>, grid, dim3(kThreads), 0, stream, a, static_cast<uint4*>(out), chunks, shared)
                                             : launch_pdl(diff_widen_kernel<ESP_BF16>, grid, dim3(kThreads), 0, stream, a, static_cast<uint4*>(out), chunks, shared);
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
