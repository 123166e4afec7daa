// E4M3 pages as 16-bit pages, for the tcgen05 kernels of differential attention, whose operands come by TMA in one 16-bit type.
//
// The codes are widened, not the values: an e4m3 number is exact in fp16 and in bf16, code * scale is not. The page scales stay fp32
// and meet the scores and the weights inside the attention kernel. Entry e of the block list becomes page e of `out`. HBM-bound:
// one byte read, two written per element; a thread takes 16 codes. 20001 keys of 8 kv heads, 128 dims: 123 MB in 28 us = 4.4 TB/s.
#include "diff.cuh"

namespace esp {
namespace {

template <int QDT>
__global__ void __launch_bounds__(256) diff_widen_kernel(const KernelArgs a, uint4* out, const int n_entries, const uint32_t chunks) {
  pdl_wait();
  pdl_launch_dependents();
  const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t e = uint32_t(i / chunks), c = uint32_t(i % chunks);
  if (e >= uint32_t(n_entries)) return;
  const int b = a.blocks[e];
  uint32_t w[4] = {0, 0, 0, 0};
  if (b >= 0 && b < a.n_blocks) {  // zeros for an entry outside the region: a padded table's, or one that the attention kernel reports when it needs it
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.kv) + a.p.kv_base + (size_t(b) * chunks + c) * 16);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  uint32_t o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    o[k] = e4m3x2_to_f16x2(uint16_t((w[k >> 1] >> (16 * (k & 1))) & 0xFFFFu));
    if constexpr (QDT == ESP_BF16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[k]));
      o[k] = Elem16<QDT>::pack2(f.x, f.y);
    }
  }
  out[2 * i] = make_uint4(o[0], o[1], o[2], o[3]);
  out[2 * i + 1] = make_uint4(o[4], o[5], o[6], o[7]);
}

}  // namespace

cudaError_t launch_diff_widen(const KernelArgs& a, void* out, int32_t n_entries, cudaStream_t stream, uint64_t* launches) {
  if (n_entries <= 0) return cudaSuccess;
  const uint32_t chunks = uint32_t(2 * size_t(a.p.bt) * size_t(a.p.kv_ld) / 16);
  const size_t total = size_t(n_entries) * chunks;
  const dim3 grid(unsigned((total + 255) / 256));
  const cudaError_t e = a.q_dtype == ESP_F16 ? launch_pdl(diff_widen_kernel<ESP_F16>, grid, dim3(256), 0, stream, a, static_cast<uint4*>(out), n_entries, chunks)
                                             : launch_pdl(diff_widen_kernel<ESP_BF16>, grid, dim3(256), 0, stream, a, static_cast<uint4*>(out), n_entries, chunks);
  if (e == cudaSuccess) ++*launches;
  return e;
}

}  // namespace esp
