// The join of a split differential pass, and the layer's lambda.
//
// A job's records of one (row, head) - two maps, `nparts` records each - become the row: per map
//   M = max m_s,  L = sum e^(m_s - M) l_s,  A = sum e^(m_s - M) O_s   (records in order, no atomics: the result does not
// depend on scheduling), then D = A_1 / L_1 - lam A_2 / L_2 and the norm. One CTA per (job row, head): 128 threads per map, HD / 4
// of them per slice of records (4 dims each), the slices joined in order through shared memory. Latency-bound: a slice asks for
// up to eight records before it folds the first.
#include "diff.cuh"

namespace esp {
namespace {

constexpr int kThreads = 256, kPerMap = 128;

template <int HD, int QDT>
__global__ void __launch_bounds__(kThreads) diff_combine_kernel(const DiffCombineArgs c) {
  using QE = Elem16<QDT>;
  constexpr int TPD = HD / 4, NSL = kPerMap / TPD;  // threads per slice, slices per map
  const DiffArgs& a = c.d;
  const KernelArgs& k = a.k;
  __shared__ float part[kThreads][6];  // 4 dims, L, M of a thread's slice
  __shared__ float sq[kPerMap / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int job_i = blockIdx.x / c.rows_max, r = blockIdx.x % c.rows_max, h = blockIdx.y, kvh = h / k.G, hg = h % k.G;
  const esp_attn_combine job = k.jobs[job_i];
  if (r >= job.rows) return;  // the whole CTA
  const int tid = threadIdx.x, map = tid / kPerMap, sl = (tid % kPerMap) / TPD, d4 = tid % TPD;
  const size_t stride = diff_record(k, 1, 0, 0, 0, 0);
  const float* rec0 = k.parts + diff_record(k, job.part0, kvh, r, hg, map);
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fold = [&](float m, float l, const float4& o) {
    if (m == -INFINITY) return;  // an empty record
    const float mn = fmaxf(M, m);
    const float f = __expf(M - mn), w = __expf(m - mn);  // M = -inf: f = 0
    L = L * f + w * l;
    acc.x = acc.x * f + w * o.x, acc.y = acc.y * f + w * o.y, acc.z = acc.z * f + w * o.z, acc.w = acc.w * f + w * o.w;
    M = mn;
  };
  for (int s = sl; s < job.nparts; s += 8 * NSL) {
    float2 ml[8], lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ml[i] = make_float2(-INFINITY, 0.0f), lo[i] = hi[i] = make_float2(0.f, 0.f);
      if (s + i * NSL < job.nparts) {
        const float* rec = rec0 + size_t(s + i * NSL) * stride;  // records are 8-byte aligned (HD + 2 floats)
        ml[i] = *reinterpret_cast<const float2*>(rec + HD);
        lo[i] = *reinterpret_cast<const float2*>(rec + 4 * d4), hi[i] = *reinterpret_cast<const float2*>(rec + 4 * d4 + 2);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) fold(ml[i].x, ml[i].y, make_float4(lo[i].x, lo[i].y, hi[i].x, hi[i].y));
  }
  float* mine = part[tid];
  mine[0] = acc.x, mine[1] = acc.y, mine[2] = acc.z, mine[3] = acc.w, mine[4] = L, mine[5] = M;
  __syncthreads();
  // the threads of slice 0 join the slices of their map, map 2's hand their result over, map 1's finish
  if (sl == 0) {
    for (int s = 1; s < NSL; ++s) {
      const float* o = part[tid + s * TPD];
      fold(o[5], o[4], make_float4(o[0], o[1], o[2], o[3]));
    }
    if (map == 1) mine[0] = acc.x, mine[1] = acc.y, mine[2] = acc.z, mine[3] = acc.w, mine[4] = L;
  }
  __syncthreads();
  const bool owner = sl == 0 && map == 0;
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  const int row = job.r0 + r;
  if (owner) {
    const float* o = part[kPerMap + d4];
    const float inv1 = L > 0.0f ? 1.0f / L : 0.0f, inv2 = o[4] > 0.0f ? diff_lam(a, row, h) / o[4] : 0.0f;
    d[0] = acc.x * inv1 - o[0] * inv2, d[1] = acc.y * inv1 - o[1] * inv2, d[2] = acc.z * inv1 - o[2] * inv2, d[3] = acc.w * inv1 - o[3] * inv2;
  }
  float ss = d[0] * d[0] + d[1] * d[1] + d[2] * d[2] + d[3] * d[3];
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (tid < kPerMap && (tid & 31) == 0) sq[tid >> 5] = ss;
  __syncthreads();
  if (!owner) return;
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kPerMap / 32; ++i) ss += sq[i];  // threads that are no owners added zeros
  const float f = diff_row_factor(a, ss, HD);
  const float4 w = a.norm_w ? *reinterpret_cast<const float4*>(a.norm_w + 4 * d4) : make_float4(1.f, 1.f, 1.f, 1.f);
  *reinterpret_cast<uint2*>(static_cast<typename QE::T*>(k.O) + size_t(row) * k.p.q_ld + size_t(h) * HD + 4 * d4) =
      make_uint2(QE::pack2(d[0] * f * w.x, d[1] * f * w.y), QE::pack2(d[2] * f * w.z, d[3] * f * w.w));
}

// One warp per head.
__global__ void diff_lambda_kernel(const float* q1, const float* k1, const float* q2, const float* k2, int H, int dim, int ld, float init, float* lam) {
  const int h = blockIdx.x, lane = threadIdx.x;
  float a = 0.0f, b = 0.0f;
  for (int d = lane; d < dim; d += 32) {
    const size_t at = size_t(h) * ld + d;
    a = fmaf(q1[at], k1[at], a), b = fmaf(q2[at], k2[at], b);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o), b += __shfl_xor_sync(0xffffffffu, b, o);
  if (lane == 0) lam[h] = expf(a) - expf(b) + init;
}

template <int QDT>
cudaError_t launch_typed(const DiffCombineArgs& c, cudaStream_t stream) {
  const dim3 grid(unsigned(c.n_jobs) * unsigned(c.rows_max), unsigned(c.d.k.p.H));
  switch (c.d.k.HD) {
    case 64: return launch_pdl(diff_combine_kernel<64, QDT>, grid, dim3(kThreads), 0, stream, c);
    case 128: return launch_pdl(diff_combine_kernel<128, QDT>, grid, dim3(kThreads), 0, stream, c);
    case 256: return launch_pdl(diff_combine_kernel<256, QDT>, grid, dim3(kThreads), 0, stream, c);
    case 512: return launch_pdl(diff_combine_kernel<512, QDT>, grid, dim3(kThreads), 0, stream, c);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_diff_combine(const DiffCombineArgs& c, cudaStream_t stream, uint64_t* launches) {
  if (c.n_jobs <= 0) return cudaSuccess;
  const cudaError_t e = c.d.k.q_dtype == ESP_F16 ? launch_typed<ESP_F16>(c, stream) : launch_typed<ESP_BF16>(c, stream);
  if (e == cudaSuccess) ++*launches;
  return e;
}

cudaError_t launch_diff_lambda(const float* q1, const float* k1, const float* q2, const float* k2, int32_t H, int32_t dim, int32_t ld,
                               float lambda_init, float* lam, cudaStream_t stream) {
  diff_lambda_kernel<<<unsigned(H), 32, 0, stream>>>(q1, k1, q2, k2, H, dim, ld, lambda_init, lam);
  return cudaGetLastError();
}

}  // namespace esp
