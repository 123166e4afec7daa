// The join of a split differential pass, and the layer's lambda.
//
// A job's records of one (row, head) - two maps, `nparts` records each - become the row: per map
//   M = max m_s,  L = sum e^(m_s - M) l_s,  A = sum e^(m_s - M) O_s   (records in order, no atomics: the result does not
// depend on scheduling), then D = A_1 / L_1 - lam A_2 / L_2 and the norm. HD / 4 threads (4 dims each) per slice of records, NSL slices
// per map, two maps per (row, head), as many (row, head) pairs as fit a CTA; the slices are joined in order through shared memory.
// A slice asks for several records before it folds the first. Few long jobs (decode) are latency-bound and take many slices;
// many short ones (chunks, trees: two records per row) are bound by the records' bytes and take one: 700 rows of 32 heads, two records,
// 93 MB in 28 us; a pass of trees split in two took 43.6 us with four slices and one pair per CTA, and a batch's maximum before its
// weights (one rescale a batch, one exponential a record) brought the former from 56 us.
#include "diff.cuh"

namespace esp {
namespace {

constexpr int kThreads = 256;

template <int HD, int QDT, int NSL>
__global__ void __launch_bounds__(kThreads) diff_combine_kernel(const DiffCombineArgs c) {
  using QE = Elem16<QDT>;
  constexpr int TPD = HD / 4, PER_MAP = TPD * NSL, PER_PAIR = 2 * PER_MAP, PAIRS = kThreads / PER_PAIR;
  const DiffArgs& a = c.d;
  const KernelArgs& k = a.k;
  __shared__ float part[kThreads][6];  // 4 dims, L, M of a thread's slice
  __shared__ float sq[kThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, t = tid % PER_PAIR, map = t / PER_MAP, sl = (t % PER_MAP) / TPD, d4 = t % TPD;
  const int64_t pair = int64_t(blockIdx.x) * PAIRS + tid / PER_PAIR;  // (job, row of the job, head), heads fastest
  const int h = int(pair % k.p.H), r = int((pair / k.p.H) % c.rows_max), job_i = int(pair / (int64_t(k.p.H) * c.rows_max));
  esp_attn_combine job{0, 0, 0, 0};
  if (job_i < c.n_jobs) job = k.jobs[job_i];
  const bool live = r < job.rows;
  const int n = live ? job.nparts : 0;
  const size_t stride = diff_record(k, 1, 0, 0, 0, 0);
  const float* rec0 = k.parts + diff_record(k, job.part0, h / k.G, live ? r : 0, h % k.G, map);
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
  // what the finish needs, asked for with the first records
  const int row = job.r0 + r;
  const float4 w = a.norm_w ? *reinterpret_cast<const float4*>(a.norm_w + 4 * d4) : make_float4(1.f, 1.f, 1.f, 1.f);
  const float lam = live ? diff_lam(a, row, h) : 0.0f;
  constexpr int AHEAD = NSL > 1 ? 8 : 4;
  for (int s = sl; s < n; s += AHEAD * NSL) {
    float2 ml[AHEAD], lo[AHEAD], hi[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      ml[i] = make_float2(-INFINITY, 0.0f), lo[i] = hi[i] = make_float2(0.f, 0.f);
      if (s + i * NSL < n) {
        const float* rec = rec0 + size_t(s + i * NSL) * stride;  // records are 8-byte aligned (HD + 2 floats)
        ml[i] = *reinterpret_cast<const float2*>(rec + HD);
        lo[i] = *reinterpret_cast<const float2*>(rec + 4 * d4), hi[i] = *reinterpret_cast<const float2*>(rec + 4 * d4 + 2);
      }
    }
    float mx = M;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) mx = fmaxf(mx, ml[i].x);
    if (mx == -INFINITY) continue;  // nothing but empty records so far
    const float f = __expf(M - mx);  // M = -inf: 0
    L *= f, acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f, M = mx;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (ml[i].x == -INFINITY) continue;  // an empty record
      const float x = __expf(ml[i].x - mx);
      L = fmaf(x, ml[i].y, L);
      acc.x = fmaf(x, lo[i].x, acc.x), acc.y = fmaf(x, lo[i].y, acc.y), acc.z = fmaf(x, hi[i].x, acc.z), acc.w = fmaf(x, hi[i].y, acc.w);
    }
  }
  float* mine = part[tid];
  if (NSL > 1) {
    mine[0] = acc.x, mine[1] = acc.y, mine[2] = acc.z, mine[3] = acc.w, mine[4] = L, mine[5] = M;
    __syncthreads();
    if (sl == 0)
      for (int s = 1; s < NSL; ++s) {
        const float* o = part[tid + s * TPD];
        fold(o[5], o[4], make_float4(o[0], o[1], o[2], o[3]));
      }
  }
  // map 2's first slice hands its result over, map 1's finishes
  if (sl == 0 && map == 1) mine[0] = acc.x, mine[1] = acc.y, mine[2] = acc.z, mine[3] = acc.w, mine[4] = L;
  __syncthreads();
  const bool owner = sl == 0 && map == 0 && live;
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  if (owner) {
    const float* o = part[tid + PER_MAP];
    const float inv1 = L > 0.0f ? 1.0f / L : 0.0f, inv2 = o[4] > 0.0f ? lam / o[4] : 0.0f;
    d[0] = acc.x * inv1 - o[0] * inv2, d[1] = acc.y * inv1 - o[1] * inv2, d[2] = acc.z * inv1 - o[2] * inv2, d[3] = acc.w * inv1 - o[3] * inv2;
  }
  // the row's sum of squares: over the TPD owners, which are whole warps or an aligned part of one
  float ss = d[0] * d[0] + d[1] * d[1] + d[2] * d[2] + d[3] * d[3];
#pragma unroll
  for (int o = (TPD < 32 ? TPD : 32) / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if constexpr (TPD > 32) {
    if ((tid & 31) == 0) sq[tid >> 5] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < TPD / 32; ++i) ss += sq[(tid - t) / 32 + i];
  }
  if (!owner) return;
  const float f = diff_row_factor(a, ss, HD);
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

template <int HD, int QDT>
cudaError_t launch_hd(const DiffCombineArgs& c, cudaStream_t stream) {
  constexpr int MOST = 128 / (HD / 4);  // slices that fill a CTA with one pair
  const bool slices = MOST > 1 && c.parts_max > 8;
  const int64_t pairs = int64_t(c.n_jobs) * c.rows_max * c.d.k.p.H, per_cta = slices ? 1 : kThreads / (HD / 2);
  const dim3 grid(unsigned((pairs + per_cta - 1) / per_cta));
  if (slices) return launch_pdl(diff_combine_kernel<HD, QDT, MOST>, grid, dim3(kThreads), 0, stream, c);
  return launch_pdl(diff_combine_kernel<HD, QDT, 1>, grid, dim3(kThreads), 0, stream, c);
}
template <int QDT>
cudaError_t launch_typed(const DiffCombineArgs& c, cudaStream_t stream) {
  switch (c.d.k.HD) {
    case 64: return launch_hd<64, QDT>(c, stream);
    case 128: return launch_hd<128, QDT>(c, stream);
    case 256: return launch_hd<256, QDT>(c, stream);
    case 512: return launch_hd<512, QDT>(c, stream);
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
