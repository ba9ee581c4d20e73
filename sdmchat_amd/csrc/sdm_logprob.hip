// sdm_logprob.hip -- log probabilities of given tokens with the rows' entropies and top alternatives
// (sdm_rt_token_logprobs), and their gradient (sdm_rt_token_logprobs_grad).
#include "sdm_vocab.h"

namespace sdmrt {

constexpr int kMaxAlternatives = 256;
constexpr float kLog2 = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogprobArgs {
  int64_t rows;
  int vocab, k;
  float inv_tau, c;   // 1 / temperature, that in units of log2
  int64_t ignore;
  const void* logits;
  int64_t l_stride;
  const int64_t* targets;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  float4* stats;   // per row: maximum, log2 of the sum against it, entropy
};

// A row's sums: with e_j = (z_j - m) / temperature in units of log2, how many logits equal the maximum m, the sum of 2^e
// over the others and that of e 2^e.  The maxima stay out of the sum: the logarithm of count + rest, taken as that of count
// plus log1p(rest / count), keeps the small log probabilities and entropies of a row that is nearly certain.
struct RowSums {
  float m, count, rest, u;
};
struct RowLogs {
  float l, l2, h;   // log of the sum, that in log2, entropy
};
__device__ __forceinline__ RowLogs row_logs(const RowSums& s) {
  const float r = s.rest / s.count;
  const float l = logf(s.count) + log1pf(r);
  return RowLogs{l, l * kLog2, l - kLn2 * (s.u / (s.count + s.rest))};
}

// greater for a greater logit, at equal logits for a lower id; 0 for -inf and NaN of either sign
__device__ __forceinline__ uint32_t ordered(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);   // -0 as 0
  if (!(z > -INFINITY)) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t logit_key(float z, int id) {
  return static_cast<uint64_t>(ordered(z)) << 32 | ~static_cast<uint32_t>(id);
}

// What becomes of a row's sums, by one thread.
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t r, const RowSums& s, const RowLogs& g) {
  const bool bad = s.m == INFINITY || s.rest != s.rest, none = !bad && s.m == -INFINITY;
  if (a.logprobs) {
    const int64_t y = a.targets[r];
    float lp = 0.f;
    if (y >= 0 && y < a.vocab && y != a.ignore) {
      const float z = to_f32(static_cast<const T*>(a.logits)[r * a.l_stride + y]);
      lp = bad ? NAN : none ? -INFINITY : (z - s.m) * a.inv_tau - g.l;
    }
    a.logprobs[r] = lp;
  }
  const float h = bad ? NAN : none ? 0.f : g.h;
  if (a.entropy) a.entropy[r] = h;
  // a row of -inf: sums that make every p 0
  if (a.stats) a.stats[r] = bad ? make_float4(NAN, NAN, NAN, 0.f) : none ? make_float4(0.f, INFINITY, 0.f, 0.f) : make_float4(s.m, g.l2, h, 0.f);
}

constexpr int kRowThreads = 256;

// One workgroup per row: its maximum, its sums, then its alternatives one by one, each the greatest below the last.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_kernel(LogprobArgs a) {
  __shared__ float red[3][kRowThreads / 64];
  __shared__ uint64_t best[kRowThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += kRowThreads) m = fmaxf(m, to_f32(z[i]));
  m = wave_max(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  for (int w = 0; w < kRowThreads / 64; ++w) m = fmaxf(m, red[0][w]);
  __syncthreads();
  float count = 0.f, rest = 0.f, u = 0.f;
  for (int i = threadIdx.x; i < a.vocab; i += kRowThreads) {
    const float x = to_f32(z[i]);
    if (x == m) {
      count += 1.f;
    } else {
      const float e = (x - m) * a.c, w = exp2f(e);
      rest += w;
      u = fmaf(w, fmaxf(e, -1000.f), u);
    }
  }
  count = wave_add(count);
  rest = wave_add(rest);
  u = wave_add(u);
  if (lane == 0) red[0][wave] = count, red[1][wave] = rest, red[2][wave] = u;
  __syncthreads();
  RowSums s{m, 0.f, 0.f, 0.f};
  for (int w = 0; w < kRowThreads / 64; ++w) s.count += red[0][w], s.rest += red[1][w], s.u += red[2][w];
  const RowLogs g = row_logs(s);
  if (threadIdx.x == 0) write_row<T>(a, r, s, g);
  const bool bad = m == INFINITY || s.rest != s.rest;
  uint64_t last = ~uint64_t{0};
  for (int q = 0; q < a.k; ++q) {
    uint64_t k = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kRowThreads) {
      const uint64_t x = logit_key(to_f32(z[i]), i);
      if (x < last && x > k) k = x;
    }
    for (int d = 32; d > 0; d >>= 1) {
      const uint64_t o = __shfl_xor(static_cast<unsigned long long>(k), d);
      k = o > k ? o : k;
    }
    __syncthreads();
    if (lane == 0) best[wave] = k;
    __syncthreads();
    for (int w = 0; w < kRowThreads / 64; ++w) k = best[w] > k ? best[w] : k;
    last = k;
    if (threadIdx.x == 0) {
      const bool there = !bad && (k >> 32) != 0;
      a.top_ids[r * a.k + q] = there ? static_cast<int64_t>(~static_cast<uint32_t>(k)) : -1;
      a.top_logprobs[r * a.k + q] = bad ? NAN : there ? (unordered(static_cast<uint32_t>(k >> 32)) - m) * a.inv_tau - g.l : -INFINITY;
    }
  }
}

struct LogprobGradArgs {
  int64_t rows;
  int vocab;
  float inv_tau, c;
  int64_t ignore;
  const void* logits;
  int64_t l_stride;
  const int64_t* targets;
  const float4* stats;
  const float* dlp;
  int64_t dlp_stride;
  const float* dh;
  int64_t dh_stride;
  void* dz;
  int64_t d_stride;
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_grad_kernel(LogprobGradArgs a) {
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
  T* d = static_cast<T*>(a.dz) + r * a.d_stride;
  const int64_t y64 = a.targets && a.dlp ? a.targets[r] : -1;
  const bool given = y64 >= 0 && y64 < a.vocab && y64 != a.ignore;
  const float ga = given ? a.dlp[r * a.dlp_stride] * a.inv_tau : 0.f;
  const float gb = a.dh ? a.dh[r * a.dh_stride] * a.inv_tau : 0.f;
  if (ga == 0.f && gb == 0.f) {
    for (int i = threadIdx.x; i < a.vocab; i += kRowThreads) d[i] = T{};
    return;
  }
  const float4 s = a.stats[r];
  const int y = given && s.y != INFINITY ? static_cast<int>(y64) : -1;
  for (int i = threadIdx.x; i < a.vocab; i += kRowThreads) {
    const float e = (to_f32(z[i]) - s.x) * a.c - s.y, p = exp2f(e);
    const float t = fmaf(gb, fmaf(fmaxf(e, -1000.f), kLn2, s.z), ga);
    d[i] = from_f32<T>((i == y ? ga : 0.f) - p * t);
  }
}

inline int check_logprob(const sdm_rt_logprob* d, const void* logits, int64_t l_stride, sdm_rt_dtype dtype) {
  int rc;
  if (!d) return set_err(SDM_RT_EINVAL, "dims is NULL");
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (d->rows < 0 || d->vocab < 1 || d->top_k < 0) return set_err(SDM_RT_EINVAL, "rows and top_k must be >= 0, vocab >= 1");
  if (d->rows > (1 << 21)) return set_err(SDM_RT_EUNSUPPORTED, "rows must be at most 2^21");
  if (d->vocab > (1 << 24)) return set_err(SDM_RT_EUNSUPPORTED, "vocab must be at most 2^24");
  if (d->top_k > kMaxAlternatives) return set_err(SDM_RT_EUNSUPPORTED, "top_k = %d must be at most %d", d->top_k, kMaxAlternatives);
  if (!(d->temperature >= 1e-18f) || !(d->temperature <= 1e18f))
    return set_err(SDM_RT_EINVAL, "temperature must be positive and finite, from 1e-18 to 1e18");
  if (d->rows > 0 && (!logits || bad_read_stride(l_stride, d->vocab)))
    return set_err(SDM_RT_EINVAL, "logits must not be NULL, their row stride 0 or >= vocab");
  return SDM_RT_OK;
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

size_t sdm_rt_token_logprobs_workspace_bytes(const sdm_rt_logprob* dims, sdm_rt_dtype dtype) {
  (void)dims;
  (void)dtype;
  return 0;
}

int sdm_rt_token_logprobs(const sdm_rt_logprob* dims, const void* logits, int64_t logits_row_stride, sdm_rt_dtype dtype,
                          const int64_t* targets, float* logprobs, float* entropy, int64_t* top_ids, float* top_logprobs,
                          float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (int rc = check_logprob(dims, logits, logits_row_stride, dtype)) return rc;
  if (dims->rows == 0) return SDM_RT_OK;
  if (logprobs && !targets) return set_err(SDM_RT_EINVAL, "logprobs need targets");
  if (dims->top_k > 0 && (!top_ids || !top_logprobs))
    return set_err(SDM_RT_EINVAL, "top_ids and top_logprobs must not be NULL with top_k above 0");
  if (stats && reinterpret_cast<uintptr_t>(stats) % 16) return set_err(SDM_RT_EINVAL, "stats must be 16-byte aligned");
  const size_t need = sdm_rt_token_logprobs_workspace_bytes(dims, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return set_err(SDM_RT_ENOSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  LogprobArgs a{};
  a.rows = dims->rows;
  a.vocab = dims->vocab;
  a.k = dims->top_k;
  a.inv_tau = 1.f / dims->temperature;
  a.c = a.inv_tau * kLog2;
  a.ignore = dims->ignore_index;
  a.logits = logits;
  a.l_stride = logits_row_stride;
  a.targets = targets;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.stats = reinterpret_cast<float4*>(stats);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(a.rows));
  if (dtype == SDM_RT_BF16)
    hipLaunchKernelGGL(logprob_kernel<bf16_t>, grid, dim3(kRowThreads), 0, st, a);
  else
    hipLaunchKernelGGL(logprob_kernel<float>, grid, dim3(kRowThreads), 0, st, a);
  return check_launch("token_logprobs");
}

int sdm_rt_token_logprobs_grad(const sdm_rt_logprob* dims, const void* logits, int64_t logits_row_stride,
                               sdm_rt_dtype dtype, const int64_t* targets, const float* stats, const float* d_logprobs,
                               int64_t d_logprobs_stride, const float* d_entropy, int64_t d_entropy_stride,
                               void* d_logits, int64_t d_logits_row_stride, void* stream) {
  g_err[0] = 0;
  if (int rc = check_logprob(dims, logits, logits_row_stride, dtype)) return rc;
  if (dims->rows == 0) return SDM_RT_OK;
  if (!stats || !d_logits) return set_err(SDM_RT_EINVAL, "stats and d_logits must not be NULL");
  if (d_logprobs && !targets) return set_err(SDM_RT_EINVAL, "d_logprobs need targets");
  if (reinterpret_cast<uintptr_t>(stats) % 16) return set_err(SDM_RT_EINVAL, "stats must be 16-byte aligned");
  if (d_logits_row_stride < dims->vocab) return set_err(SDM_RT_EINVAL, "d_logits_row_stride must be >= vocab");
  LogprobGradArgs a{};
  a.rows = dims->rows;
  a.vocab = dims->vocab;
  a.inv_tau = 1.f / dims->temperature;
  a.c = a.inv_tau * kLog2;
  a.ignore = dims->ignore_index;
  a.logits = logits;
  a.l_stride = logits_row_stride;
  a.targets = targets;
  a.stats = reinterpret_cast<const float4*>(stats);
  a.dlp = d_logprobs;
  a.dlp_stride = d_logprobs_stride;
  a.dh = d_entropy;
  a.dh_stride = d_entropy_stride;
  a.dz = d_logits;
  a.d_stride = d_logits_row_stride;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(a.rows));
  if (dtype == SDM_RT_BF16)
    hipLaunchKernelGGL(logprob_grad_kernel<bf16_t>, grid, dim3(kRowThreads), 0, st, a);
  else
    hipLaunchKernelGGL(logprob_grad_kernel<float>, grid, dim3(kRowThreads), 0, st, a);
  return check_launch("token_logprobs_grad");
}

}  // extern "C"
