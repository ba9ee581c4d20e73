// sdm_distill.hip -- the distillation loss from a teacher's top logits, joined by the cross entropy of labels
// (sdm_rt_distill_loss), and its gradient (sdm_rt_distill_grad).
#include "sdm_vocab.h"

namespace sdmrt {

struct DistillArgs {
  int64_t rows;
  int vocab, k;
  float inv_tau, kd, ce;   // 1 / temperature; alpha temperature^2; 1 - alpha (0 without labels)
  float kd_grad;           // alpha temperature
  int64_t ignore;
  const void* logits;
  int64_t l_stride;
  const int64_t* ids;   // [rows][k] the teacher's tokens (an id outside [0, vocab): no entry)
  int64_t i_stride;
  const float* top;     // [rows][k] their logits
  int64_t t_stride;
  const int64_t* labels;
  int mean;             // the loss is divided by the rows with a target
  const int* counts;    // mean: partial counts of those rows
  int n_counts;
  float* row_loss;
  float4* stats;        // per row: maximum, 1 / sum at the temperature, 1 / sum at 1, the row's weight
};

// row r has a teacher: an entry in the vocabulary whose logit over the temperature is not -inf; a label: one in the
// vocabulary
__device__ __forceinline__ bool teacher_entry(int64_t id, float t, int vocab) {
  return id >= 0 && id < vocab && !(t == -INFINITY);
}
__device__ __forceinline__ bool has_label(const DistillArgs& a, int64_t r, int* label) {
  if (!a.labels || a.ce == 0.f) return false;
  const int64_t l = a.labels[r];
  *label = static_cast<int>(l);
  return l >= 0 && l < a.vocab && l != a.ignore;
}

// counts[block]: the block's rows that have a target, a wave per row
__global__ void __launch_bounds__(1024) distill_count_kernel(DistillArgs a, int* __restrict__ counts) {
  __shared__ int red[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int n = 0;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * 16 + wave; r < a.rows; r += static_cast<int64_t>(gridDim.x) * 16) {
    int label;
    bool any = has_label(a, r, &label);
    if (a.kd > 0.f)
      for (int i = lane; i < a.k; i += 64) any |= teacher_entry(a.ids[r * a.i_stride + i], a.top[r * a.t_stride + i] * a.inv_tau, a.vocab);
    n += __ballot(any) != 0;
  }
  if (lane == 0) red[wave] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int s = 0;
    for (int w = 0; w < 16; ++w) s += red[w];
    counts[blockIdx.x] = s;
  }
}

constexpr int kDistillThreads = 256;
constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 6); ++w) v = fmaxf(v, red[w]);
  __syncthreads();
  return v;
}
template <typename V>
__device__ __forceinline__ V block_add(V v, V* red) {
  v = wave_add(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 6); ++w) v += red[w];
  __syncthreads();
  return v;
}

// The teacher's distribution of row r into LDS: tid[i], tq[i] for i < k (absent entries: id -1, 0).  Returns whether the
// row has a teacher; max and sum of its exponentials.
__device__ __forceinline__ bool load_teacher(const DistillArgs& a, int64_t r, int* tid, float* tq, float* red, float* tmax,
                                             float* tsum) {
  float m = -INFINITY;
  int any = 0;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    const int64_t id = a.ids[r * a.i_stride + i];
    const float t = a.top[r * a.t_stride + i] * a.inv_tau;
    const bool live = a.kd > 0.f && teacher_entry(id, t, a.vocab);
    tid[i] = live ? static_cast<int>(id) : -1;
    tq[i] = t;
    if (live) m = fmaxf(m, t);
    any |= live;
  }
  m = block_max(m, red);
  any = block_add(any, reinterpret_cast<int*>(red));
  float s = 0.f;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    if (tid[i] >= 0) s += expf(tq[i] - m);
  }
  s = block_add(s, red);
  *tmax = m;
  *tsum = s;
  return any != 0;
}

// one workgroup per row: the row's maximum, then its sums at the temperature and at 1, then the loss
template <typename T>
__global__ void __launch_bounds__(kDistillThreads) distill_loss_kernel(DistillArgs a) {
  __shared__ int tid[kMaxTop];
  __shared__ float tq[kMaxTop];
  __shared__ float red[kDistillThreads / 64];
  constexpr int kN = Piece<T>::kN;
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
  float w = 1.f;
  if (a.mean) {
    int c = 0;
    for (int i = threadIdx.x; i < a.n_counts; i += blockDim.x) c += a.counts[i];
    c = block_add(c, reinterpret_cast<int*>(red));
    w = 1.f / static_cast<float>(max(c, 1));
  }
  int label = 0;
  const bool has_y = has_label(a, r, &label);
  float tm, ts;
  const bool has_t = load_teacher(a, r, tid, tq, red, &tm, &ts);
  if (!has_t && !has_y) {   // no target: nothing of the row counts, whatever its logits hold
    if (threadIdx.x == 0) {
      a.row_loss[r] = 0.f;
      if (a.stats) a.stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  float m = -INFINITY;
  for (int c = threadIdx.x * kN; c < a.vocab; c += kDistillThreads * kN) {
    Piece<T> p;
    const int live = min(kN, a.vocab - c);
    if (live == kN)
      p.load(z + c);
    else
      p.load_part(z + c, live, from_f32<T>(-INFINITY));
#pragma unroll
    for (int e = 0; e < kN; ++e) m = fmaxf(m, p.get(e));
  }
  m = block_max(m, red);
  const float ct = a.inv_tau * kLog2e;
  float st = 0.f, s1 = 0.f;
  for (int c = threadIdx.x * kN; c < a.vocab; c += kDistillThreads * kN) {
    Piece<T> p;
    const int live = min(kN, a.vocab - c);
    if (live == kN)
      p.load(z + c);
    else
      p.load_part(z + c, live, from_f32<T>(-INFINITY));
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float x = p.get(e) - m;
      st += __builtin_amdgcn_exp2f(x * ct);
      s1 += __builtin_amdgcn_exp2f(x * kLog2e);
    }
  }
  st = block_add(st, red);
  s1 = block_add(s1, red);
  float loss = 0.f;
  const float lt = logf(ts), ls = logf(st);
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    if (tid[i] < 0) continue;
    const float lq = tq[i] - tm;
    const float q = expf(lq) / ts;
    if (q > 0.f || q != q) loss += q * ((lq - lt) - ((to_f32(z[tid[i]]) - m) * a.inv_tau - ls));
  }
  loss = block_add(loss, red) * a.kd;
  if (has_y) loss += a.ce * (logf(s1) - (to_f32(z[label]) - m));
  if (threadIdx.x == 0) {
    a.row_loss[r] = loss;
    if (a.stats) a.stats[r] = make_float4(m, has_t ? 1.f / st : 0.f, has_y ? 1.f / s1 : 0.f, w);
  }
}

// loss = the sum of the rows' losses (in float64, in a fixed order), divided by the rows with a target if `mean`
__global__ void __launch_bounds__(1024) distill_sum_kernel(DistillArgs a, float* __restrict__ loss) {
  __shared__ double red[16];
  __shared__ int redc[16];
  int c = 0;
  for (int i = threadIdx.x; i < a.n_counts; i += 1024) c += a.counts[i];
  c = block_add(c, redc);
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) s += static_cast<double>(a.row_loss[i]);
#pragma unroll
  for (int j = 32; j > 0; j >>= 1) s += __shfl_xor(s, j);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += red[w];
    *loss = static_cast<float>(a.mean ? s / max(c, 1) : s);
  }
}

// d_logits[r][v] = g w (kd_grad (p_v - q_v) + ce (p1_v - [v = label])), one workgroup per row; q and the label are put
// right after the pass over the row, each by one thread (ids that a row repeats all write the same sum)
template <typename T>
__global__ void __launch_bounds__(kDistillThreads) distill_grad_kernel(DistillArgs a, const float* __restrict__ grad_out,
                                                                       int per_row, T* __restrict__ dz, int64_t d_stride) {
  __shared__ int tid[kMaxTop];
  __shared__ float tq[kMaxTop];
  __shared__ float red[kDistillThreads / 64];
  constexpr int kN = Piece<T>::kN;
  const int64_t r = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
  T* dr = dz + r * d_stride;
  const float4 s = a.stats[r];
  const float g = grad_out[per_row ? r : 0];
  const bool live_row = s.w != 0.f;
  const float ct = a.inv_tau * kLog2e, m = s.x;
  const float at = g * s.w * a.kd_grad * s.y, a1 = g * s.w * a.ce * s.z;
  for (int c = threadIdx.x * kN; c < a.vocab; c += kDistillThreads * kN) {
    Piece<T> p;
    const int live = min(kN, a.vocab - c);
    if (live == kN)
      p.load(z + c);
    else
      p.load_part(z + c, live, T{});
    float v[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float x = p.get(e) - m;
      v[e] = live_row ? at * __builtin_amdgcn_exp2f(x * ct) + a1 * __builtin_amdgcn_exp2f(x * kLog2e) : 0.f;
    }
    p.set(v);
    if (live == kN)
      p.store(dr + c);
    else
      p.store_part(dr + c, live);
  }
  if (!live_row) return;
  int label = 0;
  const bool has_y = has_label(a, r, &label);
  float tm, ts;
  load_teacher(a, r, tid, tq, red, &tm, &ts);
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) tq[i] = tid[i] >= 0 ? expf(tq[i] - tm) / ts : 0.f;
  __syncthreads();   // and the row's values are written
  for (int i = threadIdx.x; i < a.k + 1; i += blockDim.x) {
    const int id = i < a.k ? tid[i] : (has_y ? label : -1);
    if (id < 0) continue;
    float q = 0.f;
    for (int j = 0; j < a.k; ++j)
      if (tid[j] == id) q += tq[j];
    const float x = to_f32(z[id]) - m;
    float v = at * __builtin_amdgcn_exp2f(x * ct) - g * s.w * a.kd_grad * q;
    v += a1 * __builtin_amdgcn_exp2f(x * kLog2e) - (has_y && id == label ? g * s.w * a.ce : 0.f);
    dr[id] = from_f32<T>(v);
  }
}

constexpr int kCountBlocks = 256;

inline int fill_distill(const sdm_rt_distill* d, const void* logits, int64_t l_stride, sdm_rt_dtype dtype,
                        const int64_t* ids, int64_t i_stride, const float* top, int64_t t_stride, const int64_t* labels,
                        DistillArgs* a) {
  int rc;
  if (!d) return set_err(SDM_RT_EINVAL, "dims is NULL");
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (d->rows < 0 || d->vocab < 1 || d->top_k < 0) return set_err(SDM_RT_EINVAL, "rows and top_k must be >= 0, vocab >= 1");
  if (d->rows > (1 << 22)) return set_err(SDM_RT_EUNSUPPORTED, "rows must be at most 2^22");
  if (d->vocab > (1 << 30)) return set_err(SDM_RT_EUNSUPPORTED, "vocab must be at most 2^30");
  if (d->top_k > kMaxTop) return set_err(SDM_RT_EUNSUPPORTED, "top_k = %d must be at most %d", d->top_k, kMaxTop);
  if (!(d->temperature > 0.f) || !(d->temperature < INFINITY) || !(1.f / d->temperature < INFINITY))
    return set_err(SDM_RT_EINVAL, "temperature must be positive and finite");
  if (!(d->alpha >= 0.f && d->alpha <= 1.f)) return set_err(SDM_RT_EINVAL, "alpha must be in [0, 1]");
  if (d->reduction < 0 || d->reduction > 2) return set_err(SDM_RT_EINVAL, "unknown reduction %d", d->reduction);
  if (d->rows > 0) {
    if (!logits || bad_read_stride(l_stride, d->vocab))
      return set_err(SDM_RT_EINVAL, "logits must not be NULL, their row stride 0 or >= vocab");
    if (d->top_k > 0 && (!ids || !top || bad_read_stride(i_stride, d->top_k) || bad_read_stride(t_stride, d->top_k)))
      return set_err(SDM_RT_EINVAL, "top_ids and top_logits must not be NULL, their row strides 0 or >= top_k");
  }
  a->rows = d->rows;
  a->vocab = d->vocab;
  a->k = d->top_k;
  a->inv_tau = 1.f / d->temperature;
  a->kd = d->alpha * d->temperature * d->temperature;
  a->kd_grad = d->alpha * d->temperature;
  a->ce = labels ? 1.f - d->alpha : 0.f;
  a->ignore = d->ignore_index;
  a->logits = logits;
  a->l_stride = l_stride;
  a->ids = ids;
  a->i_stride = i_stride;
  a->top = top;
  a->t_stride = t_stride;
  a->labels = labels;
  a->mean = d->reduction == SDM_RT_MEAN;
  return SDM_RT_OK;
}

inline size_t distill_bytes(const sdm_rt_distill* d) {
  return kCountBlocks * sizeof(int) + (d->reduction == SDM_RT_NONE ? 0 : static_cast<size_t>(d->rows) * sizeof(float));
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

size_t sdm_rt_distill_workspace_bytes(const sdm_rt_distill* dims) {
  return dims && dims->rows >= 0 ? distill_bytes(dims) : 0;
}

int sdm_rt_distill_loss(const sdm_rt_distill* dims, const void* logits, int64_t logits_row_stride, sdm_rt_dtype dtype,
                        const int64_t* top_ids, int64_t top_ids_row_stride, const float* top_logits,
                        int64_t top_logits_row_stride, const int64_t* labels, float* loss, float* stats, void* workspace,
                        size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  DistillArgs a{};
  int rc = fill_distill(dims, logits, logits_row_stride, dtype, top_ids, top_ids_row_stride, top_logits,
                        top_logits_row_stride, labels, &a);
  if (rc) return rc;
  const bool none = dims->reduction == SDM_RT_NONE;
  if (none && a.rows == 0) return SDM_RT_OK;
  if (!loss) return set_err(SDM_RT_EINVAL, "loss is NULL");
  if (stats && reinterpret_cast<uintptr_t>(stats) % 16) return set_err(SDM_RT_EINVAL, "stats must be 16-byte aligned");
  if (!workspace || workspace_bytes < distill_bytes(dims))
    return set_err(SDM_RT_ENOSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, distill_bytes(dims));
  hipStream_t st = static_cast<hipStream_t>(stream);
  int* counts = static_cast<int*>(workspace);
  a.row_loss = none ? loss : reinterpret_cast<float*>(counts + kCountBlocks);
  a.stats = reinterpret_cast<float4*>(stats);
  if (a.mean) {
    a.counts = counts;
    a.n_counts = static_cast<int>(std::min<int64_t>(kCountBlocks, (a.rows + 15) / 16));
    if (a.rows > 0)
      hipLaunchKernelGGL(distill_count_kernel, dim3(a.n_counts), dim3(1024), 0, st, a, counts);
  }
  if (a.rows > 0) {
    const dim3 grid(static_cast<unsigned>(a.rows));
    if (dtype == SDM_RT_BF16)
      hipLaunchKernelGGL((distill_loss_kernel<bf16_t>), grid, dim3(kDistillThreads), 0, st, a);
    else
      hipLaunchKernelGGL((distill_loss_kernel<float>), grid, dim3(kDistillThreads), 0, st, a);
  }
  if (!none) hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, a, loss);
  return check_launch("distill_loss");
}

int sdm_rt_distill_grad(const sdm_rt_distill* dims, const void* logits, int64_t logits_row_stride, sdm_rt_dtype dtype,
                        const int64_t* top_ids, int64_t top_ids_row_stride, const float* top_logits,
                        int64_t top_logits_row_stride, const int64_t* labels, const float* stats, const float* grad_out,
                        void* d_logits, int64_t d_logits_row_stride, void* stream) {
  g_err[0] = 0;
  DistillArgs a{};
  int rc = fill_distill(dims, logits, logits_row_stride, dtype, top_ids, top_ids_row_stride, top_logits,
                        top_logits_row_stride, labels, &a);
  if (rc) return rc;
  if (a.rows == 0) return SDM_RT_OK;
  if (!stats || !grad_out || !d_logits) return set_err(SDM_RT_EINVAL, "stats, grad_out and d_logits must not be NULL");
  if (reinterpret_cast<uintptr_t>(stats) % 16) return set_err(SDM_RT_EINVAL, "stats must be 16-byte aligned");
  if (d_logits_row_stride < a.vocab) return set_err(SDM_RT_EINVAL, "d_logits_row_stride must be >= vocab");
  a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(a.rows));
  const int per_row = dims->reduction == SDM_RT_NONE;
  if (dtype == SDM_RT_BF16)
    hipLaunchKernelGGL((distill_grad_kernel<bf16_t>), grid, dim3(kDistillThreads), 0, st, a, grad_out, per_row,
                       static_cast<bf16_t*>(d_logits), d_logits_row_stride);
  else
    hipLaunchKernelGGL((distill_grad_kernel<float>), grid, dim3(kDistillThreads), 0, st, a, grad_out, per_row,
                       static_cast<float*>(d_logits), d_logits_row_stride);
  return check_launch("distill_grad");
}

}  // extern "C"
