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
  const int* counts;    // partial counts of those rows
  int n_counts;
  float* row_loss;
  float4* stats;        // per row: maximum (or near it), 1 / sum at the temperature, 1 / sum at 1, the row's weight
};

// a row has a teacher: an entry in the vocabulary whose logit over the temperature is not -inf; a label: one in the
// vocabulary (else -1)
__device__ __forceinline__ bool teacher_entry(int64_t id, float t, int vocab) {
  return id >= 0 && id < vocab && !(t == -INFINITY);
}
__device__ __forceinline__ int has_label(const DistillArgs& a, int64_t r) {
  if (!a.labels || a.ce == 0.f) return -1;
  const int64_t l = a.labels[r];
  return l >= 0 && l < a.vocab && l != a.ignore ? static_cast<int>(l) : -1;
}

// What a row aims at, found once: whether it has a teacher and whether that may repeat an id, its label or -1; counts[block]:
// how many of the block's rows have either.  A wave takes four rows at a time.  Repeats are told by a table of 512 words
// per row in LDS: an id's hash picks a word and three of its bits, and one that finds them set may be a repeat (of 100
// distinct ids that happens in 1 row of 100; with one bit of 2^14 it was 1 of 4).  In the loss and the gradient made along with
// it only such rows compare their ids pair by pair, which they pay for at their end (512 x 151,936 with 100 entries: 93 us, 100
// if all rows did); sdm_rt_distill_grad does not know them and compares every row's.
struct Target {
  int flags;
  int label;
};
constexpr int kTaught = 1, kRepeats = 2;
constexpr int kSeenBits = 9, kSeenWords = 1 << kSeenBits;
constexpr int kTargetWaves = 16, kTargetRows = 4;
constexpr size_t kTargetLds = kTargetWaves * kTargetRows * kSeenWords * sizeof(uint32_t);   // 128 KiB

__global__ void __launch_bounds__(64 * kTargetWaves) distill_targets_kernel(DistillArgs a, Target* __restrict__ targets,
                                                                            int* __restrict__ counts) {
  extern __shared__ uint4 seen_lds[];
  __shared__ int red[kTargetWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint4* seen_own = seen_lds + wave * (kTargetRows * kSeenWords / 4);
  const int64_t waves = static_cast<int64_t>(gridDim.x) * kTargetWaves;
  int n = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kTargetWaves + wave; r0 < a.rows; r0 += waves * kTargetRows) {
    int label[kTargetRows];
    bool any[kTargetRows], twice[kTargetRows];
#pragma unroll
    for (int q = 0; q < kTargetRows; ++q) {
      any[q] = twice[q] = false;
      label[q] = has_label(a, min(r0 + q * waves, a.rows - 1));
    }
    if (a.kd > 0.f && a.k > 0) {
      for (int i = lane; i < kTargetRows * kSeenWords / 4; i += 64) seen_own[i] = make_uint4(0, 0, 0, 0);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // before the lanes' marks
      for (int i0 = 0; i0 < a.k; i0 += 64) {
        const int i = min(i0 + lane, a.k - 1);
        int64_t id[kTargetRows];
        float t[kTargetRows];
#pragma unroll
        for (int q = 0; q < kTargetRows; ++q) {
          const int64_t r = min(r0 + q * waves, a.rows - 1);
          id[q] = a.ids[r * a.i_stride + i];
          t[q] = a.top[r * a.t_stride + i];
        }
#pragma unroll
        for (int q = 0; q < kTargetRows; ++q) {
          const bool live = i0 + lane < a.k && teacher_entry(id[q], t[q] * a.inv_tau, a.vocab);
          any[q] |= live;
          if (live) {
            const uint32_t h = static_cast<uint32_t>(id[q]) * 2654435761u;
            const uint32_t bits = 1u << (h >> 18 & 31) | 1u << (h >> 13 & 31) | 1u << (h >> 8 & 31);
            uint32_t* seen = reinterpret_cast<uint32_t*>(seen_own) + q * kSeenWords;
            twice[q] |= (bits & ~atomicOr(&seen[h >> (32 - kSeenBits)], bits)) == 0;
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kTargetRows; ++q) {
      const int64_t r = r0 + q * waves;
      const bool taught = __ballot(any[q]) != 0, repeats = __ballot(twice[q]) != 0;
      if (r >= a.rows) continue;
      if (lane == 0) targets[r] = Target{(taught ? kTaught : 0) | (repeats ? kRepeats : 0), label[q]};
      n += taught || label[q] >= 0;
    }
  }
  if (lane == 0) red[wave] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int s = 0;
    for (int w = 0; w < kTargetWaves; ++w) s += red[w];
    counts[blockIdx.x] = s;
  }
}

constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

// How the exponentials at temperature 1 come from those at the temperature, where both terms need them: none (one sum
// serves: one term only, or temperature 1); by squaring, at temperature 2 (a multiplication has a quarter of an
// exponential's issue time: 16,384 x 32,768 bf16 440 us, with exponentials of their own 460; the square of a value off by r
// is off by 2 r + 2^-24); by exponentials of their own.
enum Second { kOneSum, kSquare, kOwnExp };

template <Second S>
__device__ __forceinline__ float second_exp(float et, float x) {
  if constexpr (S == kSquare) return et * et;
  if constexpr (S == kOwnExp) return __builtin_amdgcn_exp2f(x * kLog2e);
  return et;
}

// the gradient of a logit x above the maximum by the softmaxes, at p_v + a1 p1_v
template <Second S>
__device__ __forceinline__ float gradient_value(float x, float ct, float at, float a1) {
  const float et = __builtin_amdgcn_exp2f(x * ct);
  if constexpr (S == kOneSum) return at * et;
  return fmaf(a1, second_exp<S>(et, x), at * et);
}

// What a row's workgroup holds of its targets in LDS: k entries of the teacher and one of the label, their ids (-1: none),
// the teacher's exponents over the temperature (then its shares q), the student's logits at the ids, and the shares summed
// over equal ids.
struct Entries {   // arrays of k + 1, last the label's (its q is 0)
  int* id;
  float* q;
  float* z;
  float* sum;
};
__device__ __forceinline__ Entries entries_in(char* lds, int k) {
  const int n = k + 1;
  Entries t;
  t.id = reinterpret_cast<int*>(lds);
  t.q = reinterpret_cast<float*>(lds) + n;
  t.z = t.q + n;
  t.sum = t.z + n;
  return t;
}
inline size_t entries_bytes(int k) { return (static_cast<size_t>(k) + 1) * 16; }

// One wave's part of it.  first_id, first_top: the lane's first entry, loaded by the caller (before the row, so that the
// gathers below need not wait for it).  A label that the teacher names too has no entry of its own.  Returns the sum of the
// teacher's exponentials against their maximum, which t.q holds the differences to.
template <typename T>
__device__ __forceinline__ float load_entries(const DistillArgs& a, int64_t r, const T* z, bool taught, int label,
                                              int64_t first_id, float first_top, const Entries& t) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  bool named = false;
  for (int i = lane; i < a.k; i += 64) {
    const int64_t id64 = i == lane ? first_id : a.ids[r * a.i_stride + i];
    const float x = (i == lane ? first_top : a.top[r * a.t_stride + i]) * a.inv_tau;
    const bool live = taught && teacher_entry(id64, x, a.vocab);
    const int id = live ? static_cast<int>(id64) : -1;
    t.q[i] = x;
    t.id[i] = id;
    t.z[i] = to_f32(z[max(id, 0)]);
    if (live) m = fmaxf(m, x);
    named |= live && id == label;
  }
  named = __ballot(named) != 0;
  if (lane == 0) {
    t.id[a.k] = named ? -1 : label;
    t.q[a.k] = t.sum[a.k] = 0.f;
    t.z[a.k] = to_f32(z[max(label, 0)]);
  }
  m = wave_max(m);
  float s = 0.f;
  for (int i = lane; i < a.k; i += 64) {   // each lane its own entries again
    const float x = t.q[i] - m;
    t.q[i] = x;
    if (t.id[i] >= 0) s += expf(x);
  }
  return wave_add(s);
}

// Each thread its entries, where ids repeat: the shares of equal ids together.
__device__ __forceinline__ void sum_equal_ids(const DistillArgs& a, const Entries& t) {
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    const int id = t.id[i];
    float sum = 0.f;
    if (id >= 0) {
#pragma unroll 8
      for (int j = 0; j < a.k; ++j) sum += t.id[j] == id ? t.q[j] : 0.f;
    }
    t.sum[i] = sum;
  }
}

// The gradient at the entries' ids, put right after the pass over the row: base(z) less the shares (summed over equal ids)
// and the label; a repeated id's lanes all write the same.  By the waves that wrote the pieces, each after its own stores,
// so that no wave waits for another's: the threads take the row's pieces in turn, beginning anew at first_end (where the
// first chunk ends), and a thread each the values past the last whole piece.
template <typename T, typename F>
__device__ __forceinline__ void put_right(const DistillArgs& a, const Entries& t, const float* sums, int label, float kd,
                                          float ce, T* dr, int threads, int first_end, F base) {
  constexpr int kN = Piece<T>::kN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int whole = a.vocab / kN * kN;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");   // after the wave's stores
  __builtin_amdgcn_wave_barrier();
  for (int i = lane; i <= a.k; i += 64) {
    const int id = t.id[i];
    const int owner = id < whole ? (id < first_end ? id : id - first_end) / kN % threads : id - whole;
    if (id >= 0 && (owner >> 6) == wave)
      dr[id] = from_f32<T>(base(t.z[i]) - kd * sums[i] - (id == label ? ce : 0.f));
  }
}

// A row's loss and, with GRAD, its gradient for grad_out = 1, in one pass over the row by one workgroup.  A thread holds NV
// 16-byte pieces of the row in registers, so it is read once, all loads at once; every wave takes its own maximum and sums
// against it, and the workgroup joins them over LDS; then the gradient comes from the registers, and no barrier waits for
// stores.  The first wave gathers the targets meanwhile and takes the loss.  Bound by memory, a row in and a row out: what
// counts is that enough rows are under way on a compute unit while others wait for loads or stores (16,384 x 32,768 bf16,
// two sums: 8 waves to a SIMD by their registers 440 us, 6 waves 455, 5 waves 556; a copy of as many bytes 429).
//   kOne   a workgroup per row, several to a compute unit
//   kRoll  a workgroup holds a compute unit's registers: it takes rows in turn, and as a piece's gradient is stored its
//          registers take the next row's piece, so loads and stores overlap all the same
//   kMulti longer rows, or rows without a gradient, go by in chunks, with running references and sums, piece after piece as
//          they arrive (100 x 300,001: 104 us with a chunk's maximum first, now 73; of no use to a row held whole); the last
//          chunk stays in registers, the others are read again for the gradient
enum Kind { kOne, kRoll, kMulti };
constexpr int kBigThreads = 768;   // 12 waves: 168 registers a thread

template <typename T, int NV, bool GRAD, Second S, Kind K>
__global__ void __launch_bounds__(NV > 8 ? kBigThreads : 1024, NV > 8 ? 3 : K == kMulti ? 4 : 8)
    distill_kernel(DistillArgs a, const Target* __restrict__ targets, T* __restrict__ dz, int64_t d_stride) {
  constexpr bool BOTH = S != kOneSum;
  extern __shared__ char lds[];
  __shared__ float red[16][3];
  __shared__ float shared_ts;
  __shared__ int shared_count;
  constexpr int kN = Piece<T>::kN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int step = blockDim.x * kN;   // values of a piece of every thread
  const int chunk = NV * step;
  const uint32_t own = threadIdx.x * kN;
  const int whole = a.vocab / kN * kN;
  const int c_tail = whole + static_cast<int>(threadIdx.x);   // the values past the last whole piece: a thread each
  const float ct = a.kd > 0.f ? a.inv_tau * kLog2e : kLog2e;
  const bool weighted = a.mean && (GRAD || a.stats);   // a row's weight in the gradient, made here or from the stats
  const float slack = 16.f / fmaxf(ct, kLog2e);   // kMulti: a factor of up to 2^16 in the sums
  const Entries t = entries_in(lds, a.k);
  // chunks of a row, the first of them the partial one
  const int n_chunks = K == kMulti ? max((whole + chunk - 1) / chunk, 1) : 1;
  const int first_end = whole - (n_chunks - 1) * chunk;
  Piece<T> p[NV];
  // piece v of this thread in [begin, end); where it has none its registers keep the -inf they start with (a uniform address
  // and the thread's own offset: 64-bit addresses of every piece would take the registers)
#pragma unroll
  for (int v = 0; v < NV; ++v) p[v].fill(-INFINITY);
  const uint32_t own_bytes = own * sizeof(T);
  auto load_piece = [&](const T* z, int v, int begin, int end) {
    const char* at = reinterpret_cast<const char*>(z + begin + v * step);
    if (static_cast<int>(own) < end - begin - v * step) p[v].load(reinterpret_cast<const T*>(at + own_bytes));
  };
  auto load = [&](const T* z, int begin, int end) {
#pragma unroll
    for (int v = 0; v < NV; ++v) load_piece(z, v, begin, end);
  };
  if (K == kRoll) load(static_cast<const T*>(a.logits) + blockIdx.x * a.l_stride, 0, first_end);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
    T* dr = GRAD ? dz + r * d_stride : nullptr;
    const Target target = targets[r];
    const bool taught = target.flags & kTaught, repeats = target.flags & kRepeats;
    const bool live = taught || target.label >= 0;   // else nothing of the row counts, whatever its logits hold
    if (K != kRoll && !live) {
      if (GRAD) {
        Piece<T> none;
        none.r = make_uint4(0, 0, 0, 0);
        for (int c = 0; c + static_cast<int>(own) < whole; c += step) none.store(dr + c + own);
        if (c_tail < a.vocab) dr[c_tail] = T{};
      }
      if (threadIdx.x == 0) {
        a.row_loss[r] = 0.f;
        if (a.stats) a.stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      return;
    }
    int64_t first_id = -1;
    float first_top = 0.f;
    if (wave == 0 && lane < a.k && taught) {
      first_id = a.ids[r * a.i_stride + lane];
      first_top = a.top[r * a.t_stride + lane];
    }
    if (K != kRoll) load(z, 0, first_end);
    const float z_tail = c_tail < a.vocab ? to_f32(z[c_tail]) : -INFINITY;
    if (weighted && wave == waves - 1) {   // the mean's divisor
      int count = 0;
#pragma unroll 8
      for (int i = lane; i < a.n_counts; i += 64) count += a.counts[i];
      count = wave_add(count);
      if (lane == 0) shared_count = count;
    }
    if (wave == 0) {
      const float ts = load_entries(a, r, z, taught, target.label, first_id, first_top, t);
      if (lane == 0) shared_ts = ts;
    }
    float m = z_tail, st, s1 = 0.f;
    if (K != kMulti) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < kN; ++e) m = fmaxf(m, p[v].get(e));
#pragma unroll
      for (int v = 0; v < NV; ++v) p[v].forget();
      m = wave_max(m);
    }
    float ref = m == -INFINITY ? 0.f : m;   // nothing but -inf so far: sums of 0
    st = __builtin_amdgcn_exp2f((z_tail - ref) * ct);
    if (BOTH) s1 = second_exp<S>(st, z_tail - ref);
    for (int q = 0;;) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {   // a piece's values at a time: those of all pieces would take the registers
        if (K == kMulti) {   // the sums of a piece while the next ones load, against a reference of each lane's
          float pm = p[v].get(0);
#pragma unroll
          for (int e = 1; e < kN; ++e) pm = fmaxf(pm, p[v].get(e));
          if (__any(pm > m + slack)) {   // seldom: it follows a later maximum only past `slack`
            const float to = fmaxf(m, pm);
            if (m > -INFINITY) {
              st *= __builtin_amdgcn_exp2f((m - to) * ct);
              if (BOTH) s1 *= __builtin_amdgcn_exp2f((m - to) * kLog2e);
            }
            m = to;
            ref = m == -INFINITY ? 0.f : m;
          }
        }
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float x = p[v].get(e) - ref;
          const float et = __builtin_amdgcn_exp2f(x * ct);
          st += et;
          if (BOTH) s1 += second_exp<S>(et, x);
        }
        if (K == kMulti) p[v].forget();
        __builtin_amdgcn_sched_barrier(0);
      }
      if (K != kMulti || ++q == n_chunks) break;
      load(z, first_end + (q - 1) * chunk, first_end + q * chunk);
    }
    if (K != kMulti) {
#pragma unroll
      for (int v = 0; v < NV; ++v) p[v].forget();
    } else {
      const float mw = wave_max(m);
      if (m > -INFINITY) {
        st *= __builtin_amdgcn_exp2f((m - mw) * ct);
        if (BOTH) s1 *= __builtin_amdgcn_exp2f((m - mw) * kLog2e);
      }
      m = mw;
    }
    st = wave_add(st);
    if (BOTH) s1 = wave_add(s1);
    if (lane == 0) {
      red[wave][0] = m;
      red[wave][1] = st;
      red[wave][2] = s1;
    }
    lds_barrier();
    m = red[0][0];
    for (int w = 1; w < waves; ++w) m = fmaxf(m, red[w][0]);
    st = s1 = 0.f;
    for (int w = 0; w < waves; ++w) {
      // a wave of nothing but -inf has sums of 0 (NaN where it met one); a row of nothing but -inf is NaN
      const float d = red[w][0] - m;
      const bool none = red[w][0] == -INFINITY && m > -INFINITY;
      st += red[w][1] * (none ? 1.f : __builtin_amdgcn_exp2f(d * ct));
      if (BOTH) s1 += red[w][2] * (none ? 1.f : __builtin_amdgcn_exp2f(d * kLog2e));
    }
    if (!BOTH) s1 = st;
    const float inv_t = taught ? 1.f / st : 0.f, inv_1 = target.label >= 0 ? 1.f / s1 : 0.f;
    const float w = weighted ? 1.f / static_cast<float>(max(shared_count, 1)) : 1.f;
    if (wave == 0) {
      float loss = 0.f;
      const float ts = shared_ts, lt = logf(ts), ls = logf(st);
      for (int i = lane; i < a.k; i += 64) {
        if (t.id[i] < 0) continue;
        const float lq = t.q[i];
        const float q = expf(lq) / ts;
        t.q[i] = q;
        if (q > 0.f || q != q) loss += q * ((lq - lt) - ((t.z[i] - m) * a.inv_tau - ls));
      }
      loss = wave_add(loss) * a.kd;
      if (target.label >= 0) loss += a.ce * (logf(s1) - (t.z[a.k] - m));
      if (lane == 0) {
        a.row_loss[r] = live ? loss : 0.f;
        if (a.stats) a.stats[r] = live ? make_float4(m, inv_t, inv_1, w) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if (!GRAD) return;
    const float kd = taught ? w * a.kd_grad : 0.f, ce = target.label >= 0 ? w * a.ce : 0.f;
    const float at = BOTH ? kd * inv_t : kd * inv_t + ce * inv_1, a1 = ce * inv_1;
    auto value = [&](float x) {
      const float g = gradient_value<S>(x - m, ct, at, a1);
      return K == kRoll && !live ? 0.f : g;
    };
    const T* z_next = static_cast<const T*>(a.logits) + min(r + gridDim.x, a.rows - 1) * a.l_stride;   // kRoll
    for (int q = n_chunks - 1; q >= 0; --q) {
      const int begin = q == 0 ? 0 : first_end + (q - 1) * chunk, end = first_end + q * chunk;
      if (K == kMulti && q < n_chunks - 1) load(z, begin, end);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x[kN];
#pragma unroll
        for (int e = 0; e < kN; ++e) x[e] = value(p[v].get(e));
        Piece<T> o;
        o.set(x);
        char* at_v = reinterpret_cast<char*>(dr + begin + v * step);
        if (static_cast<int>(own) < end - begin - v * step) o.store(reinterpret_cast<T*>(at_v + own_bytes));
        if (K == kRoll) load_piece(z_next, v, 0, first_end);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (c_tail < a.vocab) dr[c_tail] = from_f32<T>(value(z_tail));
    lds_barrier();   // the shares are there (the stores need not be)
    if (repeats) {   // the same for the workgroup
      sum_equal_ids(a, t);
      lds_barrier();
    }
    put_right(a, t, repeats ? t.sum : t.q, target.label, kd, ce, dr, blockDim.x, first_end, value);
    if (K != kRoll) return;
    lds_barrier();   // before the next row's entries
  }
}

// loss = the sum of the rows' losses (in float64, in a fixed order), divided by the rows with a target if `mean`
__global__ void __launch_bounds__(1024) distill_sum_kernel(DistillArgs a, float* __restrict__ loss) {
  __shared__ double red[16];
  __shared__ int red_count[16];
  const int i0 = threadIdx.x;
  int count = i0 < a.n_counts ? a.counts[i0] : 0;   // at most kCountBlocks of them
  double s = 0.0;
  for (int64_t i = i0; i < a.rows; i += 16 * 1024) {
    float v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = a.row_loss[min(i + q * 1024, a.rows - 1)];   // no load behind a branch
#pragma unroll
    for (int q = 0; q < 16; ++q) s += i + q * 1024 < a.rows ? static_cast<double>(v[q]) : 0.0;
  }
#pragma unroll
  for (int j = 32; j > 0; j >>= 1) s += __shfl_xor(s, j);
  count = wave_add(count);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = s;
    red_count[threadIdx.x >> 6] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) {
      s += red[w];
      count += red_count[w];
    }
    *loss = static_cast<float>(a.mean ? s / max(count, 1) : s);
  }
}

// d_logits[r][v] = g w (kd_grad (p_v - q_v) + ce (p1_v - [v = label])) from the saved maxima and sums, a workgroup per row
// in turn.  unless_one: nothing to do where g is 1 (d_logits holds that gradient already).
constexpr int kGradThreads = 512;

template <typename T, Second S>
__global__ void __launch_bounds__(kGradThreads) distill_grad_kernel(DistillArgs a, const float* __restrict__ grad_out,
                                                                    int per_row, int unless_one, T* __restrict__ dz,
                                                                    int64_t d_stride) {
  extern __shared__ char lds[];
  constexpr int kN = Piece<T>::kN;
  if (unless_one && *grad_out == 1.f) return;
  const Entries t = entries_in(lds, a.k);
  const float ct = a.kd > 0.f ? a.inv_tau * kLog2e : kLog2e;
  const int whole = a.vocab / kN * kN;
  const int c_tail = whole + static_cast<int>(threadIdx.x);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
    T* dr = dz + r * d_stride;
    const float4 s = a.stats[r];
    const bool live_row = s.w != 0.f;
    const float g = grad_out[per_row ? r : 0] * s.w, m = s.x;
    const int label = live_row ? has_label(a, r) : -1;
    const float kd = g * a.kd_grad, ce = g * a.ce;
    const float at = S != kOneSum ? kd * s.y : kd * s.y + ce * s.z, a1 = ce * s.z;
    auto value = [&](float x) { return live_row ? gradient_value<S>(x - m, ct, at, a1) : 0.f; };
    if (live_row && threadIdx.x < 64) {
      const int lane = threadIdx.x;
      const bool one = a.kd > 0.f && lane < a.k;
      const float ts = load_entries(a, r, z, a.kd > 0.f, label, one ? a.ids[r * a.i_stride + lane] : -1,
                                    one ? a.top[r * a.t_stride + lane] : 0.f, t);
      for (int i = lane; i < a.k; i += 64) t.q[i] = t.id[i] >= 0 ? expf(t.q[i]) / ts : 0.f;
    }
#pragma unroll 4
    for (int c = threadIdx.x * kN; c < whole; c += kGradThreads * kN) {
      Piece<T> p;
      p.load(z + c);
      float v[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = value(p.get(e));
      p.set(v);
      p.store(dr + c);
    }
    if (c_tail < a.vocab) dr[c_tail] = from_f32<T>(value(to_f32(z[c_tail])));
    if (!live_row) continue;   // the same for the workgroup
    lds_barrier();
    sum_equal_ids(a, t);
    lds_barrier();
    put_right(a, t, t.sum, label, kd, ce, dr, kGradThreads, whole, value);
    lds_barrier();   // before the next row's entries
  }
}

constexpr int kCountBlocks = 256;   // one workgroup of the targets' to a compute unit

inline int fill_distill(const sdm_rt_distill* d, const void* logits, int64_t l_stride, sdm_rt_dtype dtype,
                        const int64_t* ids, int64_t i_stride, const float* top, int64_t t_stride, const int64_t* labels,
                        DistillArgs* a) {
  int rc;
  if (!d) return set_err(SDM_RT_EINVAL, "dims is NULL");
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (d->rows < 0 || d->vocab < 1 || d->top_k < 0) return set_err(SDM_RT_EINVAL, "rows and top_k must be >= 0, vocab >= 1");
  if (d->rows > (1 << 21)) return set_err(SDM_RT_EUNSUPPORTED, "rows must be at most 2^21");
  if (d->vocab > (1 << 30)) return set_err(SDM_RT_EUNSUPPORTED, "vocab must be at most 2^30");
  if (d->top_k > kMaxTop) return set_err(SDM_RT_EUNSUPPORTED, "top_k = %d must be at most %d", d->top_k, kMaxTop);
  // its square weighs the teacher's part (0 would say that there is none), its reciprocal times log2(e) the exponents
  if (!(d->temperature >= 1e-18f) || !(d->temperature <= 1e18f))
    return set_err(SDM_RT_EINVAL, "temperature must be positive and finite, from 1e-18 to 1e18");
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

// workspace: the partial counts, the rows' targets, their losses (SDM_RT_NONE keeps those in loss)
inline size_t distill_bytes(const sdm_rt_distill* d) {
  return kCountBlocks * sizeof(int) +
         static_cast<size_t>(d->rows) * (sizeof(Target) + (d->reduction == SDM_RT_NONE ? 0 : sizeof(float)));
}

template <typename F>
void by_second(const DistillArgs& a, F launch) {
  if (!(a.kd > 0.f && a.ce > 0.f) || a.inv_tau == 1.f)
    launch(std::integral_constant<Second, kOneSum>{});
  else if (a.inv_tau == 0.5f)
    launch(std::integral_constant<Second, kSquare>{});
  else
    launch(std::integral_constant<Second, kOwnExp>{});
}

template <typename T, int NV, bool GRAD, Kind K>
void launch_distill(const DistillArgs& a, int64_t groups, int threads, const Target* targets, void* dz, int64_t d_stride,
                    hipStream_t st) {
  by_second(a, [&](auto s) {
    hipLaunchKernelGGL((distill_kernel<T, NV, GRAD, decltype(s)::value, K>), dim3(static_cast<unsigned>(groups)),
                       dim3(threads), entries_bytes(a.k), st, a, targets, static_cast<T*>(dz), d_stride);
  });
}

// Threads of a row's workgroup and pieces of a thread: few pieces while a few waves hold the row (a wave computes on all its
// pieces, there or not), 8 up to 16 waves, then 16 and 25 of 12 waves, where a compute unit's registers end, then chunks
// (512 x 151,936 bf16 in chunks 1% slower, 1,200 rows 8%).
template <typename T>
void launch_distill_rows(const DistillArgs& a, const Target* targets, void* dz, int64_t d_stride, hipStream_t st) {
  const int pieces = a.vocab / Piece<T>::kN;
  auto threads = [&](int nv) { return std::max(64, std::min(1024, (pieces + 64 * nv - 1) / (64 * nv) * 64)); };
  const int64_t units = 256;   // compute units
  if (!dz)
    launch_distill<T, 8, false, kMulti>(a, a.rows, threads(8), targets, dz, d_stride, st);
  else if (pieces <= 2 * 64)
    launch_distill<T, 2, true, kOne>(a, a.rows, threads(2), targets, dz, d_stride, st);
  else if (pieces <= 4 * 256)
    launch_distill<T, 4, true, kOne>(a, a.rows, threads(4), targets, dz, d_stride, st);
  else if (pieces <= 8 * 1024)
    launch_distill<T, 8, true, kOne>(a, a.rows, threads(8), targets, dz, d_stride, st);
  else if (pieces <= 16 * kBigThreads)
    launch_distill<T, 16, true, kRoll>(a, std::min(a.rows, units), kBigThreads, targets, dz, d_stride, st);
  else if (pieces <= 25 * kBigThreads)
    launch_distill<T, 25, true, kRoll>(a, std::min(a.rows, units), kBigThreads, targets, dz, d_stride, st);
  else
    launch_distill<T, 16, true, kMulti>(a, a.rows, kBigThreads, targets, dz, d_stride, st);
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

uint64_t sdm_rt_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();   // the null stream while another one is captured: not captured itself
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
}

size_t sdm_rt_distill_workspace_bytes(const sdm_rt_distill* dims) {
  return dims && dims->rows >= 0 ? distill_bytes(dims) : 0;
}

int sdm_rt_distill_loss(const sdm_rt_distill* dims, const void* logits, int64_t logits_row_stride, sdm_rt_dtype dtype,
                        const int64_t* top_ids, int64_t top_ids_row_stride, const float* top_logits,
                        int64_t top_logits_row_stride, const int64_t* labels, float* loss, float* stats, void* d_logits,
                        int64_t d_logits_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  DistillArgs a{};
  int rc = fill_distill(dims, logits, logits_row_stride, dtype, top_ids, top_ids_row_stride, top_logits,
                        top_logits_row_stride, labels, &a);
  if (rc) return rc;
  const bool none = dims->reduction == SDM_RT_NONE;
  if (none && a.rows == 0) return SDM_RT_OK;
  if (!loss) return set_err(SDM_RT_EINVAL, "loss is NULL");
  if (stats && reinterpret_cast<uintptr_t>(stats) % 16) return set_err(SDM_RT_EINVAL, "stats must be 16-byte aligned");
  if (d_logits && d_logits_row_stride < a.vocab) return set_err(SDM_RT_EINVAL, "d_logits_row_stride must be >= vocab");
  if (!workspace || workspace_bytes < distill_bytes(dims))
    return set_err(SDM_RT_ENOSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, distill_bytes(dims));
  hipStream_t st = static_cast<hipStream_t>(stream);
  int* counts = static_cast<int*>(workspace);
  Target* targets = reinterpret_cast<Target*>(counts + kCountBlocks);
  a.row_loss = none ? loss : reinterpret_cast<float*>(targets + a.rows);
  a.stats = reinterpret_cast<float4*>(stats);
  a.counts = counts;
  a.n_counts = static_cast<int>(std::min<int64_t>(kCountBlocks, (a.rows + kTargetWaves - 1) / kTargetWaves));
  if (a.rows > 0) {
    static const bool lds = allow_lds(reinterpret_cast<const void*>(distill_targets_kernel));
    if (!lds) return lds_err("distill_loss");
    hipLaunchKernelGGL(distill_targets_kernel, dim3(a.n_counts), dim3(64 * kTargetWaves), kTargetLds, st, a, targets, counts);
    if (dtype == SDM_RT_BF16)
      launch_distill_rows<bf16_t>(a, targets, d_logits, d_logits_row_stride, st);
    else
      launch_distill_rows<float>(a, targets, d_logits, d_logits_row_stride, st);
  }
  if (!none) hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, a, loss);
  return check_launch("distill_loss");
}

int sdm_rt_distill_grad(const sdm_rt_distill* dims, const void* logits, int64_t logits_row_stride, sdm_rt_dtype dtype,
                        const int64_t* top_ids, int64_t top_ids_row_stride, const float* top_logits,
                        int64_t top_logits_row_stride, const int64_t* labels, const float* stats, const float* grad_out,
                        int32_t unless_one, void* d_logits, int64_t d_logits_row_stride, void* stream) {
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
  const int per_row = dims->reduction == SDM_RT_NONE;
  if (unless_one && per_row) return set_err(SDM_RT_EINVAL, "unless_one is for a loss of one value");
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(a.rows, unless_one ? 1024 : 65536)));
  const size_t lds = entries_bytes(a.k);
  by_second(a, [&](auto s) {
    if (dtype == SDM_RT_BF16)
      hipLaunchKernelGGL((distill_grad_kernel<bf16_t, decltype(s)::value>), grid, dim3(kGradThreads), lds, st, a, grad_out,
                         per_row, unless_one, static_cast<bf16_t*>(d_logits), d_logits_row_stride);
    else
      hipLaunchKernelGGL((distill_grad_kernel<float, decltype(s)::value>), grid, dim3(kGradThreads), lds, st, a, grad_out,
                         per_row, unless_one, static_cast<float*>(d_logits), d_logits_row_stride);
  });
  return check_launch("distill_grad");
}

}  // extern "C"
