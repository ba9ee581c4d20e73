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

// (z - max) / temperature; in halves, since the difference of two float32 of different signs may pass float32's range where its
// quotient does not
__device__ __forceinline__ float below_max(float z, float m, float inv_tau) { return (0.5f * z - 0.5f * m) * (2.f * inv_tau); }

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

// A row's target (-1: none) and its logit, loaded ahead.
struct RowTarget {
  int64_t id;
  float z;
};
__device__ __forceinline__ int64_t row_target(const LogprobArgs& a, int64_t r) {
  if (!a.logprobs) return -1;
  const int64_t y = a.targets[r];
  return y >= 0 && y < a.vocab && y != a.ignore ? y : -1;
}

// What becomes of a row's sums, by one thread.
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t r, const RowTarget& y, const RowSums& s, const RowLogs& g) {
  const bool bad = s.m == INFINITY || s.rest != s.rest, none = !bad && s.m == -INFINITY;
  if (a.logprobs) a.logprobs[r] = y.id < 0 ? 0.f : bad ? NAN : none ? -INFINITY : below_max(y.z, s.m, a.inv_tau) - g.l;
  const float h = bad ? NAN : none ? 0.f : g.h;
  if (a.entropy) a.entropy[r] = h;
  // a row of -inf: sums that make every p 0; the entropy is summed only where it is asked
  if (a.stats)
    a.stats[r] = bad    ? make_float4(NAN, NAN, NAN, 0.f)
                 : none ? make_float4(0.f, INFINITY, 0.f, 0.f)
                        : make_float4(s.m, g.l2, a.entropy ? h : NAN, 0.f);
}

// -- a row, or a slice of one, by one workgroup -------------------------------------------------------------------------
// The slice is in registers, NV 16-byte pieces a thread, so the row is read once: its maximum, its sums against that, and its
// alternatives all come from there.  At most 64 registers a thread, so that four workgroups of a 32,768-logit bf16 row are on
// a compute unit and load while others compute.  Without alternatives memory bounds it (16,384 x 32,768 bf16 with entropies
// 182 us call after call, 5.9 TB/s: what reading alone reaches here; a profiled training step's, behind a gradient, 245 in the
// median); a logit takes 4 instructions in the sums, one of them an exponential of four issue slots, and 1 in the maximum.
// With half of each row masked the entropies' sums are made twice (0 times -inf): 274 us, 192 without entropies.  With
// alternatives instructions bound it (2,048 x 151,936 bf16, 64 of them, 141 us at 4.4 TB/s: some 300 of a wave's 750
// instructions are not the sums'; with the join 64 take 143 us, 96 160, 128 186, 192 292, 256 525: a workgroup's LDS grows to
// 65 KB), and a single row the chain of its phases (32,768 logits 7 us).  Slices of 65,536 logits take the case of 64 to 189
// us, of 16,384 to 173; a row of 32,768 in two slices and a join 12.6 us in place of 8.8.
constexpr int kMaxSlots = kMaxAlternatives + kMaxAlternatives / 2 + 8;
constexpr int kCandidates = 1024;   // keys that are ranked against each other
constexpr uint32_t kLowest = 0x00800000u;   // the key of the least finite number

// What of a row's slices is joined later (slices > 1): their sums, and their alternatives' keys, falling, 0 behind the last.
struct Partial {
  RowSums* sums;    // [rows][slices]
  uint64_t* keys;   // [rows][slices][k]
};

struct RowLds {
  uint64_t keys[kCandidates];
  float top[1024];   // the threads' maxima
  float red[4][16];
  int count[16];
  uint32_t threshold;
  float log;
  int n, n_hot, n_kept;
  uint16_t hot[1024];   // threads with a logit at or above the threshold
};

// The key t for which k to 5/4 k of the threads' maxima (over 512 threads: of those of pairs of threads) have key >= t, or more
// where ties forbid that, by one wave that halves the range of keys: those maxima are k logits of the row, so all alternatives
// have keys >= t.  The key of the least finite number if fewer than k maxima are finite.
__device__ __forceinline__ uint32_t near_kth(const float* top, int threads, int k, float largest) {
  constexpr int PER = 8;
  const int lane = threadIdx.x & 63;
  uint32_t v[PER];
  float least = INFINITY;
  int n = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * 64 + lane;
    float x = at < threads ? top[at] : -INFINITY;
    if (threads > 512) x = fmaxf(x, at + 512 < threads ? top[at + 512] : -INFINITY);
    v[i] = ordered(x);
    const bool there = v[i] != 0;
    least = fminf(least, there ? x : INFINITY);
    n += __popcll(__ballot(there));
  }
  if (n < k) return kLowest;
  // k or more from lo on, fewer past hi.  The counts fall about exponentially, so the first guesses go by their logarithms (2 or 3
  // of them as a rule, where halving takes 8).
  least = -wave_max(-least);
  uint32_t lo = ordered(least), hi = max(ordered(largest), lo);
  float f_lo = least, f_hi = largest, l_lo = __builtin_amdgcn_logf(static_cast<float>(n)), l_hi = -1.f;
  const float wanted = __builtin_amdgcn_logf(1.125f * static_cast<float>(k));
  for (int tries = 0; lo < hi; ++tries) {
    uint32_t mid = lo + (hi - lo + 1) / 2;
    if (tries < 5) mid = min(max(ordered(fmaf(f_hi - f_lo, (l_lo - wanted) * __builtin_amdgcn_rcpf(l_lo - l_hi), f_lo)), lo + 1), hi);
    mid = __builtin_amdgcn_readfirstlane(mid);
    n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(v[i] >= mid));
    if (n >= k) {
      lo = mid;
      if (n <= k + k / 4) break;
      f_lo = unordered(mid);
      l_lo = __builtin_amdgcn_logf(static_cast<float>(n));
    } else {
      hi = mid - 1;
      f_hi = unordered(mid);
      l_hi = n ? __builtin_amdgcn_logf(static_cast<float>(n)) : -1.f;
    }
  }
  return lo;
}

// A thread's maximum over its pieces.  Bfloat16 values are ordered as whole numbers, two at a time: among those of the positive
// sign the signed maximum, where there are none the unsigned minimum (one instruction a value, unpacking and comparing floats
// two).  A NaN may be taken for the maximum, or passed over: the sums find it.
typedef short short2_t __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
template <typename T>
struct RunningMax;
template <>
struct RunningMax<bf16_t> {
  short2_t most = {-32768, -32768};
  ushort2_t least = {0xffff, 0xffff};
  __device__ __forceinline__ void add(const Piece<bf16_t>& p) {
    const uint32_t w[4] = {p.r.x, p.r.y, p.r.z, p.r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      most = __builtin_elementwise_max(most, __builtin_bit_cast(short2_t, w[i]));
      least = __builtin_elementwise_min(least, __builtin_bit_cast(ushort2_t, w[i]));
    }
  }
  __device__ __forceinline__ float get() const {
    const int a = max(most.x, most.y);
    const uint32_t b = min(least.x, least.y);
    return __uint_as_float((a >= 0 ? static_cast<uint32_t>(a) : b) << 16);
  }
};
template <>
struct RunningMax<float> {
  float most = -INFINITY;
  __device__ __forceinline__ void add(const Piece<float>& p) {
    most = fmaxf(fmaxf(most, p.get(0)), p.get(1));
    most = fmaxf(fmaxf(most, p.get(2)), p.get(3));
  }
  __device__ __forceinline__ float get() const { return most; }
};

// Keeps the work on a piece where it is written, so that the registers of one piece's values serve the next one's.
template <typename T>
__device__ __forceinline__ void in_turn(Piece<T>& p) {
  asm volatile("" : "+v"(p.r.x), "+v"(p.r.y), "+v"(p.r.z), "+v"(p.r.w));
}

// Ties in great number, or the best logits in a few threads' pieces: more than kCandidates logits at or above the threshold.
// The workgroup halves the range of keys until k to kCandidates logits are at or above one, or it is down to the k-th greatest
// key itself, of which it then takes as many as are wanted in the order of their ids.  The slice's pieces are read again each
// time, from the caches (held in registers they made the whole kernel spill); all threads get here together.  Returns how many
// keys it has listed.  64 x 32,768 bf16 rows of few different values, 20 alternatives: 30 us; counting from memory each time
// 210.
template <typename T, int NV>
__device__ __noinline__ int crowded(int k, const T* z, int n, int first, uint32_t lo, uint32_t hi, RowLds& lds) {
  constexpr int kN = Piece<T>::kN, kDrop = sizeof(T) == 2 ? 16 : 0;   // bits that a key of bfloat16 does not use
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, threads = blockDim.x, waves = threads >> 6;
  auto piece = [&](int v) {
    const int at = (v * threads + static_cast<int>(threadIdx.x)) * kN;
    Piece<T> p;
    if (at + kN <= n)
      p.load(z + at);
    else if (at < n)
      p.load_part(z + at, n - at, from_f32<T>(-INFINITY));
    else
      p.fill(-INFINITY);
    return p;
  };
  auto value_of = [](uint32_t key) { return unordered(key < (0x80000000u >> kDrop) ? (key << kDrop) | ((1u << kDrop) - 1) : key << kDrop); };
  auto sum_of_waves = [&](int c) {
    __syncthreads();   // the counts before these are read
    if (lane == 0) lds.count[wave] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < waves; ++w) c += lds.count[w];
    return c;
  };
  lo >>= kDrop;
  hi >>= kDrop;
  int c = kCandidates + 1;   // at or above lo: k or more
  while (lo < hi && c > kCandidates) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    const float f = value_of(mid);
    int mine = 0;
#pragma unroll 2
    for (int v = 0; v < NV; ++v) {
      const Piece<T> p = piece(v);
#pragma unroll
      for (int e = 0; e < kN; ++e) mine += p.get(e) >= f;
    }
    const int all = sum_of_waves(wave_add(mine));
    if (all >= k)
      lo = mid, c = all;
    else
      hi = mid - 1;
  }
  const float f = value_of(lo);
  __syncthreads();
  if (threadIdx.x == 0) lds.n = 0;
  __syncthreads();
#pragma unroll 1
  for (int v = 0; v < NV; ++v) {
    const Piece<T> p = piece(v);
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float x = p.get(e);
      if (c <= kCandidates ? x >= f : x > f) {
        const int at = atomicAdd(&lds.n, 1);
        if (at < kCandidates) lds.keys[at] = logit_key(x, first + (v * threads + static_cast<int>(threadIdx.x)) * kN + e);
      }
    }
  }
  __syncthreads();
  int listed = min(lds.n, kCandidates);
  if (c <= kCandidates) return listed;
  // fewer than k are greater; those equal, in the order of their ids: all threads' first pieces, then their second ones
#pragma unroll 1
  for (int v = 0; v < NV && listed < k; ++v) {
    const int at = (v * threads + static_cast<int>(threadIdx.x)) * kN;
    int equal = 0;
    for (int e = 0; e < kN && at + e < n; ++e) equal += to_f32(z[at + e]) == f;
    int before = equal;   // then of the lanes up to this one
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(before, d);
      if (lane >= d) before += o;
    }
    const int all = sum_of_waves(__shfl(before, 63));
    int to = listed + before - equal;
    for (int w = 0; w < wave; ++w) to += lds.count[w];
    for (int e = 0; e < kN && at + e < n; ++e)
      if (to_f32(z[at + e]) == f) {
        if (to < k) lds.keys[to] = logit_key(f, first + at + e);
        ++to;
      }
    listed = min(listed + all, k);
  }
  __syncthreads();
  return listed;
}

// Of n > k listed keys the k to 5/4 k greatest, by one wave that halves the range of keys (they are all different); the others
// leave the list.  Ranking all of them against each other takes n^2 steps (16,384 rows of 500 bf16 logits, 64 alternatives: 758 us).
__device__ __forceinline__ int narrowed(uint64_t* keys, int n, int k) {
  const int lane = threadIdx.x & 63;
  uint64_t lo = ~uint64_t{0}, hi = 0;
  for (int i = lane; i < n; i += 64) lo = min(lo, keys[i]), hi = max(hi, keys[i]);
  for (int d = 1; d < 64; d <<= 1) {
    lo = min(lo, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(lo), d)));
    hi = max(hi, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(hi), d)));
  }
  while (lo < hi) {   // k or more from lo on, fewer past hi
    const uint64_t mid = lo + (hi - lo) / 2 + 1;
    int c = 0;
#pragma unroll 4
    for (int i = 0; i < n; i += 64) c += __popcll(__ballot(keys[min(i + lane, n - 1)] >= mid && i + lane < n));
    if (c >= k) {
      lo = mid;
      if (c <= k + k / 4) break;
    } else {
      hi = mid - 1;
    }
  }
  int to = 0;
  for (int i = 0; i < n; i += 64) {   // the list closes up behind what has been read
    const uint64_t key = keys[min(i + lane, n - 1)];
    const bool keep = key >= lo && i + lane < n;
    const uint64_t kept = __ballot(keep);
    __builtin_amdgcn_wave_barrier();
    if (keep) keys[to + __popcll(kept & ((uint64_t{1} << lane) - 1))] = key;
    __builtin_amdgcn_wave_barrier();
    to += __popcll(kept);
  }
  return to;
}

static_assert(sizeof(RowLds) + kMaxSlots * 8 * 16 <= 65536, "LDS without asking for more");

template <typename T, int NV, bool TOP, bool ENT>
__global__ void __launch_bounds__(1024, 8) logprob_kernel(LogprobArgs a, int slices, int pieces_per_slice, Partial part, int slots) {
  constexpr int kN = Piece<T>::kN;
  extern __shared__ uint4 hot_pieces[];   // TOP: [slots][NV]
  __shared__ typename std::conditional<TOP, RowLds, float[4][16]>::type lds_;
  float(*red)[16];
  if constexpr (TOP)
    red = lds_.red;
  else
    red = lds_;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, threads = blockDim.x, waves = threads >> 6;
  const int64_t r = slices == 1 ? blockIdx.x : blockIdx.x / slices;
  const int slice = slices == 1 ? 0 : static_cast<int>(blockIdx.x - r * slices);
  const int first = slice * pieces_per_slice;
  const T* z = static_cast<const T*>(a.logits) + r * a.l_stride + static_cast<int64_t>(first) * kN;
  const int n = min(a.vocab - first * kN, pieces_per_slice * kN);   // logits of the slice
  RowTarget target{-1, 0.f};
  if (wave == 0 && slices == 1) target.id = row_target(a, r);
  Piece<T> p[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * threads + static_cast<int>(threadIdx.x)) * kN;
    if ((v + 1) * threads * kN <= n)   // all threads
      p[v].load(z + at);
    else if (at + kN <= n)
      p[v].load(z + at);
    else if (at < n)
      p[v].load_part(z + at, n - at, from_f32<T>(-INFINITY));
    else
      p[v].fill(-INFINITY);
  }
  if (target.id >= 0) target.z = to_f32(z[target.id]);
  RunningMax<T> running;
#pragma unroll
  for (int v = 0; v < NV; ++v) running.add(p[v]);
  const float mine = running.get();
  float m = wave_max(mine);
  if (lane == 0) red[0][wave] = m;
  if constexpr (TOP) {
    lds_.top[threadIdx.x] = mine;
    if (threadIdx.x == 0) lds_.n = lds_.n_hot = 0;
  }
  __syncthreads();
#pragma unroll 4
  for (int w = 0; w < waves; ++w) m = fmaxf(m, red[0][w]);
  const float ref = m == -INFINITY ? 0.f : m;
  float count = 0.f, rest = 0.f, u = 0.f;
  const bool holds = __ballot(mine == m) != 0;
  // t = z c - m c in one rounding, where m c is small enough for its own rounding (that all of them share) to be taken back after
  const float mc = ref * a.c;
  bool plain = !holds && fabsf(mc) < 256.f;
  if (plain) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      in_turn(p[v]);
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float t = fmaf(p[v].get(e), a.c, -mc), w = __builtin_amdgcn_exp2f(t);
        rest += w;
        if constexpr (ENT) u = fmaf(w, t, u);
      }
    }
    const float off = fmaf(ref, a.c, -mc), scale = __builtin_amdgcn_exp2f(-off);
    if constexpr (ENT) {
      u = scale * fmaf(-off, rest, u);
      plain = __ballot(u != u) == 0;   // 0 times -inf, if there is no NaN
    }
    rest *= scale;
  }
  if (!plain) {   // a wave that holds the maximum counts it apart
    count = rest = u = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      in_turn(p[v]);
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float x = p[v].get(e), t = (x - ref) * a.c, w = __builtin_amdgcn_exp2f(t);
        const bool top = x == m;
        count += top ? 1.f : 0.f;
        rest += top ? 0.f : w;
        if constexpr (ENT) u = fmaf(w, fmaxf(t, -1000.f), u);
      }
    }
  }
  if (holds) count = wave_add(count);
  rest = wave_add(rest);
  if constexpr (ENT) u = wave_add(u);
  if (lane == 0) red[1][wave] = count, red[2][wave] = rest, red[3][wave] = u;
  if constexpr (TOP) {
    if (wave == 0) {
      const uint32_t t = near_kth(lds_.top, threads, a.k, m);
      if (lane == 0) lds_.threshold = t;
    }
  }
  __syncthreads();
  if (wave == 0) {   // the slice's sums, by the first wave
    const bool there = lane < waves;
    const RowSums s{m, wave_add(there ? red[1][lane] : 0.f), wave_add(there ? red[2][lane] : 0.f),
                    ENT ? wave_add(there ? red[3][lane] : 0.f) : 0.f};
    if (slices > 1) {
      if (lane == 0) part.sums[r * slices + slice] = s;
    } else {
      const RowLogs g = row_logs(s);
      if (lane == 0) write_row(a, r, target, s, g);
      if constexpr (TOP) {
        if (lane == 0) lds_.log = m == INFINITY || s.rest != s.rest ? NAN : g.l;   // NaN: a row without alternatives
      }
    }
  }
  if constexpr (TOP) {
    // The threads with a logit at or above the threshold are few (k to 5/4 k of them, or somewhat more): they put their pieces
    // down in LDS, and all threads look through those.  The logits found are listed in any order.  (Read again from memory they
    // cost a line for every 16 bytes: 2,048 x 151,936 with 64 alternatives 156 us.)
    const uint32_t threshold = lds_.threshold;
    const float from = unordered(threshold);
    const uint64_t hot = __ballot(mine >= from);
    if (hot) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&lds_.n_hot, __popcll(hot));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(hot & ((uint64_t{1} << lane) - 1));
      if ((hot >> lane & 1) && at < slots) {
        lds_.hot[at] = static_cast<uint16_t>(threadIdx.x);
#pragma unroll
        for (int v = 0; v < NV; ++v) hot_pieces[at * NV + v] = p[v].r;
      }
    }
    __syncthreads();
    const int n_hot = lds_.n_hot;
    if (n_hot <= slots) {
      for (int i = threadIdx.x; i < n_hot * NV; i += threads) {
        Piece<T> q;
        q.r = hot_pieces[i];
        RunningMax<T> most;
        most.add(q);
        if (!(most.get() >= from)) continue;
        const int at = first * kN + ((i % NV) * threads + lds_.hot[i / NV]) * kN;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float x = q.get(e);
          if (x >= from) {
            const int to = atomicAdd(&lds_.n, 1);
            if (to < kCandidates) lds_.keys[to] = logit_key(x, at + e);
          }
        }
      }
      __syncthreads();
    }
    int found = n_hot <= slots ? lds_.n : kCandidates + 1;
    if (found > kCandidates) {
      found = crowded<T, NV>(a.k, z, n, first * kN, threshold, ordered(m), lds_);
    }
    if (found > 2 * a.k + 64) {
      if (wave == 0) {
        const int kept = narrowed(lds_.keys, found, a.k);
        if (lane == 0) lds_.n_kept = kept;   // not n, which other waves may be about to read: this branch hangs on it
      }
      __syncthreads();
      found = lds_.n_kept;
    }
    // each key's place among them: how many are greater, counted by four lanes
    const float log = lds_.log;
    const bool bad = log != log;
    const int quarter = lane & 3;
    for (int i = threadIdx.x / 4; i < max(found, a.k); i += threads / 4) {
      const uint64_t key = i < found ? lds_.keys[i] : 0;
      int place = 0;
      if (i < found) {
#pragma unroll 4
        for (int j = quarter; j < found; j += 4) place += lds_.keys[j] > key;
      }
      place += dpp_rows<0xb1, 0xf>(0, place);
      place += dpp_rows<0x4e, 0xf>(0, place);
      if (i >= found) place = i;
      if (place >= a.k || quarter) continue;
      if (slices > 1) {
        part.keys[(r * slices + slice) * a.k + place] = key;
      } else {
        a.top_ids[r * a.k + place] = key && !bad ? static_cast<int64_t>(~static_cast<uint32_t>(key)) : -1;
        a.top_logprobs[r * a.k + place] = bad ? NAN : key ? below_max(unordered(static_cast<uint32_t>(key >> 32)), m, a.inv_tau) - log : -INFINITY;
      }
    }
  }
}

// -- a row's slices joined ----------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 256, kJoinKeys = 2048;

// Writes the row's alternatives from its slices' lists, each falling: a key's place is the number of greater ones in all of
// them, found by halving, four lists at a time so that their reads overlap.  Every list's first ceil(k / slices) keys together
// are k or more, so those below the least of them have no place (of 5 lists of 64 keys some 90 remain; the search reads LDS at
// random, which bounds it: 2,048 rows 16.9 us with all).  Returns how many this thread wrote.
__device__ __forceinline__ int place_keys(const LogprobArgs& a, int64_t r, int slices, const uint64_t* keys, float m, float log,
                                          bool bad) {
  int there = 0;
  const int half = 1 << (31 - __builtin_clz(a.k));
  const int sure = (a.k + slices - 1) / slices - 1;
  uint64_t least = keys[sure];
#pragma unroll 4
  for (int q = 1; q < slices; ++q) least = min(least, keys[q * a.k + sure]);
  least = max(least, uint64_t{1});
  for (int i = threadIdx.x; i < slices * a.k; i += blockDim.x) {   // the lists' first keys before their second ones
    const int j = i / slices;
    const uint64_t key = keys[(i - j * slices) * a.k + j];
    if (key < least) continue;
    int place = 0;
    for (int q = 0; q < slices && place < a.k; q += 4) {
      int n[4] = {0, 0, 0, 0};
      for (int step = half; step > 0; step >>= 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = n[j] + step;
          if (keys[min(q + j, slices - 1) * a.k + min(at, a.k) - 1] > key && at <= a.k) n[j] = at;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) place += q + j < slices ? n[j] : 0;
    }
    if (place >= a.k) continue;
    ++there;
    a.top_ids[r * a.k + place] = bad ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(key));
    a.top_logprobs[r * a.k + place] = bad ? NAN : below_max(unordered(static_cast<uint32_t>(key >> 32)), m, a.inv_tau) - log;
  }
  return there;
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) logprob_join_kernel(LogprobArgs a, int slices, Partial part) {
  __shared__ uint64_t held[kJoinKeys];
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63;
  RowTarget target{-1, 0.f};
  if (threadIdx.x == 0) target.id = row_target(a, r);
  const uint64_t* keys = part.keys + r * slices * a.k;
  const bool few = slices * a.k <= kJoinKeys;
  if (few)
    for (int i = threadIdx.x; i < slices * a.k; i += blockDim.x) held[i] = keys[i];
  // a lane a slice: at most 64
  const RowSums q = lane < slices ? part.sums[r * slices + lane] : RowSums{-INFINITY, 0.f, 0.f, 0.f};
  if (target.id >= 0) target.z = to_f32(static_cast<const T*>(a.logits)[r * a.l_stride + target.id]);
  const bool bad = __ballot(q.rest != q.rest || q.m == INFINITY) != 0;
  RowSums s;
  s.m = wave_max(q.m);
  const float ref = s.m == -INFINITY ? 0.f : s.m, t = fmaxf((q.m - ref) * a.c, -1000.f), w = __builtin_amdgcn_exp2f(t);
  const bool top = q.m == s.m;
  s.count = wave_add(top ? q.count : 0.f);
  s.rest = wave_add(top ? q.rest : w * (q.count + q.rest));
  s.u = wave_add(top ? q.u : w * fmaf(t, q.count + q.rest, q.u));
  if (bad) s.rest = NAN;
  const RowLogs g = row_logs(s);
  if (threadIdx.x == 0) write_row(a, r, target, s, g);
  if (a.k == 0) return;
  __syncthreads();
  const int there = few ? place_keys(a, r, slices, held, s.m, g.l, bad) : place_keys(a, r, slices, keys, s.m, g.l, bad);
  const int mine = wave_add(there);
  __shared__ int red[kJoinThreads / 64];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mine;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x) / 64; ++w) all += red[w];
  for (int i = all + threadIdx.x; i < a.k; i += blockDim.x) {
    a.top_ids[r * a.k + i] = -1;
    a.top_logprobs[r * a.k + i] = bad ? NAN : -INFINITY;
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

// -- the gradient -------------------------------------------------------------------------------------------------------
// One workgroup per segment of a row, kGradPieces pieces a thread: a logit in, its gradient out, bound by memory (16,384 x
// 32,768 bf16 343 us in the median of a profiled step, 6.3 TB/s read and written; rows in reverse, to meet what the forward
// left in the caches, the same).
constexpr int kGradThreads = 256, kGradPieces = 4;

template <typename T, bool THROUGH>
__global__ void __launch_bounds__(kGradThreads) logprob_grad_kernel(LogprobGradArgs a, int segments, int64_t groups) {
  constexpr int kN = Piece<T>::kN;
  const int threads = blockDim.x;
  for (int64_t b = blockIdx.x; b < groups; b += gridDim.x) {
    const int64_t r = segments == 1 ? b : b / segments;
    const int first = static_cast<int>(b - r * segments) * kGradPieces * threads * kN;
    const T* z = static_cast<const T*>(a.logits) + r * a.l_stride;
    T* d = static_cast<T*>(a.dz) + r * a.d_stride;
    const int64_t y64 = a.targets && a.dlp ? a.targets[r] : -1;
    const bool given = y64 >= 0 && y64 < a.vocab && y64 != a.ignore;
    const float ga = given ? a.dlp[r * a.dlp_stride] * a.inv_tau : 0.f;
    const float gb = a.dh ? a.dh[r * a.dh_stride] * a.inv_tau : 0.f;
    const bool live = !(ga == 0.f && gb == 0.f);
    const float4 s = a.stats[r];
    const float entropy = a.dh ? s.z : 0.f;
    const int y = given && s.y != INFINITY ? static_cast<int>(y64) : -1;
    Piece<T> p[kGradPieces];
    if (live) {
#pragma unroll
      for (int v = 0; v < kGradPieces; ++v) {
        const int at = first + (v * threads + static_cast<int>(threadIdx.x)) * kN;
        if (at + kN <= a.vocab)
          p[v].load(z + at);
        else if (at < a.vocab)
          p[v].load_part(z + at, a.vocab - at, from_f32<T>(-INFINITY));
      }
    }
#pragma unroll
    for (int v = 0; v < kGradPieces; ++v) {
      const int at = first + (v * threads + static_cast<int>(threadIdx.x)) * kN;
      if (at >= a.vocab) break;
      float o[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float t = (p[v].get(e) - s.x) * a.c - s.y, w = __builtin_amdgcn_exp2f(t);
        o[e] = live ? -w * fmaf(gb, fmaf(fmaxf(t, -1000.f), kLn2, entropy), ga) : 0.f;
      }
      if (static_cast<unsigned>(y - at) < static_cast<unsigned>(kN)) {
#pragma unroll
        for (int e = 0; e < kN; ++e) o[e] += y - at == e ? ga : 0.f;
      }
      p[v].set(o);
      if (at + kN > a.vocab)
        p[v].store_part(d + at, a.vocab - at);
      else if constexpr (THROUGH)
        p[v].store_through(d + at);
      else
        p[v].store(d + at);
    }
  }
}

inline int check_logprob(const sdm_rt_logprob* d, const void* logits, int64_t l_stride, sdm_rt_dtype dtype) {
  int rc;
  if (!d) return set_err(SDM_RT_EINVAL, "dims is NULL");
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (d->rows < 0 || d->vocab < 1 || d->top_k < 0) return set_err(SDM_RT_EINVAL, "rows and top_k must be >= 0, vocab >= 1");
  if (d->rows > (1 << 21)) return set_err(SDM_RT_EUNSUPPORTED, "rows must be at most 2^21");
  if (d->vocab > (1 << 21)) return set_err(SDM_RT_EUNSUPPORTED, "vocab must be at most 2^21");
  if (d->top_k > kMaxAlternatives) return set_err(SDM_RT_EUNSUPPORTED, "top_k = %d must be at most %d", d->top_k, kMaxAlternatives);
  if (!(d->temperature >= 1e-18f) || !(d->temperature <= 1e18f))
    return set_err(SDM_RT_EINVAL, "temperature must be positive and finite, from 1e-18 to 1e18");
  if (d->rows > 0 && (!logits || bad_read_stride(l_stride, d->vocab)))
    return set_err(SDM_RT_EINVAL, "logits must not be NULL, their row stride 0 or >= vocab");
  return SDM_RT_OK;
}

// How a row is cut: at most 32,768 logits to a slice, 8 pieces a thread (2 in rows that a few waves hold).
struct RowShape {
  int slices, pieces, nv, threads;   // pieces: of a slice
};
inline RowShape row_shape(int vocab, int k, sdm_rt_dtype dtype) {
  const int kN = dtype == SDM_RT_BF16 ? 8 : 4, most = 32768 / kN;
  const int pieces = (vocab + kN - 1) / kN;
  RowShape s;
  static_assert(((1 << 21) + 32767) / 32768 <= 64, "a lane a slice");
  s.slices = (pieces + most - 1) / most;
  s.pieces = (pieces + s.slices - 1) / s.slices;
  s.nv = s.pieces <= 512 ? 2 : 8;
  s.threads = std::max(64, (s.pieces + 64 * s.nv - 1) / (64 * s.nv) * 64);
  // twice as many threads as alternatives, where the slice has the pieces: their maxima then tell the alternatives apart
  s.threads = std::max(s.threads, std::min((s.pieces + 63) / 64, (2 * k + 63) / 64) * 64);
  return s;
}
inline size_t logprob_bytes(int64_t rows, int k, int slices) {
  return slices == 1 ? 0 : static_cast<size_t>(rows) * slices * (static_cast<size_t>(k) * sizeof(uint64_t) + sizeof(RowSums));
}

template <typename T>
void launch_logprob(const LogprobArgs& a, const RowShape& s, const Partial& part, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.rows * s.slices)), threads(s.threads);
  const int slots = std::min(s.threads, a.k + a.k / 2 + 8);   // kMaxSlots at most
  auto launch = [&](auto nv, auto top, auto ent) {
    hipLaunchKernelGGL((logprob_kernel<T, decltype(nv)::value, decltype(top)::value, decltype(ent)::value>), grid, threads,
                       a.k ? static_cast<size_t>(slots) * decltype(nv)::value * 16 : 0, st, a, s.slices, s.pieces, part, slots);
  };
  auto with_nv = [&](auto top, auto ent) {
    if (s.nv == 2)
      launch(std::integral_constant<int, 2>{}, top, ent);
    else
      launch(std::integral_constant<int, 8>{}, top, ent);
  };
  auto with_top = [&](auto ent) {
    if (a.k)
      with_nv(std::true_type{}, ent);
    else
      with_nv(std::false_type{}, ent);
  };
  if (a.entropy)
    with_top(std::true_type{});
  else
    with_top(std::false_type{});
  if (s.slices > 1)
    hipLaunchKernelGGL(logprob_join_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(a.k ? kJoinThreads : 64), 0, st, a,
                       s.slices, part);
}

template <typename T>
void launch_logprob_grad(const LogprobGradArgs& a, hipStream_t st) {
  const int pieces = (a.vocab + Piece<T>::kN - 1) / Piece<T>::kN;
  const int threads = std::min(kGradThreads, (pieces + 64 * kGradPieces - 1) / (64 * kGradPieces) * 64);
  const int segments = (pieces + threads * kGradPieces - 1) / (threads * kGradPieces);
  const int64_t groups = a.rows * segments;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(groups, 1 << 22)));
  // a gradient that no cache keeps for its reader leaves the caches to the logits, which the forward has left there (1,537 x
  // 32,003 float32, forward and gradient: 107 us, 124 without; 16,384 x 32,768 bf16, 1 GB, the same either way)
  if (a.rows * a.vocab * static_cast<int64_t>(sizeof(T)) > kStreamBytes)
    hipLaunchKernelGGL((logprob_grad_kernel<T, true>), grid, dim3(threads), 0, st, a, segments, groups);
  else
    hipLaunchKernelGGL((logprob_grad_kernel<T, false>), grid, dim3(threads), 0, st, a, segments, groups);
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

size_t sdm_rt_token_logprobs_workspace_bytes(const sdm_rt_logprob* dims, sdm_rt_dtype dtype) {
  if (!dims || dims->rows < 0 || dims->vocab < 1 || dims->top_k < 0) return 0;
  return logprob_bytes(dims->rows, dims->top_k, row_shape(dims->vocab, dims->top_k, dtype).slices);
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
  const RowShape shape = row_shape(a.vocab, a.k, dtype);
  if (a.rows * shape.slices >= int64_t{1} << 22) return set_err(SDM_RT_EUNSUPPORTED, "too many rows of so large a vocabulary");
  Partial part{};
  if (shape.slices > 1) {
    if (reinterpret_cast<uintptr_t>(workspace) % 8) return set_err(SDM_RT_EINVAL, "workspace must be 8-byte aligned");
    part.keys = static_cast<uint64_t*>(workspace);
    part.sums = reinterpret_cast<RowSums*>(part.keys + a.rows * shape.slices * a.k);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SDM_RT_BF16)
    launch_logprob<bf16_t>(a, shape, part, st);
  else
    launch_logprob<float>(a, shape, part, st);
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
  if (dtype == SDM_RT_BF16)
    launch_logprob_grad<bf16_t>(a, st);
  else
    launch_logprob_grad<float>(a, st);
  return check_launch("token_logprobs_grad");
}

}  // extern "C"
