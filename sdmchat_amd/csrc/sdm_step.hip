// sdm_step.hip -- the end of a training step over a whole model's tensors: the norm of the gradients (sdm_rt_grad_norm), the
// AdamW step with its moments in 32 or in 8 bits (sdm_rt_adamw), and the values of 8-bit moments (sdm_rt_read_moments).
//
// A call takes a list of tensors.  Their addresses and sizes ride in the kernel's arguments (under 4 KB of them), some 100 to a
// launch: nothing is copied to the device, a captured launch holds all it needs, and no list has to outlive the call.  A tensor
// is cut into chunks, one a workgroup.
#include "sdm_vocab.h"

namespace sdmrt {

constexpr int kStepThreads = 256;
constexpr int kBlock = 128;                       // values of a block of 8-bit moments
constexpr int kBlockBytes = 2 * kBlock + 8;       // codes of m, codes of v, two exponents, 6 unused

// -- lists of tensors in kernel arguments -----------------------------------------------------------------------------
template <int P, int N, bool BLOCKS = false>   // addresses of a tensor, tensors at most
struct StepTable {
  static constexpr int kAddresses = P, kTensors = N, kSearched = (N + 64) / 64 * 64;
  static constexpr bool kBlocks = BLOCKS;
  char* at[P][N];
  uint32_t chunk[kSearched];         // each tensor's first chunk in the launch, then the number of all, then ~0
  uint32_t block[BLOCKS ? N : 1];    // blocks of 8-bit moments of the tensors before it in the call
  uint16_t tail[N];                  // values of its last chunk, less one; bit 15: bfloat16
};

// A workgroup's chunk: its tensor, where it begins there and how many values it has.  Every wave finds its tensor at once: a lane
// looks at each (a search by halves waits for one load after the other).
struct StepChunk {
  int tensor;
  bool bf16;
  int n;
  int64_t begin;
};
template <int CHUNK, typename TABLE>
__device__ __forceinline__ StepChunk find_chunk(const TABLE& table, uint32_t index) {
  int t = -1;
#pragma unroll
  for (int i = 0; i < TABLE::kSearched; i += 64) t += __popcll(__ballot(table.chunk[i + (threadIdx.x & 63)] <= index));
  const uint32_t first = table.chunk[t];
  const int tail = table.tail[t];
  return StepChunk{t, (tail & 0x8000) != 0, index + 1 == table.chunk[t + 1] ? (tail & 0x7fff) + 1 : CHUNK,
                   static_cast<int64_t>(index - first) * CHUNK};
}

// 8, 16 or 32 bytes at any element's address.  THROUGH: what a call streams through leaves the caches to others (a step of 110 M
// float32 values, the norm of their gradients with it, 620 us, 737 without); a model that the last-level cache holds stays there.
template <bool THROUGH, int BYTES>
__device__ __forceinline__ void load_bytes(const void* p, void* v) {
  if constexpr (!THROUGH) {
    __builtin_memcpy(v, p, BYTES);
  } else if constexpr (BYTES == 8) {
    const words2 w = __builtin_nontemporal_load(static_cast<const words2*>(p));
    __builtin_memcpy(v, &w, 8);
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const words4 w = __builtin_nontemporal_load(static_cast<const words4*>(p) + i);
      __builtin_memcpy(static_cast<char*>(v) + 16 * i, &w, 16);
    }
  }
}
template <bool THROUGH, int BYTES>
__device__ __forceinline__ void store_bytes(void* p, const void* v) {
  if constexpr (!THROUGH) {
    __builtin_memcpy(p, v, BYTES);
  } else if constexpr (BYTES == 8) {
    words2 w;
    __builtin_memcpy(&w, v, 8);
    __builtin_nontemporal_store(w, static_cast<words2*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      words4 w;
      __builtin_memcpy(&w, static_cast<const char*>(v) + 16 * i, 16);
      __builtin_nontemporal_store(w, static_cast<words4*>(p) + i);
    }
  }
}

// N values of T at p, of which the first n are there (the others 0)
template <bool THROUGH, typename T, int N>
__device__ __forceinline__ void load_values(const T* p, int64_t n, float (&v)[N]) {
  if (n >= N) {
    T x[N];
    load_bytes<THROUGH, sizeof(x)>(p, x);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = to_f32(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < n ? to_f32(p[e]) : 0.f;
  }
}
template <bool THROUGH, typename T, int N>
__device__ __forceinline__ void store_values(T* p, int64_t n, const float (&v)[N]) {
  if (n >= N) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w[N / 2];
#pragma unroll
      for (int e = 0; e < N / 2; ++e) w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      store_bytes<THROUGH, sizeof(w)>(p, w);
    } else {
      store_bytes<THROUGH, sizeof(v)>(p, v);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) p[e] = from_f32<T>(v[e]);
  }
}

// -- the gradients' norm ----------------------------------------------------------------------------------------------
using NormTable = StepTable<1, 191>;

__device__ __forceinline__ double wave_add(double v) {
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// Four pieces of a thread under way at once (220 MB of bfloat16 41 us, 5.3 TB/s): one at a time left it waiting (72), eight left
// too few waves (50).
template <typename T>
__device__ __forceinline__ double sum_squares(const T* g, int n) {
  constexpr int kN = 16 / static_cast<int>(sizeof(T)), kAtOnce = 4;
  double s = 0.0;
  for (int i = threadIdx.x * kN; i < n; i += kAtOnce * kStepThreads * kN) {
    float v[kAtOnce][kN];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      const int at = i + q * kStepThreads * kN;
      if (at < n)
        load_values<false>(g + at, n - at, v[q]);
      else
        for (int e = 0; e < kN; ++e) v[q][e] = 0.f;
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
      for (int e = 0; e < kN; ++e) s = fma(static_cast<double>(v[q][e]), static_cast<double>(v[q][e]), s);
  }
  return s;
}

// Each chunk's sum of squares in float64: no gradient is too large or too small for its square, and the order is fixed.
template <int CHUNK>
__global__ void __launch_bounds__(kStepThreads) norm_kernel(NormTable table, double* __restrict__ partial) {
  __shared__ double red[kStepThreads / 64];
  const StepChunk c = find_chunk<CHUNK>(table, blockIdx.x);
  const char* g = table.at[0][c.tensor];
  double s = c.bf16 ? sum_squares(reinterpret_cast<const bf16_t*>(g) + c.begin, c.n)
                    : sum_squares(reinterpret_cast<const float*>(g) + c.begin, c.n);
  s = wave_add(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kStepThreads / 64; ++w) s += red[w];
    partial[blockIdx.x] = s;
  }
}

__global__ void __launch_bounds__(1024) norm_join_kernel(const double* __restrict__ partial, int n, float* __restrict__ norm) {
  __shared__ double red[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = wave_add(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += red[w];
    *norm = static_cast<float>(sqrt(s));
  }
}

// -- moments in 8 bits ------------------------------------------------------------------------------------------------
// The hash that decides the rounding of a value at position i in step t: two multiplications by odd numbers (from the golden
// ratio and the square root of 3) with shifts between them.  Its upper half is for m, its lower half for v.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 2654435761u;
  x = (x ^ (x >> 15)) * 3144134277u;
  return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t step_key(uint32_t seed, int64_t t) {
  return mix(seed + static_cast<uint32_t>(t) * 2654435761u);
}

// the exponent of a block whose largest magnitude has these bits: 255 where it is above 1.875 2^126, whose codes would be infinite,
// or not finite (a NaN may have its sign set, and is then the greatest of the bits); 0 up to 0.875 2^-126
__device__ __forceinline__ uint32_t block_exponent(uint32_t bits) {
  const uint32_t e = ((bits & 0x7fffffffu) + 0xfffffu) >> 23;
  return e >= 254 ? 255 : e;
}
// 2^(E - 127), 0 for E = 0, NaN for E = 255
__device__ __forceinline__ float block_scale(uint32_t e) { return __uint_as_float(e == 255 ? 0x7fc00000u : e << 23); }

// Codes.  The bits of a code of v, put where float32 has its exponent and mantissa, are the value times a power of two, for e =
// 0 too (float32's values below its least normal one); those of m are a float16 so.  Encoding is the way back: the value
// times a power of two, random bits added below the code's last place, the bits above taken.  None of it asks for a value's
// size.
__device__ __forceinline__ float decode_v(uint32_t codes, int q, int shift) {   // shift: v_shift's
  const uint32_t bits = (q == 3 ? codes >> 4 : codes << (20 - 8 * q)) & 0x0ff00000u;
  return __builtin_amdgcn_ldexpf(__uint_as_float(bits), shift);
}
__device__ __forceinline__ int v_shift(uint32_t e) { return e == 0 ? -400 : static_cast<int>(e) - 31; }
typedef _Float16 halves __attribute__((ext_vector_type(2)));
typedef short shorts __attribute__((ext_vector_type(2)));
__device__ __forceinline__ halves decode_m(uint32_t codes, int pair) {   // without the scale of its block
  const uint32_t apart = __builtin_amdgcn_perm(0u, codes, pair ? 0x030c020cu : 0x010c000cu);   // each in the upper byte of a half
  const shorts down = __builtin_bit_cast(shorts, apart) >> 1;
  return __builtin_bit_cast(halves, __builtin_bit_cast(uint32_t, down) & 0xbfffbfffu);
}
// the code of a value in the upper byte of a word (shift: 15 - E for m, 31 - E for v, and far below for E = 0: code 0)
__device__ __forceinline__ uint32_t encode_m(float m, int shift, uint32_t random16) {
  const uint32_t t = __float_as_uint(__builtin_amdgcn_ldexpf(m, shift)) + (random16 << 4);
  return (t << 4 & 0x7fffffffu) | (t & 0x80000000u);
}
__device__ __forceinline__ uint32_t encode_v(float v, int shift, uint32_t random16) {
  const uint32_t t = __float_as_uint(__builtin_amdgcn_ldexpf(v, shift)) + (random16 << 4);
  return max(t, v > 0.f ? 0x00100000u : 0u) << 4;   // a v above 0 has no code 0
}
// the upper bytes of four words
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x07030c0cu), __builtin_amdgcn_perm(b, a, 0x0c0c0703u), 0x07060100u);
}

// the maximum over a row of 16 lanes, in each of them
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(dpp_rows<0xb1, 0xf>(0, static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(dpp_rows<0x4e, 0xf>(0, static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(dpp_rows<0x141, 0xf>(0, static_cast<int>(v))));
  return max(v, static_cast<uint32_t>(dpp_rows<0x140, 0xf>(0, static_cast<int>(v))));
}

// -- the step ---------------------------------------------------------------------------------------------------------
struct StepArgs {
  float b1, c1, b2, c2, eps;      // c: 1 - b
  float decay, size, r2;          // 1 - lr weight_decay, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  float max_norm;
  uint32_t key, seed;
  const float* norm;
  const int64_t* t_device;
  const float* lr_device;
  double lr, weight_decay, log_b1, log_b2;
};

__global__ void count_step_kernel(int64_t* t) { *t += 1; }

// What of the arguments depends on the device's step and learning rate.
__device__ __forceinline__ void read_step(StepArgs& a) {
  const int64_t t = *a.t_device;
  const double lr = a.lr_device ? static_cast<double>(*a.lr_device) : a.lr;
  a.decay = static_cast<float>(1.0 - lr * a.weight_decay);
  a.size = static_cast<float>(lr / -expm1(static_cast<double>(t) * a.log_b1));
  a.r2 = static_cast<float>(1.0 / sqrt(-expm1(static_cast<double>(t) * a.log_b2)));
  a.key = step_key(a.seed, t);
}

// One value's new moments (from the old ones times beta1 and beta2) and parameter.  Every product and sum of the moments is
// rounded by itself, as the formula is written: their codes in 8 bits then do not hang on what a compiler fuses.  The instruction
// for square roots takes a v below float32's least normal value, 2^-126, for 0: 2^-63 in the root, less than a rounding of the
// denominator unless eps is TINY.  Then the compiler's own root and quotient are taken, in kernels of their own (both in one
// kernel took a third of the 8-bit step's waves: 110 M values 368 us against 350).
template <bool TINY>
__device__ __forceinline__ void step_value(const StepArgs& a, float clip, float g, float& p, float& m, float& v) {
  {
#pragma clang fp contract(off)
    g = g * clip;
    m = m + g * a.c1;
    v = v + g * g * a.c2;
  }
  if constexpr (TINY) {
    p = fmaf(m / fmaf(sqrtf(v), a.r2, a.eps), -a.size, p * a.decay);
  } else {
    const float d = fmaf(__builtin_amdgcn_sqrtf(v), a.r2, a.eps);
    p = fmaf(m * -a.size, __builtin_amdgcn_rcpf(d), p * a.decay);
  }
}

using StepTable32 = StepTable<4, 96>;
using StepTable8 = StepTable<3, 108, true>;

// All of a thread's pieces of a chunk are loaded before the first is computed on: 16 bytes of parameters and gradients each.
template <int CHUNK, bool THROUGH, bool TINY, typename T>
__device__ __forceinline__ void step_chunk32(const StepArgs& a, float clip, T* p, const T* g, float* m, float* v, int n) {
  constexpr int kN = 4, kPieces = CHUNK / (kStepThreads * kN);
  float pv[kPieces][kN], gv[kPieces][kN], mv[kPieces][kN], vv[kPieces][kN];
#pragma unroll
  for (int q = 0; q < kPieces; ++q) {
    const int i = (q * kStepThreads + threadIdx.x) * kN;
    if (i >= n) break;
    load_values<THROUGH>(p + i, n - i, pv[q]);
    load_values<THROUGH>(g + i, n - i, gv[q]);
    load_values<THROUGH>(m + i, n - i, mv[q]);
    load_values<THROUGH>(v + i, n - i, vv[q]);
  }
#pragma unroll
  for (int q = 0; q < kPieces; ++q) {
    const int i = (q * kStepThreads + threadIdx.x) * kN;
    if (i >= n) break;
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      mv[q][e] *= a.b1;
      vv[q][e] *= a.b2;
      step_value<TINY>(a, clip, gv[q][e], pv[q][e], mv[q][e], vv[q][e]);
    }
    store_values<THROUGH>(p + i, n - i, pv[q]);
    store_values<THROUGH>(m + i, n - i, mv[q]);
    store_values<THROUGH>(v + i, n - i, vv[q]);
  }
}

// Sixteen lanes hold a block, 8 values each: its maxima come from four DPP steps.  Past a tensor's end p, g and the codes are
// 0 and stay so.  The codes do not stream past the caches: their lines are shared by neighbouring lanes' pieces (14 M values
// 43.5 us, 48.9 if they do).  Bound by memory and instructions alike: 110 M bfloat16 values 210 us call after call, 5.3 TB/s,
// 52 instructions a value (a profiled step's, behind the norm and before read_moments, 237 in the median).
template <bool THROUGH, bool TINY, typename T>
__device__ __forceinline__ void step_chunk8(const StepArgs& a, float clip, T* p, const T* g, char* chunk, uint32_t position, int n) {
  const int whole = (n + kBlock - 1) / kBlock * kBlock;
  for (int i = threadIdx.x * 8; i < whole; i += kStepThreads * 8) {
    char* state = chunk + i / kBlock * kBlockBytes;
    const int at = i % kBlock;
    uint32_t cm[2], cv[2];
    load_bytes<false, 8>(state + at, cm);
    load_bytes<false, 8>(state + kBlock + at, cv);
    const uint32_t e = *reinterpret_cast<const uint16_t*>(state + 2 * kBlock);
    float pv[8], gv[8], mv[8], vv[8];
    load_values<THROUGH>(p + i, n - i, pv);
    load_values<THROUGH>(g + i, n - i, gv);
    const float b1 = a.b1 * block_scale(e & 255), b2 = e >> 8 == 255 ? NAN : a.b2;
    const int shift = v_shift(e >> 8);
    float am = 0.f;
    uint32_t av = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const halves h = decode_m(cm[q / 4], q / 2 & 1);
      mv[q] = fmaf(static_cast<float>(q & 1 ? h.y : h.x), b1, 0.f);
      vv[q] = decode_v(cv[q / 4], q & 3, shift) * b2;
      step_value<TINY>(a, clip, gv[q], pv[q], mv[q], vv[q]);
      am = fmaxf(am, fabsf(mv[q]));   // passes over NaN: v has it then, or infinity
      av = max(av, __float_as_uint(vv[q]));
    }
    store_values<THROUGH>(p + i, n - i, pv);
    uint32_t em = block_exponent(row16_max(__float_as_uint(am)));
    const uint32_t ev = block_exponent(row16_max(av));
    em = ev == 255 ? 255 : em;
    const int sm = em == 0 ? -400 : 15 - static_cast<int>(em), sv = ev == 0 ? -400 : 31 - static_cast<int>(ev);
    const uint32_t counter = position + static_cast<uint32_t>(i) + a.key;
    uint32_t nm[8], nv[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const uint32_t u = mix(counter + q);
      nm[q] = encode_m(mv[q], sm, u >> 16);
      nv[q] = encode_v(vv[q], sv, u & 0xffff);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      cm[w] = upper_bytes(nm[4 * w], nm[4 * w + 1], nm[4 * w + 2], nm[4 * w + 3]);
      cv[w] = upper_bytes(nv[4 * w], nv[4 * w + 1], nv[4 * w + 2], nv[4 * w + 3]);
    }
    store_bytes<false, 8>(state + at, cm);
    store_bytes<false, 8>(state + kBlock + at, cv);
    if (at == 0) *reinterpret_cast<uint16_t*>(state + 2 * kBlock) = static_cast<uint16_t>(em | ev << 8);
  }
}

// a norm that is NaN makes the gradients NaN, as a product with it would
__device__ __forceinline__ float clip_factor(const StepArgs& a) {
  if (!a.norm) return 1.f;
  const float c = a.max_norm / (*a.norm + 1e-6f);
  return c > 1.f ? 1.f : c;
}

template <int CHUNK, bool DEVICE, bool THROUGH, bool TINY>
__global__ void __launch_bounds__(kStepThreads) adamw32_kernel(StepTable32 table, StepArgs a) {
  if constexpr (DEVICE) read_step(a);
  const float clip = clip_factor(a);
  const StepChunk c = find_chunk<CHUNK>(table, blockIdx.x);
  char* p = table.at[0][c.tensor];
  const char* g = table.at[1][c.tensor];
  float* m = reinterpret_cast<float*>(table.at[2][c.tensor]) + c.begin;
  float* v = reinterpret_cast<float*>(table.at[3][c.tensor]) + c.begin;
  if (c.bf16)
    step_chunk32<CHUNK, THROUGH, TINY>(a, clip, reinterpret_cast<bf16_t*>(p) + c.begin, reinterpret_cast<const bf16_t*>(g) + c.begin, m,
                                 v, c.n);
  else
    step_chunk32<CHUNK, THROUGH, TINY>(a, clip, reinterpret_cast<float*>(p) + c.begin, reinterpret_cast<const float*>(g) + c.begin, m, v,
                                 c.n);
}

template <int CHUNK, bool DEVICE, bool THROUGH, bool TINY>
__global__ void __launch_bounds__(kStepThreads) adamw8_kernel(StepTable8 table, StepArgs a) {
  if constexpr (DEVICE) read_step(a);
  const float clip = clip_factor(a);
  const StepChunk c = find_chunk<CHUNK>(table, blockIdx.x);
  char* p = table.at[0][c.tensor];
  const char* g = table.at[1][c.tensor];
  char* state = table.at[2][c.tensor] + c.begin / kBlock * kBlockBytes;
  const uint32_t position = table.block[c.tensor] * static_cast<uint32_t>(kBlock) + static_cast<uint32_t>(c.begin);
  if (c.bf16)
    step_chunk8<THROUGH, TINY>(a, clip, reinterpret_cast<bf16_t*>(p) + c.begin, reinterpret_cast<const bf16_t*>(g) + c.begin, state,
                         position, c.n);
  else
    step_chunk8<THROUGH, TINY>(a, clip, reinterpret_cast<float*>(p) + c.begin, reinterpret_cast<const float*>(g) + c.begin, state,
                         position, c.n);
}

// -- the values of 8-bit moments --------------------------------------------------------------------------------------
using ReadTable = StepTable<3, 120>;
constexpr int kReadChunk = 4096;

template <bool THROUGH, typename T>
__device__ __forceinline__ void read_chunk(T* m, T* v, const char* chunk, int n) {
  for (int i = threadIdx.x * 8; i < n; i += kStepThreads * 8) {
    const char* state = chunk + i / kBlock * kBlockBytes;
    uint32_t cm[2], cv[2];
    load_bytes<false, 8>(state + i % kBlock, cm);
    load_bytes<false, 8>(state + kBlock + i % kBlock, cv);
    const uint32_t e = *reinterpret_cast<const uint16_t*>(state + 2 * kBlock);
    const float scale = block_scale(e & 255), nan = e >> 8 == 255 ? NAN : 1.f;
    const int shift = v_shift(e >> 8);
    float mv[8], vv[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const halves h = decode_m(cm[q / 4], q / 2 & 1);
      mv[q] = fmaf(static_cast<float>(q & 1 ? h.y : h.x), scale, 0.f);
      vv[q] = decode_v(cv[q / 4], q & 3, shift) * nan;
    }
    store_values<THROUGH>(m + i, n - i, mv);
    store_values<THROUGH>(v + i, n - i, vv);
  }
}

template <bool THROUGH>
__global__ void __launch_bounds__(kStepThreads) read_moments_kernel(ReadTable table) {
  const StepChunk c = find_chunk<kReadChunk>(table, blockIdx.x);
  const char* state = table.at[0][c.tensor] + c.begin / kBlock * kBlockBytes;
  char *m = table.at[1][c.tensor], *v = table.at[2][c.tensor];
  if (c.bf16)
    read_chunk<THROUGH>(reinterpret_cast<bf16_t*>(m) + c.begin, reinterpret_cast<bf16_t*>(v) + c.begin, state, c.n);
  else
    read_chunk<THROUGH>(reinterpret_cast<float*>(m) + c.begin, reinterpret_cast<float*>(v) + c.begin, state, c.n);
}

// -- host -------------------------------------------------------------------------------------------------------------
static_assert(sizeof(StepTable32) + sizeof(StepArgs) + 16 <= 4096 && sizeof(StepTable8) + sizeof(StepArgs) + 16 <= 4096 &&
                  sizeof(NormTable) + 32 <= 4096 && sizeof(ReadTable) + 16 <= 4096,
              "kernel arguments");

inline int64_t chunks_of(int64_t n, int chunk) { return (n + chunk - 1) / chunk; }

// Every check that needs no device; values: the sum of the n.  Chunks are at least 1,024 values: not much over 2^23 in a launch.
inline int check_tensors(const sdm_rt_tensor* t, int32_t count, int64_t* values) {
  if (count < 0 || (count > 0 && !t)) return set_err(SDM_RT_EINVAL, "count must be >= 0, tensors not NULL");
  *values = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n < 0) return set_err(SDM_RT_EINVAL, "tensor %d: n must be >= 0", i);
    if (t[i].dtype != SDM_RT_F32 && t[i].dtype != SDM_RT_BF16)
      return set_err(SDM_RT_EINVAL, "tensor %d: unknown dtype %lld", i, (long long)t[i].dtype);
    if (t[i].n > (int64_t{1} << 33)) return set_err(SDM_RT_EUNSUPPORTED, "tensor %d: n must be at most 2^33", i);   // before the sum
    *values += t[i].n;
    if (*values > (int64_t{1} << 33)) return set_err(SDM_RT_EUNSUPPORTED, "more than 2^33 values in one call");
  }
  return SDM_RT_OK;
}

// launch(table, chunks of the launch, chunks before it) over the list, as many tensors at a time as a launch takes; take(tensor,
// addresses) says which addresses the kernel needs
template <typename TABLE, typename TAKE, typename LAUNCH>
void for_tables(const sdm_rt_tensor* t, int32_t count, int chunk, TAKE take, LAUNCH launch) {
  TABLE table{};
  int filled = 0;
  int64_t chunks = 0, before = 0, blocks = 0;
  auto flush = [&] {
    if (!filled) return;
    table.chunk[filled] = static_cast<uint32_t>(chunks);
    for (int i = filled + 1; i < TABLE::kSearched; ++i) table.chunk[i] = ~0u;
    launch(table, static_cast<unsigned>(chunks), before);
    before += chunks;
    chunks = filled = 0;
  };
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n == 0) continue;
    if (filled == TABLE::kTensors) flush();
    char* at[TABLE::kAddresses];
    take(t[i], at);
    for (int k = 0; k < TABLE::kAddresses; ++k) table.at[k][filled] = at[k];
    table.chunk[filled] = static_cast<uint32_t>(chunks);
    table.tail[filled] = static_cast<uint16_t>((t[i].n - 1) % chunk | (t[i].dtype == SDM_RT_BF16 ? 0x8000 : 0));
    if (TABLE::kBlocks) table.block[filled] = static_cast<uint32_t>(blocks);
    chunks += chunks_of(t[i].n, chunk);
    blocks += chunks_of(t[i].n, kBlock);
    ++filled;
  }
  flush();
}

// Few values take small chunks, so that all compute units have some: a model's 14 M float32 values' norm 13.2 us in chunks of
// 4,096, 15.0 of 16,384, their 8-bit step 40 us in chunks of 2,048, 42 of 4,096.  One bfloat16 tensor would cross over
// earlier: norms of 4, 8, 16, 32 and 105 Mi values 9.8, 10.2, 11.0, 19.6, 50.8 us in small chunks, 11.6, 9.9, 9.7, 15.7, 36.9
// in large ones, 8-bit steps 11.2, 23.2, 38.0, 73.1, 211 and 11.4, 19.4, 35.4, 66.5, 192; lists of many tensors between the
// two sizes were not compared.
constexpr int64_t kSmallStep = 16 << 20, kSmallNorm = 32 << 20;

inline int norm_chunk(int64_t values) { return values <= kSmallNorm ? 4096 : 16384; }
inline int64_t norm_partials(const sdm_rt_tensor* t, int32_t count, int64_t values) {
  int64_t n = 0;
  for (int32_t i = 0; i < count; ++i) n += chunks_of(t[i].n, norm_chunk(values));
  return n;
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

size_t sdm_rt_grad_norm_workspace_bytes(const sdm_rt_tensor* tensors, int32_t count) {
  int64_t values;
  return check_tensors(tensors, count, &values) ? 0 : static_cast<size_t>(norm_partials(tensors, count, values)) * sizeof(double);
}

int sdm_rt_grad_norm(const sdm_rt_tensor* tensors, int32_t count, float* norm, void* workspace, size_t workspace_bytes,
                     void* stream) {
  g_err[0] = 0;
  int64_t values;
  if (int rc = check_tensors(tensors, count, &values)) return rc;
  for (int32_t i = 0; i < count; ++i)
    if (tensors[i].n && !tensors[i].grad) return set_err(SDM_RT_EINVAL, "tensor %d: grad is NULL", i);
  if (!norm) return set_err(SDM_RT_EINVAL, "norm is NULL");
  const int64_t partials = norm_partials(tensors, count, values);
  const size_t need = static_cast<size_t>(partials) * sizeof(double);
  if (need && (!workspace || workspace_bytes < need))
    return set_err(SDM_RT_ENOSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return set_err(SDM_RT_EINVAL, "workspace must be 8-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  const int chunk = norm_chunk(values);
  for_tables<NormTable>(
      tensors, count, chunk,
      [](const sdm_rt_tensor& t, char** at) { at[0] = static_cast<char*>(const_cast<void*>(t.grad)); },
      [&](const NormTable& table, unsigned chunks, int64_t before) {
        if (chunk == 4096)
          hipLaunchKernelGGL(norm_kernel<4096>, dim3(chunks), dim3(kStepThreads), 0, st, table, partial + before);
        else
          hipLaunchKernelGGL(norm_kernel<16384>, dim3(chunks), dim3(kStepThreads), 0, st, table, partial + before);
      });
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(1024), 0, st, partial, static_cast<int>(partials), norm);
  return check_launch("grad_norm");
}

int sdm_rt_adamw(const sdm_rt_adamw_options* o, const sdm_rt_tensor* tensors, int32_t count, void* stream) {
  g_err[0] = 0;
  if (!o) return set_err(SDM_RT_EINVAL, "options is NULL");
  if (!(o->beta1 >= 0.0 && o->beta1 < 1.0) || !(o->beta2 >= 0.0 && o->beta2 < 1.0))
    return set_err(SDM_RT_EINVAL, "beta1 and beta2 must be in [0, 1)");
  if (!(o->eps >= 0.0) || !std::isfinite(o->eps) || !(o->weight_decay >= 0.0) || !std::isfinite(o->weight_decay))
    return set_err(SDM_RT_EINVAL, "eps and weight_decay must be finite and >= 0");
  if (!(o->lr_device && o->t_device) && (!(o->lr >= 0.0) || !std::isfinite(o->lr)))
    return set_err(SDM_RT_EINVAL, "lr must be finite and >= 0");
  if (o->lr_device && !o->t_device) return set_err(SDM_RT_EINVAL, "lr_device needs t_device");
  if (!o->t_device && o->t < 1) return set_err(SDM_RT_EINVAL, "t must be >= 1");
  if (o->norm && !(o->max_norm > 0.f)) return set_err(SDM_RT_EINVAL, "max_norm must be positive");
  if (o->state_bits != 32 && o->state_bits != 8) return set_err(SDM_RT_EINVAL, "state_bits must be 32 or 8");
  int64_t values, bytes = 0;   // bytes: of parameters, gradients and moments
  if (int rc = check_tensors(tensors, count, &values)) return rc;
  for (int32_t i = 0; i < count; ++i) {
    const sdm_rt_tensor& t = tensors[i];
    if (t.n == 0) continue;
    bytes += t.n * ((t.dtype == SDM_RT_BF16 ? 4 : 8) + (o->state_bits == 32 ? 8 : 2));
    if (!t.param || !t.grad || !t.exp_avg || (o->state_bits == 32) != (t.exp_avg_sq != nullptr))
      return set_err(SDM_RT_EINVAL, "tensor %d: param, grad and exp_avg must not be NULL, exp_avg_sq NULL for 8 bits alone", i);
    if (o->state_bits == 8 && reinterpret_cast<uintptr_t>(t.exp_avg) % 8)
      return set_err(SDM_RT_EINVAL, "tensor %d: 8-bit moments must be 8-byte aligned", i);
  }
  if (values == 0 && !o->t_device) return SDM_RT_OK;
  StepArgs a{};
  a.b1 = static_cast<float>(o->beta1);
  a.c1 = static_cast<float>(1.0 - o->beta1);
  a.b2 = static_cast<float>(o->beta2);
  a.c2 = static_cast<float>(1.0 - o->beta2);
  a.eps = static_cast<float>(o->eps);
  a.max_norm = o->max_norm;
  a.norm = o->norm;
  a.seed = o->seed;
  a.lr = o->lr;
  a.weight_decay = o->weight_decay;
  if (o->t_device) {
    a.t_device = o->t_device;
    a.lr_device = o->lr_device;
    a.log_b1 = std::log(o->beta1);
    a.log_b2 = std::log(o->beta2);
  } else {
    const double t = static_cast<double>(o->t);
    a.decay = static_cast<float>(1.0 - o->lr * o->weight_decay);
    a.size = static_cast<float>(o->lr / (1.0 - std::pow(o->beta1, t)));
    a.r2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(o->beta2, t)));
    a.key = step_key(o->seed, o->t);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (o->t_device) hipLaunchKernelGGL(count_step_kernel, dim3(1), dim3(1), 0, st, o->t_device);
  auto launch32 = [&](auto device, auto through, auto tiny) {
    constexpr int kChunk = 1024;   // 110 M float32 values 476 us, 466 with 2,048, 480 with 4,096; 285 M bfloat16 1,040, 1,075, 1,167
    for_tables<StepTable32>(
        tensors, count, kChunk,
        [](const sdm_rt_tensor& t, char** at) {
          at[0] = static_cast<char*>(t.param);
          at[1] = static_cast<char*>(const_cast<void*>(t.grad));
          at[2] = static_cast<char*>(t.exp_avg);
          at[3] = static_cast<char*>(t.exp_avg_sq);
        },
        [&](const StepTable32& table, unsigned chunks, int64_t) {
          hipLaunchKernelGGL((adamw32_kernel<kChunk, decltype(device)::value, decltype(through)::value, decltype(tiny)::value>),
                             dim3(chunks), dim3(kStepThreads), 0, st, table, a);
        });
  };
  auto launch8 = [&](auto chunk, auto device, auto through, auto tiny) {
    constexpr int kChunk = decltype(chunk)::value;
    for_tables<StepTable8>(
        tensors, count, kChunk,
        [](const sdm_rt_tensor& t, char** at) {
          at[0] = static_cast<char*>(t.param);
          at[1] = static_cast<char*>(const_cast<void*>(t.grad));
          at[2] = static_cast<char*>(t.exp_avg);
        },
        [&](const StepTable8& table, unsigned chunks, int64_t) {
          hipLaunchKernelGGL((adamw8_kernel<kChunk, decltype(device)::value, decltype(through)::value, decltype(tiny)::value>),
                             dim3(chunks), dim3(kStepThreads), 0, st, table, a);
        });
  };
  auto with_bits = [&](auto device, auto through, auto tiny) {
    if (o->state_bits == 32)
      launch32(device, through, tiny);
    else if (values <= kSmallStep)
      launch8(std::integral_constant<int, 2048>{}, device, through, tiny);
    else
      launch8(std::integral_constant<int, 4096>{}, device, through, tiny);
  };
  auto with_eps = [&](auto device, auto through) {
    if (o->eps * std::sqrt(1.0 - o->beta2) < 1.82e-12)   // 2^-39: step_value; 1 / sqrt(1 - beta2^t) is largest in the first step
      with_bits(device, through, std::true_type{});
    else
      with_bits(device, through, std::false_type{});
  };
  auto with_device = [&](auto through) {
    if (o->t_device)
      with_eps(std::true_type{}, through);
    else
      with_eps(std::false_type{}, through);
  };
  if (bytes > kStreamBytes)
    with_device(std::true_type{});
  else
    with_device(std::false_type{});
  return check_launch("adamw");
}

int64_t sdm_rt_moments_bytes(int64_t n) { return n > 0 ? (n + kBlock - 1) / kBlock * kBlockBytes : 0; }

int sdm_rt_read_moments(const sdm_rt_tensor* tensors, int32_t count, void* stream) {
  g_err[0] = 0;
  int64_t values, bytes = 0;
  if (int rc = check_tensors(tensors, count, &values)) return rc;
  for (int32_t i = 0; i < count; ++i) {
    const sdm_rt_tensor& t = tensors[i];
    if (t.n == 0) continue;
    bytes += t.n * (t.dtype == SDM_RT_BF16 ? 6 : 10);
    if (!t.param || !t.exp_avg || !t.exp_avg_sq) return set_err(SDM_RT_EINVAL, "tensor %d: a NULL pointer", i);
    if (reinterpret_cast<uintptr_t>(t.exp_avg) % 8)
      return set_err(SDM_RT_EINVAL, "tensor %d: 8-bit moments must be 8-byte aligned", i);
  }
  if (values == 0) return SDM_RT_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for_tables<ReadTable>(
      tensors, count, kReadChunk,
      [](const sdm_rt_tensor& t, char** at) {
        at[0] = static_cast<char*>(t.exp_avg);
        at[1] = static_cast<char*>(t.param);
        at[2] = static_cast<char*>(t.exp_avg_sq);
      },
      [&](const ReadTable& table, unsigned chunks, int64_t) {
        if (bytes > kStreamBytes)
          hipLaunchKernelGGL(read_moments_kernel<true>, dim3(chunks), dim3(kStepThreads), 0, st, table);
        else
          hipLaunchKernelGGL(read_moments_kernel<false>, dim3(chunks), dim3(kStepThreads), 0, st, table);
      });
  return check_launch("read_moments");
}

}  // extern "C"
