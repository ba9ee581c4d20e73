// sdm_rules.hip -- the rules of a decode step on its logits (sdm_rt_process_logits: penalties for repeated tokens, a
// bias, a grammar mask) and the token history they read (sdm_rt_append_tokens).
#include "sdm_vocab.h"

namespace sdmrt {

struct RulesArgs {
  const void* logits;
  int64_t l_stride;
  void* out;
  int64_t o_stride;
  int vocab;
  const int64_t* tokens;   // [rows][width] the streams' tokens, or nullptr
  int64_t t_stride;
  int64_t width;
  const int64_t* lengths;   // [rows] tokens a stream has had (the array is a ring of its last `width`)
  const int64_t* prompt;    // [rows] or nullptr: the tokens before it are not counted
  const float* rep;         // [rows], or nullptr: the value of *_all for every row
  const float* freq;
  const float* pres;
  float rep_all, freq_all, pres_all;
  const float* bias;        // [vocab] rows of stride bias_stride (0: one for all), or nullptr
  int64_t bias_stride;
  const uint32_t* mask;     // rows of ceil(vocab / 32) words, stride mask_stride (0: one for all), or nullptr
  int64_t mask_stride;
};

// One workgroup per (row, slice of the vocabulary).  It counts the history's tokens that fall into its slice in LDS
// (integer atomics: exact in any order), then passes over the slice once: in, rules, out.  Bit 31 of a counter says the
// token was in the prompt, the rest counts its occurrences since.  A slice reads the row's whole history again, so
// slices are as large as leaves every compute unit something to do (rules_slice).
constexpr int kRulesThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kRulesThreads) rules_kernel(RulesArgs a, int slice) {
  extern __shared__ uint32_t cnt[];
  constexpr int kN = Piece<T>::kN;
  const int row = blockIdx.y;
  const int v0 = blockIdx.x * slice;
  const int nv = min(slice, a.vocab - v0);
  const bool hist = a.tokens != nullptr;
  if (hist) {
    for (int i = threadIdx.x; i < slice; i += kRulesThreads) cnt[i] = 0;
    __syncthreads();
    const int64_t len = max(a.lengths[row], int64_t{0});
    const int64_t n = min(len, a.width);
    const int64_t prompt = a.prompt ? a.prompt[row] : 0;
    const int64_t* tk = a.tokens + row * a.t_stride;
    // the position of ring entry i: the latest one p < len with p mod width = i
    const int64_t last = len > a.width ? (len - 1) % a.width : len - 1;
    for (int64_t i = threadIdx.x; i < n; i += kRulesThreads) {
      const int64_t t = tk[i] - v0;
      if (t < 0 || t >= nv) continue;
      const int64_t pos = len - 1 - (i <= last ? last - i : last - i + a.width);
      if (pos >= prompt)
        atomicAdd(&cnt[t], 1u);
      else
        atomicOr(&cnt[t], 0x80000000u);
    }
    __syncthreads();
  }
  const float rep = a.rep ? a.rep[row] : a.rep_all;
  const float freq = a.freq ? a.freq[row] : a.freq_all;
  const float pres = a.pres ? a.pres[row] : a.pres_all;
  const T* src = static_cast<const T*>(a.logits) + row * a.l_stride + v0;
  T* dst = static_cast<T*>(a.out) + row * a.o_stride + v0;
  const float* bias = a.bias ? a.bias + row * a.bias_stride + v0 : nullptr;
  const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride + v0 / 32 : nullptr;   // slices are multiples of 32
  for (int c = static_cast<int>(threadIdx.x) * kN; c < nv; c += kRulesThreads * kN) {
    const int live = min(kN, nv - c);
    Piece<T> p;
    if (live == kN)
      p.load(src + c);
    else
      p.load_part(src + c, live, T{});
    float x[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) x[e] = p.get(e);
    if (hist) {
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const uint32_t w = cnt[c + e];   // slices are multiples of kN
        if (w) {
          x[e] = x[e] > 0.f ? x[e] / rep : x[e] * rep;
          const uint32_t k = w & 0x7fffffffu;
          if (k) x[e] -= fmaf(static_cast<float>(k), freq, pres);
        }
      }
    }
    if (bias) {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < live) x[e] += bias[c + e];
    }
    if (mask) {
      const uint32_t w = mask[c >> 5] >> (c & 31);   // a piece lies in one word
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (!((w >> e) & 1)) x[e] = -INFINITY;
    }
    p.set(x);
    if (live == kN)
      p.store(dst + c);
    else
      p.store_part(dst + c, live);
  }
}

// the slice of the vocabulary of a workgroup
inline int rules_slice(int64_t rows, int vocab, bool hist) {
  int s = 2048;
  while (s < 16384 && rows * ((vocab + 2 * s - 1) / (2 * s)) >= 512) s *= 2;
  return s;
}

// tokens[row][lengths[row] mod width] = new_ids[row], lengths[row] += 1
__global__ void __launch_bounds__(256) append_tokens_kernel(int64_t* __restrict__ tokens, int64_t t_stride, int64_t width,
                                                            int64_t* __restrict__ lengths,
                                                            const int64_t* __restrict__ new_ids, int64_t rows) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (r >= rows) return;
  const int64_t len = max(lengths[r], int64_t{0});
  tokens[r * t_stride + len % width] = new_ids[r];
  lengths[r] = len + 1;
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

int sdm_rt_process_logits(const sdm_rt_rules* rules, const void* logits, int64_t logits_row_stride, sdm_rt_dtype dtype,
                          int64_t rows, int32_t vocab, void* out, int64_t out_row_stride, void* stream) {
  g_err[0] = 0;
  int rc;
  if (!rules) return set_err(SDM_RT_EINVAL, "rules is NULL");
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (rows < 0 || vocab < 1) return set_err(SDM_RT_EINVAL, "rows must be >= 0 and vocab >= 1");
  if (rows > 65535) return set_err(SDM_RT_EUNSUPPORTED, "rows = %lld must be at most 65,535", (long long)rows);
  if (vocab > (1 << 30)) return set_err(SDM_RT_EUNSUPPORTED, "vocab must be at most 2^30");
  if (rows == 0) return SDM_RT_OK;
  if (!logits || !out) return set_err(SDM_RT_EINVAL, "logits and out must not be NULL");
  if (bad_read_stride(logits_row_stride, vocab) || out_row_stride < vocab)
    return set_err(SDM_RT_EINVAL, "out_row_stride must be >= vocab, logits_row_stride that or 0");
  if (rules->tokens && rules->width > 0 && (!rules->lengths || bad_read_stride(rules->tokens_row_stride, rules->width)))
    return set_err(SDM_RT_EINVAL, "a history needs lengths, and tokens_row_stride 0 or >= width");
  if (rules->width < 0) return set_err(SDM_RT_EINVAL, "width must be >= 0");
  if (rules->bias && bad_read_stride(rules->bias_row_stride, vocab))
    return set_err(SDM_RT_EINVAL, "bias_row_stride must be 0 or >= vocab");
  if (rules->mask && bad_read_stride(rules->mask_row_stride, (static_cast<int64_t>(vocab) + 31) / 32))
    return set_err(SDM_RT_EINVAL, "mask_row_stride must be 0 or >= ceil(vocab / 32)");
  RulesArgs a{};
  a.logits = logits;
  a.l_stride = logits_row_stride;
  a.out = out;
  a.o_stride = out_row_stride;
  a.vocab = vocab;
  if (rules->tokens && rules->width > 0) {
    a.tokens = rules->tokens;
    a.t_stride = rules->tokens_row_stride;
    a.width = rules->width;
    a.lengths = rules->lengths;
    a.prompt = rules->prompt;
  }
  a.rep = rules->repetition;
  a.freq = rules->frequency;
  a.pres = rules->presence;
  a.rep_all = rules->repetition_all;
  a.freq_all = rules->frequency_all;
  a.pres_all = rules->presence_all;
  a.bias = rules->bias;
  a.bias_stride = rules->bias_row_stride;
  a.mask = rules->mask;
  a.mask_stride = rules->mask_row_stride;
  const int slice = rules_slice(rows, vocab, a.tokens != nullptr);
  const dim3 grid(static_cast<unsigned>((vocab + slice - 1) / slice), static_cast<unsigned>(rows));
  const size_t lds = a.tokens ? static_cast<size_t>(slice) * 4 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SDM_RT_BF16)
    hipLaunchKernelGGL((rules_kernel<bf16_t>), grid, dim3(kRulesThreads), lds, st, a, slice);
  else
    hipLaunchKernelGGL((rules_kernel<float>), grid, dim3(kRulesThreads), lds, st, a, slice);
  return check_launch("process_logits");
}

int sdm_rt_append_tokens(int64_t* tokens, int64_t tokens_row_stride, int64_t width, int64_t* lengths,
                         const int64_t* new_ids, int64_t rows, void* stream) {
  g_err[0] = 0;
  if (rows < 0 || width < 1) return set_err(SDM_RT_EINVAL, "rows must be >= 0 and width >= 1");
  if (rows > (int64_t{1} << 30)) return set_err(SDM_RT_EUNSUPPORTED, "rows must be at most 2^30");
  if (rows == 0) return SDM_RT_OK;
  if (!tokens || !lengths || !new_ids) return set_err(SDM_RT_EINVAL, "tokens, lengths and new_ids must not be NULL");
  if (tokens_row_stride < width) return set_err(SDM_RT_EINVAL, "tokens_row_stride must be >= width");
  hipLaunchKernelGGL(append_tokens_kernel, dim3(static_cast<unsigned>((rows + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), tokens, tokens_row_stride, width, lengths, new_ids, rows);
  return check_launch("append_tokens");
}

}  // extern "C"
