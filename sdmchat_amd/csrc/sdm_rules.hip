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

// One workgroup per (row, slice of the vocabulary): 1,024 threads, NP pieces of 16 bytes each.  The slice's logits and mask
// words are loaded first; while they are on their way the workgroup counts the history's tokens that fall into the slice in
// LDS (integer atomics: exact in any order); then rules, out.  Bit 31 of a counter says the token was in the prompt, the
// rest counts its occurrences since.  Bound by memory, logits in and out, and by the history, which every slice of a row
// reads again: so slices are as large as leaves every compute unit two workgroups, and a row's slices run on one XCD, whose
// L2 then holds its history (workgroup i runs on XCD i mod 8).  The loads of logits, those of the history and the counting
// wait in turn, so every wave that fits is there to overlap them: 256 x 131,072 bf16 with histories of 8,192 take 36-38 us
// (a copy of as many bytes 30; rows of 131,071, which begin at any element, 40), with slices of 512 threads x 4 pieces 40, and
// with 8 tokens of a thread in flight, whose registers leave room for half the waves, 42.
constexpr int kRulesThreads = 1024, kXcds = 8;

template <typename T, int NP>
__global__ void __launch_bounds__(kRulesThreads, 8) rules_kernel(RulesArgs a, int64_t rows, int slices) {
  extern __shared__ uint4 lds[];
  uint32_t* cnt = reinterpret_cast<uint32_t*>(lds);
  constexpr int kN = Piece<T>::kN, kSlice = kRulesThreads * kN * NP;
  const int64_t group = blockIdx.x / kXcds;
  const int64_t row = group / slices * kXcds + blockIdx.x % kXcds;
  if (row >= rows) return;   // whole workgroups
  const int v0 = static_cast<int>(group % slices) * kSlice;
  const int nv = min(kSlice, a.vocab - v0);
  const bool hist = a.tokens != nullptr;
  const T* src = static_cast<const T*>(a.logits) + row * a.l_stride + v0;
  const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride + v0 / 32 : nullptr;   // slices are multiples of 32
  Piece<T> p[NP];
  uint32_t allowed[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const int c = (q * kRulesThreads + static_cast<int>(threadIdx.x)) * kN;
    allowed[q] = ~0u;
    if (c + kN <= nv)
      p[q].load(src + c);
    else if (c < nv)
      p[q].load_part(src + c, nv - c, T{});
    if (mask && c < nv) allowed[q] = mask[c >> 5] >> (c & 31);   // a piece lies in one word
  }
  if (hist) {
    for (int i = threadIdx.x; i < kSlice / 4; i += kRulesThreads) lds[i] = make_uint4(0, 0, 0, 0);
    const int64_t len = max(a.lengths[row], int64_t{0});
    const int64_t n = min(len, a.width);
    const int64_t prompt = a.prompt ? a.prompt[row] : 0;
    const int64_t* tk = a.tokens + row * a.t_stride;
    // the position of ring entry i: the latest one p < len with p mod width = i
    const int64_t last = len > a.width ? (len - 1) % a.width : len - 1;
    __syncthreads();
    constexpr int kU = 4;   // tokens of a thread in flight
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += kU * kRulesThreads) {
      int64_t t[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) t[u] = tk[min(i0 + u * kRulesThreads, n - 1)];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t i = i0 + u * kRulesThreads;
        const uint64_t at = static_cast<uint64_t>(t[u]) - static_cast<uint64_t>(v0);   // below nv: in the slice
        if (i < n && at < static_cast<uint64_t>(nv)) {
          const int64_t pos = len - 1 - (i <= last ? last - i : last - i + a.width);
          if (pos >= prompt)
            atomicAdd(&cnt[at], 1u);
          else
            atomicOr(&cnt[at], 0x80000000u);
        }
      }
    }
    __syncthreads();
  }
  const float rep = a.rep ? a.rep[row] : a.rep_all, rep_inv = 1.f / rep;
  const float freq = a.freq ? a.freq[row] : a.freq_all;
  const float pres = a.pres ? a.pres[row] : a.pres_all;
  T* dst = static_cast<T*>(a.out) + row * a.o_stride + v0;
  const float* bias = a.bias ? a.bias + row * a.bias_stride + v0 : nullptr;
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const int c = (q * kRulesThreads + static_cast<int>(threadIdx.x)) * kN;
    if (c >= nv) continue;
    const int live = min(kN, nv - c);
    float x[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) x[e] = p[q].get(e);
    if (hist) {
      uint32_t w[kN];
#pragma unroll
      for (int e = 0; e < kN; e += 4) {
        const uint4 u = lds[(c + e) / 4];
        w[e] = u.x;
        w[e + 1] = u.y;
        w[e + 2] = u.z;
        w[e + 3] = u.w;
      }
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < kN; ++e) any |= w[e];
      if (any) {
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          // x / rep: the product with the reciprocal, put right by its remainder (which is NaN for infinite x)
          const float y0 = x[e] * rep_inv, y1 = fmaf(fmaf(-y0, rep, x[e]), rep_inv, y0);
          const float y = x[e] > 0.f ? (y1 == y1 ? y1 : y0) : x[e] * rep;
          const float k = static_cast<float>(w[e] & 0x7fffffffu);
          const float z = k > 0.f ? y - fmaf(k, freq, pres) : y;
          x[e] = w[e] ? z : x[e];
        }
      }
    }
    if (bias) {
      if (live == kN) {
        float b[kN];
        __builtin_memcpy(b, bias + c, sizeof(b));
#pragma unroll
        for (int e = 0; e < kN; ++e) x[e] += b[e];
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (e < live) x[e] += bias[c + e];
      }
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) x[e] = (allowed[q] >> e) & 1 ? x[e] : -INFINITY;
    p[q].set(x);
    if (live == kN)
      p[q].store(dst + c);
    else
      p[q].store_part(dst + c, live);
  }
}

template <typename T>
void launch_rules(const RulesArgs& a, int64_t rows, hipStream_t st) {
  constexpr int kPieces = kRulesThreads * Piece<T>::kN;
  auto slices = [&](int np) { return (a.vocab + kPieces * np - 1) / (kPieces * np); };
  const int64_t rows8 = (rows + kXcds - 1) / kXcds * kXcds;
  auto launch = [&](auto np) {
    constexpr int NP = decltype(np)::value;
    hipLaunchKernelGGL((rules_kernel<T, NP>), dim3(static_cast<unsigned>(rows8 * slices(NP))), dim3(kRulesThreads),
                       a.tokens ? static_cast<size_t>(kPieces) * NP * 4 : 0, st, a, rows, slices(NP));
  };
  if (rows * slices(2) >= 512)
    launch(std::integral_constant<int, 2>{});
  else
    launch(std::integral_constant<int, 1>{});
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
  if (vocab > (1 << 21)) return set_err(SDM_RT_EUNSUPPORTED, "vocab must be at most 2^21");
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
  const int64_t groups = (rows + kXcds - 1) / kXcds * kXcds * ((vocab + 8191) / 8192);   // at most, in one launch
  if (groups >= int64_t{1} << 22) return set_err(SDM_RT_EUNSUPPORTED, "too many rows of so large a vocabulary");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SDM_RT_BF16)
    launch_rules<bf16_t>(a, rows, st);
  else
    launch_rules<float>(a, rows, st);
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
