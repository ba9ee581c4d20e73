// sdm_embed.hip -- the scaled embedding lookup (sdm_rt_embed) and its gradient by sorted tokens (sdm_rt_embed_backward).
#include "sdm_vocab.h"

namespace sdmrt {

// out[n] = scale * table[ids[n]], rounded once.  A workgroup takes a run of whole rows and its threads their 16-byte
// pieces in turn.  Bound by memory: the rows in, the rows out.
constexpr int kEmbedPieces = 1024;   // pieces of a workgroup, about

template <typename T>
__global__ void __launch_bounds__(256) embed_kernel(const int64_t* __restrict__ ids, int64_t n, const T* __restrict__ table,
                                                    int64_t t_stride, int vocab, int d, float scale,
                                                    T* __restrict__ out, int64_t o_stride, int ppr, int rows) {
  constexpr int kN = Piece<T>::kN;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows; r0 < n; r0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int live = static_cast<int>(min(static_cast<int64_t>(rows), n - r0));
    for (int i = threadIdx.x; i < live * ppr; i += 256) {
      const int r = i / ppr, c = (i - r * ppr) * kN;
      const T* src = table + clamp_token(ids[r0 + r], vocab) * t_stride + c;
      T* dst = out + (r0 + r) * o_stride + c;
      Piece<T> p;
      const bool full = c + kN <= d;
      if (full)
        p.load(src);
      else
        p.load_part(src, d - c, T{});
      float v[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = p.get(e) * scale;
      p.set(v);
      if (full)
        p.store(dst);
      else
        p.store_part(dst, d - c);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The gradient, d_table[v] = round(scale * sum over the tokens n of v of dy[n]), in the order of n: the tokens are put in
// the order of their rows, then every row sums its own.
//
// embed_order_kernel: the stable order of the tokens by row, in one launch and without a float or a global atomic.  Row v
// belongs to workgroup v mod G and is its row v / G: frequent tokens have low ids, so they are dealt out to all
// workgroups.  Every workgroup reads all the ids twice (they stay in L2).  First it counts its own rows' tokens, each
// wave its own stretch of the ids, and the tokens of the workgroups before it; that fixes where each of its (row, wave)
// begins.  Then it reads them again and places its own, each wave in order: the lanes of one row find their ranks
// among each other by ballot.
// Slot b * R + i holds row i * G + b: offsets[slot] is where its tokens begin in order[], up to offsets[slot + 1].
constexpr int kOrderWaves = 16;
constexpr int kOrderMaxRows = 2048;   // rows of a workgroup: 16 counters of 4 bytes for each, 128 KiB of LDS

__global__ void __launch_bounds__(64 * kOrderWaves) embed_order_kernel(const int64_t* __restrict__ ids, int n, int vocab,
                                                                       int pad, int lg, int R,
                                                                       int32_t* __restrict__ offsets,
                                                                       int32_t* __restrict__ order,
                                                                       int32_t* __restrict__ row_of) {
  extern __shared__ int32_t cnt[];   // [kOrderWaves][R]: tokens of a row in a wave's stretch, then where they go
  __shared__ int32_t red[kOrderWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x, mask = (1 << lg) - 1;
  for (int i = threadIdx.x; i < kOrderWaves * R; i += 64 * kOrderWaves) cnt[i] = 0;
  __syncthreads();
  const int seg = (n + 64 * kOrderWaves - 1) / (64 * kOrderWaves) * 64;
  const int begin = min(n, wave * seg), end = min(n, begin + seg);
  int32_t* mine = cnt + wave * R;
  constexpr int kU = 8;
  int below = 0;
  for (int i0 = begin; i0 < end; i0 += 64 * kU) {
    int v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + 64 * u + lane;
      v[u] = i < end ? clamp_token(ids[i], vocab) : pad;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool live = v[u] != pad && i0 + 64 * u + lane < end;
      if (live && (v[u] & mask) < b) ++below;
      if (live && (v[u] & mask) == b) atomicAdd(&mine[v[u] >> lg], 1);
    }
  }
  below = wave_add(below);
  if (lane == 0) red[wave] = below;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < kOrderWaves; ++w) base += red[w];
  __syncthreads();
  // where each row begins: thread t takes rows 2t and 2t + 1
  int tot[2] = {0, 0};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = 2 * static_cast<int>(threadIdx.x) + q;
    if (r < R)
      for (int w = 0; w < kOrderWaves; ++w) tot[q] += cnt[w * R + r];
  }
  int inc = tot[0] + tot[1];
#pragma unroll
  for (int j = 1; j < 64; j <<= 1) {
    const int u = __shfl_up(inc, j);
    if (lane >= j) inc += u;
  }
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  int at = base + inc - tot[0] - tot[1];
  for (int w = 0; w < wave; ++w) at += red[w];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = 2 * static_cast<int>(threadIdx.x) + q;
    if (r >= R) continue;
    offsets[b * R + r] = at;
    for (int w = 0; w < kOrderWaves; ++w) {
      const int c = cnt[w * R + r];
      cnt[w * R + r] = at;
      at += c;
    }
  }
  if (b == mask && threadIdx.x == 64 * kOrderWaves - 1) offsets[(b + 1) * R] = at;   // rows past R count nothing
  __syncthreads();
  for (int i0 = begin; i0 < end; i0 += 64 * kU) {
    int v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + 64 * u + lane;
      v[u] = i < end ? clamp_token(ids[i], vocab) : pad;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + 64 * u + lane;
      uint64_t todo = __ballot(i < end && v[u] != pad && (v[u] & mask) == b);
      while (todo) {   // one row of this workgroup at a time
        const int row = __shfl(v[u], __ffsll(static_cast<unsigned long long>(todo)) - 1);
        const bool same = ((todo >> lane) & 1) && v[u] == row;
        const uint64_t group = __ballot(same);
        const int start = mine[row >> lg];
        if (same) {
          const int pos = start + __popcll(group & ((1ull << lane) - 1));
          order[pos] = i;
          row_of[pos] = row;
        }
        if (lane == 0) mine[row >> lg] = start + __popcll(group);
        todo &= ~group;
      }
    }
  }
}

// d_table: a wave per slot sums its tokens' rows in order
template <typename T>
__global__ void __launch_bounds__(256) embed_rows_grad_kernel(const int32_t* __restrict__ offsets,
                                                              const int32_t* __restrict__ order, const T* __restrict__ dy,
                                                              int64_t dy_stride, int vocab, int d, float scale, int lg, int R,
                                                              T* __restrict__ d_table, int64_t dt_stride) {
  const int lane = threadIdx.x & 63;
  const int slot = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (slot >= (R << lg)) return;
  const int row = ((slot % R) << lg) + slot / R;
  if (row >= vocab) return;
  const int begin = offsets[slot], end = offsets[slot + 1];
  constexpr int kN = Piece<T>::kN;
  for (int c = lane * kN; c < d; c += 64 * kN) {
    float acc[kN] = {};
    const bool full = c + kN <= d;
    Piece<T> p;
    for (int i = begin; i < end; ++i) {
      const T* src = dy + order[i] * dy_stride + c;
      if (full)
        p.load(src);
      else
        p.load_part(src, d - c, T{});
#pragma unroll
      for (int e = 0; e < kN; ++e) acc[e] += p.get(e);
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) acc[e] *= scale;
    p.set(acc);
    T* dst = d_table + static_cast<int64_t>(row) * dt_stride + c;
    if (full)
      p.store(dst);
    else
      p.store_part(dst, d - c);
  }
}

// the split of a vocabulary's rows over workgroups: 2^lg of them, R rows each
struct OrderPlan {
  int lg, R;
  size_t off_order, off_row, total;
};
inline OrderPlan order_plan(int64_t n, int64_t vocab) {
  OrderPlan p;
  p.lg = 8;   // a workgroup for every compute unit, until a workgroup's rows outgrow its counters
  while (((vocab + (int64_t{1} << p.lg) - 1) >> p.lg) > kOrderMaxRows) ++p.lg;
  p.R = static_cast<int>((vocab + (int64_t{1} << p.lg) - 1) >> p.lg);
  const size_t offs = (static_cast<size_t>(p.R) << p.lg) + 1;
  p.off_order = (offs * 4 + 255) / 256 * 256;
  p.off_row = p.off_order + (static_cast<size_t>(n) * 4 + 255) / 256 * 256;
  p.total = p.off_row + (static_cast<size_t>(n) * 4 + 255) / 256 * 256;
  return p;
}

constexpr int64_t kEmbedMaxTokens = int64_t{1} << 30, kEmbedMaxVocab = 1 << 25;   // positions in 32 bits, one launch
constexpr int kEmbedMaxWidth = 1 << 20;

inline int check_embed(int64_t n, int64_t vocab, int32_t d, const void* ids, const void* a, const void* b,
                       int64_t a_stride, int64_t b_stride, sdm_rt_dtype dtype) {
  int rc;
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (n < 0 || vocab < 1 || d < 1) return set_err(SDM_RT_EINVAL, "n must be >= 0, vocab and d >= 1");
  if (n > kEmbedMaxTokens || vocab > kEmbedMaxVocab || d > kEmbedMaxWidth)
    return set_err(SDM_RT_EUNSUPPORTED, "at most 2^30 tokens, a vocabulary of 2^25 and rows of 2^20 values");
  if ((n > 0 && (!ids || !a)) || !b) return set_err(SDM_RT_EINVAL, "a tensor is NULL");
  if (n > 0 && bad_read_stride(a_stride, d)) return set_err(SDM_RT_EINVAL, "a read row stride must be 0 or >= d");
  if (b_stride < d) return set_err(SDM_RT_EINVAL, "the written rows' stride must be >= d");
  return SDM_RT_OK;
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

int sdm_rt_embed(const int64_t* ids, int64_t n, const void* table, int64_t table_row_stride, sdm_rt_dtype dtype,
                 int64_t vocab, int32_t d, float scale, void* out, int64_t out_row_stride, void* stream) {
  g_err[0] = 0;
  if (n == 0) return SDM_RT_OK;
  int rc = check_embed(n, vocab, d, ids, table, out, table_row_stride, out_row_stride, dtype);
  if (rc) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int kn = dtype == SDM_RT_BF16 ? 8 : 4;
  const int ppr = (d + kn - 1) / kn;
  const int rows = std::max(1, kEmbedPieces / ppr);
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((n + rows - 1) / rows, 1 << 20));
  if (dtype == SDM_RT_BF16)
    hipLaunchKernelGGL((embed_kernel<bf16_t>), dim3(blocks), dim3(256), 0, st, ids, n, static_cast<const bf16_t*>(table),
                       table_row_stride, static_cast<int>(vocab), d, scale, static_cast<bf16_t*>(out), out_row_stride, ppr,
                       rows);
  else
    hipLaunchKernelGGL((embed_kernel<float>), dim3(blocks), dim3(256), 0, st, ids, n, static_cast<const float*>(table),
                       table_row_stride, static_cast<int>(vocab), d, scale, static_cast<float*>(out), out_row_stride, ppr,
                       rows);
  return check_launch("embed");
}

size_t sdm_rt_embed_backward_workspace_bytes(int64_t n, int64_t vocab, int32_t d) {
  if (n < 0 || vocab < 1 || d < 1 || n > kEmbedMaxTokens || vocab > kEmbedMaxVocab || d > kEmbedMaxWidth) return 0;
  return order_plan(n, vocab).total;
}

int sdm_rt_embed_backward(const int64_t* ids, int64_t n, const void* dy, int64_t dy_row_stride, sdm_rt_dtype dtype,
                          int64_t vocab, int32_t d, float scale, int64_t padding_idx, void* d_table,
                          int64_t d_table_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  int rc = check_embed(n, vocab, d, ids, dy, d_table, dy_row_stride, d_table_row_stride, dtype);
  if (rc) return rc;
  const OrderPlan p = order_plan(n, vocab);
  if (!workspace) return set_err(SDM_RT_EINVAL, "workspace is NULL");
  if (workspace_bytes < p.total)
    return set_err(SDM_RT_ENOSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, p.total);
  hipStream_t st = static_cast<hipStream_t>(stream);
  static const bool lds = allow_lds(reinterpret_cast<const void*>(embed_order_kernel));
  if (!lds) return lds_err("embed_backward");
  char* ws = static_cast<char*>(workspace);
  int32_t* offsets = reinterpret_cast<int32_t*>(ws);
  int32_t* order = reinterpret_cast<int32_t*>(ws + p.off_order);
  int32_t* row_of = reinterpret_cast<int32_t*>(ws + p.off_row);
  const int pad = padding_idx >= 0 && padding_idx < vocab ? static_cast<int>(padding_idx) : -1;
  hipLaunchKernelGGL(embed_order_kernel, dim3(1u << p.lg), dim3(64 * kOrderWaves),
                     static_cast<size_t>(kOrderWaves) * p.R * 4, st, ids, static_cast<int>(n), static_cast<int>(vocab), pad,
                     p.lg, p.R, offsets, order, row_of);
  if ((rc = check_launch("embed_order"))) return rc;
  const unsigned blocks = ((static_cast<unsigned>(p.R) << p.lg) + 3) / 4;
  if (dtype == SDM_RT_BF16)
    hipLaunchKernelGGL((embed_rows_grad_kernel<bf16_t>), dim3(blocks), dim3(256), 0, st, offsets, order,
                       static_cast<const bf16_t*>(dy), dy_row_stride, static_cast<int>(vocab), d, scale, p.lg, p.R,
                       static_cast<bf16_t*>(d_table), d_table_row_stride);
  else
    hipLaunchKernelGGL((embed_rows_grad_kernel<float>), dim3(blocks), dim3(256), 0, st, offsets, order,
                       static_cast<const float*>(dy), dy_row_stride, static_cast<int>(vocab), d, scale, p.lg, p.R,
                       static_cast<float*>(d_table), d_table_row_stride);
  return check_launch("embed_rows_grad");
}

}  // extern "C"
