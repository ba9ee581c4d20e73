// sdm_embed.hip -- the scaled embedding lookup (sdm_rt_embed, sdm_rt_embed_checked) and its gradient by sorted tokens (sdm_rt_embed_backward).
#include "sdm_vocab.h"

namespace sdmrt {

// out[n] = scale * table[ids[n]], rounded once.  A workgroup takes a run of whole rows and its threads their 16-byte
// pieces in turn.  Bound by memory: the rows in, the rows out.  THROUGH: an output past kStreamBytes is stored past the
// caches, which keep the table's frequent rows (131,072 tokens of rows of 2 KB, 268 MB out: lookups one after another 88 -> 59
// us, 90 -> 63 over three tables in turn; after a backward pass that has filled the caches 93).  outside: where
// not nullptr, the last id found outside the table (a word of host memory, written only then).
constexpr int kEmbedPieces = 1024;   // pieces of a workgroup, about

template <typename T, bool THROUGH>
__global__ void __launch_bounds__(256) embed_kernel(const int64_t* __restrict__ ids, int64_t n, const T* __restrict__ table,
                                                    int64_t t_stride, int vocab, int d, float scale,
                                                    T* __restrict__ out, int64_t o_stride, int ppr, int rows,
                                                    int64_t* outside) {
  constexpr int kN = Piece<T>::kN;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows; r0 < n; r0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int live = static_cast<int>(min(static_cast<int64_t>(rows), n - r0));
    for (int i = threadIdx.x; i < live * ppr; i += 256) {
      // a row's last piece ends with the row: it may hold values of the piece before it once more
      const int r = i / ppr, c = max(0, min((i - r * ppr) * kN, d - kN));
      const int64_t id = ids[r0 + r];
      if (outside && (id < 0 || id >= vocab)) __hip_atomic_store(outside, id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
      const T* src = table + clamp_token(id, vocab) * t_stride + c;
      T* dst = out + (r0 + r) * o_stride + c;
      Piece<T> p;
      if (d >= kN)
        p.load(src);
      else
        p.load_part(src, d, T{});
      float v[kN];
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = p.get(e) * scale;
      p.set(v);
      if (d < kN)
        p.store_part(dst, d);
      else if (THROUGH)
        p.store_through(dst);
      else
        p.store(dst);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The gradient, d_table[v] = round(scale * sum over the tokens n of v of dy[n]), in the order of n: the tokens are put in
// the order of their rows, then every row sums its own.
//
// The stable order of the tokens by row, in two launches and without a global atomic.  Row v belongs to bucket v mod 256
// and is its row v / 256: frequent tokens have low ids, so they are dealt out to all buckets.  embed_tiles_kernel orders
// every tile of 1,024 tokens by bucket (lanes of one bucket find each other by ballots over its 8 bits, waves and buckets
// by a prefix sum) and keeps where the buckets begin.  embed_order_kernel, a workgroup per bucket, reads its run of every
// tile, each wave its own tiles: it counts its rows, and with the counts of the buckets before it (the sum over the tiles of
// where it begins there) places its tokens in the rows' order.  Every token is read twice; one launch whose workgroups each
// read all tokens was bound by its instructions (131,072 tokens: 106 us).
// Slot b * R + i holds row 256 i + b: offsets[slot] is where its tokens begin in order[], up to offsets[slot + 1].
constexpr int kTile = 1024, kBucketBits = 8, kBuckets = 1 << kBucketBits;
constexpr int kOrderMaxRows = 8192;

// the lanes of `live` whose `bits` low bits of v equal this lane's
__device__ __forceinline__ uint64_t same_lanes(uint64_t live, int v, int bits) {
  uint64_t m = live;
  for (int k = 0; k < bits; ++k) {
    const bool one = (v >> k) & 1;
    const uint64_t ones = __ballot(one);
    m &= one ? ones : ~ones;
  }
  return m;
}
__device__ __forceinline__ uint64_t lanes_below(int lane) { return (uint64_t{1} << lane) - 1; }

// bucket_at[b][t] (b <= 256): where bucket b begins in tile t; packed[1024 t + ...]: its tokens' rows i and places in the
// tile, i << 10 | place
__global__ void __launch_bounds__(kTile) embed_tiles_kernel(const int64_t* __restrict__ ids, int n, int vocab, int pad,
                                                            int tiles, int32_t* __restrict__ bucket_at,
                                                            uint32_t* __restrict__ packed) {
  __shared__ int32_t hist[kTile / 64][kBuckets];
  __shared__ int32_t red[kBuckets / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x;
  const int i = t * kTile + static_cast<int>(threadIdx.x);
  const int v = i < n ? clamp_token(ids[i], vocab) : pad;
  for (int k = threadIdx.x; k < kTile / 64 * kBuckets; k += kTile) hist[k / kBuckets][k % kBuckets] = 0;
  __syncthreads();
  const int b = v & (kBuckets - 1);
  const bool live = i < n && v != pad;
  const uint64_t group = same_lanes(__ballot(live), b, kBucketBits);
  const int rank = __popcll(group & lanes_below(lane));
  if (live && rank == 0) hist[wave][b] = __popcll(group);
  __syncthreads();
  int count = 0, inc = 0;
  if (threadIdx.x < kBuckets) {
    int32_t c[kTile / 64];
#pragma unroll
    for (int w = 0; w < kTile / 64; ++w) c[w] = hist[w][threadIdx.x];
#pragma unroll
    for (int w = 0; w < kTile / 64; ++w) {
      hist[w][threadIdx.x] = count;
      count += c[w];
    }
    inc = count;
#pragma unroll
    for (int j = 1; j < 64; j <<= 1) {
      const int u = __shfl_up(inc, j);
      if (lane >= j) inc += u;
    }
    if (lane == 63) red[wave] = inc;
  }
  __syncthreads();
  if (threadIdx.x < kBuckets) {
    int start = inc - count;
    for (int w = 0; w < wave; ++w) start += red[w];
    for (int w = 0; w < kTile / 64; ++w) hist[w][threadIdx.x] += start;
    bucket_at[static_cast<int64_t>(threadIdx.x) * tiles + t] = start;
    if (threadIdx.x == kBuckets - 1) bucket_at[static_cast<int64_t>(kBuckets) * tiles + t] = start + count;
  }
  __syncthreads();
  if (live) packed[static_cast<int64_t>(t) * kTile + hist[wave][b] + rank] =
      static_cast<uint32_t>(v >> kBucketBits) << 10 | threadIdx.x;
}

constexpr int kTileBatch = 8;   // tiles of a wave whose tokens are loaded together

__global__ void __launch_bounds__(1024) embed_order_kernel(const int32_t* __restrict__ bucket_at,
                                                           const uint32_t* __restrict__ packed, int tiles, int R,
                                                           int row_bits, int32_t* __restrict__ offsets,
                                                           int32_t* __restrict__ order, int32_t* __restrict__ row_of) {
  extern __shared__ int32_t cnt[];   // [waves][R]: tokens of a row in a wave's tiles, then where they go
  __shared__ int32_t red[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int b = blockIdx.x;
  const int32_t* at = bucket_at + static_cast<int64_t>(b) * tiles;
  int below = 0;
  for (int t = threadIdx.x; t < tiles; t += blockDim.x) below += at[t];
  for (int i = threadIdx.x; i < waves * R; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int per = (tiles + waves - 1) / waves;
  const int t0 = min(tiles, wave * per), t1 = min(tiles, t0 + per);
  int32_t* mine = cnt + wave * R;
  // a wave's tiles, kTileBatch at a time: lane q holds where the bucket's run of tile tb + q begins and ends
  auto for_tokens = [&](auto use) {
    for (int tb = t0; tb < t1; tb += kTileBatch) {
      const int tl = min(tb + min(lane, kTileBatch - 1), t1 - 1);
      const int from = at[tl], to = at[tiles + tl];
      uint32_t e[kTileBatch];
#pragma unroll
      for (int q = 0; q < kTileBatch; ++q) {   // the first 64 tokens of every run, in flight together
        const int tile = min(tb + q, t1 - 1);
        e[q] = packed[static_cast<int64_t>(tile) * kTile + min(__shfl(from, q) + lane, kTile - 1)];
      }
#pragma unroll
      for (int q = 0; q < kTileBatch; ++q) {
        if (tb + q >= t1) continue;   // the same for the wave
        const int begin = __shfl(from, q), end = __shfl(to, q);
        use(tb + q, e[q], begin + lane < end);
        for (int j = begin + 64; j < end; j += 64) {
          const bool live = j + lane < end;
          use(tb + q, live ? packed[static_cast<int64_t>(tb + q) * kTile + j + lane] : 0u, live);
        }
      }
    }
  };
  for_tokens([&](int, uint32_t e, bool live) {
    if (live) atomicAdd(&mine[e >> 10], 1);
  });
  below = wave_add(below);
  if (lane == 0) red[wave] = below;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < waves; ++w) base += red[w];
  __syncthreads();
  // where each row begins: a thread takes a run of rows
  const int rpt = (R + blockDim.x - 1) / blockDim.x;
  const int r0 = min(R, static_cast<int>(threadIdx.x) * rpt), r1 = min(R, r0 + rpt);
  int tot = 0;
  for (int r = r0; r < r1; ++r)
    for (int w = 0; w < waves; ++w) tot += cnt[w * R + r];
  int inc = tot;
#pragma unroll
  for (int j = 1; j < 64; j <<= 1) {
    const int u = __shfl_up(inc, j);
    if (lane >= j) inc += u;
  }
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  int pos = base + inc - tot;
  for (int w = 0; w < wave; ++w) pos += red[w];
  for (int r = r0; r < r1; ++r) {
    offsets[b * R + r] = pos;
    for (int w = 0; w < waves; ++w) {
      const int c = cnt[w * R + r];
      cnt[w * R + r] = pos;
      pos += c;
    }
  }
  if (b == kBuckets - 1 && threadIdx.x == blockDim.x - 1) offsets[kBuckets * R] = pos;   // rows past R count nothing
  __syncthreads();
  for_tokens([&](int tile, uint32_t e, bool live) {
    const int row = live ? static_cast<int>(e >> 10) : 0;
    const uint64_t group = same_lanes(__ballot(live), row, row_bits);
    const int rank = __popcll(group & lanes_below(lane));
    const int start = mine[row];
    if (live) {
      order[start + rank] = tile * kTile + static_cast<int>(e & 1023);
      row_of[start + rank] = row << kBucketBits | b;
      if (rank == 0) mine[row] = start + __popcll(group);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next tokens' lanes read what these wrote
  });
}

// The rows' sums.  The ordered tokens are cut into pieces of `len`; a group of LANES lanes sums a piece's runs of equal rows
// in order, lane l columns 4l ... 4l + 3 of its slice.  A run that is its whole row is scaled and stored; one that
// crosses an edge of a workgroup's pieces leaves a float32 partial row: part[2 b] continues a row begun before workgroup b,
// part[2 b + 1] begins one that goes on after it.  The work follows the tokens and not the rows: text repeats its tokens, and with a wave
// per row the most frequent token's chain of loads was the kernel's time (16,384 tokens of 32,768 rows of 768, a Zipf
// stream: 739 us).
template <typename T>
struct Quad4 {   // four values of a row at any element alignment
  using Raw = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
  Raw r;
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&r, p, sizeof(r)); }
  __device__ __forceinline__ void load_through(const T* p) {
    using W = typename std::conditional<sizeof(T) == 2, words2, words4>::type;
    const W w = __builtin_nontemporal_load(reinterpret_cast<const W*>(p));
    __builtin_memcpy(&r, &w, sizeof(r));
  }
  __device__ __forceinline__ void load_part(const T* p, int n) {
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = T{};
      if (e < n) v[e] = p[e];
    }
    __builtin_memcpy(&r, v, sizeof(r));
  }
  __device__ __forceinline__ float get(int e) const {
    uint32_t w[sizeof(T)];
    __builtin_memcpy(w, &r, sizeof(r));
    if constexpr (sizeof(T) == 2)
      return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    else
      return __uint_as_float(w[e]);
  }
  __device__ __forceinline__ void store(T* p, const float (&v)[4], int n) {
    if constexpr (sizeof(T) == 2)
      r = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    else
      r = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    if (n >= 4) {
      __builtin_memcpy(p, &r, sizeof(r));
      return;
    }
    T t[4];
    __builtin_memcpy(t, &r, sizeof(r));
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) p[e] = t[e];
  }
};

// The four columns of a lane that would begin at column c: the row's last four where they would pass its end, so every load
// and store is whole and none is behind a branch (two lanes then hold some columns, with the same sums).  Rows of less
// than four values begin at 0.
__device__ __forceinline__ int quad_column(int c, int d) { return max(0, min(c, d - 4)); }

struct RowsGrad {
  const int32_t* offsets;
  const int32_t* order;
  const int32_t* row_of;
  float* part;        // [2 blocks][pitch]
  int pitch;          // d rounded up to 4
  int n_tokens;       // all of them, the padding's too
  int n_slots;        // 256 R
  int R, vocab, d;
  int blocks, slices;   // workgroups on the pieces, on the columns of a row
  int len;            // a piece's tokens
  int2* edge;         // [blocks] the row that leaves a workgroup and the last workgroup that has a part of it, or -1
  float scale;
  const void* dy;
  int64_t dy_stride;
  void* d_table;
  int64_t dt_stride;
};

// Workgroups past the pieces' clear the rows without a token meanwhile, each wave those among kClearRows slots.
constexpr int kClearRows = 8;

template <typename T>
__device__ __forceinline__ void clear_rows(const RowsGrad& a, int first) {
  constexpr int kN = Piece<T>::kN;
  const int lane = threadIdx.x & 63;
  const int off = a.offsets[min(first + min(lane, kClearRows), a.n_slots)];
  Piece<T> none;
  none.r = make_uint4(0, 0, 0, 0);
  for (int q = 0; q < kClearRows; ++q) {
    const int slot = first + q;
    if (slot >= a.n_slots || __shfl(off, q) != __shfl(off, q + 1)) continue;
    const int row = slot % a.R * kBuckets + slot / a.R;
    if (row >= a.vocab) continue;
    T* dst = static_cast<T*>(a.d_table) + static_cast<int64_t>(row) * a.dt_stride;
    for (int c = lane * kN; c < a.d; c += 64 * kN) {
      if (c + kN <= a.d)
        none.store(dst + c);
      else
        none.store_part(dst + c, a.d - c);
    }
  }
}

// A workgroup of 256 threads takes 256 / LANES pieces side by side, and of their rows one slice of 4 LANES columns,
// a lane four of them: the code that ends a run stands behind every row of a batch, and with a wave on 1,024
// columns fetching it once each took a third of the kernel (16,384 tokens: 13 us).  A group's cut runs go to LDS, head (a run
// begun before its piece) and tail (one that goes on after it); a run cut inside the workgroup is then put together there by
// the group it begins in, and only one that enters or leaves the workgroup becomes a partial row in memory: with a
// partial row for every cut piece they were a sixth of the kernel's traffic and their join took as long again as the sums
// of 16,384 tokens (9.6 us).  THROUGH: gradients past kStreamBytes, each read once, are read past the caches (131,072 rows of
// 2 KB: the backward 156 -> 125 us).
template <typename T, int LANES, bool THROUGH>
__global__ void __launch_bounds__(256) embed_rows_grad_kernel(RowsGrad a) {
  constexpr int QS = 16;   // rows in flight
  constexpr int kGroups = 256 / LANES;
  __shared__ float4 heads[kGroups][LANES];
  __shared__ float4 tails[kGroups][LANES];
  __shared__ int through[kGroups];   // the group's head run goes on after its piece
  const int lane = threadIdx.x % LANES, mine = threadIdx.x / LANES;
  if (static_cast<int>(blockIdx.x) >= a.blocks * a.slices) {
    clear_rows<T>(a, ((blockIdx.x - a.blocks * a.slices) * 4 + (threadIdx.x >> 6)) * kClearRows);
    return;
  }
  const int block = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;   // a row's slices side by side
  const int group = static_cast<int>(threadIdx.x & 63) & ~(LANES - 1);
  // one trip for everything the piece needs to know: lane l holds token l of the piece (len is at most LANES), the rows
  // before and after it, and how many tokens there are (n_tokens but for the padding's; what lies past them is not used)
  const int total = a.offsets[a.n_slots];
  const int64_t block_begin = static_cast<int64_t>(block) * kGroups * a.len;
  const int begin = static_cast<int>(min(block_begin + mine * a.len, static_cast<int64_t>(a.n_tokens)));
  const int own_at = min(begin + min(lane, a.len - 1), a.n_tokens - 1);
  const int tok = a.order[own_at], row = a.row_of[own_at];
  const int row_before = a.row_of[max(begin - 1, 0)], row_after = a.row_of[min(begin + a.len, a.n_tokens - 1)];
  const bool first_slice = slice == 0;
  if (block_begin >= total) {   // whole workgroups
    if (first_slice && threadIdx.x == 0) a.edge[block] = make_int2(-1, 0);
    return;
  }
  const int n = max(0, min(a.len, total - begin));   // none for groups past the end
  const int before = begin > 0 && n > 0 ? row_before : -1;
  const int after = begin + n < total ? row_after : -1;
  const int row0 = __shfl(row, group), row_last = __shfl(row, group + max(n, 1) - 1);
  const bool head = n > 0 && row0 == before;               // its first run began before it
  const bool whole = head && row0 == row_last && row0 == after;   // and goes on after it
  const bool tail = n > 0 && row_last == after && !whole && !(head && row0 == row_last);   // its last begins here, goes on
  if (lane == 0) through[mine] = whole;
  const int col = slice * 4 * LANES + 4 * lane, c = quad_column(col, a.d);
  const bool live = col < a.d, narrow = a.d < 4;
  auto store_row = [&](int to, float4 x) {
    const float v[4] = {x.x * a.scale, x.y * a.scale, x.z * a.scale, x.w * a.scale};
    Quad4<T> o;
    if (live) o.store(static_cast<T*>(a.d_table) + static_cast<int64_t>(to) * a.dt_stride + c, v, a.d - c);
  };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  int cur = row0;
  bool first = true;   // the run of cur is the piece's first
  for (int i0 = 0; i0 < n; i0 += QS) {
    Quad4<T> g[QS];
#pragma unroll
    for (int q = 0; q < QS; ++q) {
      const T* src = static_cast<const T*>(a.dy) + __shfl(tok, group + min(i0 + q, n - 1)) * a.dy_stride;
      if (narrow)
        g[q].load_part(src, a.d);
      else if (THROUGH)
        g[q].load_through(src + c);
      else
        g[q].load(src + c);
    }
#pragma unroll
    for (int q = 0; q < QS; ++q) {
      const int r = __shfl(row, group + min(i0 + q, n - 1));
      if (r != cur) {
        if (first && head)
          heads[mine][lane] = acc;
        else
          store_row(cur, acc);
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        cur = r;
        first = false;
      }
      if (i0 + q < n) {   // past the piece's end nothing is added
        acc.x += g[q].get(0);
        acc.y += g[q].get(1);
        acc.z += g[q].get(2);
        acc.w += g[q].get(3);
      }
    }
  }
  if (n > 0) {
    if (first && head)
      heads[mine][lane] = acc;
    else if (tail)
      tails[mine][lane] = acc;
    else
      store_row(cur, acc);
  }
  __syncthreads();
  // the runs cut by the groups' edges: group 0 takes the one that enters the workgroup, every group the one it begins
  const bool enters = mine == 0 && head;
  float* part = a.part + 2 * static_cast<int64_t>(block) * a.pitch;
  auto join = [&](float4& x, int g, bool on) {   // adds the heads from group g while the run goes on; whether it leaves
    for (; on && g < kGroups; ++g) {
      const float4 v = heads[g][lane];
      x.x += v.x;
      x.y += v.y;
      x.z += v.z;
      x.w += v.w;
      on = through[g] != 0;
    }
    return on;
  };
  if (enters) {
    float4 x = heads[0][lane];
    join(x, 1, through[0] != 0);
    if (live) __builtin_memcpy(part + c, &x, 16);
  }
  bool leaves = false;
  if (tail) {
    float4 x = tails[mine][lane];
    leaves = join(x, mine + 1, true);
    if (!leaves)
      store_row(row_last, x);   // begun and ended in this workgroup
    else if (live)
      __builtin_memcpy(part + a.pitch + c, &x, 16);
  }
  // the run that begins in this workgroup and leaves it, for the join: its row and the last workgroup it reaches
  if (first_slice) {
    if (leaves && lane == 0) {
      const int slot = (row_last & (kBuckets - 1)) * a.R + (row_last >> kBucketBits);
      a.edge[block] = make_int2(row_last, (a.offsets[slot + 1] - 1) / (kGroups * a.len));
    }
    if (!__syncthreads_or(leaves) && threadIdx.x == 0) a.edge[block] = make_int2(-1, 0);
  }
}

// The rows cut over several workgroups: for each workgroup of the sums that one leaves, a workgroup adds that row's partial
// rows, its four quarters of 256 threads a quarter of the partial rows each, in order.
template <typename T>
__global__ void __launch_bounds__(1024) embed_rows_join_kernel(RowsGrad a) {
  __shared__ float4 red[3][256];
  const int s = blockIdx.x;
  const int2 edge = a.edge[s];
  if (edge.x < 0) return;   // whole workgroups
  const int row = edge.x, last = edge.y;   // workgroups s (its second partial row), s + 1 ... last (their first)
  const int n = last - s + 1, quarter = threadIdx.x >> 8, per = (n + 3) / 4;
  const int p0 = s + min(n, quarter * per), p1 = s + min(n, (quarter + 1) * per);
  for (int cb = 0; cb < a.d; cb += 1024) {
    const int col = cb + 4 * static_cast<int>(threadIdx.x & 255), c = quad_column(col, a.d);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < a.d) {
      constexpr int kB = 16;
      for (int p = p0; p < p1; p += kB) {
        float4 v[kB];
#pragma unroll
        for (int q = 0; q < kB; ++q) {
          const int at = min(p + q, p1 - 1);
          __builtin_memcpy(&v[q], a.part + (2 * static_cast<int64_t>(at) + (at == s)) * a.pitch + c, 16);
        }
#pragma unroll
        for (int q = 0; q < kB; ++q) {
          if (p + q < p1) {
            acc.x += v[q].x;
            acc.y += v[q].y;
            acc.z += v[q].z;
            acc.w += v[q].w;
          }
        }
      }
    }
    if (quarter) red[quarter - 1][threadIdx.x & 255] = acc;
    __syncthreads();
    if (quarter == 0 && col < a.d) {
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        const float4 v = red[q][threadIdx.x];
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
      }
      const float v[4] = {acc.x * a.scale, acc.y * a.scale, acc.z * a.scale, acc.w * a.scale};
      Quad4<T> o;
      o.store(static_cast<T*>(a.d_table) + static_cast<int64_t>(row) * a.dt_stride + c, v, a.d - c);
    }
    __syncthreads();
  }
}

// Few tokens: the whole gradient in one launch.  A workgroup per bucket and 256 columns reads all ids itself, every wave a run
// of them, puts its own tokens in the order of their rows in LDS (counts per wave and row, their prefix sums, places by
// ballots: the tokens of a row stay in their order), clears its rows without one and sums the others: rows of up to kAlone
// tokens by a wave each, the frequent ones by all waves, which share a row's tokens and join over LDS.  What bounds it is
// the table's gradient going out and one compute unit's loads of a frequent token's rows (410 of 5,003 in a Zipf stream: 9 us),
// which the four launches share evenly: 64 tokens of 32,768 rows of 768 in bfloat16 take 13 us against their 18, 2,048 18
// against 23, 4,096 22 against 23, 6,144 26 against 24.  A call that waits for the host also saves three launches.
// Every slice of 256 columns orders the tokens anew, so wide rows are left to the four launches: Zipf streams of 640 and
// 5,120 tokens of 8,192 float32 rows take 8 and 14 us against 19 and 21 with 256 columns, 20 and 26 against 21 and 26 with
// 1,024, but 29 and 41 against 27 and 36 with 2,048, 45 and 76 against 39 and 57 with 4,096.  One token all along is the
// worst stream for one launch: 5,120 times 131 us against 40 with 1,024 columns, 188 against 77 with 4,096.
constexpr int kFewTokens = 5120, kFewRows = 1024, kFewWidth = 1024, kFewWaves = 16, kAlone = 32;
inline size_t few_lds(int R, int64_t n) {
  return (static_cast<size_t>(kFewWaves) * R + R + 1 + kFewTokens / kAlone) * 4 + static_cast<size_t>(n) * 2;
}

template <typename T>
__global__ void __launch_bounds__(64 * kFewWaves, 8) embed_few_grad_kernel(const int64_t* __restrict__ ids, int n, int vocab,
                                                                        int pad, int R, int row_bits,
                                                                        const T* __restrict__ dy, int64_t dy_stride,
                                                                        float scale, T* __restrict__ d_table,
                                                                        int64_t dt_stride, int d) {
  extern __shared__ int32_t cnt[];   // [waves][R]: tokens of a row in a wave's run, then where they go
  __shared__ float4 part[kFewWaves][64];
  __shared__ int32_t red[kFewWaves];
  __shared__ int32_t n_many;
  constexpr int kRun = kFewTokens / kFewWaves / 64;   // tokens of a lane, at most
  int32_t* off = cnt + kFewWaves * R;                 // [R + 1]: where a row's tokens begin in list
  int32_t* many = off + R + 1;                        // rows of more than kAlone
  uint16_t* list = reinterpret_cast<uint16_t*>(many + kFewTokens / kAlone);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x;
  const int run = (n + 64 * kFewWaves - 1) / (64 * kFewWaves);   // 64 tokens each
  int64_t id[kRun];
  int row[kRun];   // of the bucket, or -1
#pragma unroll
  for (int k = 0; k < kRun; ++k)   // all on their way together
    if (k < run) id[k] = ids[min((wave * run + k) * 64 + lane, n - 1)];
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    row[k] = -1;
    if (k >= run || (wave * run + k) * 64 + lane >= n) continue;
    const int v = clamp_token(id[k], vocab);
    if (v != pad && (v & (kBuckets - 1)) == b) row[k] = v >> kBucketBits;
  }
  for (int i = threadIdx.x; i < kFewWaves * R; i += 64 * kFewWaves) cnt[i] = 0;
  if (threadIdx.x == 0) n_many = 0;
  __syncthreads();
  int32_t* mine = cnt + wave * R;
#pragma unroll
  for (int k = 0; k < kRun; ++k)
    if (row[k] >= 0) atomicAdd(&mine[row[k]], 1);
  __syncthreads();
  {   // a thread per row (R is at most their number)
    const int r = threadIdx.x;
    int tot = 0;
    if (r < R)
      for (int w = 0; w < kFewWaves; ++w) tot += cnt[w * R + r];
    int inc = tot;
#pragma unroll
    for (int j = 1; j < 64; j <<= 1) {
      const int u = __shfl_up(inc, j);
      if (lane >= j) inc += u;
    }
    if (lane == 63) red[wave] = inc;
    __syncthreads();
    int pos = inc - tot;
    for (int w = 0; w < wave; ++w) pos += red[w];
    if (r < R) {
      off[r] = pos;
      if (r == R - 1) off[R] = pos + tot;
      if (tot > kAlone) many[atomicAdd(&n_many, 1)] = r;
      for (int w = 0; w < kFewWaves; ++w) {
        const int c = cnt[w * R + r];
        cnt[w * R + r] = pos;
        pos += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const bool live = row[k] >= 0;
    const uint64_t all = __ballot(live);
    if (!all) continue;   // the same for the wave
    const int r = live ? row[k] : 0;
    const uint64_t group = same_lanes(all, r, row_bits);
    const int rank = __popcll(group & lanes_below(lane));
    const int start = mine[r];
    if (live) {
      list[start + rank] = static_cast<uint16_t>((wave * run + k) * 64 + lane);
      if (rank == 0) mine[r] = start + __popcll(group);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next tokens' lanes read what these wrote
  }
  __syncthreads();
  const bool narrow = d < 4;
  const int col = blockIdx.y * 256 + 4 * lane, c = quad_column(col, d);
  // the sum of the rows of m tokens from list[first] on
  auto sum = [&](int first, int m) {
    constexpr int kB = 4;   // rows in flight (8: no gain, the waves are many)
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < m; j += kB) {
      const int t = list[first + min(j + min(lane, kB - 1), m - 1)];
      Quad4<T> g[kB];
#pragma unroll
      for (int q = 0; q < kB; ++q) {
        const T* src = dy + __builtin_amdgcn_readlane(t, q) * dy_stride;
        if (narrow)
          g[q].load_part(src, d);
        else
          g[q].load(src + c);
      }
#pragma unroll
      for (int q = 0; q < kB; ++q) {
        if (j + q < m) {
          acc.x += g[q].get(0);
          acc.y += g[q].get(1);
          acc.z += g[q].get(2);
          acc.w += g[q].get(3);
        }
      }
    }
    return acc;
  };
  auto store = [&](int r, float4 x) {
    const float v[4] = {x.x * scale, x.y * scale, x.z * scale, x.w * scale};
    Quad4<T> o;
    if (col < d) o.store(d_table + (static_cast<int64_t>(r) << kBucketBits | b) * dt_stride + c, v, d - c);
  };
  const int r_own = kFewWaves * lane + wave;   // a wave's rows: 16 lane + wave
  const bool there = r_own < R && (r_own << kBucketBits | b) < vocab;
  const int first = there ? off[r_own] : 0, m = there ? off[r_own + 1] - first : -1;
  for (uint64_t left = __ballot(m == 0); left; left &= left - 1)
    store(kFewWaves * (__ffsll(static_cast<unsigned long long>(left)) - 1) + wave, make_float4(0.f, 0.f, 0.f, 0.f));
  for (uint64_t left = __ballot(m > 0 && m <= kAlone); left; left &= left - 1) {
    const int l = __ffsll(static_cast<unsigned long long>(left)) - 1;
    store(kFewWaves * l + wave, sum(__builtin_amdgcn_readlane(first, l), __builtin_amdgcn_readlane(m, l)));
  }
  for (int e = 0; e < n_many; ++e) {
    const int r = many[e], from = off[r], k = off[r + 1] - from, per = (k + kFewWaves - 1) / kFewWaves;
    const int j0 = min(k, wave * per);
    part[wave][lane] = sum(from + j0, min(k, j0 + per) - j0);
    __syncthreads();
    if (wave == 0) {
      float4 x = part[0][lane];
      for (int q = 1; q < kFewWaves; ++q) {
        const float4 y = part[q][lane];
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      store(r, x);
    }
    __syncthreads();
  }
}

// the shape of the order and the sums
struct OrderPlan {
  int R, row_bits, waves, tiles;          // rows of a bucket, the bits of their numbers, waves that order them
  int lanes, len, block, blocks, pitch;   // lanes of a piece, its tokens, those of a workgroup, workgroups
  size_t off_bucket, off_packed, off_order, off_row, off_edge, off_part, total;
};
inline OrderPlan order_plan(int64_t n, int64_t vocab, int d) {
  OrderPlan p;
  p.R = static_cast<int>((vocab + kBuckets - 1) / kBuckets);
  p.row_bits = 0;
  while ((p.R - 1) >> p.row_bits) ++p.row_bits;
  p.waves = p.R <= 2048 ? 16 : 4;   // counters of 4 bytes per wave and row, 128 KiB of LDS
  p.tiles = static_cast<int>((n + kTile - 1) / kTile);
  p.lanes = d <= 64 ? 16 : d <= 128 ? 32 : 64;   // four columns a lane
  // pieces of 16 tokens, two batches of rows in flight, for every SIMD; past 4,096 pieces longer ones, so that the partial
  // rows of a frequent token stay few
  p.len = 16;
  while (p.len < p.lanes && n / p.len > 4096) p.len *= 2;
  p.block = 256 / p.lanes * p.len;
  p.blocks = static_cast<int>((n + p.block - 1) / p.block);
  p.pitch = (d + 3) / 4 * 4;
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  take((static_cast<size_t>(p.R) * kBuckets + 1) * 4);   // offsets
  p.off_bucket = take((static_cast<size_t>(kBuckets) + 1) * p.tiles * 4);
  p.off_packed = take(static_cast<size_t>(p.tiles) * kTile * 4);
  p.off_order = take(static_cast<size_t>(n) * 4);
  p.off_row = take(static_cast<size_t>(n) * 4);
  p.off_edge = take(static_cast<size_t>(p.blocks) * 8);
  p.off_part = take(2 * static_cast<size_t>(p.blocks) * p.pitch * 4);
  p.total = o;
  return p;
}

constexpr int64_t kEmbedMaxTokens = 1 << 27, kEmbedMaxVocab = kOrderMaxRows * kBuckets;   // positions in 32 bits, one launch
constexpr int kEmbedMaxWidth = 1 << 20;

inline int check_embed(int64_t n, int64_t vocab, int32_t d, const void* ids, const void* a, const void* b,
                       int64_t a_stride, int64_t b_stride, sdm_rt_dtype dtype) {
  int rc;
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if (n < 0 || vocab < 1 || d < 1) return set_err(SDM_RT_EINVAL, "n must be >= 0, vocab and d >= 1");
  if (n > kEmbedMaxTokens || vocab > kEmbedMaxVocab || d > kEmbedMaxWidth)
    return set_err(SDM_RT_EUNSUPPORTED, "at most 2^27 tokens, a vocabulary of 2^21 and rows of 2^20 values");
  if ((n > 0 && (!ids || !a)) || !b) return set_err(SDM_RT_EINVAL, "a tensor is NULL");
  if (n > 0 && bad_read_stride(a_stride, d)) return set_err(SDM_RT_EINVAL, "a read row stride must be 0 or >= d");
  if (b_stride < d) return set_err(SDM_RT_EINVAL, "the written rows' stride must be >= d");
  return SDM_RT_OK;
}

}  // namespace sdmrt

using namespace sdmrt;

extern "C" {

int sdm_rt_embed_checked(const int64_t* ids, int64_t n, const void* table, int64_t table_row_stride, sdm_rt_dtype dtype,
                         int64_t vocab, int32_t d, float scale, void* out, int64_t out_row_stride, int64_t* outside,
                         void* stream) {
  g_err[0] = 0;
  if (n == 0) return SDM_RT_OK;
  int rc = check_embed(n, vocab, d, ids, table, out, table_row_stride, out_row_stride, dtype);
  if (rc) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int kn = dtype == SDM_RT_BF16 ? 8 : 4;
  const int ppr = (d + kn - 1) / kn;
  const int rows = std::max(1, kEmbedPieces / ppr);
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((n + rows - 1) / rows, 1 << 20));
  const bool through = n * d * (dtype == SDM_RT_BF16 ? 2 : 4) > kStreamBytes;
#define SDM_RT_EMBED(T, THROUGH)                                                                                            \
  hipLaunchKernelGGL((embed_kernel<T, THROUGH>), dim3(blocks), dim3(256), 0, st, ids, n, static_cast<const T*>(table),      \
                     table_row_stride, static_cast<int>(vocab), d, scale, static_cast<T*>(out), out_row_stride, ppr, rows, \
                     outside)
  if (dtype == SDM_RT_BF16) {
    if (through) SDM_RT_EMBED(bf16_t, true);
    else SDM_RT_EMBED(bf16_t, false);
  } else {
    if (through) SDM_RT_EMBED(float, true);
    else SDM_RT_EMBED(float, false);
  }
#undef SDM_RT_EMBED
  return check_launch("embed");
}

int sdm_rt_embed(const int64_t* ids, int64_t n, const void* table, int64_t table_row_stride, sdm_rt_dtype dtype,
                 int64_t vocab, int32_t d, float scale, void* out, int64_t out_row_stride, void* stream) {
  return sdm_rt_embed_checked(ids, n, table, table_row_stride, dtype, vocab, d, scale, out, out_row_stride, nullptr, stream);
}

size_t sdm_rt_embed_backward_workspace_bytes(int64_t n, int64_t vocab, int32_t d) {
  if (n < 0 || vocab < 1 || d < 1 || n > kEmbedMaxTokens || vocab > kEmbedMaxVocab || d > kEmbedMaxWidth) return 0;
  return order_plan(n, vocab, d).total;
}

int sdm_rt_embed_backward(const int64_t* ids, int64_t n, const void* dy, int64_t dy_row_stride, sdm_rt_dtype dtype,
                          int64_t vocab, int32_t d, float scale, int64_t padding_idx, void* d_table,
                          int64_t d_table_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  int rc = check_embed(n, vocab, d, ids, dy, d_table, dy_row_stride, d_table_row_stride, dtype);
  if (rc) return rc;
  const OrderPlan p = order_plan(n, vocab, d);
  if (!workspace) return set_err(SDM_RT_EINVAL, "workspace is NULL");
  if (workspace_bytes < p.total)
    return set_err(SDM_RT_ENOSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, p.total);
  const int slices = (d + 4 * p.lanes - 1) / (4 * p.lanes);
  const int64_t groups = static_cast<int64_t>(p.blocks) * slices + (p.R * kBuckets + 4 * kClearRows - 1) / (4 * kClearRows);
  if (groups >= 1 << 24)
    return set_err(SDM_RT_EUNSUPPORTED, "too many tokens of so wide rows for one launch");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int pad = padding_idx >= 0 && padding_idx < vocab ? static_cast<int>(padding_idx) : -1;
  if (n <= kFewTokens && p.R <= kFewRows && d <= kFewWidth) {
    auto few = [&](auto zero) -> int {
      using T = decltype(zero);
      static const bool lds = allow_lds(reinterpret_cast<const void*>(embed_few_grad_kernel<T>));
      if (!lds) return lds_err("embed_backward");
      hipLaunchKernelGGL((embed_few_grad_kernel<T>), dim3(kBuckets, (d + 255) / 256), dim3(64 * kFewWaves), few_lds(p.R, n), st, ids,
                         static_cast<int>(n), static_cast<int>(vocab), pad, p.R, p.row_bits, static_cast<const T*>(dy),
                         dy_row_stride, scale, static_cast<T*>(d_table), d_table_row_stride, d);
      return check_launch("embed_few_grad");
    };
    return dtype == SDM_RT_BF16 ? few(bf16_t{}) : few(float{});
  }
  static const bool lds = allow_lds(reinterpret_cast<const void*>(embed_order_kernel));
  if (!lds) return lds_err("embed_backward");
  char* ws = static_cast<char*>(workspace);
  int32_t* offsets = reinterpret_cast<int32_t*>(ws);
  int32_t* order = reinterpret_cast<int32_t*>(ws + p.off_order);
  int32_t* row_of = reinterpret_cast<int32_t*>(ws + p.off_row);
  int32_t* bucket_at = reinterpret_cast<int32_t*>(ws + p.off_bucket);
  uint32_t* packed = reinterpret_cast<uint32_t*>(ws + p.off_packed);
  if (p.tiles > 0)
    hipLaunchKernelGGL(embed_tiles_kernel, dim3(p.tiles), dim3(kTile), 0, st, ids, static_cast<int>(n),
                       static_cast<int>(vocab), pad, p.tiles, bucket_at, packed);
  hipLaunchKernelGGL(embed_order_kernel, dim3(kBuckets), dim3(64 * p.waves), static_cast<size_t>(p.waves) * p.R * 4, st,
                     bucket_at, packed, p.tiles, p.R, p.row_bits, offsets, order, row_of);
  if ((rc = check_launch("embed_order"))) return rc;
  RowsGrad a{};
  a.offsets = offsets;
  a.order = order;
  a.row_of = row_of;
  a.part = reinterpret_cast<float*>(ws + p.off_part);
  a.pitch = p.pitch;
  a.n_slots = p.R * kBuckets;
  a.R = p.R;
  a.vocab = static_cast<int>(vocab);
  a.d = d;
  a.len = p.len;
  a.n_tokens = static_cast<int>(n);
  a.edge = reinterpret_cast<int2*>(ws + p.off_edge);
  a.scale = scale;
  a.dy = dy;
  a.dy_stride = dy_row_stride;
  a.d_table = d_table;
  a.dt_stride = d_table_row_stride;
  a.slices = slices;
  a.blocks = p.blocks;
  const dim3 grid(static_cast<unsigned>(groups));
  const dim3 edges(static_cast<unsigned>(std::max(1, p.blocks - 1)));
  const bool through = n * d * (dtype == SDM_RT_BF16 ? 2 : 4) > kStreamBytes;
  auto launch = [&](auto zero, auto lanes) {
    using T = decltype(zero);
    constexpr int LANES = decltype(lanes)::value;
    if (through)
      hipLaunchKernelGGL((embed_rows_grad_kernel<T, LANES, true>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((embed_rows_grad_kernel<T, LANES, false>), grid, dim3(256), 0, st, a);
  };
  auto launch_type = [&](auto zero) {
    using T = decltype(zero);
    if (p.lanes == 16)
      launch(zero, std::integral_constant<int, 16>{});
    else if (p.lanes == 32)
      launch(zero, std::integral_constant<int, 32>{});
    else
      launch(zero, std::integral_constant<int, 64>{});
    if (p.blocks > 1) hipLaunchKernelGGL((embed_rows_join_kernel<T>), edges, dim3(1024), 0, st, a);
  };
  if (dtype == SDM_RT_BF16)
    launch_type(bf16_t{});
  else
    launch_type(float{});
  return check_launch("embed_rows_grad");
}

}  // extern "C"
