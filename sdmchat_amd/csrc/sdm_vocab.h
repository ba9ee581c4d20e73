// sdm_vocab.h -- what the operators on token ids and vocabulary rows share (sdm_embed.hip, sdm_distill.hip,
// sdm_rules.hip): 16-byte pieces of a row at any element alignment, and the sums and maxima of a workgroup.
#pragma once
#include "sdm_common.h"

namespace sdmrt {

// 8 and 16 bytes at any element's address, for loads and stores that leave the caches to others (nontemporal)
typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));

// What passes once through a kernel and is larger than this does not stay in the 256 MB last-level cache until its next
// reader anyway: then it should not drive out what the kernel reads again.
constexpr int64_t kStreamBytes = int64_t{128} << 20;

// 16 bytes of a row: kN values of T.  A row of an odd vocabulary starts at any multiple of its element's size; gfx950
// loads and stores 16 bytes at any address, so full pieces take the same instruction wherever the row starts, and only
// a row's last, partial piece goes value by value.
template <typename T>
struct Piece {
  static constexpr int kN = 16 / static_cast<int>(sizeof(T));
  uint4 r;

  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&r, p, 16); }
  // the first n (< kN) values at p, the rest `fill`
  __device__ __forceinline__ void load_part(const T* p, int n, T fill) {
    T v[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      v[e] = fill;
      if (e < n) v[e] = p[e];
    }
    __builtin_memcpy(&r, v, 16);
  }
  // makes the compiler forget what it knows of the bits: values unpacked before are unpacked again after, instead of
  // staying in twice the registers of the piece
  __device__ __forceinline__ void forget() {
    if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w));
  }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, &r, 16); }
  __device__ __forceinline__ void store_through(T* p) const {
    const words4 w = {r.x, r.y, r.z, r.w};
    __builtin_nontemporal_store(w, reinterpret_cast<words4*>(p));
  }
  __device__ __forceinline__ void store_part(T* p, int n) const {
    T v[kN];
    __builtin_memcpy(v, &r, 16);
#pragma unroll
    for (int e = 0; e < kN; ++e)
      if (e < n) p[e] = v[e];
  }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if constexpr (sizeof(T) == 2)
      return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    else
      return __uint_as_float(w[e]);
  }
  __device__ __forceinline__ void fill(float x) {
    float v[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) v[e] = x;
    set(v);
  }
  // kN floats, each rounded once to T
  __device__ __forceinline__ void set(const float (&v)[kN]) {
    if constexpr (sizeof(T) == 2)
      r = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    else
      r = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

// rows that are only read may also be one row repeated (stride 0)
inline bool bad_read_stride(int64_t stride, int64_t width) { return stride != 0 && stride < width; }

// The row of a [vocab] table that a token id stands for: ids outside are clamped into it (the host reads none).
__device__ __forceinline__ int clamp_token(int64_t id, int vocab) {
  return static_cast<int>(min(max(id, int64_t{0}), static_cast<int64_t>(vocab) - 1));
}

// the maximum and the sum over a wave's 64 lanes, in every lane, by DPP: swap neighbours, swap pairs, mirror the halves and
// the rows of 16, then the last lane of rows 0 and 2 into rows 1 and 3, and lane 31 into rows 2 and 3
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_rows(int old, int v) {
  return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ float wave_max(float v) {
  auto step = [](float x, int y) { return fmaxf(x, __int_as_float(y)); };
  v = step(v, dpp_rows<0xb1, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x4e, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x141, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x140, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x142, 0xa>(__float_as_int(v), __float_as_int(v)));
  v = step(v, dpp_rows<0x143, 0xc>(__float_as_int(v), __float_as_int(v)));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_add(float v) {
  auto step = [](float x, int y) { return x + __int_as_float(y); };
  v = step(v, dpp_rows<0xb1, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x4e, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x141, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x140, 0xf>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x142, 0xa>(0, __float_as_int(v)));
  v = step(v, dpp_rows<0x143, 0xc>(0, __float_as_int(v)));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ int wave_add(int v) {
  v += dpp_rows<0xb1, 0xf>(0, v);
  v += dpp_rows<0x4e, 0xf>(0, v);
  v += dpp_rows<0x141, 0xf>(0, v);
  v += dpp_rows<0x140, 0xf>(0, v);
  v += dpp_rows<0x142, 0xa>(0, v);
  v += dpp_rows<0x143, 0xc>(0, v);
  return __builtin_amdgcn_readlane(v, 63);
}

}  // namespace sdmrt
