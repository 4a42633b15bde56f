// The paged key-value cache's handle and what its kernels share (include/tq4_paged.h).
#pragma once

#include "../../include/tq4_paged.h"
#include "internal.cuh"

// Memory stays the caller's: the handle only describes it.
struct tq4_paged {
  tq4_paged_desc desc{};
  int device = 0;
  int page_log2 = 0;
  void* k_pages = nullptr;
  void* v_pages = nullptr;
  const int32_t* page_table = nullptr;
};

namespace tq4 {

// The pool as a kernel sees it.
struct PagedView {
  const int32_t* table;  // [max_seqs][max_pages]
  int64_t num_pages;
  int64_t max_slots;  // max_pages << page_log2
  int32_t max_seqs, max_pages;
  int32_t kv_heads, head_dim, page_log2;

  // Element offset of row (page, kv_head, row-in-page); 64 bits, since a pool passes 2^31 values.
  __device__ __forceinline__ int64_t row_offset(int page, int kv_head, int in_page) const {
    return ((((int64_t)page * kv_heads + kv_head) << page_log2) + in_page) * head_dim;
  }
  __device__ __forceinline__ bool page_ok(int page) const { return page >= 0 && page < num_pages; }
};

inline PagedView view_of(const tq4_paged& c) {
  PagedView v;
  v.table = c.page_table;
  v.num_pages = c.desc.num_pages;
  v.max_slots = (int64_t)c.desc.max_pages << c.page_log2;
  v.max_seqs = c.desc.max_seqs;
  v.max_pages = c.desc.max_pages;
  v.kv_heads = c.desc.kv_heads;
  v.head_dim = c.desc.head_dim;
  v.page_log2 = c.page_log2;
  return v;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether [a, a + a_bytes) and [b, b + b_bytes) share a byte.
inline bool overlaps(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + (uint64_t)b_bytes && y < x + (uint64_t)a_bytes;
}

// Two values rounded to 16 bits in a word, and back.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t x);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
// The values of a 16-byte chunk, and back.
template <typename T> __device__ __forceinline__ void unpack16(const uint4& x, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else {
      const float2 v = unpack2<T>(w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// The length of sequence b, 0 (and the device status set) where it cannot be one.
__device__ __forceinline__ int64_t paged_length(const PagedView& c, const int32_t* lengths, int64_t b) {
  const int64_t n = lengths[b];
  if (n >= 0 && n <= c.max_slots) return n;
  report(kDevBadArgument);
  return 0;
}

}  // namespace tq4
