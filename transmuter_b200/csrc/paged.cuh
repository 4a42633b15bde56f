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
// N values of a type in 4, 8 or 16 bytes, as they are loaded and stored.
template <typename T, int N> struct Packed {
  static constexpr int kWords = N * (int)sizeof(T) / 4;
  using Raw = std::conditional_t<kWords == 4, uint4, std::conditional_t<kWords == 2, uint2, uint32_t>>;
  union {
    Raw raw;
    uint32_t w[kWords];
  };
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const Raw*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void get(float (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 v = unpack2<T>(w[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
      else w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
  }
};

// The length of sequence b, 0 (and the device status set) where it cannot be one.
__device__ __forceinline__ int64_t paged_length(const PagedView& c, const int32_t* lengths, int64_t b) {
  const int64_t n = lengths[b];
  if (n >= 0 && n <= c.max_slots) return n;
  report(kDevBadArgument);
  return 0;
}

}  // namespace tq4
