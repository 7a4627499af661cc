// Device helpers over the paged key-value cache of serve.h.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serve.h"

namespace tc {

enum { kErrAppend = 51, kErrAttend = 52, kErrPrompt = 53, kErrEvict = 54, kErrPromptWait = 55 };

__device__ __forceinline__ void kv_fail(const KvCache& c, int code) { atomicCAS(c.err, 0, code); }

// Sequence b's slots in use; a length beyond the page list counts up to its end.
__device__ __forceinline__ int kv_length(const KvCache& c, int b, int code) {
  const int n = __ldg(c.length + b), cap = c.max_pages << c.shift;
  if (n > cap) {
    kv_fail(c, code);
    return cap;
  }
  return n < 0 ? 0 : n;
}
// The page that holds `slot` of sequence b, or -1 for an id outside the pool. slot >> shift is
// below max_pages.
__device__ __forceinline__ int kv_page(const KvCache& c, int b, int slot, int code) {
  const int p = __ldg(c.table + (int64_t)b * c.ts + (slot >> c.shift));
  if ((unsigned)p >= (unsigned)c.n_pages) {
    kv_fail(c, code);
    return -1;
  }
  return p;
}
// Element offset of head h of `slot`, which lies in `page` (64 bits: a pool may pass 2^32 elements).
__device__ __forceinline__ int64_t kv_offset(const KvCache& c, int page, int slot, int h) {
  return (int64_t)page * c.sp + (int64_t)(slot & ((1 << c.shift) - 1)) * c.ss + (int64_t)h * c.sh;
}
// The sequence that owns row i (cu[b] <= i < cu[b + 1]), or -1 behind the last one. cu NULL: row i.
__device__ __forceinline__ int seq_of(const int* cu, int batch, int i) {
  if (!cu) return i < batch ? i : -1;
  if (i >= __ldg(cu + batch)) return -1;
  int lo = 0, hi = batch;                       // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The visible slots of a row whose last one is end - 1: [0, min(sinks, first)) and [first, end).
__device__ __forceinline__ int first_in_window(int end, int window) { return window < end ? end - window : 0; }

// 2^x to 2 units in the last place (0 below 2^-126).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xFF800000); }

template <class T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float2 f2(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float2 f2(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

}  // namespace tc
