// One query row of attention by one warp on the CUDA cores, key by key over the visible slots only.
#pragma once
#include "paged.cuh"

namespace tc {

// 32 lanes hold a row of HD elements, HD / 32 consecutive ones each.
template <class T, int HD>
__device__ __forceinline__ void row_load(const uint8_t* base, int64_t at, int lane, float (&x)[HD / 32]) {
  const T* p = reinterpret_cast<const T*>(base) + at + lane * (HD / 32);
  uint32_t w[HD / 64];
  if constexpr (HD == 64) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (HD == 128) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < HD / 64; ++i) {
    const float2 f = Elem<T>::f2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <class T, int HD>
__device__ __forceinline__ void row_store(uint8_t* base, int64_t at, int lane, const float (&x)[HD / 32]) {
  T* p = reinterpret_cast<T*>(base) + at + lane * (HD / 32);
#pragma unroll
  for (int i = 0; i < HD / 64; ++i) reinterpret_cast<uint32_t*>(p)[i] = Elem<T>::pack(x[2 * i], x[2 * i + 1]);
}

// o = the attention of query q (head g's keys of sequence b) over the visible slots before `end`.
// Statistics and sums in fp32.
template <class T, int HD>
__device__ void attend_row(const KvCache& c, int b, int g, const float (&q)[HD / 32], float scale2, int end, int window,
                           int sinks, int code, float (&o)[HD / 32]) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  float m = __int_as_float(0xFF800000), l = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.0f;
  const int first = first_in_window(end, window), head = min(sinks, first);
  bool any = false;
  for (int j = 0; j < end; ++j) {
    if (j >= head && j < first) j = first;
    const int page = kv_page(c, b, j, code);
    if (page < 0) {
      j |= (1 << c.shift) - 1;
      continue;
    }
    const int64_t at = kv_offset(c, page, j, g);
    float k[E], v[E];
    row_load<T, HD>(c.k, at, lane, k);
    row_load<T, HD>(c.v, at, lane, v);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
    s *= scale2;
    any = true;
    const float m2 = fmaxf(m, s), base = m2 == __int_as_float(0xFF800000) ? 0.0f : m2;
    const float f = exp2f(m - base), p = exp2f(s - base);
    m = m2;
    l = fmaf(l, f, p);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(o[i], f, p * v[i]);
  }
  if (any) {
    const float r = 1.0f / l;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] *= r;
  }
}

}  // namespace tc
