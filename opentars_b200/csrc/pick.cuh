// The greedy pick's candidates (np.argmax): NaN first, then the larger value, then the smaller
// index - an order-free rule, so candidates may be combined in any grouping.
#pragma once
#include "fp32.cuh"

namespace tc {

struct Pick {
  float v;
  int i;       // -1: no element yet
  int nan;
};
// elements of one chain arrive in increasing index order, so a tie keeps the earlier one
__device__ __forceinline__ void pick_step(Pick& p, float v, int j) {
  const int vn = is_nan(v);
  const bool take = (p.i < 0) | (vn & !p.nan) | (!p.nan & !vn & (v > p.v));
  p.v = take ? v : p.v;
  p.i = take ? j : p.i;
  p.nan = take ? vn : p.nan;
}
__device__ __forceinline__ Pick pick_comb(Pick a, Pick b) {
  bool take_b;
  if (b.i < 0) take_b = false;
  else if (a.i < 0) take_b = true;
  else if (a.nan != b.nan) take_b = b.nan;
  else if (a.nan) take_b = b.i < a.i;
  else take_b = b.v > a.v || (b.v == a.v && b.i < a.i);
  return take_b ? b : a;
}
__device__ __forceinline__ Pick pick_shfl(Pick p, int o) {
  Pick q;
  q.v = __shfl_xor_sync(0xFFFFFFFFu, p.v, o);
  q.i = __shfl_xor_sync(0xFFFFFFFFu, p.i, o);
  q.nan = __shfl_xor_sync(0xFFFFFFFFu, p.nan, o);
  return q;
}

}  // namespace tc
