// Attention of the rows of a prompt over the paged cache (tc_attend_prompt), one warp per (row, head).
#include <cuda_runtime.h>

#include "attend_row.cuh"

namespace tc {
namespace {

constexpr int kRowThreads = 128;

template <class T, int HD>
__global__ void __launch_bounds__(kRowThreads) k_prompt_rows(AttendArgs a) {
  const KvCache& c = a.c;
  const int64_t u = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (u >= (int64_t)a.tokens * a.nh) return;
  const int i = (int)(u / a.nh), h = (int)(u - (int64_t)i * a.nh);
  const int b = seq_of(a.cu, c.batch, i);
  if (b < 0) return;
  const int end = kv_length(c, b, kErrPrompt) - (__ldg(a.cu + b + 1) - i) + 1;
  float q[HD / 32], o[HD / 32];
  row_load<T, HD>(a.q, (int64_t)i * a.qr + (int64_t)h * a.qh, lane, q);
  attend_row<T, HD>(c, b, h / (a.nh / c.n_kv), q, a.scale2, max(end, 0), a.window, a.sinks, kErrPrompt, o);
  row_store<T, HD>(a.out, (int64_t)i * a.orow + (int64_t)h * a.oh, lane, o);
}

template <class T>
cudaError_t rows_of(const AttendArgs& a, cudaStream_t st) {
  const int64_t blocks = ((int64_t)a.tokens * a.nh * 32 + kRowThreads - 1) / kRowThreads;
  switch (a.c.hd) {
    case 64: k_prompt_rows<T, 64><<<blocks, kRowThreads, 0, st>>>(a); break;
    case 128: k_prompt_rows<T, 128><<<blocks, kRowThreads, 0, st>>>(a); break;
    default: k_prompt_rows<T, 256><<<blocks, kRowThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attend_prompt(const AttendArgs& a, cudaStream_t st) {
  if (a.tokens == 0) return cudaSuccess;
  return a.dtype == TC_BF16 ? rows_of<__nv_bfloat16>(a, st) : rows_of<__half>(a, st);
}

}  // namespace tc
