// Attention over the paged cache: one query row per sequence (tc_attend) and the rows of a prompt
// (tc_attend_prompt), one warp per (row, head).
#include <cuda_runtime.h>

#include <algorithm>

#include "attend_row.cuh"
#include "mma.h"

namespace tc {
namespace {

constexpr int kRowThreads = 128;

template <class T, int HD>
__global__ void __launch_bounds__(kRowThreads) k_attend_rows(AttendArgs a, int rows, bool prompt, float* scores, float2* ml) {
  const KvCache& c = a.c;
  const int64_t u = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (u >= (int64_t)rows * a.nh) return;
  const int i = (int)(u / a.nh), h = (int)(u - (int64_t)i * a.nh);
  const int b = prompt ? seq_of(a.cu, c.batch, i) : i;
  if (b < 0) return;
  const int code = prompt ? kErrPrompt : kErrAttend;
  const int len = kv_length(c, b, code), end = prompt ? len - (__ldg(a.cu + b + 1) - i) + 1 : len;
  float q[HD / 32], o[HD / 32];
  row_load<T, HD>(a.q, (int64_t)i * a.qr + (int64_t)h * a.qh, lane, q);
  attend_row<T, HD>(c, b, h / (a.nh / c.n_kv), q, a.scale2, max(end, 0), a.window, a.sinks, code, o,
                    scores ? scores + u * c.track : nullptr, ml ? &ml[u].x : nullptr, ml ? &ml[u].y : nullptr);
  row_store<T, HD>(a.out, (int64_t)i * a.orow + (int64_t)h * a.oh, lane, o);
}

// weight_out = weight + the visible slots' probabilities, summed over the heads that share a key-value head.
constexpr int kWeightThreads = 256;
__global__ void __launch_bounds__(kWeightThreads) k_weights(AttendArgs a, const float* scores, const float2* ml) {
  const KvCache& c = a.c;
  const int row = blockIdx.x, b = row / c.n_kv, g = row - b * c.n_kv, G = a.nh / c.n_kv;
  const int len = kv_length(c, b, kErrAttend), first = first_in_window(len, a.window);
  const int64_t at = (int64_t)row * c.track;
  for (int j = blockIdx.y * kWeightThreads + threadIdx.x; j < len; j += gridDim.y * kWeightThreads) {
    float w = c.weight[at + j];
    if ((j < a.sinks || j >= first) && kv_page(c, b, j, kErrAttend) >= 0) {
      float sum = 0.0f;
      for (int i = 0; i < G; ++i) {
        const int64_t u = (int64_t)b * a.nh + g * G + i;
        const float2 f = ml[u];
        sum += exp2f(scores[u * c.track + j] - f.x) / f.y;
      }
      w += sum;
    }
    a.weight_out[at + j] = w;
  }
}

template <class T>
cudaError_t rows_of(const AttendArgs& a, bool prompt, cudaStream_t st) {
  const int rows = prompt ? a.tokens : a.c.batch;
  const int64_t blocks = ((int64_t)rows * a.nh * 32 + kRowThreads - 1) / kRowThreads;
  float2* ml = nullptr;
  float* scores = nullptr;
  if (a.weight_out) {
    ml = reinterpret_cast<float2*>(a.ws);
    scores = reinterpret_cast<float*>(a.ws + ((int64_t)rows * a.nh * 8 + 255) / 256 * 256);
  }
  switch (a.c.hd) {
    case 64: k_attend_rows<T, 64><<<blocks, kRowThreads, 0, st>>>(a, rows, prompt, scores, ml); break;
    case 128: k_attend_rows<T, 128><<<blocks, kRowThreads, 0, st>>>(a, rows, prompt, scores, ml); break;
    default: k_attend_rows<T, 256><<<blocks, kRowThreads, 0, st>>>(a, rows, prompt, scores, ml); break;
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !a.weight_out) return e;
  const int kvrows = a.c.batch * a.c.n_kv;
  k_weights<<<dim3(kvrows, std::max(1, 148 * 4 / kvrows)), kWeightThreads, 0, st>>>(a, scores, ml);
  return cudaGetLastError();
}

}  // namespace

uint64_t attend_workspace(const KvCache& c, int nh, bool weights) {
  const uint64_t rows = (uint64_t)c.batch * nh;
  return weights ? (rows * 8 + 255) / 256 * 256 + rows * c.track * 4 : 0;
}
cudaError_t launch_attend(const AttendArgs& a, cudaStream_t st) {
  return a.dtype == TC_BF16 ? rows_of<__nv_bfloat16>(a, false, st) : rows_of<__half>(a, false, st);
}
cudaError_t launch_attend_prompt(const AttendArgs& a, cudaStream_t st) {
  if (a.tokens == 0) return cudaSuccess;
  return a.dtype == TC_BF16 ? rows_of<__nv_bfloat16>(a, true, st) : rows_of<__half>(a, true, st);
}

}  // namespace tc
