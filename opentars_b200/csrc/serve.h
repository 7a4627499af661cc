// Kernel launch interfaces of the serving operators (include/tarscuda_serve.h has their definitions).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/tarscuda_serve.h"

namespace tc {

// tc_kv_cache as the kernels take it.
struct KvCache {
  uint8_t* k;
  uint8_t* v;
  int64_t sp, ss, sh;                // page, slot and head strides in elements
  int n_pages, shift, n_kv, hd;      // page_size = 1 << shift
  int batch, max_pages;
  const int* table;
  int64_t ts;
  int* length;
  float* weight;
  int* pos;
  int64_t track;
  const int* seen;
  int* err;                          // device word for what only the device sees
};

struct AppendArgs {
  KvCache c;
  int dtype;                         // the cache's element type
  const uint8_t* k;
  const uint8_t* v;
  int src;
  int64_t rs, hs;
  const int* cu;
  int tokens;
};
cudaError_t launch_append(const AppendArgs& a, cudaStream_t st);

struct AttendArgs {
  KvCache c;
  int dtype;
  const uint8_t* q;  int64_t qr, qh;
  uint8_t* out;      int64_t orow, oh;
  int nh;
  float scale2;                      // scale * log2(e): scores are kept as powers of two
  int window, sinks;                 // window: INT32_MAX for all
  float* weight_out;
  uint8_t* ws;
  const int* cu;                     // prompt only
  int tokens;
  uint32_t spin;                     // poll limit of the bounded waits
  int block, code;                   // set by the launchers: tokens of an MMA, the error code of bad pages
};
uint64_t attend_workspace(const KvCache& c, int nh, bool weights);
cudaError_t launch_attend(AttendArgs a, cudaStream_t st);
// Chunks of few rows: the tokens of an MMA's block, or 0 where the prompt kernel takes the call.
int chunk_block(const KvCache& c, int nh, int tokens, int window, int sinks);
uint64_t chunk_workspace(const KvCache& c, int nh, int tokens, int window, int sinks);
cudaError_t launch_attend_chunk(AttendArgs a, cudaStream_t st);
cudaError_t launch_attend_prompt(const AttendArgs& a, cudaStream_t st);

struct EvictArgs {
  KvCache c;
  int budget, sinks, recent;
  int* length_out;
  float* weight_out;
  int* pos_out;
  uint8_t* ws;
};
uint64_t evict_workspace(const KvCache& c, int budget);
cudaError_t launch_evict(const EvictArgs& a, cudaStream_t st);

cudaError_t launch_adjust(const tc_logits_rules& r, cudaStream_t st);

}  // namespace tc
