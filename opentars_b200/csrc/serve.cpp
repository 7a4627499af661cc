// The C entry points of the serving operators (include/tarscuda_serve.h): argument checks, then one
// launch function each. Nothing throws and nothing is kept between calls.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>

#include "mma.h"
#include "serve.h"

using namespace tc;

namespace {

constexpr double kLog2e = 1.4426950408889634;
constexpr int64_t kMaxStride = 1ll << 40;

bool al16(const void* p) { return (uintptr_t)p % 16 == 0; }
// A stride in elements of `bytes` each that keeps rows 16-byte aligned.
bool stride_ok(int64_t s, int bytes) { return s >= 0 && s < kMaxStride && s * bytes % 16 == 0; }

// Whether two sets of rows, rows x heads runs of `width` elements with strides of their own, may share an element.
// Exact for two of the same nested strides (interleaved parts of one buffer are apart); with different strides they
// may as soon as their ranges meet. `ahead`: how many elements the second set starts behind the first.
bool may_share(int64_t ahead, int64_t ra, int64_t ha, int64_t rb, int64_t hb, int64_t rows, int64_t heads,
               int64_t width) {
  if (rows == 1) ra = rb = 0;                    // a dimension of one entry is never stepped over
  if (heads == 1) ha = hb = 0;
  const auto reach = [&](int64_t r, int64_t h) { return (double)(rows - 1) * r + (double)(heads - 1) * h + width; };
  if ((double)ahead >= reach(ra, ha) || -(double)ahead >= reach(rb, hb)) return false;
  if (ra != rb || ha != hb) return true;
  const int64_t big = std::max(ra, ha), small = std::min(ra, ha);
  const int64_t nb = ra >= ha ? rows : heads, ns = ra >= ha ? heads : rows;
  if ((nb > 1 && (double)(ns - 1) * small + width > (double)big) || (ns > 1 && small < width)) return true;
  const int64_t d = std::abs(ahead), i0 = big ? d / big : 0;
  for (int64_t i = i0; i <= i0 + (big > 0); ++i) {
    const int64_t left = d - i * big, j0 = small ? std::abs(left) / small : 0;
    if (i >= nb) break;
    for (int64_t j = j0; j <= j0 + (small > 0); ++j)
      if (j < ns && std::abs(left) - j * small < width && j * small - std::abs(left) < width) return true;
  }
  return false;
}
int64_t ahead_of(const void* a, const void* b, int bytes) {
  return ((int64_t)(uintptr_t)b - (int64_t)(uintptr_t)a) / bytes;
}
// An output of n 4-byte elements that may be the array it is computed from, but no shifted part of it.
bool same_or_apart(const void* a, const void* b, int64_t n) {
  const int64_t ahead = ahead_of(a, b, 4);
  return a == b || ahead >= n || -ahead >= n;
}

// Whether a pool's rows of head_dim elements lie apart, its dimensions nested in any order (a stride of 0 or
// one that steps into the next row has rows share memory; a dimension of one entry is never stepped over).
bool pool_apart(const tc_kv_cache* c) {
  int64_t stride[3] = {c->page_stride, c->slot_stride, c->head_stride}, n[3] = {c->n_pages, c->page_size, c->n_kv};
  int64_t width = c->head_dim;                   // elements from the first to behind the last of the dimensions so far
  for (int left = 3; left > 0; --left) {
    int at = 0;
    for (int i = 1; i < left; ++i)
      if (stride[i] < stride[at]) at = i;
    if (n[at] > 1) {
      if (stride[at] < width) return false;
      width = std::min(kMaxStride, stride[at] > kMaxStride / n[at] ? kMaxStride : (n[at] - 1) * stride[at] + width);
    }
    stride[at] = stride[left - 1];
    n[at] = n[left - 1];
  }
  return true;
}

// Entries of a cache's weight and pos.
int64_t tracked(const tc_kv_cache* c) { return (int64_t)c->batch * c->n_kv * c->track_stride; }

// Everything of a cache that the host can check.
bool take_cache(const tc_kv_cache* c, KvCache* o) {
  if (!c || !c->k || !c->v || !c->table || !c->length) return false;
  if (c->dtype != TC_BF16 && c->dtype != TC_FP16) return false;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return false;
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page_size) ++shift;
  if ((1 << shift) != c->page_size) return false;
  if (c->n_pages < 1 || c->n_kv < 1 || c->n_kv > 1024 || c->batch < 1 || c->batch > (1 << 20)) return false;
  if (c->max_pages < 1 || c->max_pages > (INT_MAX >> 1 >> shift) || c->table_stride < c->max_pages) return false;
  if (!al16(c->k) || !al16(c->v)) return false;
  if (!stride_ok(c->page_stride, 2) || !stride_ok(c->slot_stride, 2) || !stride_ok(c->head_stride, 2)) return false;
  if (!pool_apart(c)) return false;
  const bool any = c->weight || c->pos || c->seen, all = c->weight && c->pos && c->seen;
  if (any && (!all || c->track_stride < (int64_t)c->max_pages << shift)) return false;
  o->k = static_cast<uint8_t*>(c->k);
  o->v = static_cast<uint8_t*>(c->v);
  o->sp = c->page_stride; o->ss = c->slot_stride; o->sh = c->head_stride;
  o->n_pages = c->n_pages; o->shift = shift; o->n_kv = c->n_kv; o->hd = c->head_dim;
  o->batch = c->batch; o->max_pages = c->max_pages;
  o->table = c->table; o->ts = c->table_stride; o->length = c->length;
  o->weight = c->weight; o->pos = c->pos; o->track = c->track_stride; o->seen = c->seen;
  o->err = nullptr;
  return true;
}

// The error word belongs to the current device: looked up after every check has passed.
bool take_error(KvCache* c) { return (c->err = wait_error_flag()) != nullptr; }

bool take_attend(const tc_kv_cache* c, const void* q, int64_t qr, int64_t qh, void* out, int64_t orow, int64_t oh,
                 int32_t nh, float scale, int32_t window, int32_t sinks, int64_t rows, AttendArgs* a) {
  if (!take_cache(c, &a->c) || !q || !out || !al16(q) || !al16(out)) return false;
  if (!stride_ok(qr, 2) || !stride_ok(qh, 2) || !stride_ok(orow, 2) || !stride_ok(oh, 2)) return false;
  if (nh < 1 || nh % c->n_kv || nh > (1 << 16) || window < 0 || sinks < 0 || !std::isfinite(scale)) return false;
  // (a row is read again after its output is stored where that is not finite)
  if (may_share(ahead_of(q, out, 2), qr, qh, orow, oh, rows, nh, c->head_dim)) return false;
  a->dtype = c->dtype;
  a->q = static_cast<const uint8_t*>(q); a->qr = qr; a->qh = qh;
  a->out = static_cast<uint8_t*>(out); a->orow = orow; a->oh = oh;
  a->nh = nh;
  a->scale2 = (float)(scale * kLog2e);
  a->window = window ? window : INT_MAX;
  a->sinks = sinks;
  a->weight_out = nullptr; a->ws = nullptr; a->cu = nullptr; a->tokens = 0;
  a->spin = spin_limit();
  return true;
}

int done(cudaError_t e) { return e == cudaSuccess ? TC_OK : TC_ERR_CUDA; }

}  // namespace

extern "C" {

int tc_kv_append(const tc_kv_cache* c, const void* k, const void* v, int32_t src, int64_t row_stride,
                 int64_t head_stride, const int32_t* cu, int32_t tokens, void* stream) {
  AppendArgs a{};
  if (!take_cache(c, &a.c) || tokens < 0 || (src != TC_FP32 && src != TC_BF16 && src != TC_FP16)) return TC_ERR_ARG;
  if (tokens == 0) return TC_OK;
  const int bytes = src == TC_FP32 ? 4 : 2;
  if (!k || !v || !al16(k) || !al16(v) || !stride_ok(row_stride, bytes) || !stride_ok(head_stride, bytes))
    return TC_ERR_ARG;
  if (!cu && tokens > c->batch) return TC_ERR_ARG;
  a.dtype = c->dtype;
  a.k = static_cast<const uint8_t*>(k); a.v = static_cast<const uint8_t*>(v);
  a.src = src; a.rs = row_stride; a.hs = head_stride; a.cu = cu; a.tokens = tokens;
  if (!take_error(&a.c)) return TC_ERR_CUDA;
  return done(launch_append(a, static_cast<cudaStream_t>(stream)));
}

uint64_t tc_attend_workspace(const tc_kv_cache* c, int32_t n_heads, int32_t weights) {
  KvCache o{};
  if (!take_cache(c, &o) || n_heads < 1 || n_heads % c->n_kv || n_heads > (1 << 16)) return 0;
  return attend_workspace(o, n_heads, weights != 0);
}

int tc_attend(const tc_kv_cache* c, const void* q, int64_t q_row_stride, int64_t q_head_stride, void* out,
              int64_t out_row_stride, int64_t out_head_stride, int32_t n_heads, float scale, int32_t window,
              int32_t sinks, float* weight_out, void* ws, uint64_t ws_bytes, void* stream) {
  AttendArgs a{};
  if (!take_attend(c, q, q_row_stride, q_head_stride, out, out_row_stride, out_head_stride, n_heads, scale, window,
                   sinks, c ? c->batch : 1, &a))
    return TC_ERR_ARG;
  if (weight_out && (!c->weight || !same_or_apart(c->weight, weight_out, tracked(c)))) return TC_ERR_ARG;
  const uint64_t need = attend_workspace(a.c, n_heads, weight_out != nullptr);
  if (need && (!ws || (uintptr_t)ws % 256 || ws_bytes < need)) return TC_ERR_ARG;
  a.weight_out = weight_out;
  a.ws = static_cast<uint8_t*>(ws);
  if (!take_error(&a.c)) return TC_ERR_CUDA;
  return done(launch_attend(a, static_cast<cudaStream_t>(stream)));
}

int tc_attend_prompt(const tc_kv_cache* c, const void* q, int64_t q_row_stride, int64_t q_head_stride, void* out,
                     int64_t out_row_stride, int64_t out_head_stride, int32_t n_heads, const int32_t* cu,
                     int32_t tokens, float scale, int32_t window, int32_t sinks, void* ws, uint64_t ws_bytes,
                     void* stream) {
  AttendArgs a{};
  if (tokens < 0 || tokens > (1 << 28) || !cu) return TC_ERR_ARG;
  if (tokens == 0) return take_cache(c, &a.c) ? TC_OK : TC_ERR_ARG;
  if (!take_attend(c, q, q_row_stride, q_head_stride, out, out_row_stride, out_head_stride, n_heads, scale, window,
                   sinks, tokens, &a))
    return TC_ERR_ARG;
  const uint64_t need = chunk_workspace(a.c, n_heads, tokens, a.window, a.sinks);
  if (need && (!ws || (uintptr_t)ws % 256 || ws_bytes < need)) return TC_ERR_ARG;
  a.cu = cu;
  a.tokens = tokens;
  a.ws = static_cast<uint8_t*>(ws);
  if (!take_error(&a.c)) return TC_ERR_CUDA;
  return done(need ? launch_attend_chunk(a, static_cast<cudaStream_t>(stream))
                   : launch_attend_prompt(a, static_cast<cudaStream_t>(stream)));
}

uint64_t tc_attend_prompt_workspace(const tc_kv_cache* c, int32_t n_heads, int32_t tokens, int32_t window,
                                    int32_t sinks) {
  KvCache o{};
  if (!take_cache(c, &o) || n_heads < 1 || n_heads % c->n_kv || n_heads > (1 << 16) || tokens < 1 ||
      tokens > (1 << 28) || window < 0 || sinks < 0)
    return 0;
  return chunk_workspace(o, n_heads, tokens, window ? window : INT_MAX, sinks);
}

uint64_t tc_kv_evict_workspace(const tc_kv_cache* c, int32_t budget) {
  KvCache o{};
  if (!take_cache(c, &o) || budget < 1) return 0;
  return evict_workspace(o, budget);
}

int tc_kv_evict(const tc_kv_cache* c, int32_t budget, int32_t sinks, int32_t recent, int32_t* length_out,
                float* weight_out, int32_t* pos_out, void* ws, uint64_t ws_bytes, void* stream) {
  EvictArgs a{};
  if (!take_cache(c, &a.c) || !c->weight || budget < 1 || sinks < 0 || recent < 0 ||
      (int64_t)sinks + recent > budget || !length_out || !weight_out || !pos_out)
    return TC_ERR_ARG;
  if (!same_or_apart(c->weight, weight_out, tracked(c)) || !same_or_apart(c->pos, pos_out, tracked(c)) ||
      !same_or_apart(c->length, length_out, c->batch))
    return TC_ERR_ARG;
  if (!ws || (uintptr_t)ws % 256 || ws_bytes < evict_workspace(a.c, budget)) return TC_ERR_ARG;
  a.budget = budget; a.sinks = sinks; a.recent = recent;
  a.length_out = length_out; a.weight_out = weight_out; a.pos_out = pos_out;
  a.ws = static_cast<uint8_t*>(ws);
  if (!take_error(&a.c)) return TC_ERR_CUDA;
  return done(launch_evict(a, static_cast<cudaStream_t>(stream)));
}

int tc_adjust_logits(const tc_logits_rules* r, void* stream) {
  if (!r || !r->logits || !r->out || r->rows < 1 || r->rows > (1 << 24) || r->vocab < 1 || r->vocab > (1 << 28) ||
      r->logits_stride < r->vocab || r->out_stride < r->vocab)
    return TC_ERR_ARG;
  tc_logits_rules a = *r;
  if ((a.logits != a.out || (a.rows > 1 && a.logits_stride != a.out_stride)) &&
      may_share(ahead_of(a.logits, a.out, 4), a.logits_stride, 0, a.out_stride, 0, a.rows, 1, a.vocab))
    return TC_ERR_ARG;
  if (a.history) {
    if (a.max_history < 0 || a.max_history >= (1 << 20) || a.history_stride < a.max_history) return TC_ERR_ARG;
  } else if (a.n_history || a.n_prompt || a.repetition || a.presence || a.frequency) {
    return TC_ERR_ARG;
  }
  if (!a.bias != !a.bias_ids) return TC_ERR_ARG;
  if (a.bias && (a.n_bias < 0 || a.n_bias > 2047 || a.bias_stride < a.n_bias)) return TC_ERR_ARG;
  if (a.mask && (a.mask_stride < 0 || (a.mask_stride && a.mask_stride < (a.vocab + 31) / 32))) return TC_ERR_ARG;
  return done(launch_adjust(a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
