/* libtarscuda serving operators: a paged key-value cache, the attention that reads it, a bound on
 * its size, and rules on logits before the greedy pick. They serve conversations longer than the
 * decode engine's dense fp32 cache (tarscuda_engine.h) holds, in bf16 or fp16, for any model with
 * grouped-query attention; the reference has no counterpart (its attention reads one dense cache
 * of max_tokens positions, llm.py:735-746, and its pick is np.argmax, llm.py:834).
 *
 * Every pointer is a device pointer of the current device; work is enqueued on `stream` (a
 * cudaStream_t, NULL: the default stream) and can be captured into a CUDA graph. Calls keep
 * nothing: what one needs beyond its outputs is in the workspace it is given, which calls that
 * may overlap must not share. Return values: TC_OK, TC_ERR_ARG (before anything is enqueued), or
 * TC_ERR_CUDA. What only the device can see is checked there, and the first code found stays in
 * the word that tc_wait_error reads: 51 append, 52 attend, 53 attend_prompt, 54 evict - a page id
 * outside the pool or a length beyond the page list. A key on such a page is left out of the
 * attention, a row for it is not written, a length counts up to the page list's end. 55
 * (attend_prompt) is a bounded wait that gave up, as tc_wait_error describes.
 */
#ifndef TARSCUDA_SERVE_H
#define TARSCUDA_SERVE_H
#include <stdint.h>

#include "tarscuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types: the contract's output format codes (contract.py EPI OUT field). */
#define TC_FP32 0
#define TC_BF16 1
#define TC_FP16 3

/* A paged key-value cache of `batch` sequences. Slot s of sequence b is row s % page_size of page
 * table[b * table_stride + s / page_size] of both pools; key-value head h of a row is `head_dim`
 * contiguous elements at page * page_stride + row * slot_stride + h * head_stride (elements; bases
 * and strides 16-byte aligned, the three dimensions nested in any order so that no two rows share
 * memory; the stride of a dimension of one entry is not used). length[b] slots are in use. Entries
 * of the page list behind the used slots, and rows of a page behind them, may hold anything: they
 * never reach a result. */
typedef struct {
  void* k;
  void* v;
  int64_t page_stride, slot_stride, head_stride;
  int32_t n_pages, page_size;   /* page_size: 16, 32, 64, 128 or 256 */
  int32_t n_kv, head_dim;       /* head_dim: 64, 128 or 256 */
  int32_t dtype;                /* TC_BF16 or TC_FP16 */
  int32_t batch, max_pages;
  const int32_t* table;
  int64_t table_stride;
  int32_t* length;              /* [batch] */
  /* What eviction needs (all NULL without it): the attention weight each slot has drawn and the
   * position its token had, per sequence and head at (b * n_kv + h) * track_stride + slot, and the
   * number of tokens each sequence has taken in all. */
  float* weight;
  int32_t* pos;
  int64_t track_stride;
  const int32_t* seen;          /* [batch] */
} tc_kv_cache;

/* The new tokens' key and value rows into the cache, rounded to its type (to nearest, ties to even).
 * Rows are [tokens][n_kv][head_dim] of type src (TC_FP32, TC_BF16 or TC_FP16, k and v with the same
 * strides in elements, 16-byte aligned); sequence b owns rows cu[b] .. cu[b+1] - 1 (cu: batch + 1
 * ascending row numbers from 0; NULL: one row per sequence, row b), and length[b] and seen[b] count
 * them already: row i of n lands in slot length[b] - n + i. Rows at and behind cu[batch], and rows
 * whose slot would be negative, are ignored. With tracking their weight is set to 0 and their
 * position to seen[b] - n + i. */
int tc_kv_append(const tc_kv_cache* c, const void* k, const void* v, int32_t src, int64_t row_stride,
                 int64_t head_stride, const int32_t* cu, int32_t tokens, void* stream);

/* Attention of one query row per sequence over its cache: out[b][h] = sum_j p_j v_j with
 * p = softmax over the visible slots j of scale * q[b][h] . k_j; head h reads key-value head
 * h / (n_heads / n_kv). Slot j of length[b] = L is visible if j >= L - window or j < sinks (window 0:
 * all). A sequence of length 0 gets zeros. q and out have the cache's type, rows [batch][n_heads]
 * [head_dim] with strides in elements, 16-byte aligned, and share no memory. With weight_out (laid
 * out as the cache's weight, which may be it, but no shifted part of it) weight_out[b][g][j] =
 * weight[b][g][j] + the p_j of the heads of key-value head g, for j < L; slots behind are left alone.
 * ws: tc_attend_workspace bytes, 256-byte aligned; with weights they hold a score for every sequence,
 * head and slot that the page lists have room for (batch * n_heads * max_pages * page_size * 4
 * bytes), whatever the lengths. */
int tc_attend(const tc_kv_cache* c, const void* q, int64_t q_row_stride, int64_t q_head_stride, void* out,
              int64_t out_row_stride, int64_t out_head_stride, int32_t n_heads, float scale, int32_t window,
              int32_t sinks, float* weight_out, void* ws, uint64_t ws_bytes, void* stream);
uint64_t tc_attend_workspace(const tc_kv_cache* c, int32_t n_heads, int32_t weights);

/* Attention of the tokens of a prompt, or of a chunk of one, whose key and value rows are in the
 * cache already: rows cu[b] .. cu[b+1] - 1 of q are the last tokens of sequence b, row i of n at
 * position p = length[b] - n + i. It sees slot j if j <= p and (p - j < window or j < sinks; window
 * 0: all). Rows at a negative position get zeros; rows at and behind cu[batch] are left alone. q and out
 * share no memory.
 * ws: tc_attend_prompt_workspace bytes, 256-byte aligned (0 bytes, and NULL, for calls of many
 * rows). */
int tc_attend_prompt(const tc_kv_cache* c, const void* q, int64_t q_row_stride, int64_t q_head_stride, void* out,
                     int64_t out_row_stride, int64_t out_head_stride, int32_t n_heads, const int32_t* cu,
                     int32_t tokens, float scale, int32_t window, int32_t sinks, void* ws, uint64_t ws_bytes,
                     void* stream);
uint64_t tc_attend_prompt_workspace(const tc_kv_cache* c, int32_t n_heads, int32_t tokens, int32_t window, int32_t sinks);

/* Cuts every sequence longer than `budget` slots to budget, separately for each key-value head. The
 * slots whose position is below `sinks` or at least seen[b] - recent stay first (sinks + recent <=
 * budget), then those with the largest weight (a NaN before all numbers, ties to the lowest slot).
 * The slots that stay but lie at or behind budget move, in ascending order, into the evicted slots
 * before it, in ascending order: every other slot stays where it is, nothing is read that was
 * written, and attention without a window is unchanged but for what was evicted. Afterwards
 * length_out[b] = min(length[b], budget), and weight_out and pos_out hold the slots' weights and
 * positions (each may be the cache's own array, but no shifted part of it; otherwise all slots before
 * length_out[b] are written). Pages of such a sequence must not be shared with another one.
 * ws: tc_kv_evict_workspace bytes, 256-byte aligned. */
int tc_kv_evict(const tc_kv_cache* c, int32_t budget, int32_t sinks, int32_t recent, int32_t* length_out,
                float* weight_out, int32_t* pos_out, void* ws, uint64_t ws_bytes, void* stream);
uint64_t tc_kv_evict_workspace(const tc_kv_cache* c, int32_t budget);

/* Rules on rows of fp32 logits, then the greedy pick. Every pointer but logits and out may be NULL
 * (the rule is then left out; penalties need the history, and presence and frequency count its
 * tokens from n_prompt on). In this order, each step rounded to fp32:
 *   a token of the history   x = x > 0 ? x / repetition : x * repetition
 *   c > 0 generated times    x = x - frequency * c, then x = x - presence
 *   a listed token           x = x + bias (the last entry, where a token is listed twice)
 *   a token not allowed      x = -infinity  (bit t % 32 of mask word t / 32 clear)
 * token[r] is the first NaN, else the first largest value, among the allowed tokens (np.argmax's
 * order); `none` when the mask allows no token. Ids outside the vocabulary are ignored. */
typedef struct {
  const float* logits;          /* [rows][vocab], rows logits_stride elements apart */
  float* out;                   /* the same logits, or rows that share no memory with them */
  int64_t logits_stride, out_stride;
  int32_t rows, vocab;
  const int32_t* history;       /* [rows][max_history] token ids: the prompt's, then the generated ones */
  int64_t history_stride;
  int32_t max_history;          /* at most 2^20 - 1 */
  const int32_t* n_history;     /* [rows] ids in use (NULL: max_history) */
  const int32_t* n_prompt;      /* [rows] of them the prompt's (NULL: 0) */
  const float* repetition;      /* [rows] */
  const float* presence;        /* [rows] */
  const float* frequency;       /* [rows] */
  const int32_t* bias_ids;      /* [rows][n_bias] */
  const float* bias;            /* [rows][n_bias] */
  int64_t bias_stride;
  int32_t n_bias;               /* at most 2047 */
  const uint32_t* mask;         /* [rows][(vocab + 31) / 32] */
  int64_t mask_stride;          /* 0: one mask for all rows */
  int32_t* token;               /* [rows] */
  int32_t none;
} tc_logits_rules;
int tc_adjust_logits(const tc_logits_rules* r, void* stream);

#ifdef __cplusplus
}
#endif
#endif
