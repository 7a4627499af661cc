// The serving operators that move and rank: appending rows to the paged cache, evicting slots by
// accumulated attention weight, and the rules on logits with the greedy pick.
#include <cuda_runtime.h>

#include <algorithm>

#include "fp32.cuh"
#include "mma.h"
#include "paged.cuh"
#include "pdl.cuh"
#include "pick.cuh"
#include "umma.cuh"

namespace tc {
namespace {

// ----------------------------------------------------------------------------------- append
// One thread rounds 8 consecutive elements of a key row and of its value row: 16-byte stores, a
// row's threads side by side. Bound by the launch and one trip to memory and back: a step's 64 rows and four
// prompts of up to 2048 rows of 256 (10.5 MB, 1.6 us at the copy rate) both take 3.4 us.
constexpr int kAppendThreads = 256;

template <class S>
__device__ __forceinline__ void load8(const uint8_t* p, int64_t at, float (&x)[8]) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const S*>(p) + at));
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<S>::f2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const uint8_t* p, int64_t at, float (&x)[8]) {
  const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
  const float4 a = __ldg(s), b = __ldg(s + 1);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

template <class S, class T>
__global__ void __launch_bounds__(kAppendThreads) k_append(AppendArgs a) {
  const KvCache& c = a.c;
  const int per_head = c.hd / 8, per_row = c.n_kv * per_head;
  const int64_t all = (int64_t)a.tokens * per_row;
  for (int64_t u = (int64_t)blockIdx.x * kAppendThreads + threadIdx.x; u < all;
       u += (int64_t)gridDim.x * kAppendThreads) {
    const int i = (int)(u / per_row), r = (int)(u - (int64_t)i * per_row);
    const int h = r / per_head, e = (r - h * per_head) * 8;
    const int b = seq_of(a.cu, c.batch, i);
    if (b < 0) continue;
    const int back = a.cu ? __ldg(a.cu + b + 1) - i : 1;          // rows from this one to the sequence's end
    const int len = __ldg(c.length + b), slot = len - back;
    if (slot < 0) continue;
    if ((slot >> c.shift) >= c.max_pages) {
      kv_fail(c, kErrAppend);
      continue;
    }
    const int page = kv_page(c, b, slot, kErrAppend);
    if (page >= 0) {
      float k[8], v[8];
      load8<S>(a.k, (int64_t)i * a.rs + (int64_t)h * a.hs + e, k);
      load8<S>(a.v, (int64_t)i * a.rs + (int64_t)h * a.hs + e, v);
      const int64_t at = kv_offset(c, page, slot, h) + e;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(c.k) + at) =
          make_uint4(Elem<T>::pack(k[0], k[1]), Elem<T>::pack(k[2], k[3]), Elem<T>::pack(k[4], k[5]),
                     Elem<T>::pack(k[6], k[7]));
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(c.v) + at) =
          make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]),
                     Elem<T>::pack(v[6], v[7]));
    }
    if (c.weight && e == 0) {
      const int64_t t = ((int64_t)b * c.n_kv + h) * c.track + slot;
      c.weight[t] = 0.0f;
      c.pos[t] = __ldg(c.seen + b) - back;
    }
  }
}

template <class T>
cudaError_t append_to(const AppendArgs& a, cudaStream_t st) {
  const int64_t all = (int64_t)a.tokens * a.c.n_kv * (a.c.hd / 8);
  const int grid = (int)std::min<int64_t>((all + kAppendThreads - 1) / kAppendThreads, 148 * 8);
  switch (a.src) {
    case TC_FP32: k_append<float, T><<<grid, kAppendThreads, 0, st>>>(a); break;
    case TC_BF16: k_append<__nv_bfloat16, T><<<grid, kAppendThreads, 0, st>>>(a); break;
    default: k_append<__half, T><<<grid, kAppendThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------ evict
// One CTA ranks the slots of one (sequence, key-value head). A slot's rank key is a 32-bit number
// (protected slots highest, then a NaN weight, then the weight's bits made monotonic), computed once
// and kept in shared memory while it fits there. The budget-th largest key is found digit by digit
// from the top (11, 11 and 10 bits, counted in shared memory), and of the slots with that key as many
// stay as are needed, from the lowest slot on. Threads own contiguous runs of slots, so the lists of
// leaving and arriving slots come out in ascending order from one scan over the threads.
// A few rows are moved at once (a cache one slot over its budget moves one); more of them in a second
// kernel over the lists. Bound by the chain of block-wide steps (some 0.5 us each with 1024 threads): 16 x 8
// heads one slot over a budget of 1024, 10 us with the second launch; the rows' move by memory: six sequences
// of up to 8192 slots cut to 2048, 27 us: 13 us of ranking on 32 CTAs, then as long for moving 75 MB.
constexpr int kRankThreads = 1024, kRankWarps = kRankThreads / 32, kBins = 2048, kKeysMax = 49152, kFewMoves = 32;

__device__ __forceinline__ uint32_t rank_key(float w, int pos, int sinks, int64_t recent_from) {
  if (pos < sinks || pos >= recent_from) return 0xFFFFFFFFu;
  const uint32_t u = fb(w + 0.0f);                               // -0 ranks as 0
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFEu;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// One entry per evicted slot that a kept one fills.
struct Moves {
  int* n;              // [batch * n_kv]
  int2* at;            // [batch * n_kv][most]: source slot, destination slot
  int most;
};
__host__ __device__ inline Moves moves_of(uint8_t* ws, int rows, int most) {
  return Moves{reinterpret_cast<int*>(ws), reinterpret_cast<int2*>(ws + ((int64_t)rows * 4 + 255) / 256 * 256), most};
}
__host__ __device__ inline int most_moves(int capacity, int budget) {
  return capacity <= budget ? 0 : (budget < capacity - budget ? budget : capacity - budget);
}

// Exclusive sums over the threads of the CTA of (x, y), and the totals. s_warp is not reused before a barrier.
__device__ __forceinline__ int2 threads_before(int x, int y, int2* s_warp, int2* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int2 sum = make_int2(x, y);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, sum.x, o), v = __shfl_up_sync(0xFFFFFFFFu, sum.y, o);
    if (lane >= o) {
      sum.x += u;
      sum.y += v;
    }
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  int2 w = s_warp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xFFFFFFFFu, w.x, o), v = __shfl_up_sync(0xFFFFFFFFu, w.y, o);
    if (lane >= o) {
      w.x += u;
      w.y += v;
    }
  }
  *all = make_int2(__shfl_sync(0xFFFFFFFFu, w.x, 31), __shfl_sync(0xFFFFFFFFu, w.y, 31));
  const int bx = __shfl_sync(0xFFFFFFFFu, w.x, (warp + 31) & 31), by = __shfl_sync(0xFFFFFFFFu, w.y, (warp + 31) & 31);
  return make_int2((warp ? bx : 0) + sum.x - x, (warp ? by : 0) + sum.y - y);
}

// One 16-byte piece of a moved row, keys and values. Sources lie at or behind the budget, destinations before it.
__device__ __forceinline__ void move_piece(const KvCache& c, int b, int h, int2 m, int e) {
  const int ps = kv_page(c, b, m.x, kErrEvict), pd = kv_page(c, b, m.y, kErrEvict);
  if (ps < 0 || pd < 0) return;
  const int64_t s = kv_offset(c, ps, m.x, h) + e, d = kv_offset(c, pd, m.y, h) + e;
  const uint4 k = *reinterpret_cast<const uint4*>(c.k + 2 * s), v = *reinterpret_cast<const uint4*>(c.v + 2 * s);
  *reinterpret_cast<uint4*>(c.k + 2 * d) = k;
  *reinterpret_cast<uint4*>(c.v + 2 * d) = v;
}

__global__ void __launch_bounds__(kRankThreads) k_rank(EvictArgs a, Moves mv, int room) {
  const KvCache& c = a.c;
  extern __shared__ __align__(16) uint32_t s_key[];              // `room` keys, a multiple of four
  __shared__ int s_hist[2][kBins];
  __shared__ int2 s_warp[2][kRankWarps];
  __shared__ int2 s_few[kFewMoves];
  __shared__ int s_digit[3], s_left[3], s_count;
  griddep_launch();
  const int row = blockIdx.x, b = row / c.n_kv;
  const int len = kv_length(c, b, kErrEvict);
  const float* w = c.weight + (int64_t)row * c.track;
  const int* pos = c.pos + (int64_t)row * c.track;
  float* wo = a.weight_out + (int64_t)row * c.track;
  int* po = a.pos_out + (int64_t)row * c.track;
  const bool copy_w = wo != w, copy_p = po != pos;
  if (len <= a.budget) {
    for (int i = threadIdx.x; i < len; i += kRankThreads) {
      if (copy_w) wo[i] = w[i];
      if (copy_p) po[i] = pos[i];
    }
    if (threadIdx.x == 0) mv.n[row] = 0;
    return;
  }
  const int64_t recent_from = (int64_t)__ldg(c.seen + b) - a.recent;
  const bool held = len <= room;
  for (int i = threadIdx.x; i < kBins; i += kRankThreads) s_hist[0][i] = 0;
  if (held)
#pragma unroll 4
    for (int i = threadIdx.x; i < len; i += kRankThreads) s_key[i] = rank_key(w[i], pos[i], a.sinks, recent_from);
  // every slot before the budget as it is; those that are evicted are overwritten below
  if (copy_w)
#pragma unroll 4
    for (int i = threadIdx.x; i < a.budget; i += kRankThreads) wo[i] = w[i];
  if (copy_p)
#pragma unroll 4
    for (int i = threadIdx.x; i < a.budget; i += kRankThreads) po[i] = pos[i];
  __syncthreads();
  // this thread's run of slots, four at a time: f(slot, key)
  const int run = ((len + kRankThreads - 1) / kRankThreads + 3) / 4 * 4;
  const int from = min(len, (int)threadIdx.x * run), to = min(len, from + run);
  auto each = [&](auto f) {
    for (int i = from; i < to; i += 4) {
      uint4 k;
      if (held) {
        k = *reinterpret_cast<const uint4*>(s_key + i);
      } else {
        auto at = [&](int j) { return j < len ? rank_key(w[j], pos[j], a.sinks, recent_from) : 0; };
        k = make_uint4(at(i), at(i + 1), at(i + 2), at(i + 3));
      }
      f(i, k.x);
      if (i + 1 < to) f(i + 1, k.y);
      if (i + 2 < to) f(i + 2, k.z);
      if (i + 3 < to) f(i + 3, k.w);
    }
  };
  uint32_t prefix = 0, known = 0;
  int need = a.budget;                                           // slots still wanted among those with this prefix
  int2 all = make_int2(0, 0);
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const uint32_t bins = digit < 2 ? 2047u : 1023u;
    int* hist = s_hist[digit & 1];
    each([&](int, uint32_t k) {
      if ((k & known) == prefix) atomicAdd(&hist[k >> shift & bins], 1);
    });
    if (digit < 2)
      for (int i = threadIdx.x; i < kBins; i += kRankThreads) s_hist[~digit & 1][i] = 0;
    __syncthreads();
    // thread t takes bins 2047 - 2t and the one below: the digit is the bin where the count from the top reaches need
    const int hi = hist[kBins - 1 - 2 * threadIdx.x], lo = hist[kBins - 2 - 2 * threadIdx.x];
    const int above = threads_before(hi + lo, 0, s_warp[digit & 1], &all).x;
    if (above < need && above + hi + lo >= need) {
      const bool first = above + hi >= need;
      s_digit[digit] = kBins - 1 - 2 * threadIdx.x - !first;
      s_left[digit] = need - above - (first ? 0 : hi);
      if (digit == 2) s_count = first ? hi : lo;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit[digit] << shift;
    known |= bins << shift;
    need = s_left[digit];
  }
  // every slot of a larger key than `prefix` stays, and `need` of the s_count slots with that key, from the lowest on
  int ties0 = 0;
  if (need < s_count) {
    int ties = 0;
    each([&](int, uint32_t k) { ties += k == prefix; });
    ties0 = threads_before(ties, 0, s_warp[1], &all).x;
  }
  int t = ties0, out = 0, in = 0;
  each([&](int i, uint32_t k) {
    const bool stay = k > prefix || (k == prefix && t++ < need);
    out += !stay && i < a.budget;
    in += stay && i >= a.budget;
  });
  // (s_warp[0] was last read before the last digit's second barrier)
  const int2 at0 = threads_before(out, in, s_warp[0], &all);
  const int n = all.y;
  const bool few = n <= kFewMoves;
  int2* at = few ? s_few : mv.at + (int64_t)row * mv.most;
  t = ties0;
  out = at0.x;
  in = at0.y;
  each([&](int i, uint32_t k) {
    const bool stay = k > prefix || (k == prefix && t++ < need);
    if (!stay && i < a.budget) at[out++].y = i;
    if (stay && i >= a.budget) at[in++].x = i;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kRankThreads) {
    const int2 m = at[i];
    wo[m.y] = w[m.x];
    po[m.y] = pos[m.x];
  }
  if (few) {
    const int pieces = c.hd / 8;
    for (int u = threadIdx.x; u < n * pieces; u += kRankThreads)
      move_piece(c, b, row - b * c.n_kv, s_few[u / pieces], u % pieces * 8);
  }
  if (threadIdx.x == 0) mv.n[row] = few ? 0 : n;
}

// The rows of the longer lists, 16 bytes a thread, and the new lengths (every CTA of k_rank has read the old ones).
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads) k_move(EvictArgs a, Moves mv) {
  const KvCache& c = a.c;
  griddep_wait();
  const int row = blockIdx.x, b = row / c.n_kv, h = row - b * c.n_kv;
  if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    const int len = kv_length(c, b, kErrEvict);
    a.length_out[b] = min(len, a.budget);
  }
  const int pieces = c.hd / 8, n = mv.n[row];
  const int64_t all = (int64_t)n * pieces;
  for (int64_t u = (int64_t)blockIdx.y * kMoveThreads + threadIdx.x; u < all; u += (int64_t)gridDim.y * kMoveThreads) {
    const int i = (int)(u / pieces);
    move_piece(c, b, h, mv.at[(int64_t)row * mv.most + i], (int)(u - (int64_t)i * pieces) * 8);
  }
}

// ------------------------------------------------------------------------------ logits rules
// A row is spread over a cluster of CTAs. A CTA first fills, in shared memory, one word per token of its
// share (or of a slice of it): how often it was generated, whether it is in the prompt, whether a bias
// lists it; the tokens met for the first time go on a list. That reads the whole history (a few KB out
// of L2) and keeps what falls into the share. Then the logits are masked and stored as they stream,
// without a barrier, and the listed tokens, few of many, are changed afterwards, a thread each
// (divisions and bias reads inside the stream made it three times as long). Each thread keeps its
// best group of four; the candidates are combined over the cluster and the winning group is read once
// more for the token. Words of 16 bits for histories below 2^14 ids: 32768 tokens in 64 KB.
// 64 rows of 262144 with histories of up to 4000 ids take 39 us, 21 us at the copy rate (8 bytes a token and the
// mask): bound by the filling, seven or eight steps behind a barrier each before a slice streams, and twice
// where a share is two slices as here (DRAM at 26 %, barriers the first stall). One row of 151936: 9.3 us (a
// chain of latencies). Tried and not kept: a prefetch of the share to L2 (48 us), eight groups in flight (109
// us, with the penalties in the stream).
template <class Word>
struct Bits {
  static constexpr uint32_t kListed = 1u << (8 * sizeof(Word) - 1), kPrompt = kListed >> 1, kCount = kPrompt - 1;
};

struct RowRules {
  float rep, pres, freq;
};
template <class Word>
__device__ __forceinline__ float penalties(float x, uint32_t w, const RowRules& r) {
  const uint32_t n = w & Bits<Word>::kCount;
  if (w & (Bits<Word>::kPrompt | Bits<Word>::kCount)) x = x > 0.0f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, (float)n)), r.pres);
  return x;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// The words of a slice's tokens and the list of those that are not zero (16-bit words are changed in pairs).
template <class Word>
struct Slice {
  uint32_t* word;
  uint16_t* list;
  int* listed;
  int s0, n;
  __device__ __forceinline__ uint32_t get(int t) const { return reinterpret_cast<const Word*>(word)[t]; }
  __device__ __forceinline__ void set(int t, uint32_t v) const { reinterpret_cast<Word*>(word)[t] = (Word)v; }
  __device__ __forceinline__ void mark(int id, uint32_t bit, bool add) const {
    const unsigned t = (unsigned)id - (unsigned)s0;
    if (t >= (unsigned)n) return;
    const int at = sizeof(Word) == 2 ? t >> 1 : t, shift = sizeof(Word) == 2 ? (t & 1) * 16 : 0;
    const uint32_t was = add ? atomicAdd(&word[at], 1u << shift) : atomicOr(&word[at], bit << shift);
    if (!(Word)(was >> shift)) list[atomicAdd(listed, 1)] = (uint16_t)t;
  }
};

// VEC: rows of logits and out start on 16-byte boundaries.
constexpr int kRuleThreads = 512, kGroups = 4;         // a thread has kGroups groups of four tokens in flight
constexpr int kSliceBytes = 65536;               // of words
template <bool VEC, class Word>
__global__ void __launch_bounds__(kRuleThreads, 2)
    k_adjust(const __grid_constant__ tc_logits_rules a, int cluster, int share, int slice) {
  extern __shared__ uint32_t s_word[];
  __shared__ Pick s_warp[kRuleThreads / 32];
  __shared__ int s_cand[3], s_listed;
  const int row = blockIdx.x / cluster, rank = (int)cluster_rank(), lane = threadIdx.x & 31;
  const int lo = min(a.vocab, rank * share), hi = min(a.vocab, lo + share);
  const float* x = a.logits + (int64_t)row * a.logits_stride;
  float* y = a.out + (int64_t)row * a.out_stride;
  const uint32_t* mask = a.mask ? a.mask + (int64_t)row * a.mask_stride : nullptr;
  const int* hist = a.history ? a.history + (int64_t)row * a.history_stride : nullptr;
  const bool hist4 = ((uintptr_t)hist & 15) == 0;
  int n_all = 0, n_first = 0;
  if (hist) {
    n_all = a.n_history ? min(max(__ldg(a.n_history + row), 0), a.max_history) : a.max_history;
    n_first = a.n_prompt ? min(max(__ldg(a.n_prompt + row), 0), n_all) : 0;
  }
  const int* ids = a.bias_ids ? a.bias_ids + (int64_t)row * a.bias_stride : nullptr;
  const float* bias = ids ? a.bias + (int64_t)row * a.bias_stride : nullptr;
  RowRules r;
  r.rep = a.repetition ? __ldg(a.repetition + row) : 1.0f;
  r.pres = a.presence ? __ldg(a.presence + row) : 0.0f;
  r.freq = a.frequency ? __ldg(a.frequency + row) : 0.0f;
  const bool any = n_all > 0 || ids;
  const float none = __int_as_float(0xFF800000);
  float best = none;                             // the best group's value and first token (-1: all -infinity so far)
  int best_at = -1;
  auto take = [&](float v, int j) {
    best = v;
    best_at = j;
  };
  // a group of the stream: a thread meets these in ascending order, so that of equal ones the first is held
  auto consider = [&](float v, int j) {
    if (!is_nan(best) && !(v <= best)) take(v, j);
  };
  // a listed token's group: of two of one value, or of two with a NaN, the first counts
  auto consider_any = [&](float v, int j) {
    if (is_nan(v) ? !is_nan(best) || j < best_at
                  : !is_nan(best) && (v > best || (v == best && best_at >= 0 && j < best_at)))
      take(v, j);
  };
  for (int s0 = lo; s0 < hi; s0 += slice) {
    const int s1 = min(hi, s0 + slice), n = s1 - s0;
    float e[kGroups][4];
    uint32_t bits[kGroups];
    auto request = [&](int j0) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int j = j0 + 4 * (threadIdx.x + g * kRuleThreads);      // slices begin at multiples of 32: one mask word a group
        bits[g] = mask && j < s1 ? __ldg(mask + (j >> 5)) : ~0u;
        if (VEC && j + 4 <= s1) {
          const float4 f = *reinterpret_cast<const float4*>(x + j);
          e[g][0] = f.x; e[g][1] = f.y; e[g][2] = f.z; e[g][3] = f.w;
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) e[g][u] = j + u < s1 ? x[j + u] : none;
        }
      }
    };
    request(s0);                                 // on their way while the words are filled
    int* last = reinterpret_cast<int*>(s_word) + slice * (int)sizeof(Word) / 4;     // of a listed token: its last bias entry
    const Slice<Word> sl{s_word, reinterpret_cast<uint16_t*>(last + a.n_bias), &s_listed, s0, n};
    int biased = 0;
    if (any) {
      const int words = (n * (int)sizeof(Word) + 15) / 16;       // (a slice's words are a multiple of 16 bytes)
      for (int i = threadIdx.x; i < words; i += kRuleThreads) reinterpret_cast<uint4*>(s_word)[i] = make_uint4(0, 0, 0, 0);
      if (threadIdx.x == 0) s_listed = 0;
      __syncthreads();
      if (ids) {
        // the listed tokens come first on the list; each one's last entry is found by its place there, which
        // its word holds meanwhile
        for (int i = threadIdx.x; i < a.n_bias; i += kRuleThreads) sl.mark(__ldg(ids + i), Bits<Word>::kListed, false);
        __syncthreads();
        biased = s_listed;
        for (int i = threadIdx.x; i < biased; i += kRuleThreads) {
          sl.set(sl.list[i], i);
          last[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.n_bias; i += kRuleThreads) {
          const unsigned t = (unsigned)__ldg(ids + i) - (unsigned)s0;
          if (t < (unsigned)n) atomicMax(&last[sl.get(t)], i);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < biased; i += kRuleThreads) sl.set(sl.list[i], Bits<Word>::kListed);
        __syncthreads();
      }
      int i0 = 0;
      if (hist4) {
        i0 = n_all & ~3;
#pragma unroll 2
        for (int i = 4 * threadIdx.x; i < i0; i += 4 * kRuleThreads) {
          const int4 t = __ldg(reinterpret_cast<const int4*>(hist + i));
          sl.mark(t.x, Bits<Word>::kPrompt, i >= n_first);
          sl.mark(t.y, Bits<Word>::kPrompt, i + 1 >= n_first);
          sl.mark(t.z, Bits<Word>::kPrompt, i + 2 >= n_first);
          sl.mark(t.w, Bits<Word>::kPrompt, i + 3 >= n_first);
        }
      }
#pragma unroll 4
      for (int i = i0 + threadIdx.x; i < n_all; i += kRuleThreads) sl.mark(__ldg(hist + i), Bits<Word>::kPrompt, i >= n_first);
      __syncthreads();
    }
    for (int j0 = s0; j0 < s1; j0 += 4 * kGroups * kRuleThreads) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int j = j0 + 4 * (threadIdx.x + g * kRuleThreads);
        if (j < s1) {
#pragma unroll
          for (int u = 0; u < 4; ++u) e[g][u] = bits[g] >> ((j & 31) + u) & 1 ? e[g][u] : none;
          if (VEC && j + 4 <= s1) {
            *reinterpret_cast<float4*>(y + j) = make_float4(e[g][0], e[g][1], e[g][2], e[g][3]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (j + u < s1) y[j + u] = e[g][u];
          }
          if (any) {                             // listed tokens come below
            uint32_t w[4];
            if constexpr (sizeof(Word) == 2) {
              const uint2 v = *reinterpret_cast<const uint2*>(s_word + (j - s0) / 2);
              w[0] = v.x & 0xFFFFu; w[1] = v.x >> 16; w[2] = v.y & 0xFFFFu; w[3] = v.y >> 16;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(s_word + (j - s0));
              w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) e[g][u] = w[u] ? none : e[g][u];
          }
          consider(max_nan(max_nan(e[g][0], e[g][1]), max_nan(e[g][2], e[g][3])), j);
        }
      }
      request(j0 + 4 * kGroups * kRuleThreads);
    }
    if (any) {
      __syncthreads();                           // the slice is stored
      const int listed = s_listed;
      for (int i = threadIdx.x; i < listed; i += kRuleThreads) {
        const int t = sl.list[i], j = s0 + t;
        const float was = *(volatile const float*)(y + j);
        const uint32_t word = mask ? __ldg(mask + (j >> 5)) : ~0u;
        if (word >> (j & 31) & 1) {
          float v = penalties<Word>(was, sl.get(t), r);
          if (i < biased) v = __fadd_rn(v, __ldg(bias + last[i]));
          y[j] = v;
          consider_any(v, j & ~3);
        }
      }
      __syncthreads();
    }
  }
  if (!a.token) return;
  Pick m{best, best_at, is_nan(best)};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = pick_comb(m, pick_shfl(m, o));
  if (lane == 0) s_warp[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    Pick t = threadIdx.x < kRuleThreads / 32 ? s_warp[threadIdx.x] : Pick{0.0f, -1, 0};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = pick_comb(t, pick_shfl(t, o));
    if (threadIdx.x == 0) {
      s_cand[0] = __float_as_int(t.v);
      s_cand[1] = t.i;
      s_cand[2] = t.nan;
    }
  }
  cluster_sync();                                // (orders the stores of out before the read below as well)
  if (rank == 0 && threadIdx.x < 32) {
    Pick t{0.0f, -1, 0};
    if (lane < cluster)
      t = Pick{__int_as_float(dsmem_ld_s32(smem_u32(&s_cand[0]), lane)), dsmem_ld_s32(smem_u32(&s_cand[1]), lane),
               dsmem_ld_s32(smem_u32(&s_cand[2]), lane)};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = pick_comb(t, pick_shfl(t, o));
    int token = a.none;
    if (t.i >= 0) {                              // the group's first NaN, or first entry of its value
      const float v = lane < 4 && t.i + lane < a.vocab ? *(volatile const float*)(y + t.i + lane) : none;
      const bool is = lane < 4 && t.i + lane < a.vocab && (t.nan ? is_nan(v) : v == t.v);
      token = t.i + __ffs(__ballot_sync(0xFFFFFFFFu, is)) - 1;
    } else if (!mask) {
      token = 0;                                 // a row of -infinity alone: the first token
    } else {
      for (int i = 0; i < (a.vocab + 31) / 32; ++i) {
        const uint32_t word = __ldg(mask + i) & (a.vocab - 32 * i >= 32 ? ~0u : (1u << (a.vocab - 32 * i)) - 1);
        if (word) {
          token = 32 * i + __ffs(word) - 1;      // allowed tokens that are all -infinity: the first of them
          break;
        }
      }
    }
    if (lane == 0) a.token[row] = token;
  }
  cluster_sync();                                // no CTA leaves while its candidate is read
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, cudaStream_t st) {
  if (a.tokens == 0) return cudaSuccess;
  return a.dtype == TC_BF16 ? append_to<__nv_bfloat16>(a, st) : append_to<__half>(a, st);
}

uint64_t evict_workspace(const KvCache& c, int budget) {
  const uint64_t rows = (uint64_t)c.batch * c.n_kv;
  return (rows * 4 + 255) / 256 * 256 + rows * most_moves(c.max_pages << c.shift, budget) * sizeof(int2);
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t st) {
  const int rows = a.c.batch * a.c.n_kv;
  const Moves mv = moves_of(a.ws, rows, most_moves(a.c.max_pages << a.c.shift, a.budget));
  const int room = std::min(a.c.max_pages << a.c.shift, kKeysMax);
  cudaError_t e = allow_smem<k_rank>(kKeysMax * 4);
  if (e != cudaSuccess) return e;
  k_rank<<<rows, kRankThreads, room * 4, st>>>(a, mv, room);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t pieces = (int64_t)std::max(1, mv.most) * (a.c.hd / 8);
  const int blocks = (int)std::min<int64_t>((pieces + kMoveThreads - 1) / kMoveThreads, std::max(1, 148 * 8 / rows));
  return launch_dependent(k_move, dim3(rows, blocks), dim3(kMoveThreads), st, a, mv);
}

namespace {
template <bool VEC, class Word>
cudaError_t adjust_of(const tc_logits_rules& r, cudaStream_t st) {
  constexpr auto kern = k_adjust<VEC, Word>;
  // As many CTAs a row as fit on the SMs at once, two to an SM, with 4096 tokens or more each. Measured on rows of
  // 151936 (us for clusters of 16, 8, 4, 2): 1 row 9.5, 11.8, 17.3; 16 rows 20, 15, 18; 64 rows 59, 34, 28, 35;
  // 128 rows 113, 63, 53, 45; 128 rows of 32000 90, 42, 24, 15.
  int cluster = r.rows <= 4 ? 16 : 8;
  while (cluster > 1 && ((int64_t)r.rows * cluster > 2 * 148 || r.vocab < 4096 * cluster)) cluster /= 2;
  const int share = ((r.vocab + cluster - 1) / cluster + 31) / 32 * 32;
  const int slice = std::min(share, kSliceBytes / (int)sizeof(Word));
  // a word a token, a place a bias entry, and list entries for as many tokens as the history and the biases can name
  const int n_bias = r.bias ? r.n_bias : 0;
  const int64_t names = (r.history ? r.max_history : 0) + (int64_t)n_bias;
  const int smem = slice * (int)sizeof(Word) + 4 * n_bias + 2 * (int)std::min<int64_t>(slice, names);
  static std::atomic<uint64_t> ready{0};         // devices on which clusters of 16 and the shared memory are allowed
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kSliceBytes + 8192);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  tc_logits_rules a = r;
  a.n_bias = n_bias;
  return launch_ex(kern, dim3((unsigned)r.rows * cluster), dim3(kRuleThreads), smem, st, cluster, a, cluster, share, slice);
}
}  // namespace

cudaError_t launch_adjust(const tc_logits_rules& r, cudaStream_t st) {
  const bool vec = ((uintptr_t)r.logits | (uintptr_t)r.out) % 16 == 0 && r.logits_stride % 4 == 0 && r.out_stride % 4 == 0;
  if (r.history && r.max_history > (int)Bits<uint16_t>::kCount)
    return vec ? adjust_of<true, uint32_t>(r, st) : adjust_of<false, uint32_t>(r, st);
  return vec ? adjust_of<true, uint16_t>(r, st) : adjust_of<false, uint16_t>(r, st);
}

}  // namespace tc
