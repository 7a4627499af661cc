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
// row's threads side by side. Bound by memory (each source element read once, each cache element
// written once); a single step's rows are bound by the launch.
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
// (protected slots highest, then a NaN weight, then the weight's bits made monotonic); the budget-th
// largest key is found digit by digit from the top (8 bits a pass, counted in shared memory), and of
// the slots with that key as many stay as are needed, from the lowest slot on. Warps own contiguous
// runs of slots, so the lists of leaving and arriving slots come out in ascending order from
// ballots and one scan over the warps. The rows move in a second kernel over the lists.
constexpr int kRankThreads = 1024, kRankWarps = kRankThreads / 32;

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

// Exclusive sum over the warps of the CTA of each warp's x (same x in a warp's lanes); *all gets the total.
__device__ __forceinline__ int warps_before(int x, int* s_warp, int* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) s_warp[warp] = x;
  __syncthreads();
  const int mine = s_warp[lane];
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += y;
  }
  *all = __shfl_sync(0xFFFFFFFFu, sum, 31);
  return __shfl_sync(0xFFFFFFFFu, sum - mine, warp);
}

__global__ void __launch_bounds__(kRankThreads) k_rank(EvictArgs a, Moves mv) {
  const KvCache& c = a.c;
  __shared__ int s_hist[256];
  __shared__ int s_warp[kRankWarps];
  __shared__ uint32_t s_digit;
  __shared__ int s_left;
  const int row = blockIdx.x, b = row / c.n_kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  auto key = [&](int i) { return rank_key(w[i], pos[i], a.sinks, recent_from); };
  uint32_t prefix = 0, known = 0;
  int need = a.budget;                                           // slots still wanted among those with this prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kRankThreads) s_hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < len; i += kRankThreads) {
      const uint32_t k = key(i);
      if ((k & known) == prefix) atomicAdd(&s_hist[k >> shift & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = need, d = 255;
      while (d > 0 && s_hist[d] < left) left -= s_hist[d--];
      s_digit = d;
      s_left = left;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    known |= 255u << shift;
    need = s_left;
  }
  // `need` slots of key `prefix` stay, from the lowest on, and every slot of a larger key
  const int run = (len + 32 * kRankWarps - 1) / (32 * kRankWarps) * 32;
  const int from = min(len, warp * run), to = min(len, from + run);
  int ties = 0, all = 0;
  for (int i = from + lane; i - lane < to; i += 32)
    ties += __popc(__ballot_sync(0xFFFFFFFFu, i < to && key(i) == prefix));
  const int ties0 = warps_before(ties, s_warp, &all);
  const uint32_t below = (1u << lane) - 1;
  int n_out = 0, n_in = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int t = ties0, out0 = 0, in0 = 0;
    if (pass) {
      out0 = warps_before(n_out, s_warp, &all);
      in0 = warps_before(n_in, s_warp, &all);
      if (threadIdx.x == 0) mv.n[row] = all;
    }
    for (int i = from + lane; i - lane < to; i += 32) {
      const bool on = i < to;
      const uint32_t k = on ? key(i) : 0;
      const uint32_t tie = __ballot_sync(0xFFFFFFFFu, on && k == prefix);
      const bool stay = on && (k > prefix || (k == prefix && t + __popc(tie & below) < need));
      t += __popc(tie);
      const uint32_t leave = __ballot_sync(0xFFFFFFFFu, on && !stay && i < a.budget);
      const uint32_t move = __ballot_sync(0xFFFFFFFFu, stay && i >= a.budget);
      if (pass) {
        int2* at = mv.at + (int64_t)row * mv.most;
        if (leave >> lane & 1) at[out0 + __popc(leave & below)].y = i;
        if (move >> lane & 1) at[in0 + __popc(move & below)].x = i;
        if (stay && i < a.budget) {
          if (copy_w) wo[i] = w[i];
          if (copy_p) po[i] = pos[i];
        }
      }
      out0 += __popc(leave);
      in0 += __popc(move);
    }
    n_out = out0;
    n_in = in0;
  }
  __syncthreads();
  const int2* at = mv.at + (int64_t)row * mv.most;
  for (int i = threadIdx.x; i < all; i += kRankThreads) {
    const int2 m = at[i];
    wo[m.y] = w[m.x];
    po[m.y] = pos[m.x];
  }
}

// The rows of the moves: a quarter of a warp's lanes (or as many as a row has 16-byte pieces) per
// row, keys and values. Sources lie at or behind the budget, destinations before it.
constexpr int kMoveThreads = 256;
__global__ void __launch_bounds__(kMoveThreads) k_move(EvictArgs a, Moves mv) {
  const KvCache& c = a.c;
  const int row = blockIdx.x, b = row / c.n_kv, h = row - b * c.n_kv;
  if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    const int len = kv_length(c, b, kErrEvict);
    a.length_out[b] = min(len, a.budget);
  }
  const int pieces = c.hd / 8, n = mv.n[row];
  const int64_t all = (int64_t)n * pieces;
  for (int64_t u = (int64_t)blockIdx.y * kMoveThreads + threadIdx.x; u < all; u += (int64_t)gridDim.y * kMoveThreads) {
    const int i = (int)(u / pieces), e = (int)(u - (int64_t)i * pieces) * 8;
    const int2 m = mv.at[(int64_t)row * mv.most + i];
    const int ps = kv_page(c, b, m.x, kErrEvict), pd = kv_page(c, b, m.y, kErrEvict);
    if (ps < 0 || pd < 0) continue;
    const int64_t s = kv_offset(c, ps, m.x, h) + e, d = kv_offset(c, pd, m.y, h) + e;
    const uint4 k = *reinterpret_cast<const uint4*>(c.k + 2 * s), v = *reinterpret_cast<const uint4*>(c.v + 2 * s);
    *reinterpret_cast<uint4*>(c.k + 2 * d) = k;
    *reinterpret_cast<uint4*>(c.v + 2 * d) = v;
  }
}

// ------------------------------------------------------------------------------ logits rules
// A row is spread over a cluster of kRuleCluster CTAs; a CTA takes its share in slices. A slice has one
// word per token in shared memory: bits 0-19 how often it was generated, bit 20 that it is in the
// prompt, bits 21-31 the last bias entry that lists it. Filling the words reads the whole history (a
// few KB out of L2) and keeps what falls into the slice; then the logits pass once, read and
// written, and the greedy candidates are combined over the cluster.
constexpr int kRuleCluster = 8, kRuleThreads = 512;
constexpr uint32_t kRulePrompt = 1u << 20, kRuleCount = kRulePrompt - 1;

struct RowRules {
  float rep, pres, freq;
  const float* bias;
  bool any;
};
__device__ __forceinline__ float rule(float x, uint32_t w, const RowRules& r) {
  if (w) {
    const uint32_t n = w & kRuleCount;
    if (w & (kRulePrompt | kRuleCount)) x = x > 0.0f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
    if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, (float)n)), r.pres);
    if (w >> 21) x = __fadd_rn(x, __ldg(r.bias + (w >> 21) - 1));
  }
  return x;
}
__device__ __forceinline__ void pick_allowed(Pick& p, float v, int j, uint32_t allowed) {
  const int vn = is_nan(v);
  const bool take = allowed & ((p.i < 0) | (vn & !p.nan) | (!p.nan & !vn & (v > p.v)));
  p.v = take ? v : p.v;
  p.i = take ? j : p.i;
  p.nan = take ? vn : p.nan;
}

template <bool VEC>
__global__ void __launch_bounds__(kRuleThreads) k_adjust(tc_logits_rules a, int share, int slice) {
  extern __shared__ uint32_t s_word[];
  __shared__ Pick s_warp[kRuleThreads / 32];
  __shared__ int s_cand[3];
  const int row = blockIdx.x / kRuleCluster, rank = (int)cluster_rank();
  const int lo = min(a.vocab, rank * share), hi = min(a.vocab, lo + share);
  const float* x = a.logits + (int64_t)row * a.logits_stride;
  float* y = a.out + (int64_t)row * a.out_stride;
  const uint32_t* mask = a.mask ? a.mask + (int64_t)row * a.mask_stride : nullptr;
  const int* hist = a.history ? a.history + (int64_t)row * a.history_stride : nullptr;
  int n_all = 0, n_first = 0;
  if (hist) {
    n_all = a.n_history ? min(max(__ldg(a.n_history + row), 0), a.max_history) : a.max_history;
    n_first = a.n_prompt ? min(max(__ldg(a.n_prompt + row), 0), n_all) : 0;
  }
  const int* ids = a.bias_ids ? a.bias_ids + (int64_t)row * a.bias_stride : nullptr;
  RowRules r;
  r.rep = a.repetition ? __ldg(a.repetition + row) : 1.0f;
  r.pres = a.presence ? __ldg(a.presence + row) : 0.0f;
  r.freq = a.frequency ? __ldg(a.frequency + row) : 0.0f;
  r.bias = ids ? a.bias + (int64_t)row * a.bias_stride : nullptr;
  r.any = n_all > 0 || ids;
  Pick p[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) p[u] = Pick{0.0f, -1, 0};
  for (int s0 = lo; s0 < hi; s0 += slice) {
    const int s1 = min(hi, s0 + slice), n = s1 - s0;
    if (r.any) {
      for (int i = threadIdx.x; i < n; i += kRuleThreads) s_word[i] = 0;
      __syncthreads();
      if (ids) {
        for (int i = threadIdx.x; i < a.n_bias; i += kRuleThreads) {
          const unsigned t = (unsigned)__ldg(ids + i) - (unsigned)s0;
          if (t < (unsigned)n) atomicMax(&s_word[t], (uint32_t)(i + 1) << 21);
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < n_all; i += kRuleThreads) {
        const unsigned t = (unsigned)__ldg(hist + i) - (unsigned)s0;
        if (t < (unsigned)n) {
          if (i < n_first) atomicOr(&s_word[t], kRulePrompt);
          else atomicAdd(&s_word[t], 1u);
        }
      }
      __syncthreads();
    }
    if (VEC) {
      // s0 is a multiple of 32: a vector's four tokens share a mask word
      for (int j = s0 + 4 * threadIdx.x; j < s1; j += 4 * kRuleThreads) {
        const uint32_t bits = mask ? __ldg(mask + (j >> 5)) >> (j & 31) : 15u;
        if (j + 4 <= s1) {
          float4 f = *reinterpret_cast<const float4*>(x + j);
          float e[4] = {f.x, f.y, f.z, f.w};
          if (r.any) {
            const uint4 w = *reinterpret_cast<const uint4*>(s_word + (j - s0));
            e[0] = rule(e[0], w.x, r);
            e[1] = rule(e[1], w.y, r);
            e[2] = rule(e[2], w.z, r);
            e[3] = rule(e[3], w.w, r);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            pick_allowed(p[u], e[u], j + u, bits >> u & 1);
            if (!(bits >> u & 1)) e[u] = __int_as_float(0xFF800000);
          }
          *reinterpret_cast<float4*>(y + j) = make_float4(e[0], e[1], e[2], e[3]);
        } else {
          for (int u = 0; j + u < s1; ++u) {
            float e = x[j + u];
            if (r.any) e = rule(e, s_word[j + u - s0], r);
            pick_allowed(p[0], e, j + u, bits >> u & 1);
            y[j + u] = bits >> u & 1 ? e : __int_as_float(0xFF800000);
          }
        }
      }
    } else {
      for (int j = s0 + threadIdx.x; j < s1; j += kRuleThreads) {
        const uint32_t ok = mask ? __ldg(mask + (j >> 5)) >> (j & 31) & 1 : 1u;
        float e = x[j];
        if (r.any) e = rule(e, s_word[j - s0], r);
        pick_allowed(p[0], e, j, ok);
        y[j] = ok ? e : __int_as_float(0xFF800000);
      }
    }
    __syncthreads();
  }
  if (!a.token) return;
  Pick m = pick_comb(pick_comb(p[0], p[1]), pick_comb(p[2], p[3]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = pick_comb(m, pick_shfl(m, o));
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    Pick t = s_warp[0];
    for (int w = 1; w < kRuleThreads / 32; ++w) t = pick_comb(t, s_warp[w]);
    s_cand[0] = __float_as_int(t.v);
    s_cand[1] = t.i;
    s_cand[2] = t.nan;
  }
  cluster_sync();
  if (rank == 0 && threadIdx.x == 0) {
    Pick t{__int_as_float(s_cand[0]), s_cand[1], s_cand[2]};
    for (int q = 1; q < kRuleCluster; ++q) {
      const Pick u{__int_as_float(dsmem_ld_s32(smem_u32(&s_cand[0]), q)), dsmem_ld_s32(smem_u32(&s_cand[1]), q),
                   dsmem_ld_s32(smem_u32(&s_cand[2]), q)};
      t = pick_comb(t, u);
    }
    a.token[row] = t.i < 0 ? a.none : t.i;
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
  k_rank<<<rows, kRankThreads, 0, st>>>(a, mv);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t pieces = (int64_t)std::max(1, mv.most) * (a.c.hd / 8);
  const int blocks = (int)std::min<int64_t>((pieces + kMoveThreads - 1) / kMoveThreads, std::max(1, 148 * 8 / rows));
  k_move<<<dim3(rows, blocks), kMoveThreads, 0, st>>>(a, mv);
  return cudaGetLastError();
}

cudaError_t launch_adjust(const tc_logits_rules& r, cudaStream_t st) {
  const int share = ((r.vocab + kRuleCluster - 1) / kRuleCluster + 31) / 32 * 32;
  // 32 KB of words leave room for several CTAs an SM, so that one fills its words while another streams
  const int slice = std::min(share, 8192);
  const bool vec = ((uintptr_t)r.logits | (uintptr_t)r.out) % 16 == 0 && r.logits_stride % 4 == 0 && r.out_stride % 4 == 0;
  auto kern = vec ? k_adjust<true> : k_adjust<false>;
  const int smem = slice * 4;
  return launch_ex(kern, dim3(r.rows * kRuleCluster), dim3(kRuleThreads), smem, st, kRuleCluster, r, share, slice);
}

}  // namespace tc
