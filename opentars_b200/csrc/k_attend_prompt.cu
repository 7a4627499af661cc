// Attention of the rows of a prompt over the paged cache (tc_attend_prompt), on the 5th-generation
// tensor cores.
//
// A tile is 128 query rows: the heads of one key-value head (at most 32 of them) for 128 / heads
// consecutive tokens, so a group's heads share every key and value tile that is staged. A CTA takes
// two tiles (one for head dim 256, whose output alone fills half of TMEM) of one sequence and walks
// the blocks of key slots that any of its rows sees: the sinks' blocks, then those of the windows.
//   loaders    a block's keys and values into a ring, rows behind the sequence's end, which may hold
//              anything, as zeros (0 x NaN is not 0). Pages of 64 slots and more: one warp, by TMA (64
//              columns x page rows boxes, 128-byte swizzle). Smaller pages: three warps, by cp.async
//              (16-byte pieces, eight slots of one page at a time, placed as the swizzle wants them),
//              because boxes of 2 or 4 KB are TMA's limit: 16000 tokens of a window of 512 at head dim
//              256 take 131 us by TMA against 101 over 16-slot pages, and 92 against 99 over 64-slot
//              ones; three prompts of up to 8192 tokens at head dim 128 364 against 413 over the latter
//   MMA        one thread: S = Q K^T into TMEM (tcgen05 kind::f16), then O += P V with P as the
//              TMEM operand where S was; with two tiles one is multiplied while the other is
//              exponentiated, with one tile S is double-buffered
//   softmax    a warpgroup per tile, a thread per row: the row's scores stay in registers, the
//              running maximum is only moved (and O rescaled) when it grows by more than 2^8, and
//              P is rounded once to the cache's type, whose range holds that: the output's error against
//              64 bits is 1.29 (bf16) and 1.40 (fp16) times that of the output's own rounding alone. A second
//              part, as attend keeps, would add half to the 2048 cycles that the MMAs of a pair of tiles
//              take (below). The row's sum is of the unrounded fp32 values
// Three prompts of up to 8192 tokens, 16 heads on 8 of 128, bf16: 365 us (1005 TFLOP/s; 430 us in long runs under
// the power limit). A pair of tiles takes 3400 cycles for 128 slots, of which its MMAs are 2048: the rest is the
// way of one tile's scores to its softmax and of its probabilities back (some 1500 cycles besides the work).
// Parts of 64 slots, which put twice as many tiles' steps in flight, took 432 us: S at N = 64 is bound by the
// reads of Q from shared memory.
// A row with a NaN in its output, and every row of a CTA that met a page id outside the pool, is computed
// again by attend_row over its visible slots alone: a NaN or an infinity in a slot that the mask hides from
// this row but not from its tile reaches it as 0 x inf. Not so a row whose sum is NaN or whose scores are all
// -infinity: only visible scores do that (but for scale 0, where a hidden one is -infinity x 0), and its output is
// NaN whatever else there is. Nor an infinity without a NaN: a hidden value would have made a NaN. A key row of
// NaN at the front of a prompt of 2048 tokens, 16 heads on 8 of 128: 55 us as without it (34 ms, a row a warp).
#include <cuda_runtime.h>

#include <algorithm>

#include "attend_row.cuh"
#include "fp32.cuh"
#include "mma.h"
#include "paged_map.h"
#include "pdl.cuh"
#include "umma.cuh"

namespace tc {
namespace {

constexpr int kRows = 128, kMaxHeads = 32;

template <int HD>
struct PromptShape {
  static constexpr int kTiles = HD == 256 ? 1 : 2;           // query tiles of a CTA
  static constexpr int kBlock = HD == 256 ? 64 : 128;        // key slots of a block
  static constexpr int kQ = kRows * HD * 2, kMat = kBlock * HD * 2;
  static constexpr int kParts = kTiles;                      // a block's probabilities are handed over in parts
  static constexpr int kSlots = HD == 64 ? 8 : 5;            // ring of key / value blocks
  static constexpr int kThreads = 128 * kTiles + 128;        // softmax, MMA, loaders
  static constexpr int kSmem = 1024 + kTiles * kQ + kSlots * kMat;
  static constexpr uint32_t kS = 0, kO = 256;                // TMEM columns: two S (and P) buffers, the outputs
};

struct PromptMaps {
  CUtensorMap k, v;
};
constexpr int kLoaders = 3, kTmaPage = 64;       // loader warps without TMA; the smallest page it takes

// What a CTA works on, the same in every thread.
struct Work {
  int b, kvh, h0, hb;               // sequence, key-value head, first query head and how many
  int row0, n, len;                 // first row of the sequence in q, its rows, its slots
  int tok[2];                       // first token (of the sequence's n) of each tile
  int ntok[2], end[2], nb[2];       // its tokens, one past its last position, its blocks
  int first, head, na, t0, nmax;    // visible slots [0, head) and [first, end): blocks 0 .. na - 1, t0 on
  __device__ __forceinline__ int block(int j) const { return j < na ? j : t0 + j - na; }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

// Two fp32 values in a register pair, one instruction for both.
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b));
  return v;
}
__device__ __forceinline__ uint64_t pair(float a) { return pair(__float_as_uint(a), __float_as_uint(a)); }
__device__ __forceinline__ float2 halves(uint64_t v) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x of two values <= 16 on the FMA units: x = n + f with n the nearest integer (1.5 x 2^23 + 127 is added, so that
// n + 127, the exponent field of 2^n, stands in the sum's low bits) and f in [-1/2, 1/2]; 2^f by a polynomial fitted
// to least relative error (2.6e-6), times 2^n. From 2^-126.5 down the field is 0 and so is the result. A NaN stays
// one (its low bits make a factor of 0 or -infinity).
__device__ __forceinline__ uint64_t ex2_fma(uint64_t x2) {
  const float2 x = halves(x2);
  x2 = pair(__float_as_uint(max_nan(x.x, -127.0f)), __float_as_uint(max_nan(x.y, -127.0f)));
  const uint64_t t = add2(x2, pair(12583039.0f)), f = add2(x2, fma2(t, pair(-1.0f), pair(12583039.0f)));
  uint64_t p = fma2(f, pair(0.009570101276040077f), pair(0.05591785907745361f));
  p = fma2(p, f, pair(0.240247443318367f));
  p = fma2(p, f, pair(0.6931217908859253f));
  p = fma2(p, f, pair(0.9999992847442627f));
  const float2 n = halves(t);
  return mul2(p, pair(__float_as_uint(n.x) << 23, __float_as_uint(n.y) << 23));
}
// v[i] = 2^(v[i] scale - base) for N scores, rounded to T two by two into out; their sum (of the unrounded values).
// MIX: every fourth pair goes to the FMA units, which are idle while the others wait for the special function
// unit (8 cycles a warp and instruction); not where masked scores of -infinity have to become 0.
template <class T, int N, bool MIX>
__device__ __forceinline__ float exponentials(const uint32_t* v, uint32_t* out, float scale2, float base) {
  const uint64_t s2 = pair(scale2), b2 = pair(-base);
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int x = 0; x < N; x += 2) {
    const uint64_t y = fma2(pair(v[x], v[x + 1]), s2, b2);
    uint64_t p;
    if (MIX && (x >> 1 & 3) == 3) {
      p = ex2_fma(y);
    } else {
      const float2 f = halves(y);
      p = pair(__float_as_uint(ex2(f.x)), __float_as_uint(ex2(f.y)));
    }
    sum[x >> 1 & 1] = add2(sum[x >> 1 & 1], p);
    const float2 f = halves(p);
    out[x >> 1] = Elem<T>::pack(f.x, f.y);
  }
  const float2 f = halves(add2(sum[0], sum[1]));
  return f.x + f.y;
}

template <class T, int HD>
__device__ __noinline__ void redo_row(const AttendArgs& a, int b, int kvh, int64_t row, int h, int end) {
  float q[HD / 32], o[HD / 32];
  const int lane = threadIdx.x & 31;
  row_load<T, HD>(a.q, row * a.qr + (int64_t)h * a.qh, lane, q);
  attend_row<T, HD>(a.c, b, kvh, q, a.scale2, end, a.window, a.sinks, kErrPrompt, o);
  row_store<T, HD>(a.out, row * a.orow + (int64_t)h * a.oh, lane, o);
}

template <class T, int HD, bool TMA>
__global__ void __launch_bounds__(PromptShape<HD>::kThreads, 1)
    k_prompt(const __grid_constant__ PromptMaps maps, const __grid_constant__ AttendArgs a, int gblocks, int hb, int tokens) {
  using Sh = PromptShape<HD>;
  constexpr int NT = Sh::kTiles, BN = Sh::kBlock;
  extern __shared__ uint8_t s_raw[];
  __shared__ __align__(8) uint64_t s_full[Sh::kSlots], s_free[Sh::kSlots], s_sfull[2], s_pfull[4], s_odone[2], s_fix, s_end;
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[16], s_found[2], s_bad, s_dead;
  const KvCache& c = a.c;
  uint8_t* s_q = s_raw + (1024 - (smem_u32(s_raw) & 1023)) % 1024;
  uint8_t* s_kv = s_q + NT * Sh::kQ;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMma = 4 * NT;                    // warps 0 .. 4 NT - 1 softmax, then the MMA's, then the loaders

  // ---- which rows: pairs of tiles, sequence by sequence; the last pairs (the longest rows) go first
  Work w;
  {
    const int nsub = c.n_kv * gblocks, span = NT * tokens;
    const int pairs = gridDim.x / nsub, pr = pairs - 1 - (int)(blockIdx.x / nsub), sub = blockIdx.x % nsub;
    const int per = (c.batch + Sh::kThreads - 1) / Sh::kThreads, lo = min(c.batch, (int)threadIdx.x * per), hi = min(c.batch, lo + per);
    if (threadIdx.x == 0) s_found[0] = -1;
    int mine = 0;
    for (int b = lo; b < hi; ++b) mine += (max(__ldg(a.cu + b + 1) - __ldg(a.cu + b), 0) + span - 1) / span;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) s_scan[warp] = sum;
    __syncthreads();
    int at = sum - mine;
    for (int k = 0; k < warp; ++k) at += s_scan[k];
    if (pr >= at && pr < at + mine) {
      int b = lo;
      for (; b < hi - 1; ++b) {
        const int k = (max(__ldg(a.cu + b + 1) - __ldg(a.cu + b), 0) + span - 1) / span;
        if (pr < at + k) break;
        at += k;
      }
      s_found[0] = b;
      s_found[1] = pr - at;
    }
    __syncthreads();
    w.b = s_found[0];
    if (w.b < 0) return;
    w.kvh = sub / gblocks;
    const int G = a.nh / c.n_kv, g0 = (sub - w.kvh * gblocks) * hb;
    w.h0 = w.kvh * G + g0;
    w.hb = min(hb, G - g0);
    w.row0 = __ldg(a.cu + w.b);
    w.n = __ldg(a.cu + w.b + 1) - w.row0;
    const int rows = w.row0 < 0 ? 0 : min(w.n, a.tokens - w.row0);       // (rows outside q are left out)
    w.len = kv_length(c, w.b, kErrPrompt);
    const int tok0 = s_found[1] * span, p0 = w.len - w.n + tok0;
    w.first = p0 + 1 > 0 ? first_in_window(p0 + 1, a.window) : 0;
    w.head = min(a.sinks, w.first);
    w.t0 = w.first / BN;
    w.na = min((w.head + BN - 1) / BN, w.t0);
    w.nmax = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      w.tok[t] = tok0 + t * tokens;
      w.ntok[t] = t < NT ? min(max(rows - w.tok[t], 0), tokens) : 0;
      w.end[t] = w.ntok[t] ? max(w.len - w.n + w.tok[t] + w.ntok[t], 0) : 0;
      w.nb[t] = w.end[t] ? w.na + (w.end[t] + BN - 1) / BN - w.t0 : 0;
      w.nmax = max(w.nmax, w.nb[t]);
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < Sh::kSlots; ++i) {
      mbar_init(&s_full[i], TMA ? 1 : kLoaders);
      mbar_init(&s_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_sfull[i], 1);
      mbar_init(&s_pfull[2 * i], 4);
      mbar_init(&s_pfull[2 * i + 1], 4);
      mbar_init(&s_odone[i], 1);
    }
    mbar_init(&s_fix, 1);
    mbar_init(&s_end, 1);
    mbar_fence_init();
    s_bad = s_dead = 0;
  }
  if (warp == kMma) tmem_alloc(&s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  // With two tiles the launch's 168 registers a thread (3 warpgroups) are split 208 + 208 + 88, their sum unchanged
  if (warp >= kMma) {
    if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (TMA && warp == kMma + 1) {
      // one loader: a block page by page in boxes of 64 columns, a lane a box
      int slot = 0, phase = 0, issued = 0, fixes = 0;
      const int end = max(w.end[0], w.end[1]), box = min(BN, 1 << c.shift), per = box / 16;
      auto load = [&](int j, bool is_v) {
        if (issued >= Sh::kSlots &&
            !__all_sync(0xFFFFFFFFu, mbar_wait(&s_free[slot], phase ^ 1, c.err, kErrPromptWait, a.spin)))
          return false;
        const int j0 = w.block(j) * BN, js = j0 + 16 * lane;
        int page = -1;
        if (lane < BN / 16 && js < end) {
          page = __ldg(c.table + (int64_t)w.b * c.ts + (js >> c.shift));
          if ((unsigned)page >= (unsigned)c.n_pages) {
            page = -1;
            if (js + 16 > w.first || js < w.head) {      // (a page that no row sees may be gone)
              kv_fail(c, kErrPrompt);
              s_bad = 1;
            }
          }
        }
        const uint32_t have = __ballot_sync(0xFFFFFFFFu, page >= 0);
        const bool fix = is_v && (have != (1u << BN / 16) - 1 || j0 + BN > w.len);
        uint64_t* bar = fix ? &s_fix : &s_full[slot];
        auto groups = [&](int u) { return have >> (u * per) & ((1u << per) - 1); };   // of box u
        uint32_t bytes = 0;
        for (int u = 0; u < BN / box; ++u) bytes += groups(u) ? box * HD * 2 : 0;
        if (lane == 0) mbar_expect_tx(bar, bytes);
        __syncwarp();
        uint8_t* dst = s_kv + slot * Sh::kMat;
        const int boxes = BN / box * (HD / 64), x = min(lane, boxes - 1), u = x / (HD / 64), half = x - u * (HD / 64);
        const uint32_t here = groups(u);
        const int pg = __shfl_sync(0xFFFFFFFFu, page, here ? u * per + __ffs(here) - 1 : 0);
        if (here && lane < boxes)
          tma_load_4d(smem_u32(dst) + half * BN * 128 + u * box * 128, is_v ? &maps.v : &maps.k, 64 * half,
                      (j0 + u * box) & ((1 << c.shift) - 1), w.kvh, pg, bar);
        if (fix) {
          const bool ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_fix, fixes & 1, c.err, kErrPromptWait));
          ++fixes;
          if (!ok) return false;
          for (int r = 0; r < BN; ++r)
            if (!(have >> (r >> 4) & 1) || j0 + r >= w.len)
              for (int y = lane; y < HD / 8; y += 32)
                *reinterpret_cast<uint4*>(dst + (y >> 3) * BN * 128 + r * 128 + (y & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_full[slot]);
        }
        ++issued;
        if (++slot == Sh::kSlots) { slot = 0; phase ^= 1; }
        return true;
      };
      bool ok = w.nmax == 0 || load(0, false);
      for (int j = 0; ok && j < w.nmax; ++j) {
        // in the order of use: with two tiles V(j), K(j + 1); with one K(j + 1), V(j)
        if (NT == 2) ok = load(j, true) && (j + 1 == w.nmax || load(j + 1, false));
        else ok = (j + 1 == w.nmax || load(j + 1, false)) && load(j, true);
      }
      if (!ok) s_dead = 1;
      // no copy is in flight when the block ends: the last use of every slot has arrived
      for (int k = 0; k < Sh::kSlots && k < issued; ++k) {
        if (--slot < 0) { slot = Sh::kSlots - 1; phase ^= 1; }
        mbar_wait(&s_full[slot], phase, c.err, kErrPromptWait);
      }
    } else if (!TMA && warp > kMma) {
      // A loader takes every kLoaders-th unit of 8 slots of a block; a lane copies piece lane % kLanes of rows r0,
      // r0 + kAtOnce, ..: row r of a 64-column group is 128 bytes, its piece p at place p ^ (r % 8)
      constexpr int kPieces = HD / 8, kLanes = kPieces < 32 ? kPieces : 32, kAtOnce = 32 / kLanes, kLag = 2;
      const int piece = lane % kLanes, r0 = lane / kLanes, me = warp - kMma - 1;
      const uint32_t put = smem_u32(s_kv) + (piece >> 3) * BN * 128 + r0 * 128 + (((piece & 7) ^ r0) << 4);
      const int64_t step = 2 * kAtOnce * c.ss;
      const int end = max(w.end[0], w.end[1]);
      int slot = 0, phase = 0, issued = 0, full = 0;
      auto arrive = [&] {                          // the oldest block still on its way is here
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_full[full]);
        if (++full == Sh::kSlots) full = 0;
      };
      auto load = [&](int j, const uint8_t* pool) {
        if (issued >= Sh::kSlots &&
            !__all_sync(0xFFFFFFFFu, mbar_wait(&s_free[slot], phase ^ 1, c.err, kErrPromptWait, a.spin)))
          return false;
        const int j0 = w.block(j) * BN;
        int page = -1;                             // lane u: of unit u
        if (lane < BN / 8 && j0 + 8 * lane < end) {
          const int js = j0 + 8 * lane;
          page = __ldg(c.table + (int64_t)w.b * c.ts + (js >> c.shift));
          if ((unsigned)page >= (unsigned)c.n_pages) {
            page = -1;
            if (js + 8 > w.first || js < w.head) { // (a page that no row sees may be gone)
              kv_fail(c, kErrPrompt);
              s_bad = 1;
            }
          }
        }
        for (int u = me; u < BN / 8; u += kLoaders) {
          const int pg = __shfl_sync(0xFFFFFFFFu, page, u), js = j0 + 8 * u + r0;
          const uint8_t* from = pool + 2 * (kv_offset(c, max(pg, 0), js, w.kvh) + 8 * piece);
          const uint32_t to = put + slot * Sh::kMat + u * 1024;
          const int rows = pg >= 0 ? w.len - js : 0;         // of them exist, counted from this lane's first
#pragma unroll
          for (int x = 0; x < 8 / kAtOnce; ++x)
            asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"((to ^ (x * kAtOnce << 4)) + x * kAtOnce * 128),
                         "l"(from + x * step), "r"(x * kAtOnce < rows ? 16 : 0)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++issued > kLag) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
          arrive();
        }
        if (++slot == Sh::kSlots) { slot = 0; phase ^= 1; }
        return true;
      };
      bool ok = w.nmax == 0 || load(0, c.k);
      for (int j = 0; ok && j < w.nmax; ++j) {
        // in the order of use: with two tiles V(j), K(j + 1); with one K(j + 1), V(j)
        if (NT == 2) ok = load(j, c.v) && (j + 1 == w.nmax || load(j + 1, c.k));
        else ok = (j + 1 == w.nmax || load(j + 1, c.k)) && load(j, c.v);
      }
      if (!ok) s_dead = 1;
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (ok)
        for (int x = min(issued, kLag); x > 0; --x) arrive();
    } else if (warp == kMma) {
      asm volatile("bar.sync 1, %0;" ::"n"(128 * NT + 32) : "memory");       // Q is in shared memory
      tc_fence_after();
      constexpr bool bf16 = __is_same(T, __nv_bfloat16);
      constexpr uint32_t id_s = idesc_f16(kRows, BN, bf16, false), id_o = idesc_f16(kRows, HD, bf16, true);
      constexpr uint32_t kGroup = kRows * 128 / 16, kKeys = BN * 128 / 16;   // a 64-column group's bytes in descriptor units
      // (the whole warp runs this part: the elected lane issues, and commits what it issued)
      const uint32_t leader = elect_one();
      const uint64_t q_desc = sdesc_k128(smem_u32(s_q)), k_desc = sdesc_k128(smem_u32(s_kv)),
                     v_desc = sdesc_mn128(smem_u32(s_kv), BN * 128);
      int slot = 0, phase = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, int parity) {
        return ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, c.err, kErrPromptWait, a.spin));
      };
      auto next = [&] {
        if (++slot == Sh::kSlots) { slot = 0; phase ^= 1; }
      };
      // S = Q K^T of tile t with the keys in `at`, into buffer `buf`
      auto scores = [&](int t, int at, int buf) {
        const uint64_t q = q_desc + t * (Sh::kQ / 16), k = k_desc + at * (Sh::kMat / 16);
#pragma unroll
        for (int x = 0; x < HD / 16; ++x)
          mma_f16(tmem + Sh::kS + buf * BN, q + (x >> 2) * kGroup + 2 * (x & 3), k + (x >> 2) * kKeys + 2 * (x & 3), id_s,
                  x > 0, leader);
        mma_commit_if(&s_sfull[buf], leader);
      };
      // part h of O += P V: the probabilities come in kParts, so that the first can be multiplied while the
      // rest is still being exponentiated
      auto values = [&](int t, int at, int buf, bool more, int h) {
        const uint64_t v = v_desc + at * (Sh::kMat / 16);
#pragma unroll
        for (int x = h * (BN / 16 / Sh::kParts); x < (h + 1) * (BN / 16 / Sh::kParts); ++x)
          mma_f16_ta(tmem + Sh::kO + t * HD, tmem + Sh::kS + buf * BN + 8 * x, v + x * 128, id_o, more || x > 0, leader);
        if (h == Sh::kParts - 1) mma_commit_if(&s_odone[t], leader);
      };
      if (w.nmax && wait(&s_full[0], 0)) {
        tc_fence_after();
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (w.nb[t]) scores(t, 0, t);
        mma_commit_if(&s_free[0], leader);
        next();
      }
      for (int j = 0; ok && j < w.nmax; ++j) {
        if constexpr (NT == 2) {
          const int vs = slot, vph = phase;
          next();
          const int ks = slot, kph = phase;
          const bool more = j + 1 < w.nmax;
          if (more) next();
          bool have_v = false, have_k = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || j >= w.nb[t]) continue;
            if (!have_v && !wait(&s_full[vs], vph)) continue;
            have_v = true;
#pragma unroll
            for (int h = 0; h < Sh::kParts; ++h)
              if (wait(&s_pfull[2 * t + h], j & 1)) {
                tc_fence_after();
                values(t, vs, t, j > 0, h);
              }
            if (t == 1 || j >= w.nb[1]) mma_commit_if(&s_free[vs], leader);       // the last tile that reads it
            if (ok && j + 1 < w.nb[t] && (have_k || wait(&s_full[ks], kph))) {
              have_k = true;
              scores(t, ks, t);
            }
          }
          if (more) mma_commit_if(&s_free[ks], leader);
        } else {
          if (j + 1 < w.nmax) {
            if (!wait(&s_full[slot], phase)) break;
            tc_fence_after();
            scores(0, slot, (j + 1) & 1);
            mma_commit_if(&s_free[slot], leader);
            next();
          }
          if (!wait(&s_full[slot], phase) || !wait(&s_pfull[2 * (j & 1)], j >> 1 & 1)) break;
          tc_fence_after();
          values(0, slot, j & 1, j > 0, 0);
          mma_commit_if(&s_free[slot], leader);
          next();
        }
      }
      if (!ok) s_dead = 1;
      mma_commit_if(&s_end, leader);               // nothing this warp issued is still running when the block ends
      mbar_wait(&s_end, 0, c.err, kErrPromptWait);
    }
    __syncthreads();
    __syncthreads();                               // the outputs are out of TMEM
    tc_fence_after();
    if (warp == kMma) tmem_dealloc(tmem, 512);
    return;
  }

  // ---- softmax: thread = row
  if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
  const int t = NT == 2 ? warp >> 2 : 0, r = threadIdx.x & 127;
  // (this tile's entries by selection: an index known only at run time would put them into local memory)
  const int w_tok = t ? w.tok[1] : w.tok[0], w_ntok = t ? w.ntok[1] : w.ntok[0], w_end = t ? w.end[1] : w.end[0],
            n = t ? w.nb[1] : w.nb[0];
  const uint32_t lanes = (uint32_t)(warp & 3) << 21;                     // this warp's TMEM lanes, 32 (warp % 4) on
  const int tok = r / w.hb, h = w.h0 + r - tok * w.hb;
  const bool mine = tok < w_ntok;
  const int p = mine ? w.len - w.n + w_tok + tok : -1;
  float l = 0.0f;
  // the query rows into shared memory (16-byte pieces, 128-byte swizzle); a negative scale goes into their signs
  const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0u;
  // A warp copies its 32 rows, consecutive lanes consecutive pieces; rows without a token read as zeros
  constexpr int kPieces = HD / 8, kLanes = kPieces < 32 ? kPieces : 32, kAtOnce = 32 / kLanes;
  const int64_t row = w.row0 + w_tok + tok;
  const int64_t from_q = 2 * (mine ? row * a.qr + (int64_t)h * a.qh : 0);
  const uint32_t live = __ballot_sync(0xFFFFFFFFu, mine);
#pragma unroll 8
  for (int x = 0; x < 32; x += kAtOnce) {
    const int lr = x + lane / kLanes, rr = (warp & 3) * 32 + lr, piece = lane % kLanes;
    const uint32_t to = smem_u32(s_q) + t * Sh::kQ + (piece >> 3) * kRows * 128 + rr * 128 + (((piece & 7) ^ (rr & 7)) << 4);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to),
                 "l"(a.q + __shfl_sync(0xFFFFFFFFu, from_q, lr) + 16 * piece), "r"(live >> lr & 1 ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (flip) {
    __syncwarp();
    for (int x = 0; x < kPieces; ++x) {
      uint4* v = reinterpret_cast<uint4*>(s_q + t * Sh::kQ + (x >> 3) * kRows * 128 + r * 128 + (x & 7) * 16);
      v->x ^= flip; v->y ^= flip; v->z ^= flip; v->w ^= flip;
    }
  }
  fence_async_shared();
  asm volatile("bar.sync 1, %0;" ::"n"(128 * NT + 32) : "memory");
  const float scale2 = fabsf(a.scale2);
  const int pmin = w.len - w.n + w_tok, pmax = w_end - 1;
  const int from = first_in_window(p + 1, a.window);
  // fp16 probabilities are kept 2^7 times as large (the running maximum may be behind by 2^8: below 2^15), which takes
  // the smallest that is not lost from 2^-25 of the maximum to 2^-32; the sum is 2^7 times as large as well
  constexpr float lift = __is_same(T, __half) ? 7.0f : 0.0f;
  float m = neg_inf();
  bool ok = true;
  for (int j = 0; j < n; ++j) {
    const int buf = NT == 2 ? t : j & 1, ph = NT == 2 ? j & 1 : j >> 1 & 1;
    ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_sfull[buf], ph, c.err, kErrPromptWait, a.spin));
    if (!ok) break;
    tc_fence_after();
    const uint32_t st = tmem + lanes + Sh::kS + buf * BN;
    uint32_t v[BN];
#pragma unroll
    for (int x = 0; x < BN; x += 32) tmem_ld32(st + x, v + x);
    tmem_wait_ld();
#pragma unroll
    for (int x = 0; x < BN; ++x) asm volatile("" : "+r"(v[x]));        // no use moves before the wait
    const int j0 = w.block(j) * BN;
    const bool masked = j0 + BN - 1 > pmin || (pmax - j0 >= a.window && j0 + BN > a.sinks);
    if (masked) {
      const int hi = p + 1 - j0, lo = from - j0, sk = a.sinks - j0;
#pragma unroll
      for (int x = 0; x < BN; ++x)
        if (!(x < hi && (x >= lo || x < sk))) v[x] = 0xFF800000u;
    }
    float mx[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
    for (int x = 0; x < BN; x += 2) mx[x >> 1 & 3] = max3(mx[x >> 1 & 3], __uint_as_float(v[x]), __uint_as_float(v[x + 1]));
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
    const bool grow = top > m + 8.0f || (m == neg_inf() && top > m);
    if (__any_sync(0xFFFFFFFFu, grow)) {
      const float f = grow ? ex2(m - top) : 1.0f;
      if (grow) m = top;
      l *= f;
      if (j > 0) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_odone[t], (j - 1) & 1, c.err, kErrPromptWait, a.spin));
        if (!ok) break;
        tc_fence_after();
        const uint32_t ot = tmem + lanes + Sh::kO + t * HD;
#pragma unroll
        for (int x = 0; x < HD; x += 32) {
          uint32_t o[32];
          tmem_ld32(ot + x, o);
          tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 32; ++y) {
            asm volatile("" : "+r"(o[y]));
            o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
          }
          tmem_st32(ot + x, o);
        }
      }
    }
    const float base = m == neg_inf() ? 0.0f : m - lift;
    constexpr int kN = BN / Sh::kParts;
#pragma unroll
    for (int h = 0; h < Sh::kParts; ++h) {
      l += masked ? exponentials<T, kN, false>(v + h * kN, v + h * kN / 2, scale2, base)
                  : exponentials<T, kN, true>(v + h * kN, v + h * kN / 2, scale2, base);
      tmem_st32(st + h * kN / 2, v + h * kN / 2);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_pfull[2 * buf + h]);
    }
  }
  if (ok && n) ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s_odone[t], (n - 1) & 1, c.err, kErrPromptWait, a.spin));
  if (!ok) s_dead = 1;
  __syncthreads();
  tc_fence_after();
  if (!s_dead) {
    const bool any = p >= 0;
    const float inv = any ? 1.0f / l : 0.0f;       // (scores of -infinity alone: 0 / 0)
    const bool sure = m == neg_inf() || (l != l && scale2 != 0.0f);
    float most = 0.0f;                             // NaN once an output is
    // the warp's rows go out through the query tile's place (no tensor core reads it any more), so
    // that consecutive lanes store consecutive pieces of a row
    uint8_t* mine_at = s_q + t * Sh::kQ + r * 128;
#pragma unroll
    for (int x = 0; x < HD; x += 32) {
      uint32_t o[32];
      if (n) {
        tmem_ld32(tmem + lanes + Sh::kO + t * HD + x, o);
        tmem_wait_ld();
      }
      uint32_t pk[16];
#pragma unroll
      for (int y = 0; y < 32; y += 2) {
        asm volatile("" : "+r"(o[y]), "+r"(o[y + 1]));
        const float o0 = any ? __uint_as_float(o[y]) * inv : 0.0f, o1 = any ? __uint_as_float(o[y + 1]) * inv : 0.0f;
        most = max3_nan(most, o0, o1);
        pk[y >> 1] = Elem<T>::pack(o0, o1);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int piece = x / 8 + y;
        *reinterpret_cast<uint4*>(mine_at + (piece >> 3) * kRows * 128 + (((piece & 7) ^ (r & 7)) << 4)) =
            make_uint4(pk[4 * y], pk[4 * y + 1], pk[4 * y + 2], pk[4 * y + 3]);
      }
    }
    __syncwarp();
    const int64_t to_out = 2 * (mine ? row * a.orow + (int64_t)h * a.oh : 0);
#pragma unroll 8
    for (int x = 0; x < 32; x += kAtOnce) {
      const int lr = x + lane / kLanes, rr = (warp & 3) * 32 + lr, piece = lane % kLanes;
      const int64_t to = __shfl_sync(0xFFFFFFFFu, to_out, lr) + 16 * piece;
      if (live >> lr & 1)
        *reinterpret_cast<uint4*>(a.out + to) = *reinterpret_cast<const uint4*>(
            s_q + t * Sh::kQ + (piece >> 3) * kRows * 128 + rr * 128 + (((piece & 7) ^ (rr & 7)) << 4));
    }
    __syncwarp();
    uint32_t redo = __ballot_sync(0xFFFFFFFFu, mine && any && (s_bad || (is_nan(most) && !sure)));
    while (redo) {
      const int from_lane = __ffs(redo) - 1;
      redo &= redo - 1;
      redo_row<T, HD>(a, w.b, w.kvh, __shfl_sync(0xFFFFFFFFu, row, from_lane), __shfl_sync(0xFFFFFFFFu, h, from_lane),
                      __shfl_sync(0xFFFFFFFFu, p, from_lane) + 1);
    }
  }
  tc_fence_before();
  __syncthreads();
}

template <class T, int HD, bool TMA>
cudaError_t prompt_hd(const AttendArgs& a, cudaStream_t st) {
  using Sh = PromptShape<HD>;
  const KvCache& c = a.c;
  PromptMaps maps{};
  const int box = std::min(Sh::kBlock, 1 << c.shift);
  if (TMA && (!make_map_pool(&maps.k, c, c.k, box) || !make_map_pool(&maps.v, c, c.v, box))) return cudaErrorInvalidValue;
  const cudaError_t e = allow_smem<k_prompt<T, HD, TMA>>(Sh::kSmem);
  if (e != cudaSuccess) return e;
  // a group's heads in blocks of nearly equal size; as many tokens as fill a tile with them
  const int G = a.nh / c.n_kv, gblocks = (G + kMaxHeads - 1) / kMaxHeads, hb = (G + gblocks - 1) / gblocks;
  const int tokens = kRows / hb, span = Sh::kTiles * tokens;
  // every sequence ends in at most one span that is not full
  const int64_t pairs = std::min<int64_t>(a.tokens, a.tokens / span + std::min(a.tokens, c.batch));
  const int64_t grid = pairs * c.n_kv * gblocks;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  k_prompt<T, HD, TMA><<<(unsigned)grid, Sh::kThreads, Sh::kSmem, st>>>(maps, a, gblocks, hb, tokens);
  return cudaGetLastError();
}

template <class T>
cudaError_t prompt_of(const AttendArgs& a, cudaStream_t st) {
  const bool tma = 1 << a.c.shift >= kTmaPage;
  switch (a.c.hd) {
    case 64: return tma ? prompt_hd<T, 64, true>(a, st) : prompt_hd<T, 64, false>(a, st);
    case 128: return tma ? prompt_hd<T, 128, true>(a, st) : prompt_hd<T, 128, false>(a, st);
    default: return tma ? prompt_hd<T, 256, true>(a, st) : prompt_hd<T, 256, false>(a, st);
  }
}

}  // namespace

cudaError_t launch_attend_prompt(const AttendArgs& a, cudaStream_t st) {
  return a.dtype == TC_BF16 ? prompt_of<__nv_bfloat16>(a, st) : prompt_of<__half>(a, st);
}

}  // namespace tc
