// Attention of one query row per sequence over the paged cache (tc_attend).
//
// The G = n_heads / n_kv heads of a key-value head read the same rows, so they are the rows of one
// warp MMA (m16n8k16; more than 16 go in blocks of 16): each key and value row crosses HBM once and the
// kernel is bound by that stream. The work of a call is one list of tiles of 64 slots - sequence by
// sequence, key-value head by key-value head, only tiles with a visible slot - cut into equal runs,
// one per CTA and one CTA per SM: ragged batches and a single long sequence fill the GPU alike. Every
// CTA derives its run from the lengths (a scan of the batch); nothing is planned on the host.
//   warp 4     producer: the tile's key and value rows by TMA (64 x page rows boxes, 128-byte
//              swizzle) into a ring of stages; a lane per box
//   warps 0-3  16 of a tile's 64 slots each, with running maximum, sum and output of their own:
//              S = Q K^T from ldmatrix, p = 2^(s - m), O += P V with P split in two 16-bit parts (the
//              probabilities keep 16 bits and more at the price of MMAs that the memory bound hides)
// At an item's end the four warps' states are joined through shared memory. An item that lies in one
// CTA's run is stored at once; of the others every CTA writes its state (maximum, sum, 16 x HD fp32)
// to the workspace, and k_join, launched early as a dependent, combines them in run order: no atomics,
// the same bits every time.
#include <cuda_runtime.h>

#include <algorithm>

#include "attend_row.cuh"
#include "mma.h"
#include "paged_map.h"
#include "pdl.cuh"
#include "umma.cuh"

namespace tc {
namespace {

constexpr int kTile = 64, kConsumers = 4, kAttendThreads = 32 * (kConsumers + 1), kRowsMma = 16, kMaxGrid = 148;

template <int HD>
struct AttendShape {
  static constexpr int kHalves = HD / 64;                    // 128-byte column groups of a row
  static constexpr int kMat = kTile * HD * 2;                // bytes of a tile's keys (or values)
  static constexpr int kStages = HD == 64 ? 8 : HD == 128 ? 5 : 3;
  static constexpr int kJoin = 2 * kRowsMma * HD * 4;        // two warps' outputs
  static constexpr int kSmem = 1024 + kStages * 2 * kMat + kJoin;
  static constexpr int kPart = kRowsMma * HD + 2 * kRowsMma; // floats of a CTA's state of an item
};

// Where one sequence's visible slots lie: [0, head) and [first, len), in nt tiles: tiles 0 .. na - 1,
// then from t0 on.
struct SeqTiles {
  int len, first, head, na, t0, nt;
  __device__ __forceinline__ SeqTiles(const AttendArgs& a, int b) {
    len = kv_length(a.c, b, kErrAttend);
    first = first_in_window(len, a.window);
    head = min(a.sinks, first);
    t0 = first / kTile;
    na = min((head + kTile - 1) / kTile, t0);
    nt = len ? na + (len + kTile - 1) / kTile - t0 : 0;
  }
  __device__ __forceinline__ int tile(int i) const { return i < na ? i : t0 + i - na; }
  __device__ __forceinline__ bool visible(int j) const { return j < len && (j >= first || j < head); }
};

struct PlanShared {
  long long warp[8];
  long long into;
  int b;
};
// The tiles of the whole call are cut into runs of total / runs (rounded down) and one more; there are
// never more runs than tiles, so none is empty.
__device__ __forceinline__ int runs_of(long long total, int grid) { return (int)min(total, (long long)grid); }
__device__ __forceinline__ long long run_begin(long long total, int runs, int i) { return total * i / runs; }
// The run that holds tile t: the last one that begins at or before it.
__device__ __forceinline__ int run_of(long long total, int runs, long long t) { return (int)(((t + 1) * runs - 1) / total); }

// The tiles of the whole call (every thread of the CTA calls it; at most 256 threads), and *before: the
// tiles before sequence `want`; or, want < 0, s.b = the sequence that holds the first tile of run
// `run` and the tiles of it before that one.
__device__ __forceinline__ long long plan(const AttendArgs& a, int nsub, PlanShared& s, int want, int run, int grid,
                                          long long* before) {
  const int T = blockDim.x, t = threadIdx.x, B = a.c.batch, per = (B + T - 1) / T;
  const int lo = min(B, t * per), hi = min(B, lo + per), warp = t >> 5, lane = t & 31;
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += (long long)SeqTiles(a, b).nt * nsub;
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += y;
  }
  if (lane == 31) s.warp[warp] = sum;
  __syncthreads();
  long long base = 0, total = 0;
  for (int w = 0; w < T / 32; ++w) {
    if (w < warp) base += s.warp[w];
    total += s.warp[w];
  }
  long long at = base + sum - mine;                          // tiles before this thread's sequences
  const int runs = runs_of(total, grid);
  const long long find = want < 0 && run < runs ? run_begin(total, runs, run) : total;
  if (want < 0 ? mine && find >= at && find < at + mine : want >= lo && want < hi) {
    int b = lo;
    for (;; ++b) {
      if (b == want) break;
      const long long n = (long long)SeqTiles(a, b).nt * nsub;
      if (want < 0 && find < at + n) break;
      at += n;
    }
    s.b = b;
    s.into = want < 0 ? find - at : at;
  }
  __syncthreads();
  *before = s.into;
  return total;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The factor a state kept at maximum m takes at maximum m2 >= m (1 where both are still -infinity).
__device__ __forceinline__ float shrink(float m, float m2) { return m2 == neg_inf() ? 1.0f : ex2(m - m2); }

struct AttendMaps {
  CUtensorMap k, v;
};
// What a call keeps in its workspace: the CTAs' states, the scores and the final statistics.
struct AttendWs {
  float* part;
  int* redo;                         // per item that one CTA holds whole: an output is not finite
  float2* ml;
  float* scores;
  int64_t cap;                       // slots a row of scores holds
};

// A warp's running state over its slots: rows r = lane / 4 and r + 8 of the head block.
template <int HD>
struct State {
  float o[HD / 8][4];
  float m[2], l[2];                  // l: this lane's share of the row's sum
  bool any;                          // a visible slot was met
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    m[0] = m[1] = neg_inf();
    l[0] = l[1] = 0.0f;
    any = false;
  }
  __device__ __forceinline__ void scale(float f0, float f1) {
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      o[n][0] *= f0; o[n][1] *= f0;
      o[n][2] *= f1; o[n][3] *= f1;
    }
    l[0] *= f0;
    l[1] *= f1;
  }
};

template <class T, int HD>
__global__ void __launch_bounds__(kAttendThreads, 1)
    k_attend(const __grid_constant__ AttendMaps maps, const __grid_constant__ AttendArgs a, AttendWs ws, int rows_box) {
  using Sh = AttendShape<HD>;
  extern __shared__ uint8_t s_raw[];
  __shared__ __align__(8) uint64_t s_full[Sh::kStages], s_free[Sh::kStages];
  __shared__ uint32_t s_valid[Sh::kStages];
  __shared__ float s_ml[kConsumers][2][kRowsMma];
  __shared__ PlanShared s_plan;
  __shared__ int s_dead;
  griddep_launch();                               // k_join may take its place and wait
  const KvCache& c = a.c;
  uint8_t* s_tiles = s_raw + (1024 - (smem_u32(s_raw) & 1023)) % 1024;
  float* s_join = reinterpret_cast<float*>(s_tiles + Sh::kStages * 2 * Sh::kMat);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Sh::kStages; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kConsumers);
    }
    mbar_fence_init();
    s_dead = 0;
  }
  const int G = a.nh / c.n_kv, gblocks = (G + kRowsMma - 1) / kRowsMma, nsub = c.n_kv * gblocks;
  long long into = 0;
  const long long total = plan(a, nsub, s_plan, -1, blockIdx.x, gridDim.x, &into);   // (also orders the barriers' setup)
  const int runs = runs_of(total, gridDim.x);
  if ((int)blockIdx.x >= runs) return;
  int b = s_plan.b, left = (int)(run_begin(total, runs, blockIdx.x + 1) - run_begin(total, runs, blockIdx.x));
  SeqTiles sq(a, b);
  int sub = (int)(into / sq.nt), i = (int)(into - (long long)sub * sq.nt);
  int stage = 0, phase = 0;
  if (warp == kConsumers) {
    int issued = 0;
    bool dead = false;
    for (; left > 0 && !dead; --left) {
      const int kvh = sub / gblocks, j0 = sq.tile(i) * kTile;
      // one lane per box: rows_box slots of one 64-column group of the keys or the values
      const int chunks = kTile / rows_box, boxes = 2 * chunks * Sh::kHalves;
      bool ok = issued < Sh::kStages || mbar_wait(&s_free[stage], phase ^ 1, c.err, kErrAttendWait, a.spin);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) {
        dead = true;
        break;
      }
      // 16-slot groups with a visible slot on a page of the pool; a box is loaded if it has one
      uint32_t mine = 0;
      int page = -1;
      if (lane < 4) {
        const int j = j0 + 16 * lane;
        const bool seen = j < sq.len && (j + 16 > sq.first || j < sq.head);
        if (seen) page = kv_page(c, b, j, kErrAttend);
        mine = page >= 0;
      }
      const uint32_t valid = __ballot_sync(0xFFFFFFFFu, mine);
      auto groups = [&](int u) { return valid >> (u * rows_box / 16) & ((1u << rows_box / 16) - 1); };   // of box u
      uint32_t bytes = 0;
      for (int u = 0; u < chunks; ++u) bytes += groups(u) ? rows_box * HD * 4 : 0;
      if (lane == 0) {
        s_valid[stage] = valid;
        mbar_expect_tx(&s_full[stage], bytes);
      }
      __syncwarp();
      const uint32_t base = smem_u32(s_tiles) + stage * 2 * Sh::kMat;
      for (int x0 = 0; x0 < boxes; x0 += 32) {
        const int x = min(x0 + lane, boxes - 1);
        const int u = x / (2 * Sh::kHalves), r = x - u * 2 * Sh::kHalves, half = r >> 1, is_v = r & 1;
        const uint32_t here = groups(u);                     // a box lies in one page: that of its first seen group
        const int pg = __shfl_sync(0xFFFFFFFFu, page, here ? u * rows_box / 16 + __ffs(here) - 1 : 0);
        if (here && x0 + lane < boxes)
          tma_load_4d(base + is_v * Sh::kMat + half * kTile * 128 + u * rows_box * 128, is_v ? &maps.v : &maps.k,
                      64 * half, (j0 + u * rows_box) & ((1 << c.shift) - 1), kvh, pg, &s_full[stage]);
      }
      ++issued;
      if (++stage == Sh::kStages) { stage = 0; phase ^= 1; }
      if (++i == sq.nt) {
        i = 0;
        if (++sub == nsub && left > 1) {
          sub = 0;
          do sq = SeqTiles(a, ++b);
          while (sq.nt == 0);
        }
      }
    }
    // no copy is in flight when the block ends: the last use of every stage has arrived
    for (int k = 0; k < Sh::kStages && k < issued; ++k) {
      if (--stage < 0) { stage = Sh::kStages - 1; phase ^= 1; }
      mbar_wait(&s_full[stage], phase, c.err, kErrAttendWait);
    }
    return;
  }

  bool dead = false;
  while (left > 0) {
    const int kvh = sub / gblocks, h0 = kvh * G + (sub - kvh * gblocks) * kRowsMma, rows = min(kRowsMma, (kvh + 1) * G - h0);
    // the query rows' fragments: rows lane / 4 and + 8, columns 2 (lane % 4) (+ 1, + 8, + 9) of each 16
    uint32_t q[HD / 16][4];
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = (lane >> 2) + (x & 1) * 8, col = 16 * kk + 2 * (lane & 3) + (x >> 1) * 8;
        q[kk][x] = 0;
        if (r < rows)
          q[kk][x] = __ldg(reinterpret_cast<const uint32_t*>(a.q + 2 * ((int64_t)b * a.qr + (int64_t)(h0 + r) * a.qh + col)));
      }
    State<HD> st;
    st.clear();
    const int i0 = i, n = min(left, sq.nt - i);
    for (int k = 0; k < n; ++k, ++i) {
      if (!dead) dead = !__all_sync(0xFFFFFFFFu, mbar_wait(&s_full[stage], phase, c.err, kErrAttendWait, a.spin));
      if (!dead && (s_valid[stage] >> warp & 1)) {
        const int j0 = sq.tile(i) * kTile + 16 * warp;
        const uint32_t kt = smem_u32(s_tiles) + stage * 2 * Sh::kMat + 16 * warp * 128, vt = kt + Sh::kMat;
        st.any = true;
        const bool whole = j0 + 16 <= sq.len && (j0 >= sq.first || j0 + 16 <= sq.head);
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          // matrices: slots 0-7 | 8-15 x columns 0-7 | 8-15
          const int r = (lane & 7) + (lane >> 4) * 8, c16 = (kk & 3) * 2 + (lane >> 3 & 1);
          uint32_t f[4];
          ldsm4(kt + (kk >> 2) * kTile * 128 + r * 128 + ((c16 ^ (r & 7)) << 4), f);
          mma16816<T>(s[0], q[kk], f[0], f[1]);
          mma16816<T>(s[1], q[kk], f[2], f[3]);
        }
        bool show[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) show[t][e] = whole || sq.visible(j0 + 8 * t + 2 * (lane & 3) + e);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] = show[t][e & 1] ? s[t][e] * a.scale2 : neg_inf();
        if (ws.scores) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int r = (lane >> 2) + 8 * y;
            if (r < rows) {
              float* to = ws.scores + ((int64_t)b * a.nh + h0 + r) * ws.cap + j0 + 2 * (lane & 3);
              *reinterpret_cast<float2*>(to) = make_float2(s[0][2 * y], s[0][2 * y + 1]);
              *reinterpret_cast<float2*>(to + 8) = make_float2(s[1][2 * y], s[1][2 * y + 1]);
            }
          }
        }
        if (!whole) {
          // a hidden slot's value row may hold anything, and 0 x NaN is not 0: it is cleared here
          for (int r = 0; r < 16; ++r)
            if (!sq.visible(j0 + r))
              for (int x = lane; x < HD / 8; x += 32)
                *reinterpret_cast<uint4*>(s_tiles + stage * 2 * Sh::kMat + Sh::kMat + (x >> 3) * kTile * 128 +
                                          (16 * warp + r) * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_async_shared();
          __syncwarp();
        }
        float m2[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float m = fmaxf(fmaxf(s[0][2 * y], s[0][2 * y + 1]), fmaxf(s[1][2 * y], s[1][2 * y + 1]));
          m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
          m2[y] = fmaxf(st.m[y], m);
        }
        if (__any_sync(0xFFFFFFFFu, m2[0] > st.m[0] || m2[1] > st.m[1])) {
          st.scale(shrink(st.m[0], m2[0]), shrink(st.m[1], m2[1]));
          st.m[0] = m2[0];
          st.m[1] = m2[1];
        }
        const float at[2] = {m2[0] == neg_inf() ? 0.0f : m2[0], m2[1] == neg_inf() ? 0.0f : m2[1]};
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) p[t][e] = show[t][e & 1] ? ex2(s[t][e] - at[e >> 1]) : 0.0f;
        st.l[0] += (p[0][0] + p[0][1]) + (p[1][0] + p[1][1]);
        st.l[1] += (p[0][2] + p[0][3]) + (p[1][2] + p[1][3]);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float p0 = p[x >> 1][(x & 1) * 2], p1 = p[x >> 1][(x & 1) * 2 + 1];
          hi[x] = Elem<T>::pack(p0, p1);
          const float2 f = Elem<T>::f2(hi[x]);
          lo[x] = Elem<T>::pack(p0 - f.x, p1 - f.y);
        }
#pragma unroll
        for (int nn = 0; nn < HD / 16; ++nn) {
          // matrices: slots 0-7 | 8-15 of columns 0-7, then of columns 8-15
          const int r = lane & 15, c16 = (nn & 3) * 2 + (lane >> 4);
          uint32_t f[4];
          ldsm4t(vt + (nn >> 2) * kTile * 128 + r * 128 + ((c16 ^ (r & 7)) << 4), f);
          mma16816<T>(st.o[2 * nn], hi, f[0], f[1]);
          mma16816<T>(st.o[2 * nn + 1], hi, f[2], f[3]);
          mma16816<T>(st.o[2 * nn], lo, f[0], f[1]);
          mma16816<T>(st.o[2 * nn + 1], lo, f[2], f[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[stage]);
      if (++stage == Sh::kStages) { stage = 0; phase ^= 1; }
    }
    // the four warps' states, joined at their common maximum: 2 into 0 and 3 into 1, then 1 into 0
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      st.l[y] += __shfl_xor_sync(0xFFFFFFFFu, st.l[y], 1);
      st.l[y] += __shfl_xor_sync(0xFFFFFFFFu, st.l[y], 2);
      if ((lane & 3) == 0) s_ml[warp][0][(lane >> 2) + 8 * y] = st.m[y];
    }
    if (dead && lane == 0) s_dead = 1;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    float m[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int r = (lane >> 2) + 8 * y;
      m[y] = fmaxf(fmaxf(s_ml[0][0][r], s_ml[1][0][r]), fmaxf(s_ml[2][0][r], s_ml[3][0][r]));
    }
    st.scale(shrink(st.m[0], m[0]), shrink(st.m[1], m[1]));
    if ((lane & 3) == 0) {
      s_ml[warp][1][lane >> 2] = st.any ? st.l[0] : -1.0f;
      s_ml[warp][1][(lane >> 2) + 8] = st.any ? st.l[1] : -1.0f;
    }
    float4* mine = reinterpret_cast<float4*>(s_join) + (warp & 1) * (kRowsMma * HD / 4);
    auto give = [&] {
#pragma unroll
      for (int x = 0; x < HD / 8; ++x) mine[x * 32 + lane] = make_float4(st.o[x][0], st.o[x][1], st.o[x][2], st.o[x][3]);
    };
    auto take = [&](const float4* from) {
#pragma unroll
      for (int x = 0; x < HD / 8; ++x) {
        const float4 f = from[x * 32 + lane];
        st.o[x][0] += f.x; st.o[x][1] += f.y; st.o[x][2] += f.z; st.o[x][3] += f.w;
      }
    };
    if (warp >= 2) give();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (warp < 2) take(mine);
    if (warp == 1) {
      __syncwarp();
      give();
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (warp == 0 && !s_dead) {
      take(mine + kRowsMma * HD / 4);
      const bool all = i0 == 0 && n == sq.nt;
      float* part = ws.part + ((int64_t)blockIdx.x * 2 + (i0 == 0)) * Sh::kPart;
      bool good = true;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int r = (lane >> 2) + 8 * y;
        float l = 0.0f;
        bool any = false;
#pragma unroll
        for (int w = 0; w < kConsumers; ++w) {
          const float x = s_ml[w][1][r];
          if (!(x < 0.0f)) {                     // (a warp that met no visible slot says -1)
            l += x;
            any = true;
          }
        }
        const float inv = any ? 1.0f / l : 0.0f;
        if (r < rows) {
          uint8_t* to = a.out + 2 * ((int64_t)b * a.orow + (int64_t)(h0 + r) * a.oh);
#pragma unroll
          for (int x = 0; x < HD / 8; ++x) {
            const int col = 8 * x + 2 * (lane & 3);
            const float o0 = st.o[x][2 * y], o1 = st.o[x][2 * y + 1];
            if (all) {
              good &= fabsf(o0 * inv) + fabsf(o1 * inv) < __int_as_float(0x7F800000);
              *reinterpret_cast<uint32_t*>(to + 2 * col) = Elem<T>::pack(o0 * inv, o1 * inv);
            } else {
              *reinterpret_cast<float2*>(part + r * HD + col) = make_float2(o0, o1);
            }
          }
          if ((lane & 3) == 0) {
            if (!all) {
              part[kRowsMma * HD + r] = m[y];
              part[kRowsMma * HD + kRowsMma + r] = any ? l : -1.0f;
            } else if (ws.ml) {
              ws.ml[(int64_t)b * a.nh + h0 + r] = make_float2(m[y], l);
            }
          }
        }
      }
      good = __all_sync(0xFFFFFFFFu, good);
      if (all && lane == 0) ws.redo[(int64_t)b * nsub + sub] = !good;
    }
    left -= n;
    if (i == sq.nt) {
      i = 0;
      if (++sub == nsub && left > 0) {
        sub = 0;
        do sq = SeqTiles(a, ++b);
        while (sq.nt == 0);
      }
    }
  }
}

// The items whose tiles lie in several CTAs' runs: their states at the common maximum, in run order.
// Sequences without a slot get zeros. One CTA per (sequence, head block), a warp per row in turn. A row
// with a NaN or an infinity is computed again key by key: the second half of a split probability times
// an infinite value would make a NaN of it.
constexpr int kJoinThreads = 256;
template <class T, int HD>
__global__ void __launch_bounds__(kJoinThreads) k_join(const __grid_constant__ AttendArgs a, AttendWs ws, int grid) {
  using Sh = AttendShape<HD>;
  __shared__ PlanShared s_plan;
  griddep_launch();
  const KvCache& c = a.c;
  const int G = a.nh / c.n_kv, gblocks = (G + kRowsMma - 1) / kRowsMma, nsub = c.n_kv * gblocks;
  const int b = blockIdx.x / nsub, sub = blockIdx.x - b * nsub;
  const int kvh = sub / gblocks, h0 = kvh * G + (sub - kvh * gblocks) * kRowsMma, rows = min(kRowsMma, (kvh + 1) * G - h0);
  long long at = 0;
  const long long total = plan(a, nsub, s_plan, b, 0, 1, &at);
  const int nt = SeqTiles(a, b).nt;
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (nt == 0) {
    for (int r = warp; r < rows; r += kJoinThreads / 32)
      for (int x = lane; x < HD / 2; x += 32)
        *reinterpret_cast<uint32_t*>(a.out + 2 * ((int64_t)b * a.orow + (int64_t)(h0 + r) * a.oh) + 4 * x) = 0;
    return;
  }
  const long long t0 = at + (long long)sub * nt;
  const int runs = runs_of(total, grid), c0 = run_of(total, runs, t0), c1 = run_of(total, runs, t0 + nt - 1);
  const bool redo = c0 == c1 && ws.redo[blockIdx.x];
  if (c0 == c1 && !redo) return;
  for (int r = warp; r < rows; r += kJoinThreads / 32) {
    float m = neg_inf(), l = 0.0f, o[HD / 32] = {};
    bool any = false;
    for (int k = c0; k <= c1 && !redo; ++k) {
      const float* part = ws.part + ((int64_t)k * 2 + (k == c0)) * Sh::kPart;
      const float mk = part[kRowsMma * HD + r], lk = part[kRowsMma * HD + kRowsMma + r];
      if (lk < 0.0f) continue;
      any = true;
      const float m2 = fmaxf(m, mk), f = shrink(m, m2), g = shrink(mk, m2);
      m = m2;
      l = l * f + lk * g;
#pragma unroll
      for (int x = 0; x < HD / 64; ++x) {
        const float2 v = *reinterpret_cast<const float2*>(part + r * HD + 2 * (lane + 32 * x));
        o[2 * x] = o[2 * x] * f + v.x * g;
        o[2 * x + 1] = o[2 * x + 1] * f + v.y * g;
      }
    }
    const float inv = any ? 1.0f / l : 0.0f;
    bool good = true;
#pragma unroll
    for (int x = 0; x < HD / 32; ++x) {
      o[x] *= inv;
      good &= fabsf(o[x]) < __int_as_float(0x7F800000);
    }
    const int64_t at_out = (int64_t)b * a.orow + (int64_t)(h0 + r) * a.oh;
    if (ws.ml && lane == 0 && !redo) ws.ml[(int64_t)b * a.nh + h0 + r] = make_float2(m, l);
    if (redo || !__all_sync(0xFFFFFFFFu, good)) {
      float q[HD / 32];
      row_load<T, HD>(a.q, (int64_t)b * a.qr + (int64_t)(h0 + r) * a.qh, lane, q);
      attend_row<T, HD>(c, b, kvh, q, a.scale2, SeqTiles(a, b).len, a.window, a.sinks, kErrAttend, o);
      row_store<T, HD>(a.out, at_out, lane, o);
    } else {
      uint32_t* to = reinterpret_cast<uint32_t*>(a.out + 2 * at_out);
#pragma unroll
      for (int x = 0; x < HD / 64; ++x) to[lane + 32 * x] = Elem<T>::pack(o[2 * x], o[2 * x + 1]);
    }
  }
}

// weight_out = weight + the visible slots' probabilities, summed over the heads that share a key-value head.
constexpr int kWeightThreads = 256;
__global__ void __launch_bounds__(kWeightThreads) k_weights(const __grid_constant__ AttendArgs a, AttendWs ws) {
  griddep_wait();
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
        const float2 f = ws.ml[u];
        sum += ex2(ws.scores[u * ws.cap + j] - f.x) / f.y;
      }
      w += sum;
    }
    a.weight_out[at + j] = w;
  }
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
AttendWs ws_of(const KvCache& c, int nh, bool weights, uint8_t* ws, uint64_t* bytes) {
  AttendWs w{};
  int64_t at = 0;
  w.part = reinterpret_cast<float*>(ws);
  at += up256((int64_t)kMaxGrid * 2 * (kRowsMma * c.hd + 2 * kRowsMma) * 4);
  w.redo = reinterpret_cast<int*>(ws + at);
  at += up256((int64_t)c.batch * c.n_kv * ((nh / c.n_kv + kRowsMma - 1) / kRowsMma) * 4);
  if (weights) {
    w.ml = reinterpret_cast<float2*>(ws + at);
    at += up256((int64_t)c.batch * nh * 8);
    w.scores = reinterpret_cast<float*>(ws + at);
    w.cap = (int64_t)c.max_pages << c.shift;
    at += up256((int64_t)c.batch * nh * w.cap * 4);
  }
  *bytes = at;
  return w;
}

template <class T, int HD>
cudaError_t attend_hd(const AttendArgs& a, cudaStream_t st) {
  using Sh = AttendShape<HD>;
  const KvCache& c = a.c;
  uint64_t bytes = 0;
  const AttendWs ws = ws_of(c, a.nh, a.weight_out != nullptr, a.ws, &bytes);
  AttendMaps maps;
  const int rows_box = std::min(kTile, 1 << c.shift);
  if (!make_map_pool(&maps.k, c, c.k, rows_box) || !make_map_pool(&maps.v, c, c.v, rows_box)) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(k_attend<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
  if (e != cudaSuccess) return e;
  // no more CTAs than the page lists can hold tiles
  const int G = a.nh / c.n_kv, nsub = c.n_kv * ((G + kRowsMma - 1) / kRowsMma);
  const int64_t most = (int64_t)c.batch * nsub * ((((int64_t)c.max_pages << c.shift) + kTile - 1) / kTile);
  const int grid = (int)std::min<int64_t>(kMaxGrid, most);
  k_attend<T, HD><<<grid, kAttendThreads, Sh::kSmem, st>>>(maps, a, ws, rows_box);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = launch_dependent(k_join<T, HD>, dim3(c.batch * nsub), dim3(kJoinThreads), st, a, ws, grid)) != cudaSuccess) return e;
  if (!a.weight_out) return cudaSuccess;
  const int kvrows = c.batch * c.n_kv;
  return launch_dependent(k_weights, dim3(kvrows, std::max(1, 148 * 4 / kvrows)), dim3(kWeightThreads), st, a, ws);
}

template <class T>
cudaError_t attend_of(const AttendArgs& a, cudaStream_t st) {
  switch (a.c.hd) {
    case 64: return attend_hd<T, 64>(a, st);
    case 128: return attend_hd<T, 128>(a, st);
    default: return attend_hd<T, 256>(a, st);
  }
}

}  // namespace

uint64_t attend_workspace(const KvCache& c, int nh, bool weights) {
  uint64_t bytes = 0;
  ws_of(c, nh, weights, nullptr, &bytes);
  return bytes;
}
cudaError_t launch_attend(const AttendArgs& a, cudaStream_t st) {
  return a.dtype == TC_BF16 ? attend_of<__nv_bfloat16>(a, st) : attend_of<__half>(a, st);
}

}  // namespace tc
