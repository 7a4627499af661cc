// Attention of few query rows per sequence over the paged cache: one token each (tc_attend), or short
// chunks of a prompt (tc_attend_prompt takes longer ones to the tensor cores, k_attend_prompt.cu).
//
// The G = n_heads / n_kv heads of a key-value head read the same rows, so the heads of a token, or of a
// block of consecutive tokens, are the columns of one warp MMA (m16n8k16: 16 slots x 8 rows of q; blocks
// of at most 8 or 16 rows): each key and value row crosses HBM once and the kernel is bound by that
// stream. The work of a call is one list of chunks of 16 slots - sequence by sequence, block by block,
// key-value head by key-value head, only chunks with a visible slot - cut into equal runs, one per CTA
// and one CTA per SM: ragged batches and a single long sequence fill the GPU alike. Every CTA derives
// its run from the lengths (a scan of the batch); nothing is planned on the host. The warps of a CTA
// take the chunks of its run in turn, each with a ring of its own that it fills by cp.async (16-byte
// pieces, hidden rows as zeros: 0 x NaN is not 0) and a running maximum, sum and output of its own, so
// no warp waits for another within an item:
//   S^T = K Q^T (ldmatrix), p = 2^(s - m), O^T += V^T P^T (ldmatrix.trans) with P split in two 16-bit
//   parts: the probabilities keep 16 bits and more at the price of MMAs that the memory bound hides
// (Boxes of TMA over 16-slot pages were tried in place of cp.async: 3.46 against 4.84 TB/s with
// 64-slot pages, the boxes of 2 KB being the limit.) 64 ragged conversations of up to 8192 slots, 16
// heads on 8 of 128, bf16: 204 us over 16-slot pages, 190 us over 64-slot ones (5.4 and 5.75 TB/s).
// At an item's end the warps' states are joined through shared memory. An item that lies in one
// CTA's run is stored at once; of the others every CTA writes its state (maximum, sum, 16 x HD fp32)
// to the workspace, and k_join, launched early as a dependent, combines them in run order: no atomics,
// the same bits every time.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "attend_row.cuh"
#include "mma.h"
#include "pdl.cuh"
#include "umma.cuh"

namespace tc {
namespace {

constexpr int kTile = 16, kRowsMma = 16, kMaxGrid = 148;

template <int HD>
struct AttendShape {
  // a warp's ring: kUnits times a chunk's keys or a chunk's values
  static constexpr int kWarps = 8, kThreads = 32 * kWarps, kUnits = HD == 64 ? 10 : HD == 128 ? 6 : 3;
  static constexpr int kMat = kTile * HD * 2, kRing = kUnits * kMat;
  static constexpr int kCols = HD < 128 ? HD : 128;          // columns joined in one pass
  static constexpr int kSlot = 8 * (kCols + 4);              // floats of a warp's outputs of 8 heads, rows padded
  static constexpr int kSmem = 512 + kWarps * (kRing + kSlot * 4);
  static constexpr int kPart = kRowsMma * HD + 2 * kRowsMma; // floats of a CTA's state of an item
};

// ONE in what follows: one token per sequence (tc_attend); what chunks need besides is then left out of the code.
// A sequence's query tokens in blocks of a.block: rows row0 .. row0 + rows - 1 of q are the last n of its
// len tokens (rows < n where q ends before them).
template <bool ONE>
struct Seq {
  int b, len, n, row0, rows, nblk;
  __device__ __forceinline__ Seq(const AttendArgs& a, int b_) : b(b_) {
    len = kv_length(a.c, b, a.code);
    n = 1;
    row0 = b;
    rows = 1;
    if (!ONE) {
      row0 = __ldg(a.cu + b);
      n = max(__ldg(a.cu + b + 1) - row0, 0);
      rows = row0 < 0 ? 0 : max(min(n, a.tokens - row0), 0);
    }
    nblk = ONE ? 1 : a.block == 1 ? rows : (rows + a.block - 1) / a.block;
  }
};
// A block of tokens: the first one's position, how many, and the slots that any of them sees, [0, head) and
// [first, end), in nt chunks: chunks 0 .. na - 1, then from t0 on.
template <bool ONE>
struct Block {
  int tb, pos, ntok, end, first, head, na, t0, nt;
  __device__ __forceinline__ Block(const AttendArgs& a, const Seq<ONE>& q, int tb_) : tb(tb_) {
    pos = ONE ? q.len - 1 : q.len - q.n + tb * a.block;
    ntok = ONE ? 1 : min(a.block, q.rows - tb * a.block);
    end = max(pos + ntok, 0);
    first = pos >= 0 ? first_in_window(pos + 1, a.window) : 0;
    head = min(a.sinks, first);
    t0 = first / kTile;
    na = min((head + kTile - 1) / kTile, t0);
    nt = ntok > 0 && end > 0 ? na + (end + kTile - 1) / kTile - t0 : 0;
  }
  __device__ __forceinline__ int tile(int i) const { return i < na ? i : t0 + i - na; }
  __device__ __forceinline__ bool visible(int j) const { return j < end && (j >= first || j < head); }
  // every row sees all slots of the chunk
  __device__ __forceinline__ bool whole(const AttendArgs& a, int j0) const {
    return j0 + kTile <= pos + 1 && (j0 >= (ONE ? first : first_in_window(end, a.window)) || j0 + kTile <= a.sinks);
  }
};

// x * i / n rounded down, i <= n, n at most a few hundred: 32-bit arithmetic (a quarter of the time) while it serves.
__device__ __forceinline__ long long part_of(long long x, int i, int n) {
  return x < (1 << 22) ? (long long)((uint32_t)x * (uint32_t)i / (uint32_t)n) : x * i / n;
}
// The chunks of the whole call are cut into runs of total / runs (rounded down) or one more; there are
// no more runs than leave every warp of a CTA a chunk, so none is empty.
__device__ __forceinline__ int runs_of(long long total, int grid, int warps) {
  return (int)min((total + warps - 1) / warps, (long long)grid);
}
__device__ __forceinline__ long long run_begin(long long total, int runs, int i) { return part_of(total, i, runs); }
// The run that holds chunk t: the last one that begins at or before it.
__device__ __forceinline__ int run_of(long long total, int runs, long long t) {
  const long long x = (t + 1) * runs - 1;
  return max(x, total) <= 0x7FFFFFFF ? (int)((uint32_t)x / (uint32_t)total) : (int)(x / total);
}

// What plan() finds: the chunks of the whole call, a block of tokens by its number in the batch, its sequence
// (-1: there is none) and its place in that, and a number of chunks before something.
struct Plan {
  long long total, before;
  int b, tb, group;
};
struct PlanShared {
  long long warp[8];
  int groups[8];
  Plan found;
};
constexpr int kSolo = 64;            // up to this many sequences every warp scans the batch for itself, without a barrier
// Every thread of the CTA calls it (at most 256 threads). Finds block number `want` and the chunks before it; or,
// want < 0, the block that holds the first chunk of run `run` and the chunks of it before that one.
template <bool ONE>
__device__ __forceinline__ Plan plan(const AttendArgs& a, int nsub, PlanShared& s, int want, int run, int grid, int warps) {
  const int B = a.c.batch, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool solo = B <= kSolo;
  const int T = solo ? 32 : blockDim.x, t = solo ? lane : threadIdx.x, per = (B + T - 1) / T;
  const int lo = min(B, t * per), hi = min(B, lo + per);
  long long mine = 0;
  int groups = 0;
  for (int b = lo; b < hi; ++b) {
    const Seq<ONE> q(a, b);
    groups += q.nblk;
    for (int tb = 0; tb < q.nblk; ++tb) mine += (long long)Block<ONE>(a, q, tb).nt * nsub;
  }
  long long sum = mine;
  int gsum = groups;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    const int z = __shfl_up_sync(0xFFFFFFFFu, gsum, o);
    if (lane >= o) {
      sum += y;
      gsum += z;
    }
  }
  Plan p{0, 0, -1, 0, 0};
  long long at = sum - mine;                                 // chunks and blocks before this thread's sequences
  int group = gsum - groups;
  if (solo) {
    p.total = __shfl_sync(0xFFFFFFFFu, sum, 31);
  } else {
    if (lane == 31) {
      s.warp[warp] = sum;
      s.groups[warp] = gsum;
    }
    if (t == 0) s.found.b = -1;
    __syncthreads();
    for (int w = 0; w < T / 32; ++w) {
      if (w < warp) {
        at += s.warp[w];
        group += s.groups[w];
      }
      p.total += s.warp[w];
    }
  }
  const int runs = runs_of(p.total, grid, warps);
  const long long find = want < 0 && run < runs ? run_begin(p.total, runs, run) : p.total;
  if (want < 0 ? mine && find >= at && find < at + mine : want >= group && want < group + groups) {
    for (int b = lo; b < hi && p.b < 0; ++b) {
      const Seq<ONE> q(a, b);
      for (int tb = 0; tb < q.nblk && p.b < 0; ++tb) {
        const long long n = (long long)Block<ONE>(a, q, tb).nt * nsub;
        if (want < 0 ? find < at + n : group == want) {
          p.b = b;
          p.tb = tb;
          p.group = group;
          p.before = want < 0 ? find - at : at;
        }
        at += n;
        ++group;
      }
    }
  }
  if (solo) {
    const uint32_t who = __ballot_sync(0xFFFFFFFFu, p.b >= 0);
    const int from = who ? __ffs(who) - 1 : 0;
    p.b = __shfl_sync(0xFFFFFFFFu, p.b, from);
    p.tb = __shfl_sync(0xFFFFFFFFu, p.tb, from);
    p.group = __shfl_sync(0xFFFFFFFFu, p.group, from);
    p.before = __shfl_sync(0xFFFFFFFFu, p.before, from);
  } else {
    if (p.b >= 0) s.found = p;
    __syncthreads();
    p.b = s.found.b;
    p.tb = s.found.tb;
    p.group = s.found.group;
    p.before = s.found.before;
  }
  return p;
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

// Probabilities and sums are kept 2^kLift times as large: fp16 ends at 2^-25, and slots of less than that share
// of a warp's maximum, tens of thousands of them, would count in the sum but not in the output. From 2^14 on two
// parts reach 2^-39.
template <class T>
constexpr float kLift = __is_same(T, __half) ? 14.0f : 0.0f;

// What a call keeps in its workspace: the CTAs' states, the scores and the final statistics.
struct AttendWs {
  float* part;
  int* redo;                         // per item that one CTA holds whole: an output is not finite
  int64_t items;
  float2* ml;
  float* scores;
  int64_t cap;                       // slots a row of scores holds
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The parts of items that a CTA's run consists of, one after the other: chunks [i0, i1) of an item.
template <bool ONE>
struct Walk {
  int left, group, sub, i0, i1;      // left: chunks of the run from this part on
  Seq<ONE> q;
  Block<ONE> sq;
  __device__ __forceinline__ Walk(const AttendArgs& a, int left_, const Plan& p)
      : left(left_), group(p.group), sub(0), i0(0), i1(0), q(a, p.b), sq(a, q, p.tb) {
    sub = p.before <= 0x7FFFFFFF ? (int)((uint32_t)p.before / (uint32_t)sq.nt) : (int)(p.before / sq.nt);
    i0 = (int)(p.before - (long long)sub * sq.nt);
    i1 = min(sq.nt, i0 + left);
  }
  __device__ __forceinline__ bool next(const AttendArgs& a, int nsub) {
    left -= i1 - i0;
    if (left <= 0) return false;
    if (++sub == nsub) {
      sub = 0;
      do {                                        // (a sequence without rows has no block to count)
        int tb = sq.tb + 1;
        if (q.nblk > 0) ++group;
        if (tb >= q.nblk) {
          if (q.b + 1 >= a.c.batch) return false;  // (only if the lengths changed under the call)
          q = Seq<ONE>(a, q.b + 1);
          tb = 0;
        }
        sq = Block<ONE>(a, q, tb);
      } while (sq.nt == 0);
    }
    i0 = 0;
    i1 = min(sq.nt, left);
    return true;
  }
};

template <class T, int HD, int NB, bool ONE>
__global__ void __launch_bounds__(AttendShape<HD>::kThreads, 1)
    k_attend(const __grid_constant__ AttendArgs a, AttendWs ws, int gblocks, int hb) {
  using Sh = AttendShape<HD>;
  constexpr int W = Sh::kWarps, U = Sh::kUnits, kPieces = HD / 8;
  extern __shared__ __align__(16) uint8_t s_raw[];
  __shared__ float s_m[W][kRowsMma], s_l[W][kRowsMma];
  __shared__ PlanShared s_plan;
  griddep_launch();                               // k_join may take its place and wait
  const KvCache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.nh / c.n_kv, nsub = c.n_kv * gblocks;
  const Plan p = plan<ONE>(a, nsub, s_plan, -1, blockIdx.x, gridDim.x, W);
  const int runs = runs_of(p.total, gridDim.x, W);
  if ((int)blockIdx.x >= runs) return;
  Walk<ONE> w(a, (int)(run_begin(p.total, runs, blockIdx.x + 1) - run_begin(p.total, runs, blockIdx.x)), p);
  const uint32_t s_at = smem_u32(s_raw), pad = (512 - (s_at & 511)) % 512, ring = s_at + pad + warp * Sh::kRing;
  float* s_out = reinterpret_cast<float*>(s_raw + pad + W * Sh::kRing);

  // ---- the copies: a chunk's keys, its values, the next chunk's keys ..., U - 1 units ahead of their
  // use. A chunk's page id is loaded one chunk earlier still and only looked at when it is copied.
  Walk<ONE> pw = w;
  int pi = w.i0 + warp, page = -1, to_slot = 0;
  uint32_t held = 0;                              // bit x: the unit copied x copies ago is in the ring
  bool more = true;
  // A row's 16-byte piece p is kept at place p ^ (row % 8) of its 128 bytes (no bank conflicts in ldmatrix);
  // a lane copies piece lane % kLanes of rows r0, r0 + kAtOnce, .. and r0 < kAtOnce divides 8, so the
  // place is that of row r0 with constant bits flipped. The ring starts on a multiple of 512 bytes.
  constexpr int kLanes = kPieces < 32 ? kPieces : 32, kAtOnce = 32 / kLanes;
  const int r0 = lane / kLanes;
  const uint32_t put = ring + r0 * HD * 2 + ((lane % kLanes ^ r0) << 4);
  const int64_t step = 2 * kAtOnce * c.ss;
  auto find = [&] {
    while (more && pi >= pw.i1) {
      more = pw.next(a, nsub);
      pi = pw.i0 + warp;
    }
    if (more) page = __ldg(c.table + (int64_t)pw.q.b * c.ts + (pw.sq.tile(pi) * kTile >> c.shift));
  };
  auto copy = [&](const uint8_t* pool, bool last) {
    const bool good = more && (unsigned)page < (unsigned)c.n_pages;
    if (more && !good) kv_fail(c, a.code);
    held = held << 1 | good;
    if (good) {
      const int j0 = pw.sq.tile(pi) * kTile;
      const uint8_t* from = pool + 2 * ((int64_t)page * c.sp + (int64_t)((j0 & ((1 << c.shift) - 1)) + r0) * c.ss +
                                        (int64_t)(pw.sub / gblocks) * c.sh) + 16 * (lane % kLanes);
      const uint32_t to = put + to_slot * Sh::kMat;
      if (j0 + kTile <= pw.sq.end && (j0 >= pw.sq.first || j0 + kTile <= pw.sq.head)) {
#pragma unroll
        for (int x = 0; x < kTile / kAtOnce; ++x)
          asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"((to ^ (x * kAtOnce % 8 << 4)) + x * kAtOnce * HD * 2),
                       "l"(from + x * step) : "memory");
      } else {                                    // a hidden row may hold anything: it reads as zeros
#pragma unroll
        for (int x = 0; x < kTile / kAtOnce; ++x)
          asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"((to ^ (x * kAtOnce % 8 << 4)) + x * kAtOnce * HD * 2),
                       "l"(from + x * step), "r"(pw.sq.visible(j0 + r0 + x * kAtOnce) ? 16 : 0) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++to_slot == U) to_slot = 0;
    if (last) {
      pi += W;
      find();
    }
  };
  find();
#pragma unroll
  for (int x = 0; x < U - 1; ++x) copy(x & 1 ? c.v : c.k, x & 1);

  int slot = 0;
  // where ldmatrix reads: keys, slots 0-15 of columns 0-7 then 8-15; values, slots 0-7 of columns 0-7 and 8-15,
  // then slots 8-15. The next 16 columns are 32 bytes on, which flips bits of the place.
  const uint32_t k_at = ring + (lane & 15) * HD * 2 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_at = ring + ((lane & 7) + (lane >> 4) * 8) * HD * 2 + (((lane >> 3 & 1) ^ (lane & 7)) << 4);
  do {
    // row r of the item is head h0 + r % heads of token r / heads of the block
    const int kvh = w.sub / gblocks, g0 = (w.sub - kvh * gblocks) * hb, h0 = kvh * G + g0, heads = min(hb, G - g0),
              rows = heads * w.sq.ntok, row0 = w.q.row0 + w.sq.tb * a.block;
    // the query rows as the MMA's second operand: row lane / 4, columns 2 (lane % 4) (+ 1, + 8, + 9) of each 16
    uint32_t q[NB][HD / 16][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = 8 * nb + (lane >> 2), rr = min(r, rows - 1), tok = ONE ? 0 : rr / heads;
      const uint32_t* from = reinterpret_cast<const uint32_t*>(
          a.q + 2 * ((int64_t)(row0 + tok) * a.qr + (int64_t)(h0 + rr - tok * heads) * a.qh + 2 * (lane & 3)));
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int x = 0; x < 2; ++x) q[nb][kk][x] = __ldg(from + 8 * kk + 4 * x);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int x = 0; x < 2; ++x) q[nb][kk][x] = r < rows ? q[nb][kk][x] : 0;
    }
    // rows 2 (lane % 4) (+ 1) of each block of 8 are this lane's in the scores and outputs: what they see
    int last[NB][2], from[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        last[nb][y] = w.sq.pos + (ONE ? 0 : (8 * nb + 2 * (lane & 3) + y) / heads);
        from[nb][y] = ONE ? w.sq.first : first_in_window(last[nb][y] + 1, a.window);
      }
    // this warp's state: rows (lane / 4, + 8) of each 16 columns of O^T, those two rows of q in each block of 8
    float o[HD / 16][NB][4], m[NB][2], l[NB][2];
    bool any = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int x = 0; x < HD / 16; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[x][nb][e] = 0.0f;
      m[nb][0] = m[nb][1] = neg_inf();
      l[nb][0] = l[nb][1] = 0.0f;
    }
    for (int i = w.i0 + warp; i < w.i1; i += W) {
      asm volatile("cp.async.wait_group %0;" ::"n"(U - 2) : "memory");
      __syncwarp();                               // the keys are here, and the unit before them is used up
      const uint32_t kt = k_at + slot * Sh::kMat;
      if (++slot == U) slot = 0;
      copy((U - 1) & 1 ? c.v : c.k, (U - 1) & 1);
      const int j0 = w.sq.tile(i) * kTile;
      const bool here = held >> (U - 1) & 1;      // (not on a page outside the pool)
      any |= here;
      float s[NB][4], s2[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nb][e] = s2[nb][e] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t f[4];
        ldsm4(kt ^ (kk << 5), f);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16816<T>(kk & 1 ? s2[nb] : s[nb], f, q[nb][kk][0], q[nb][kk][1]);
      }
      const bool whole = w.sq.whole(a, j0);
      const int r = lane >> 2;
      // bit 4 nb + e: element e of block nb is visible (with one token the same bits for every block and row)
      constexpr int kShow = ONE ? 1 : NB;
      uint32_t show = here ? ~0u : 0;
      if (here && !whole) {
        show = 0;
#pragma unroll
        for (int nb = 0; nb < kShow; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + r + 8 * (e >> 1);
            if (j <= last[nb][e & 1] && (j >= from[nb][e & 1] || j < a.sinks)) show |= 1u << (4 * nb + e);
          }
      }
      auto seen = [&](int nb, int e) { return show >> (4 * (ONE ? 0 : nb) + (ONE ? e & 2 : e)) & 1; };
      float top[NB][2];
      bool grow = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nb][e] = seen(nb, e) ? (s[nb][e] + s2[nb][e]) * a.scale2 : neg_inf();
        if (ws.scores && here) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = 8 * nb + 2 * (lane & 3) + (e & 1);  // (scores are kept for one token a sequence: row = head)
            if (h < rows) ws.scores[((int64_t)w.q.b * a.nh + h0 + h) * ws.cap + j0 + r + 8 * (e >> 1)] = s[nb][e];
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float t = fmaxf(s[nb][y], s[nb][y + 2]);
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 4));
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 8));
          t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 16));
          top[nb][y] = fmaxf(m[nb][y], t);
          grow |= top[nb][y] > m[nb][y];
        }
      }
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float f[2] = {shrink(m[nb][0], top[nb][0]), shrink(m[nb][1], top[nb][1])};
#pragma unroll
          for (int x = 0; x < HD / 16; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[x][nb][e] *= f[e & 1];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            l[nb][y] *= f[y];
            m[nb][y] = top[nb][y];
          }
        }
      }
      uint32_t hi[NB][2], lo[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float base = m[nb][e & 1] == neg_inf() ? 0.0f : m[nb][e & 1] - kLift<T>;
          p[e] = seen(nb, e) ? ex2(s[nb][e] - base) : 0.0f;
        }
        l[nb][0] += p[0] + p[2];
        l[nb][1] += p[1] + p[3];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t h = Elem<T>::pack(p[2 * y], p[2 * y + 1]);
          const float2 f = Elem<T>::f2(h);
          hi[nb][y] = transpose8x8(h);
          lo[nb][y] = transpose8x8(Elem<T>::pack(p[2 * y] - f.x, p[2 * y + 1] - f.y));
        }
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(U - 2) : "memory");
      __syncwarp();                               // the values are here, and the keys are used up
      const uint32_t vt = v_at + slot * Sh::kMat;
      if (++slot == U) slot = 0;
      copy(U & 1 ? c.v : c.k, U & 1);
      if (here)
#pragma unroll
      for (int x = 0; x < HD / 16; ++x) {
        uint32_t f[4];
        ldsm4t(vt ^ (x << 5), f);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma16816<T>(o[x][nb], f, hi[nb][0], hi[nb][1]);
          mma16816<T>(o[x][nb], f, lo[nb][0], lo[nb][1]);
        }
      }
    }

    // ---- the warps' states at their common maximum; a warp that met no slot says so by a sum of -1
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nb][y] += __shfl_xor_sync(0xFFFFFFFFu, l[nb][y], x);
        if (lane < 4) {
          s_m[warp][8 * nb + 2 * lane + y] = m[nb][y];
          s_l[warp][8 * nb + 2 * lane + y] = any ? l[nb][y] : -1.0f;
        }
      }
    __syncthreads();
    const bool all = w.i0 == 0 && w.i1 == w.sq.nt;
    float* part = ws.part + ((int64_t)blockIdx.x * 2 + (w.i0 == 0)) * Sh::kPart;
    bool good = true;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float f[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int h = 8 * nb + 2 * (lane & 3) + y;
        float mm = s_m[0][h];
#pragma unroll
        for (int k = 1; k < W; ++k) mm = fmaxf(mm, s_m[k][h]);
        f[y] = shrink(m[nb][y], mm);
      }
#pragma unroll
      for (int c0 = 0; c0 < HD; c0 += Sh::kCols) {
        if (nb + c0 > 0) __syncthreads();         // the pass before is read
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int x = 0; x < Sh::kCols / 16; ++x) {
            float* to = s_out + warp * Sh::kSlot + (2 * (lane & 3) + y) * (Sh::kCols + 4) + 16 * x + (lane >> 2);
            to[0] = o[c0 / 16 + x][nb][y] * f[y];
            to[8] = o[c0 / 16 + x][nb][y + 2] * f[y];
          }
        __syncthreads();
        for (int u = threadIdx.x; u < 8 * Sh::kCols / 4; u += Sh::kThreads) {
          const int hh = u / (Sh::kCols / 4), at = 4 * (u - hh * (Sh::kCols / 4)), col = c0 + at, h = 8 * nb + hh;
          if (h >= rows) break;
          float mm = s_m[0][h], sum = 0.0f;
#pragma unroll
          for (int k = 1; k < W; ++k) mm = fmaxf(mm, s_m[k][h]);
          bool met = false;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int k = 0; k < W; ++k) {
            const float lk = s_l[k][h];
            if (!(lk < 0.0f)) {
              sum = fmaf(lk, shrink(s_m[k][h], mm), sum);
              met = true;
            }
            const float4 g = *reinterpret_cast<const float4*>(s_out + k * Sh::kSlot + hh * (Sh::kCols + 4) + at);
            v.x += g.x; v.y += g.y; v.z += g.z; v.w += g.w;
          }
          if (all) {
            const float inv = met ? 1.0f / sum : 0.0f;
            v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
            // (a sum that is NaN makes a NaN of every output, as the formula does)
            good &= sum != sum || fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) < __int_as_float(0x7F800000);
            const int tok = ONE ? 0 : h / heads;
            *reinterpret_cast<uint2*>(a.out + 2 * ((int64_t)(row0 + tok) * a.orow + (int64_t)(h0 + h - tok * heads) * a.oh +
                                                   col)) = make_uint2(Elem<T>::pack(v.x, v.y), Elem<T>::pack(v.z, v.w));
            if (col == 0 && ws.ml) ws.ml[(int64_t)w.q.b * a.nh + h0 + h] = make_float2(mm - kLift<T>, sum);
          } else {
            *reinterpret_cast<float4*>(part + h * HD + col) = v;
            if (col == 0) {
              part[kRowsMma * HD + h] = mm;
              part[kRowsMma * HD + kRowsMma + h] = met ? sum : -1.0f;
            }
          }
        }
      }
    }
    const int bad = __syncthreads_or(!good);
    const int64_t item = (int64_t)w.group * nsub + w.sub;         // (beyond the workspace only if cu is not ascending)
    if (all && threadIdx.x == 0 && item < ws.items) ws.redo[item] = bad;
  } while (w.next(a, nsub));
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// The items whose tiles lie in several CTAs' runs: their states at the common maximum. One CTA per
// (block, head block, row): its warps take the pieces in turn, and their sums are added in warp
// order. Blocks that see no slot get zeros. A row with a NaN or an infinity and a sum that is a
// number is computed again key by key: the second half of a split probability times an infinite value would
// make a NaN of it.
constexpr int kJoinWarps = 8, kJoinThreads = 32 * kJoinWarps;
template <class T, int HD, bool ONE>
__global__ void __launch_bounds__(kJoinThreads)
    k_join(const __grid_constant__ AttendArgs a, AttendWs ws, int grid, int gblocks, int hb) {
  using Sh = AttendShape<HD>;
  __shared__ PlanShared s_plan;
  __shared__ float2 s_o[kJoinWarps][HD / 2];
  griddep_launch();
  const KvCache& c = a.c;
  const int G = a.nh / c.n_kv, nsub = c.n_kv * gblocks;
  const int most = ONE ? hb : hb * a.block, item = blockIdx.x / most, r = blockIdx.x - item * most, sub = item % nsub;
  const int kvh = sub / gblocks, g0 = (sub - kvh * gblocks) * hb, heads = min(hb, G - g0);
  const Plan p = plan<ONE>(a, nsub, s_plan, item / nsub, 0, 1, Sh::kWarps);
  const long long total = p.total;
  griddep_wait();                                // (before any return: what follows in the stream counts on it)
  if (p.b < 0) return;
  const Seq<ONE> q(a, p.b);
  const Block<ONE> sq(a, q, p.tb);
  const int nt = sq.nt, tok = ONE ? r >= heads : r / heads, h = kvh * G + g0 + r - tok * heads, row = q.row0 + sq.tb * a.block + tok;
  if (tok >= sq.ntok) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t at_out = (int64_t)row * a.orow + (int64_t)h * a.oh;
  uint32_t* to = reinterpret_cast<uint32_t*>(a.out + 2 * at_out);
  if (nt == 0) {
    for (int x = threadIdx.x; x < HD / 2; x += kJoinThreads) to[x] = 0;
    return;
  }
  const long long t0 = p.before + (long long)sub * nt;
  const int runs = runs_of(total, grid, Sh::kWarps), c0 = run_of(total, runs, t0), c1 = run_of(total, runs, t0 + nt - 1);
  bool redo = c0 == c1;
  if (redo && !ws.redo[item]) return;
  if (!redo) {
    // every warp: the pieces' statistics, a lane each (at most kMaxGrid = 148 pieces)
    constexpr int kEach = (kMaxGrid + 31) / 32;
    float m = neg_inf(), l = 0.0f, f[kEach], lk[kEach];
    const int pieces = c1 - c0 + 1;
    auto piece = [&](int k) { return ws.part + ((int64_t)(c0 + k) * 2 + (k == 0)) * Sh::kPart; };
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const int k = lane + 32 * x;
      f[x] = neg_inf();
      lk[x] = -1.0f;                             // a piece without a visible slot
      if (k < pieces) {
        f[x] = piece(k)[kRowsMma * HD + r];
        lk[x] = piece(k)[kRowsMma * HD + kRowsMma + r];
      }
    }
#pragma unroll
    for (int x = 0; x < kEach; ++x) m = lk[x] < 0.0f ? m : fmaxf(m, f[x]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
    bool any = false;
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const bool met = !(lk[x] < 0.0f);
      any |= met;
      f[x] = met ? shrink(f[x], m) : 0.0f;
      if (met) l = fmaf(lk[x], f[x], l);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
    any = __any_sync(0xFFFFFFFFu, any);
    float2 o[HD / 64];
#pragma unroll
    for (int z = 0; z < HD / 64; ++z) o[z] = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int x = 0; x < kEach; ++x)
#pragma unroll
      for (int y = 0; y < 32 / kJoinWarps; ++y) {
        const int k = 32 * x + y * kJoinWarps + warp;
        const float g = __shfl_sync(0xFFFFFFFFu, f[x], y * kJoinWarps + warp);
        if (k < pieces && g != 0.0f) {
          const float2* from = reinterpret_cast<const float2*>(piece(k) + r * HD);
#pragma unroll
          for (int z = 0; z < HD / 64; ++z) {
            const float2 v = from[lane + 32 * z];
            o[z].x = fmaf(v.x, g, o[z].x);
            o[z].y = fmaf(v.y, g, o[z].y);
          }
        }
      }
#pragma unroll
    for (int z = 0; z < HD / 64; ++z) s_o[warp][lane + 32 * z] = o[z];
    __syncthreads();
    bool good = true;
    const float inv = any ? 1.0f / l : 0.0f;
    if (threadIdx.x < HD / 2) {
      float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < kJoinWarps; ++k) {
        v.x += s_o[k][threadIdx.x].x;
        v.y += s_o[k][threadIdx.x].y;
      }
      v.x *= inv;
      v.y *= inv;
      good = l != l || fabsf(v.x) + fabsf(v.y) < __int_as_float(0x7F800000);
      to[threadIdx.x] = Elem<T>::pack(v.x, v.y);
    }
    if (ws.ml && threadIdx.x == 0) ws.ml[(int64_t)q.b * a.nh + h] = make_float2(m - kLift<T>, l);
    redo = __syncthreads_or(!good);
  }
  if (redo && warp == 0) {
    float x[HD / 32], o[HD / 32];
    row_load<T, HD>(a.q, (int64_t)row * a.qr + (int64_t)h * a.qh, lane, x);
    attend_row<T, HD>(c, q.b, kvh, x, a.scale2, max(sq.pos + tok + 1, 0), a.window, a.sinks, a.code, o);
    row_store<T, HD>(a.out, at_out, lane, o);
  }
}

// weight_out = weight + the visible slots' probabilities, summed over the heads that share a key-value head, a
// slot a thread: the scores of k_attend once more (4 bytes a head and slot) and the final statistics.
constexpr int kWeightThreads = 256, kWeightHeads = 64;
__global__ void __launch_bounds__(kWeightThreads) k_weights(const __grid_constant__ AttendArgs a, AttendWs ws) {
  __shared__ float2 s_ml[kWeightHeads];          // a head's maximum, and 1 / its sum
  const KvCache& c = a.c;
  const int row = blockIdx.x, b = row / c.n_kv, g = row - b * c.n_kv, G = a.nh / c.n_kv;
  const int len = kv_length(c, b, kErrAttend), first = first_in_window(len, a.window);
  const int64_t at = (int64_t)row * c.track, u = (int64_t)b * a.nh + g * G;
  griddep_wait();
  for (int i0 = 0; i0 < G; i0 += kWeightHeads) {
    const int n = min(kWeightHeads, G - i0);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kWeightThreads) {
      const float2 f = ws.ml[u + i0 + i];
      s_ml[i] = make_float2(f.x, 1.0f / f.y);
    }
    __syncthreads();
    for (int j = blockIdx.y * kWeightThreads + threadIdx.x; j < len; j += gridDim.y * kWeightThreads) {
      float w = i0 ? a.weight_out[at + j] : c.weight[at + j];
      if (j < a.sinks || j >= first) {
        const bool here = (unsigned)__ldg(c.table + (int64_t)b * c.ts + (j >> c.shift)) < (unsigned)c.n_pages;
        const float* from = ws.scores + (u + i0) * ws.cap + j;
        float sum = 0.0f;
#pragma unroll 4
        for (int i = 0; i < n; ++i) sum = fmaf(ex2(from[i * ws.cap] - s_ml[i].x), s_ml[i].y, sum);
        if (here) w += sum;
      }
      a.weight_out[at + j] = w;
    }
  }
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
// A group's heads in blocks of nearly equal size (at most 16), and the blocks of tokens a call may have.
struct Shape {
  int gblocks, hb, nsub;
  int64_t groups;
};
Shape shape_of(const KvCache& c, int nh, int block, int tokens) {
  const int G = nh / c.n_kv, gblocks = (G + kRowsMma - 1) / kRowsMma;
  // (every sequence ends in at most one block that is not full; tokens < 0: one token a sequence)
  const int64_t groups = tokens < 0 ? c.batch : std::min<int64_t>(tokens, tokens / block + std::min(tokens, c.batch));
  return Shape{gblocks, (G + gblocks - 1) / gblocks, c.n_kv * gblocks, groups};
}
AttendWs ws_of(const KvCache& c, int nh, int64_t items, bool weights, uint8_t* ws, uint64_t* bytes) {
  AttendWs w{};
  int64_t at = 0;
  w.part = reinterpret_cast<float*>(ws);
  at += up256((int64_t)kMaxGrid * 2 * (kRowsMma * c.hd + 2 * kRowsMma) * 4);
  w.redo = reinterpret_cast<int*>(ws + at);
  w.items = items;
  at += up256(items * 4);
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

template <class T, int HD, bool ONE>
cudaError_t attend_hd(const AttendArgs& a, cudaStream_t st) {
  using Sh = AttendShape<HD>;
  const KvCache& c = a.c;
  const Shape sh = shape_of(c, a.nh, a.block, ONE ? -1 : a.tokens);
  uint64_t bytes = 0;
  const AttendWs ws = ws_of(c, a.nh, sh.groups * sh.nsub, a.weight_out != nullptr, a.ws, &bytes);
  const bool one = sh.hb * a.block <= 8;         // rows of an item
  auto kern = one ? k_attend<T, HD, 1, ONE> : k_attend<T, HD, 2, ONE>;
  cudaError_t e = one ? allow_smem<k_attend<T, HD, 1, ONE>>(Sh::kSmem) : allow_smem<k_attend<T, HD, 2, ONE>>(Sh::kSmem);
  if (e != cudaSuccess) return e;
  // no more CTAs than the page lists can hold chunks for
  const int64_t chunks = ((int64_t)c.max_pages << c.shift) / kTile;
  const int grid = (int)std::min<int64_t>(kMaxGrid, (sh.groups * sh.nsub * chunks + Sh::kWarps - 1) / Sh::kWarps);
  const int64_t joins = sh.groups * sh.nsub * sh.hb * a.block;
  if (joins > INT32_MAX) return cudaErrorInvalidValue;
  kern<<<grid, Sh::kThreads, Sh::kSmem, st>>>(a, ws, sh.gblocks, sh.hb);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  e = launch_dependent(k_join<T, HD, ONE>, dim3((unsigned)joins), dim3(kJoinThreads), st, a, ws, grid, sh.gblocks, sh.hb);
  if (e != cudaSuccess || !a.weight_out) return e;
  const int kvrows = c.batch * c.n_kv;
  const int64_t blocks = (((int64_t)c.max_pages << c.shift) + kWeightThreads - 1) / kWeightThreads;
  return launch_dependent(k_weights, dim3(kvrows, (unsigned)std::min<int64_t>(blocks, std::max(1, 148 * 8 / kvrows))),
                          dim3(kWeightThreads), st, a, ws);
}

template <class T, bool ONE>
cudaError_t attend_of(const AttendArgs& a, cudaStream_t st) {
  switch (a.c.hd) {
    case 64: return attend_hd<T, 64, ONE>(a, st);
    case 128: return attend_hd<T, 128, ONE>(a, st);
    default: return attend_hd<T, 256, ONE>(a, st);
  }
}

}  // namespace

uint64_t attend_workspace(const KvCache& c, int nh, bool weights) {
  const Shape sh = shape_of(c, nh, 1, -1);
  uint64_t bytes = 0;
  ws_of(c, nh, sh.groups * sh.nsub, weights, nullptr, &bytes);
  return bytes;
}
cudaError_t launch_attend(AttendArgs a, cudaStream_t st) {
  a.block = 1;
  a.code = kErrAttend;
  return a.dtype == TC_BF16 ? attend_of<__nv_bfloat16, true>(a, st) : attend_of<__half, true>(a, st);
}

// Which of the two kernels takes a chunk of a prompt, by their times on a B200 in microseconds, fitted to
// measurements at 1 to 128 tokens of 1, 8 and 32 sequences behind 1000 and 16000 slots (16 heads on 8 of 128,
// 4 on 1 of 256). This one passes over a sequence's slots once for each block of rows and head block
// (8 x 4 tokens behind 1000 slots, 16 heads on 8: 20 us against 24; 8 x 16: 49 against 25; behind 16000
// slots 95 against 251 and 200 against 252); the prompt kernel's time is that of its blocks of 128 (64) slots
// one after the other while its CTAs fit on the SMs. The lengths are the device's: the page lists' room
// stands in for them.
int chunk_block(const KvCache& c, int nh, int tokens, int window, int sinks) {
  const Shape sh = shape_of(c, nh, 1, tokens);
  const int each = (tokens + c.batch - 1) / c.batch, rows = sh.hb * each;
  const int block = std::max(1, (rows <= 8 ? 8 : kRowsMma) / sh.hb);
  const double keys = std::min((double)((int64_t)c.max_pages << c.shift), (double)window + sinks + each);
  const double items = (double)std::min(tokens, c.batch) * sh.nsub, passes = items * ((each + block - 1) / block);
  const double few = 10 + passes * ((rows <= 8 ? 0.12 : 0.2) + keys * c.hd * (rows <= 8 ? 0.6e-6 : 0.7e-6));
  const double spans = items * ((each * sh.hb + 255) / 256), waves = std::ceil(spans / kMaxGrid);
  const double many = 8 + waves * keys * (c.hd == 256 ? 24e-3 : 15e-3);
  return few < many ? block : 0;
}
uint64_t chunk_workspace(const KvCache& c, int nh, int tokens, int window, int sinks) {
  const int block = chunk_block(c, nh, tokens, window, sinks);
  if (!block) return 0;
  const Shape sh = shape_of(c, nh, block, tokens);
  uint64_t bytes = 0;
  ws_of(c, nh, sh.groups * sh.nsub, false, nullptr, &bytes);
  return bytes;
}
cudaError_t launch_attend_chunk(AttendArgs a, cudaStream_t st) {
  a.block = chunk_block(a.c, a.nh, a.tokens, a.window, a.sinks);
  a.code = kErrPrompt;
  return a.dtype == TC_BF16 ? attend_of<__nv_bfloat16, false>(a, st) : attend_of<__half, false>(a, st);
}

}  // namespace tc
