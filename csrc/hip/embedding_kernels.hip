// K22: embedding lookup with a scale, and its weight gradient from tokens sorted by id.
//
//   forward   out[i, :] = scale * W[id_i, :]; an id outside [0, V) gives a row of zeros
//   gradient  dW[v, :]  = scale * sum over { i : id_i = v } of dy[i, :], all V rows written
//
// The sum over a token's rows is taken in fp32 and does not depend on scheduling: the positions are sorted by id with a
// stable radix sort (no floating-point atomics) and cut into pieces, walked in order, whose sums are joined in a fixed
// grouping. Sizes and types alone choose that grouping: the same call gives the same bits.
//
// All of it is bound by memory. 131071 tokens, 1536 columns, fp32 table of 100003 rows under bf16 rows: lookup 130 us
// (402 MB written, 805 MB of rows read of which the caches serve the frequent ones), gradient 302 us = sort 30 + sums 266
// (402 MB read, 614 MB written, 3.8 TB/s) + joins 6; on another card lookup 145, sums 238, joins 10. 8192 tokens of 1024
// bf16 columns, 32768 rows: lookup 7 us, gradient 37 us = sort 18 (one workgroup: its latency) + sums 15 (5.6 TB/s) +
// joins 4.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "vec_types.h"

namespace rmm {
namespace hip {

namespace {

template <typename TI>
__device__ __forceinline__ uint32_t embed_key(TI id, int64_t V, int64_t pad) {
  const int64_t v = int64_t(id);
  return uint32_t(v < 0 || v >= V || v == pad ? V : v);  // V: no gradient, sorts behind every row
}

// ------------------------------------------------------------------------------------------ lookup
// Everywhere below, a lane has VEC neighbouring columns at any alignment, and the last lane of a row whose length is no
// multiple of VEC begins early enough to end with it: columns that two lanes have get the same value from both.
__device__ __forceinline__ int64_t run_start(int64_t c, int64_t D, int vec) { return c + vec <= D ? c : D - vec; }

// 2^lpr lanes share a row (up to kRun times); a workgroup has 256 >> lpr rows in flight.
constexpr int kRun = 4;

template <typename TI, typename TW, typename TO, int VEC>
__global__ __launch_bounds__(256) void k_embed_fwd(const TI* __restrict__ ids, const TW* __restrict__ w, int64_t ws,
                                                   TO* __restrict__ out, int64_t n, int64_t V, int64_t D, float scale,
                                                   int lpr) {
  const int lane = threadIdx.x & ((1 << lpr) - 1);
  const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> lpr, step = int64_t(VEC) << lpr;
  if (i >= n) return;
  const int64_t id = int64_t(ids[i]);
  const bool ok = id >= 0 && id < V;
  const TW* row = w + (ok ? id : 0) * ws;
  for (int64_t c0 = int64_t(lane) * VEC; c0 < D; c0 += kRun * step) {
    RunOf<TW, VEC> r[kRun];
#pragma unroll
    for (int q = 0; q < kRun; q++)
      if (ok && c0 + q * step < D)
        r[q] = *reinterpret_cast<const RunOf<TW, VEC>*>(row + run_start(c0 + q * step, D, VEC));
#pragma unroll
    for (int q = 0; q < kRun; q++) {
      if (c0 + q * step >= D) break;
      float v[VEC];
#pragma unroll
      for (int k = 0; k < VEC; k++) v[k] = ok ? to_f32(r[q].v[k]) * scale : 0.f;
      store_run<TO, VEC>(out + i * D + run_start(c0 + q * step, D, VEC), v);
    }
  }
}

// ------------------------------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (key, position). Batches of up to kSmall ids are sorted by one workgroup
// in LDS (one launch); larger ones in tiles, a count and a scatter launch for each digit of up to 9 bits.

// Lanes of this wave whose digit equals mine (inactive lanes excluded).
__device__ __forceinline__ uint64_t match_digit(uint32_t d, int bits, bool active) {
  const uint64_t all = __ballot(active);
  uint32_t lo = uint32_t(all), hi = uint32_t(all >> 32);
  for (int b = 0; b < bits; b++) {
    const uint32_t mine = uint32_t(int32_t(d << (31 - b)) >> 31);  // this bit in every place
    const uint64_t v = __ballot(mine != 0);
    lo &= ~(uint32_t(v) ^ mine);
    hi &= ~(uint32_t(v >> 32) ^ mine);
  }
  return (uint64_t(hi) << 32) | lo;
}

// Orders LDS accesses of one wave (its lanes run in step; this holds the compiler to that order).
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The place of this lane's element behind slots[d]: that counter (moved on for the whole wave) plus the element's rank
// among the lanes with the same digit, in lane order.
__device__ __forceinline__ uint32_t take_slot(uint32_t* slots, uint32_t d, int bits, bool active) {
  const uint64_t same = match_digit(d, bits, active);
  uint32_t at = 0;
  if (active) {
    const int rank = __builtin_amdgcn_mbcnt_hi(uint32_t(same >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(same), 0u));
    at = slots[d] + rank;
    wave_fence();  // all lanes have read the slot before its first lane moves it on
    if (rank == 0) slots[d] += __popcll(same);
  }
  wave_fence();
  return at;
}

constexpr int kSmall = 8192, kSmallThreads = 1024, kSmallWaves = kSmallThreads / kWave, kSmallBits = 8;
constexpr int kSmallRadix = 1 << kSmallBits;

template <typename TI>
__global__ __launch_bounds__(kSmallThreads) void k_sort_small(const TI* __restrict__ ids, int n, int64_t V, int64_t pad,
                                                              int passes, int bits, uint32_t* __restrict__ okeys,
                                                              uint32_t* __restrict__ opos) {
  constexpr int kPer = kSmall / kSmallThreads;  // elements a thread
  __shared__ uint32_t key[2][kSmall];
  __shared__ uint16_t pos[2][kSmall];
  __shared__ uint32_t slot[kSmallWaves][kSmallRadix];
  __shared__ uint32_t wsum[kSmallWaves];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, radix = 1 << bits;
  const int seg = (n + kSmallThreads - 1) / kSmallThreads * kWave, lo = min(n, wave * seg), hi = min(n, lo + seg);
  for (int i = tid; i < n; i += kSmallThreads) {
    key[0][i] = embed_key(ids[i], V, pad);
    pos[0][i] = uint16_t(i);
  }
  for (int s = 0; s < passes; s++) {
    const int from = s & 1, to = from ^ 1, shift = s * bits;
    for (int r = lane; r < radix; r += kWave) slot[wave][r] = 0;
    __syncthreads();
    uint32_t k[kPer], rank[kPer];  // each element's rank among its digit's in this wave; slot becomes their count
#pragma unroll
    for (int q = 0; q < kPer; q++) {
      const int i = lo + q * kWave + lane;
      k[q] = i < hi ? key[from][i] : 0u;
      rank[q] = 0;
      if (lo + q * kWave < hi) rank[q] = take_slot(slot[wave], (k[q] >> shift) & (radix - 1), bits, i < hi);
    }
    __syncthreads();
    // exclusive sums in the order (digit, wave): 4 threads a digit, 4 waves each
    const int d = tid / 4, w0 = tid % 4 * 4;
    uint32_t c[4] = {}, sum = 0;
    if (d < radix) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        c[j] = slot[w0 + j][d];
        sum += c[j];
      }
    }
    uint32_t incl = sum;
    for (int off = 1; off < kWave; off <<= 1) {
      const uint32_t up = __shfl_up(incl, off);
      if (lane >= off) incl += up;
    }
    if (lane == kWave - 1) wsum[wave] = incl;
    __syncthreads();
    uint32_t at = incl - sum;
    for (int w = 0; w < wave; w++) at += wsum[w];
    if (d < radix) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        slot[w0 + j][d] = at;
        at += c[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; q++) {
      const int i = lo + q * kWave + lane;
      if (i < hi) {
        const uint32_t dst = slot[wave][(k[q] >> shift) & (radix - 1)] + rank[q];
        key[to][dst] = k[q];
        pos[to][dst] = pos[from][i];
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += kSmallThreads) {
    okeys[i] = key[passes & 1][i];
    opos[i] = pos[passes & 1][i];
  }
}

constexpr int kHistThreads = 256, kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kMaxBits = 9, kMaxRadix = 1 << kMaxBits, kMaxTiles = 256;

// Digit counts of each tile: counts[tile][radix].
template <typename TI>
__global__ __launch_bounds__(kHistThreads) void k_sort_hist(const TI* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                            int64_t n, int64_t tile, int64_t V, int64_t pad, int shift,
                                                            int bits, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kMaxRadix];
  const int radix = 1 << bits;
  for (int r = threadIdx.x; r < radix; r += kHistThreads) hist[r] = 0;
  __syncthreads();
  const int64_t lo = int64_t(blockIdx.x) * tile, hi = min(n, lo + tile);
  for (int64_t i = lo + threadIdx.x; i < hi; i += kHistThreads) {
    const uint32_t k = ids ? embed_key(ids[i], V, pad) : keys[i];
    atomicAdd(&hist[(k >> shift) & (radix - 1)], 1u);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < radix; r += kHistThreads) counts[int64_t(blockIdx.x) * radix + r] = hist[r];
}

// One stable pass: tile after tile, wave after wave, round after round, lane after lane is the input order,
// and the slot of an element is (smaller digits anywhere) + (same digit in earlier tiles, waves, rounds, lanes).
template <typename TI>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(const TI* __restrict__ ids,
                                                               const uint32_t* __restrict__ keys,
                                                               const uint32_t* __restrict__ pos, int64_t n, int64_t tile,
                                                               int64_t V, int64_t pad, int shift, int bits,
                                                               const uint32_t* __restrict__ counts,
                                                               uint32_t* __restrict__ okeys, uint32_t* __restrict__ opos) {
  __shared__ uint32_t base[kMaxRadix];               // slot of the digit's first element of this tile
  __shared__ uint32_t slot[kSortWaves][kMaxRadix];   // counts, then running slots, of each wave
  __shared__ uint4 part[4][kMaxRadix / 2];
  __shared__ uint32_t wsum[kSortWaves];
  const int radix = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int64_t lo = int64_t(blockIdx.x) * tile, hi = min(n, lo + tile);
  const int64_t seg = tile / kSortWaves, wlo = min(hi, lo + wave * seg), whi = min(hi, wlo + seg);
  for (int r = lane; r < radix; r += kWave) slot[wave][r] = 0;
  wave_fence();
  for (int64_t i = wlo + lane; i < whi; i += kWave) {  // this wave's counts
    const uint32_t k = ids ? embed_key(ids[i], V, pad) : keys[i];
    atomicAdd(&slot[wave][(k >> shift) & (radix - 1)], 1u);
  }
  // digit totals over all tiles, and the part of the tiles before this one: two digits a thread, and the tiles dealt out
  // to four groups of threads
  const int pair = tid % (kMaxRadix / 2), quarter = tid / (kMaxRadix / 2), r0 = 2 * pair;
  uint32_t total[2] = {0, 0}, before[2] = {0, 0};
  if (r0 < radix) {
    const uint2* col = reinterpret_cast<const uint2*>(counts + r0);  // radix is even: bits >= 1
    const int tiles = int(gridDim.x), mine = int(blockIdx.x);
    for (int b0 = quarter; b0 < tiles; b0 += 4 * 8) {
      uint2 c[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int b = b0 + 4 * k;
        c[k] = col[int64_t(b < tiles ? b : 0) * (radix / 2)];
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int b = b0 + 4 * k;
        if (b < tiles) total[0] += c[k].x, total[1] += c[k].y;
        if (b < mine) before[0] += c[k].x, before[1] += c[k].y;
      }
    }
  }
  part[quarter][pair] = uint4{total[0], total[1], before[0], before[1]};
  __syncthreads();
  // exclusive sums of the totals in the order of the digits, by the first group
  uint32_t incl = 0;
  if (quarter == 0) {
    for (int q = 1; q < 4; q++) {
      const uint4 o = part[q][pair];
      total[0] += o.x, total[1] += o.y, before[0] += o.z, before[1] += o.w;
    }
    incl = total[0] + total[1];
    for (int off = 1; off < kWave; off <<= 1) {
      const uint32_t up = __shfl_up(incl, off);
      if (lane >= off) incl += up;
    }
    if (lane == kWave - 1) wsum[wave] = incl;
  }
  __syncthreads();
  if (quarter == 0 && r0 < radix) {
    uint32_t excl = incl - total[0] - total[1];
    for (int w = 0; w < wave; w++) excl += wsum[w];
    base[r0] = excl + before[0];
    base[r0 + 1] = excl + total[0] + before[1];
  }
  __syncthreads();
  for (int r = tid; r < radix; r += kSortThreads) {
    uint32_t at = base[r];
    for (int w = 0; w < kSortWaves; w++) {
      const uint32_t c = slot[w][r];
      slot[w][r] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = wlo; i0 < whi; i0 += kWave) {
    const int64_t i = i0 + lane;
    const bool active = i < whi;
    const uint32_t k = !active ? 0u : ids ? embed_key(ids[i], V, pad) : keys[i];
    const uint32_t at = take_slot(slot[wave], (k >> shift) & (radix - 1), bits, active);
    if (active) {
      okeys[at] = k;
      opos[at] = ids ? uint32_t(i) : pos[i];
    }
  }
}

// ------------------------------------------------------------------------------------------ segment sums
// The sorted positions are cut into pieces of one length, and 2^lpr lanes walk a piece for a chunk of 2^lpr VEC columns:
// the reads of dy are spread evenly however the tokens are distributed. A token whose segment lies inside a piece is
// written at once. One that crosses pieces leaves its sum in each: part[2p] for the segment that entered piece p,
// part[2p + 1] for one that starts in p and goes on; k_embed_join adds those up in order. Rows without a token are
// written by the same launch's further workgroups.
struct SumPlan {
  int64_t piece = 0, pieces = 0;  // positions in a piece, pieces
  int lpr = 0;
  int64_t chunks = 0;             // of columns
};

constexpr int kAhead = 8;        // rows of dy in flight per lane
constexpr int kZeroRows = 64;    // rows that a zero-writing workgroup looks at at a time
constexpr int64_t kZeroGroups = 1 << 22;  // such workgroups at most: they go on in steps of all of them

__device__ __forceinline__ uint32_t lower_bound(const uint32_t* __restrict__ keys, uint32_t n, uint32_t v) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <typename TW, int VEC>
__device__ __forceinline__ void write_row(TW* __restrict__ dw, int64_t at, const float (&acc)[VEC], float scale) {
  float o[VEC];
#pragma unroll
  for (int k = 0; k < VEC; k++) o[k] = acc[k] * scale;
  store_run<TW, VEC>(dw + at, o);
}

template <typename TW, typename TO, int VEC>
__global__ __launch_bounds__(256) void k_embed_sum(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                   uint32_t n, const TO* __restrict__ dy, int64_t dys,
                                                   TW* __restrict__ dw, float* __restrict__ part, int64_t V, int64_t D,
                                                   float scale, SumPlan s, uint32_t sum_blocks) {
  if (blockIdx.x >= sum_blocks) {
    __shared__ bool used[kZeroRows];
    float zero[VEC] = {};
    const int lane = threadIdx.x & ((1 << s.lpr) - 1);
    const int64_t step = int64_t(gridDim.x - sum_blocks) * kZeroRows;
    for (int64_t v0 = int64_t(blockIdx.x - sum_blocks) * kZeroRows; v0 < V; v0 += step) {
      const int rows = int(min(int64_t(kZeroRows), V - v0));
      if (threadIdx.x < rows) {
        const uint32_t v = uint32_t(v0 + threadIdx.x), at = lower_bound(keys, n, v);
        used[threadIdx.x] = at < n && keys[at] == v;
      }
      __syncthreads();
      for (int r = threadIdx.x >> s.lpr; r < rows; r += 256 >> s.lpr) {
        if (used[r]) continue;
        for (int64_t c = int64_t(lane) * VEC; c < D; c += int64_t(VEC) << s.lpr)
          store_run<TW, VEC>(dw + (v0 + r) * D + run_start(c, D, VEC), zero);
      }
      __syncthreads();
    }
    return;
  }
  const int64_t unit = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> s.lpr;
  const int64_t p = unit / s.chunks;
  const int64_t c0 = ((unit - p * s.chunks) << s.lpr) * VEC + (threadIdx.x & ((1 << s.lpr) - 1)) * VEC;
  if (p >= s.pieces || c0 >= D) return;
  const int64_t c = run_start(c0, D, VEC);
  const uint32_t lo = uint32_t(p * s.piece), hi = uint32_t(min(int64_t(n), int64_t(lo) + s.piece));
  uint32_t cur = keys[lo];
  bool entered = lo > 0 && keys[lo - 1] == cur;  // the segment at hand began in an earlier piece
  const bool leaves = hi < n && keys[hi] == keys[hi - 1];
  float acc[VEC] = {};
  for (uint32_t j0 = lo; j0 < hi; j0 += kAhead) {
    uint32_t k[kAhead];
    RunOf<TO, VEC> row[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; q++) {
      const uint32_t j = min(j0 + q, hi - 1);
      k[q] = keys[j];
      row[q] = *reinterpret_cast<const RunOf<TO, VEC>*>(dy + int64_t(pos[j]) * dys + c);
    }
#pragma unroll
    for (int q = 0; q < kAhead; q++) {
      if (j0 + q >= hi) break;
      if (k[q] != cur) {
        if (entered) {
          store_run<float, VEC>(part + 2 * p * D + c, acc);
        } else {
          write_row<TW, VEC>(dw, int64_t(cur) * D + c, acc, scale);
        }
        entered = false;
        cur = k[q];
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[e] = 0.f;
      }
      if (cur >= uint32_t(V)) return;  // only places without a gradient are left
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[e] += to_f32(row[q].v[e]);
    }
  }
  if (entered || leaves)
    store_run<float, VEC>(part + (2 * p + (entered ? 0 : 1)) * D + c, acc);
  else
    write_row<TW, VEC>(dw, int64_t(cur) * D + c, acc, scale);
}

// A workgroup per piece and chunk: the row whose segment starts in piece p and goes on behind it. The waves add up
// consecutive runs of the pieces it covers; the runs are joined in order.
constexpr int kJoinWaves = 8;

template <typename TW, int VEC>
__global__ __launch_bounds__(kJoinWaves* kWave) void k_embed_join(const uint32_t* __restrict__ keys, uint32_t n,
                                                    const float* __restrict__ part, TW* __restrict__ dw, int64_t V,
                                                    int64_t D, float scale, SumPlan s) {
  __shared__ float run[kJoinWaves][kWave * VEC];
  const int64_t p = blockIdx.x / s.chunks, ch = blockIdx.x - p * s.chunks;
  const uint32_t lo = uint32_t(p * s.piece), hi = uint32_t(min(int64_t(n), int64_t(lo) + s.piece));
  if (hi >= n) return;
  const uint32_t v = keys[hi];
  if (v >= uint32_t(V) || keys[hi - 1] != v || (lo > 0 && keys[lo - 1] == v)) return;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int64_t count = 1;  // pieces covered: p and those whose first position still has token v
  for (bool more = true; more; ) {
    const int64_t at = (p + count + lane) * s.piece;
    const int got = __popcll(__ballot(at < n && keys[at < n ? at : 0] == v));
    count += got;
    more = got == kWave;
  }
  const int64_t c0 = ((ch << s.lpr) + lane) * VEC, c = run_start(c0, D, VEC);
  const bool live = lane < (1 << s.lpr) && c0 < D;
  const int64_t per = (count + kJoinWaves - 1) / kJoinWaves, q0 = min(count, wave * per), q1 = min(count, q0 + per);
  float acc[VEC] = {};
  if (live) {
    // piece p left its sum in slot 2p + 1, the pieces p + 1, p + 2, .. in slots 2p + 2, 2p + 4, ..
#pragma unroll 16
    for (int64_t q = q0; q < q1; q++) {
      float x[VEC];
      load_run<float, VEC>(part + (2 * (p + q) + (q == 0 ? 1 : 0)) * D + c, x);
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[e] += x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; e++) run[wave][lane * VEC + e] = acc[e];
  __syncthreads();
  if (wave == 0 && live) {
#pragma unroll
    for (int w = 1; w < kJoinWaves; w++)
#pragma unroll
      for (int e = 0; e < VEC; e++) acc[e] += run[w][lane * VEC + e];
    write_row<TW, VEC>(dw, int64_t(v) * D + c, acc, scale);
  }
}

int lanes_log2(int64_t D, int vec) {
  int lpr = 0;
  while (lpr < 8 && (int64_t(vec) << lpr) < D) lpr++;
  return lpr;
}

struct SortPlan {
  bool small = false;
  int64_t tile = 0;
  int tiles = 0, passes = 0, bits = 0;
};

SortPlan sort_plan(int64_t n, int64_t V) {
  SortPlan p;
  int nb = 1;
  while ((int64_t(1) << nb) <= V) nb++;  // keys are 0 .. V
  p.small = n <= kSmall;
  const int most = p.small ? kSmallBits : kMaxBits;
  p.passes = (nb + most - 1) / most;
  p.bits = (nb + p.passes - 1) / p.passes;
  const int64_t per = (n + kMaxTiles - 1) / kMaxTiles;
  p.tile = std::max<int64_t>(1, (per + kSortThreads - 1) / kSortThreads) * kSortThreads;
  p.tiles = int((n + p.tile - 1) / p.tile);
  return p;
}

// Pieces of 16 to 256 positions: short enough that about 1500 waves walk them (twice as many where a lane has less than
// 16 bytes of a row), long enough that the sums left between pieces (8 bytes a column and piece, written and read) stay
// below the rows themselves. 131072 rows of 1024 bytes on two tokens take 96 us so, and 153 in twice as many pieces.
SumPlan sum_plan(int64_t n, int64_t D, int vec, bool wide) {
  SumPlan s;
  s.lpr = std::min(6, lanes_log2(D, vec));
  s.chunks = (D + (int64_t(vec) << s.lpr) - 1) / (int64_t(vec) << s.lpr);
  const int64_t lanes = s.chunks << s.lpr, waves = wide ? 1500 : 3000;
  s.piece = 16;
  while (s.piece < 256 && n / (2 * s.piece) * lanes >= waves * kWave) s.piece *= 2;
  s.pieces = (n + s.piece - 1) / s.piece;
  return s;
}

template <typename TI, typename TW, typename TO>
void embed_fwd_t(const TI* ids, const void* w, int64_t ws, void* out, int64_t n, int64_t V, int64_t D, float scale,
                 hipStream_t stream) {
  const TW* wp = static_cast<const TW*>(w);
  TO* op = static_cast<TO*>(out);
  const auto run = [&](auto width) {
    constexpr int VEC = decltype(width)::value;
    // a wave a row where there are rows enough to fill the card, else up to a workgroup a row; less where n passes a launch
    int lpr = std::min(lanes_log2(D, VEC), n >= 4096 ? 6 : 8);
    while (lpr > 0 && (n << lpr) > (int64_t(1) << 31)) lpr--;
    const dim3 grid = grid_of((n + (256 >> lpr) - 1) / (256 >> lpr), 256, "embedding", "ids");
    hipLaunchKernelGGL((k_embed_fwd<TI, TW, TO, VEC>), grid, dim3(256), 0, stream, ids, wp, ws, op, n, V, D, scale, lpr);
    RMM_HIP_CHECK(hipGetLastError());
  };
  if (D >= 8)
    run(std::integral_constant<int, 8>{});
  else
    run(std::integral_constant<int, 1>{});
}

template <typename TI>
void embed_sort(const TI* ids, int64_t n, int64_t V, int64_t pad, uint32_t* ws, const uint32_t** keys,
                const uint32_t** pos, hipStream_t stream) {
  const SortPlan p = sort_plan(n, V);
  uint32_t* buf[2][2] = {{ws, ws + n}, {ws + 2 * n, ws + 3 * n}};
  const uint32_t *kin = nullptr, *pin = nullptr;
  if (p.small) {
    hipLaunchKernelGGL((k_sort_small<TI>), dim3(1), dim3(kSmallThreads), 0, stream, ids, int(n), V, pad, p.passes, p.bits,
                       buf[0][0], buf[0][1]);
    RMM_HIP_CHECK(hipGetLastError());
    kin = buf[0][0];
    pin = buf[0][1];
  }
  uint32_t* counts = ws + (4 * n + 1) / 2 * 2;  // read in pairs
  for (int s = 0; s < p.passes && !p.small; s++) {
    const TI* src = s == 0 ? ids : nullptr;
    hipLaunchKernelGGL((k_sort_hist<TI>), dim3(p.tiles), dim3(kHistThreads), 0, stream, src, kin, n, p.tile, V, pad,
                       s * p.bits, p.bits, counts);
    hipLaunchKernelGGL((k_sort_scatter<TI>), dim3(p.tiles), dim3(kSortThreads), 0, stream, src, kin, pin, n, p.tile, V,
                       pad, s * p.bits, p.bits, counts, buf[s & 1][0], buf[s & 1][1]);
    RMM_HIP_CHECK(hipGetLastError());
    kin = buf[s & 1][0];
    pin = buf[s & 1][1];
  }
  *keys = kin;
  *pos = pin;
}

int64_t sort_words(int64_t n, int64_t V) {
  const SortPlan p = sort_plan(n, V);
  return p.small ? 2 * n : (4 * n + 1) / 2 * 2 + (int64_t(p.tiles) << p.bits);
}

template <typename TW, typename TO, int VEC>
void embed_sum_t(const uint32_t* keys, const uint32_t* pos, int64_t n, const TO* dy, int64_t dys, TW* dw, float* part,
                 int64_t V, int64_t D, float scale, hipStream_t stream) {
  const SumPlan s = sum_plan(n, D, VEC, VEC * sizeof(TO) >= 16);
  const int64_t sums = ((s.pieces * s.chunks << s.lpr) + 255) / 256;
  const int64_t zeros = std::min(kZeroGroups, (V + kZeroRows - 1) / kZeroRows);
  const dim3 grid = grid_of(sums + zeros, 256, "embedding_grad", "elements");
  hipLaunchKernelGGL((k_embed_sum<TW, TO, VEC>), grid, dim3(256), 0, stream, keys, pos, uint32_t(n), dy, dys, dw, part, V, D,
                     scale, s, uint32_t(sums));
  if (s.pieces > 1)
    hipLaunchKernelGGL((k_embed_join<TW, VEC>), grid_of(s.pieces * s.chunks, kJoinWaves * kWave, "embedding_grad", "ids"),
                       dim3(kJoinWaves * kWave), 0, stream, keys, uint32_t(n), part, dw, V, D, scale, s);
  RMM_HIP_CHECK(hipGetLastError());
}

// 16 bytes of dy a lane, or single elements of rows shorter than that.
template <typename TW, typename TO>
void embed_sum_any(const uint32_t* keys, const uint32_t* pos, int64_t n, const void* dy, int64_t dys, void* dw,
                   float* part, int64_t V, int64_t D, float scale, hipStream_t stream) {
  constexpr int VEC = 16 / sizeof(TO);
  const auto sum = D >= VEC ? embed_sum_t<TW, TO, VEC> : embed_sum_t<TW, TO, 1>;
  sum(keys, pos, n, static_cast<const TO*>(dy), dys, static_cast<TW*>(dw), part, V, D, scale, stream);
}

}  // namespace

void embedding_fwd(const void* ids, bool ids64, const void* w, int wtype, int64_t wstride, void* out, int otype,
                   int64_t n, int64_t V, int64_t D, float scale, hipStream_t stream) {
  if (n <= 0 || D <= 0) return;
  dispatch_types(wtype, otype, "embedding", [&](auto tw, auto to) {
    using TW = decltype(tw);
    using TO = decltype(to);
    if (ids64)
      embed_fwd_t<int64_t, TW, TO>(static_cast<const int64_t*>(ids), w, wstride, out, n, V, D, scale, stream);
    else
      embed_fwd_t<int32_t, TW, TO>(static_cast<const int32_t*>(ids), w, wstride, out, n, V, D, scale, stream);
  });
}

int64_t embedding_grad_workspace(int64_t n, int64_t V, int64_t D) {
  if (n <= 0 || D <= 0) return 0;
  int64_t pieces = 0;  // of whichever width the launch will have
  for (int vec : {8, 4, 1}) pieces = std::max(pieces, sum_plan(n, D, vec, vec >= 4).pieces);
  return (sort_words(n, V) + 3) / 4 * 16 + (pieces > 1 ? 2 * pieces * D * int64_t(sizeof(float)) : 0);
}

void embedding_grad(const void* ids, bool ids64, const void* dy, int otype, int64_t dystride, void* dw, int wtype,
                    int64_t n, int64_t V, int64_t D, int64_t pad, float scale, void* workspace, hipStream_t stream) {
  if (V <= 0 || D <= 0) return;
  constexpr int64_t kMax = (int64_t(1) << 31) - 1;
  if (n >= kMax || V >= kMax) throw std::invalid_argument("embedding_grad: fewer than 2^31 - 1 tokens and rows");
  if (n > 0 && workspace == nullptr) throw std::invalid_argument("embedding_grad: no workspace");
  const uint32_t *keys = nullptr, *pos = nullptr;
  float* part = nullptr;
  if (n > 0) {
    uint32_t* ws = static_cast<uint32_t*>(workspace);
    part = reinterpret_cast<float*>(ws + (sort_words(n, V) + 3) / 4 * 4);
    if (ids64)
      embed_sort(static_cast<const int64_t*>(ids), n, V, pad, ws, &keys, &pos, stream);
    else
      embed_sort(static_cast<const int32_t*>(ids), n, V, pad, ws, &keys, &pos, stream);
  }
  dispatch_types(wtype, otype, "embedding_grad", [&](auto tw, auto to) {
    embed_sum_any<decltype(tw), decltype(to)>(keys, pos, n, dy, dystride, dw, part, V, D, scale, stream);
  });
}

}  // namespace hip
}  // namespace rmm
