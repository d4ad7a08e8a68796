// K22: embedding lookup with a scale, and its weight gradient from tokens sorted by id.
//
//   forward   out[i, :] = scale * W[id_i, :]; an id outside [0, V) gives a row of zeros
//   gradient  dW[v, :]  = scale * sum over { i : id_i = v } of dy[i, :], all V rows written
//
// The sum over a token's rows is taken in fp32 in the order of the positions, so the result does not
// depend on scheduling: the positions are sorted by id with a stable radix sort (no floating-point
// atomics) and each row of dW is one walk over its segment of the sorted positions.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

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
// 2^lpr lanes share a row (VEC elements each); a workgroup has 256 >> lpr rows in flight.
template <typename TI, typename TW, typename TO, int VEC>
__global__ __launch_bounds__(256) void k_embed_fwd(const TI* __restrict__ ids, const TW* __restrict__ w, int64_t ws,
                                                   TO* __restrict__ out, int64_t n, int64_t V, int64_t D, float scale,
                                                   int lpr) {
  const int lane = threadIdx.x & ((1 << lpr) - 1);
  const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> lpr;
  if (i >= n) return;
  const int64_t id = int64_t(ids[i]);
  const bool ok = id >= 0 && id < V;
  const TW* row = w + (ok ? id : 0) * ws;
  for (int64_t c = int64_t(lane) * VEC; c < D; c += int64_t(VEC) << lpr) {
    float v[VEC];
    if (ok) {
      load_vec<TW, VEC>(row + c, v);
#pragma unroll
      for (int k = 0; k < VEC; k++) v[k] *= scale;
    } else {
#pragma unroll
      for (int k = 0; k < VEC; k++) v[k] = 0.f;
    }
    store_vec<TO, VEC>(out + i * D + c, v);
  }
}

// ------------------------------------------------------------------------------------------ sort
constexpr int kSortThreads = 256, kSortWaves = kSortThreads / kWave, kMaxBits = 9, kMaxRadix = 1 << kMaxBits;
constexpr int kMaxTiles = 256;

// Digit counts of each tile: counts[tile][radix].
template <typename TI>
__global__ __launch_bounds__(kSortThreads) void k_sort_hist(const TI* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                            int64_t n, int64_t tile, int64_t V, int64_t pad, int shift,
                                                            int bits, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[kMaxRadix];
  const int radix = 1 << bits;
  for (int r = threadIdx.x; r < radix; r += kSortThreads) hist[r] = 0;
  __syncthreads();
  const int64_t lo = int64_t(blockIdx.x) * tile, hi = min(n, lo + tile);
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    const uint32_t k = ids ? embed_key(ids[i], V, pad) : keys[i];
    atomicAdd(&hist[(k >> shift) & (radix - 1)], 1u);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < radix; r += kSortThreads) counts[int64_t(blockIdx.x) * radix + r] = hist[r];
}

// Lanes of this wave whose digit equals mine (inactive lanes excluded).
__device__ __forceinline__ uint64_t match_digit(uint32_t d, int bits, bool active) {
  uint64_t m = __ballot(active);
  for (int b = 0; b < bits; b++) {
    const bool one = (d >> b) & 1;
    const uint64_t v = __ballot(one && active);
    m &= one ? v : ~v;
  }
  return m;
}

// Orders LDS accesses of one wave (its lanes run in step; this holds the compiler to that order).
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// One stable pass: tile after tile, wave after wave, round after round, lane after lane is the input order,
// and the slot of an element is (smaller digits anywhere) + (same digit in earlier tiles, waves, rounds, lanes).
template <typename TI>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(const TI* __restrict__ ids,
                                                               const uint32_t* __restrict__ keys,
                                                               const uint32_t* __restrict__ pos, int64_t n, int64_t tile,
                                                               int64_t V, int64_t pad, int shift, int bits,
                                                               const uint32_t* __restrict__ counts,
                                                               uint32_t* __restrict__ okeys, uint32_t* __restrict__ opos) {
  __shared__ uint32_t base[kMaxRadix];                // slot of the digit's first element of this tile
  __shared__ uint32_t whist[kSortWaves][kMaxRadix];   // counts, then running slots, of each wave
  __shared__ uint32_t wsum[kSortWaves];
  const int radix = 1 << bits, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int64_t lo = int64_t(blockIdx.x) * tile, hi = min(n, lo + tile);
  const int64_t seg = tile / kSortWaves, wlo = lo + wave * seg, whi = min(hi, wlo + seg);
  for (int r = lane; r < radix; r += kWave) whist[wave][r] = 0;
  for (int64_t i = wlo + lane; i < whi; i += kWave) {  // this wave's counts
    const uint32_t k = ids ? embed_key(ids[i], V, pad) : keys[i];
    atomicAdd(&whist[wave][(k >> shift) & (radix - 1)], 1u);
  }
  // digits 2t and 2t+1 belong to thread t: totals over all tiles, and the part of the earlier tiles
  const int r0 = 2 * tid;
  uint32_t total[2] = {0, 0}, before[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (r0 + k < radix) {
      for (uint32_t b = 0; b < gridDim.x; b++) {
        const uint32_t c = counts[int64_t(b) * radix + r0 + k];
        total[k] += c;
        if (b < blockIdx.x) before[k] += c;
      }
    }
  }
  uint32_t incl = total[0] + total[1];
  for (int off = 1; off < kWave; off <<= 1) {
    const uint32_t up = __shfl_up(incl, off);
    if (lane >= off) incl += up;
  }
  if (lane == kWave - 1) wsum[wave] = incl;
  __syncthreads();
  uint32_t excl = incl - total[0] - total[1];
  for (int w = 0; w < wave; w++) excl += wsum[w];
  if (r0 < radix) base[r0] = excl + before[0];
  if (r0 + 1 < radix) base[r0 + 1] = excl + total[0] + before[1];
  __syncthreads();
  for (int r = tid; r < radix; r += kSortThreads) {
    uint32_t at = base[r];
    for (int w = 0; w < kSortWaves; w++) {
      const uint32_t c = whist[w][r];
      whist[w][r] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = wlo; i0 < whi; i0 += kWave) {
    const int64_t i = i0 + lane;
    const bool active = i < whi;
    const uint32_t k = !active ? 0u : ids ? embed_key(ids[i], V, pad) : keys[i];
    const uint32_t d = (k >> shift) & (radix - 1);
    const uint64_t same = match_digit(d, bits, active);
    if (active) {
      const int rank = __popcll(same & ((uint64_t(1) << lane) - 1));
      const uint32_t at = whist[wave][d] + rank;
      wave_fence();  // all lanes have read the slot before its first lane moves it on
      if (rank == 0) whist[wave][d] += __popcll(same);
      okeys[at] = k;
      opos[at] = ids ? uint32_t(i) : pos[i];
    }
    wave_fence();
  }
}

// ------------------------------------------------------------------------------------------ segment sums
__device__ __forceinline__ uint32_t lower_bound(const uint32_t* __restrict__ keys, uint32_t n, uint32_t v) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <typename TW, typename TO, int VEC>
__global__ __launch_bounds__(256) void k_embed_rows(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                    uint32_t n, const TO* __restrict__ dy, int64_t dys,
                                                    TW* __restrict__ dw, int64_t V, int64_t D, float scale, int lpr) {
  const int lane = threadIdx.x & ((1 << lpr) - 1);
  const int64_t v = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> lpr;
  if (v >= V) return;
  const uint32_t first = lower_bound(keys, n, uint32_t(v));
  for (int64_t c = int64_t(lane) * VEC; c < D; c += int64_t(VEC) << lpr) {
    float acc[VEC] = {};
    for (uint32_t j = first; j < n && keys[j] == uint32_t(v); j++) {
      float x[VEC];
      load_vec<TO, VEC>(dy + int64_t(pos[j]) * dys + c, x);
#pragma unroll
      for (int k = 0; k < VEC; k++) acc[k] += x[k];
    }
#pragma unroll
    for (int k = 0; k < VEC; k++) acc[k] *= scale;
    store_vec<TW, VEC>(dw + v * D + c, acc);
  }
}

int lanes_log2(int64_t D, int vec) {
  int lpr = 0;
  while (lpr < 8 && (int64_t(vec) << lpr) < D) lpr++;
  return lpr;
}

uint32_t row_blocks(int64_t rows, int lpr, const char* who) {
  const int64_t blocks = (rows + (256 >> lpr) - 1) / (256 >> lpr);
  if (blocks > (int64_t(1) << 31) - 1) throw std::invalid_argument(std::string(who) + ": too many rows");
  return uint32_t(blocks);
}

struct SortPlan {
  int64_t tile = 0;
  int tiles = 0, passes = 0, bits = 0;
};

SortPlan sort_plan(int64_t n, int64_t V) {
  SortPlan p;
  int nb = 1;
  while ((int64_t(1) << nb) <= V) nb++;  // keys are 0 .. V
  p.passes = (nb + kMaxBits - 1) / kMaxBits;
  p.bits = (nb + p.passes - 1) / p.passes;
  const int64_t per = (n + kMaxTiles - 1) / kMaxTiles;
  p.tile = std::max<int64_t>(2048, (per + kSortThreads - 1) / kSortThreads * kSortThreads);
  p.tiles = int((n + p.tile - 1) / p.tile);
  return p;
}

template <typename TI, typename TW, typename TO>
void embed_fwd_t(const TI* ids, const void* w, int64_t ws, void* out, int64_t n, int64_t V, int64_t D, float scale,
                 hipStream_t stream) {
  const TW* wp = static_cast<const TW*>(w);
  TO* op = static_cast<TO*>(out);
  constexpr int VEC = 8;
  const bool wide = D % VEC == 0 && ws % VEC == 0 && vec_aligned<TW, VEC>(w) && vec_aligned<TO, VEC>(out);
  const int lpr = lanes_log2(D, wide ? VEC : 1);
  const uint32_t blocks = row_blocks(n, lpr, "embedding");
  if (wide)
    hipLaunchKernelGGL((k_embed_fwd<TI, TW, TO, VEC>), dim3(blocks), dim3(256), 0, stream, ids, wp, ws, op, n, V, D,
                       scale, lpr);
  else
    hipLaunchKernelGGL((k_embed_fwd<TI, TW, TO, 1>), dim3(blocks), dim3(256), 0, stream, ids, wp, ws, op, n, V, D,
                       scale, lpr);
  RMM_HIP_CHECK(hipGetLastError());
}

template <typename TI>
void embed_sort(const TI* ids, int64_t n, int64_t V, int64_t pad, uint32_t* ws, const uint32_t** keys,
                const uint32_t** pos, hipStream_t stream) {
  const SortPlan p = sort_plan(n, V);
  uint32_t* buf[2][2] = {{ws, ws + n}, {ws + 2 * n, ws + 3 * n}};
  uint32_t* counts = ws + 4 * n;
  const uint32_t *kin = nullptr, *pin = nullptr;
  for (int s = 0; s < p.passes; s++) {
    const TI* src = s == 0 ? ids : nullptr;
    hipLaunchKernelGGL((k_sort_hist<TI>), dim3(p.tiles), dim3(kSortThreads), 0, stream, src, kin, n, p.tile, V, pad,
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

template <typename TW, typename TO>
void embed_rows_t(const uint32_t* keys, const uint32_t* pos, int64_t n, const void* dy, int64_t dys, void* dw, int64_t V,
                  int64_t D, float scale, hipStream_t stream) {
  constexpr int VEC = 8;
  const bool wide = D % VEC == 0 && dys % VEC == 0 && vec_aligned<TO, VEC>(dy) && vec_aligned<TW, VEC>(dw);
  const int lpr = lanes_log2(D, wide ? VEC : 1);
  const uint32_t blocks = row_blocks(V, lpr, "embedding_grad");
  const TO* yp = static_cast<const TO*>(dy);
  TW* wp = static_cast<TW*>(dw);
  if (wide)
    hipLaunchKernelGGL((k_embed_rows<TW, TO, VEC>), dim3(blocks), dim3(256), 0, stream, keys, pos, uint32_t(n), yp, dys,
                       wp, V, D, scale, lpr);
  else
    hipLaunchKernelGGL((k_embed_rows<TW, TO, 1>), dim3(blocks), dim3(256), 0, stream, keys, pos, uint32_t(n), yp, dys,
                       wp, V, D, scale, lpr);
  RMM_HIP_CHECK(hipGetLastError());
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

int64_t embedding_grad_workspace(int64_t n, int64_t V) {
  if (n <= 0) return 0;
  const SortPlan p = sort_plan(n, V);
  return (4 * n + (int64_t(p.tiles) << p.bits)) * int64_t(sizeof(uint32_t));
}

void embedding_grad(const void* ids, bool ids64, const void* dy, int otype, int64_t dystride, void* dw, int wtype,
                    int64_t n, int64_t V, int64_t D, int64_t pad, float scale, void* workspace, hipStream_t stream) {
  if (V <= 0 || D <= 0) return;
  constexpr int64_t kMax = (int64_t(1) << 31) - 1;
  if (n > kMax || V >= kMax) throw std::invalid_argument("embedding_grad: at most 2^31 - 1 tokens and rows");
  if (n > 0 && workspace == nullptr) throw std::invalid_argument("embedding_grad: no workspace");
  const uint32_t *keys = nullptr, *pos = nullptr;
  if (n > 0) {
    uint32_t* ws = static_cast<uint32_t*>(workspace);
    if (ids64)
      embed_sort(static_cast<const int64_t*>(ids), n, V, pad, ws, &keys, &pos, stream);
    else
      embed_sort(static_cast<const int32_t*>(ids), n, V, pad, ws, &keys, &pos, stream);
  }
  dispatch_types(wtype, otype, "embedding_grad", [&](auto tw, auto to) {
    embed_rows_t<decltype(tw), decltype(to)>(keys, pos, n, dy, dystride, dw, V, D, scale, stream);
  });
}

}  // namespace hip
}  // namespace rmm
