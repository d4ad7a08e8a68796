// K24: gated linear recurrence over [B, L, D], forward, backward and the single-step form.
//
//   z_t = sigmoid(g_t),  h_t = (1 - z_t) h_{t-1} + z_t x_t,  y_t = h_t      (element by element, state in fp32)
//
// A reset at t takes h_{t-1} as 0 there. Steps at or behind a sequence's length leave the state as it is, and
// their y, dx and dg are 0 whatever x, g and dy hold. Backward, with dh the gradient of the state:
//
//   dh_t = dy_t + (1 - z_{t+1}) dh_{t+1}  (0 across a reset),    dx_t = z_t dh_t,
//   dg_t = dh_t (x_t - h_{t-1}) z_t (1 - z_t),                   dh0  = (1 - z_0) dh_0
//
// The forward pass leaves the fp32 state at the start of every chunk of K steps (K = 16, for fp32 tensors 8), from
// which the backward pass recomputes h_{t-1}: that reads less than a stored h would (4 / K bytes an element against the
// element itself) and keeps the rounding of y out of the gradient.
//
// Split. Either pass is a composition of affine maps s -> A s + H, one per step. A wave takes a chunk of K steps of
// 64 VEC channels, loads it whole into registers (every load in flight at once) and composes its K maps per lane; the
// 1 to 4 waves of a workgroup, consecutive chunks, exchange their compositions through LDS; and where a sequence is
// longer than that, workgroups pass the state on in one launch: each publishes its composition as soon as it has it,
// looks back over its predecessors' until it meets a finished state (each wave at other segments), publishes its own
// finished state, and writes its rows. So x, g (and dy) cross the memory bus once for any L, and few channels still fill the card.
//
// Waiting. A published word is one 64-bit atomic (A, H) that carries its own readiness in A: all ones before it is
// written, -1 for a finished state, else in [0, 1]. The workgroups of a chain (one sequence's 64 VEC channels) take their
// segments from the chain's ticket counter, and wait only for lower tickets of that counter, whose workgroups therefore
// run already: by induction over the tickets every wait ends.
//
// A = 0 stands for a reset alone: what is before it is dropped, not multiplied by zero (it may be infinite or NaN).
// Products that underflow are held at the smallest denormal instead, so an infinite state stays infinite.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "common.h"
#include "kernels.h"
#include "vec_types.h"

namespace rmm {
namespace hip {

namespace {

constexpr int kScanWaves = 4;  // most waves of a workgroup
constexpr float kTiny = 1.4e-45f;

template <typename T>
constexpr int chunk_steps() {
  return sizeof(T) == 4 ? 8 : 16;
}

// z = sigmoid(g) and a = 1 - z, both to full relative precision: from exp(-|g|), which cannot overflow.
__device__ __forceinline__ void gate_of(float g, float& z, float& a) {
  const float e = __expf(-fabsf(g));
  const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
  z = g >= 0.f ? big : small;
  a = g >= 0.f ? small : big;
}

__device__ __forceinline__ int length_of(const int64_t* __restrict__ lengths, int64_t b, int L) {
  if (lengths == nullptr) return L;
  const int64_t n = lengths[b];
  return __builtin_amdgcn_readfirstlane(n < 0 ? 0 : n > L ? L : int(n));
}

struct Map {  // s -> A s + H, A = 0: s is dropped
  float A, H;
};

__device__ __forceinline__ float apply(const Map& m, float s) { return m.A == 0.f ? m.H : fmaf(m.A, s, m.H); }

// `later` after `first`
__device__ __forceinline__ Map then(const Map& first, const Map& later) {
  if (later.A == 0.f) return later;
  return Map{first.A == 0.f ? 0.f : fmaxf(first.A * later.A, kTiny), fmaf(later.A, first.H, later.H)};
}

__device__ __forceinline__ uint64_t pack(float a, float h) {
  return (uint64_t(__float_as_uint(a)) << 32) | __float_as_uint(h);
}

__device__ __forceinline__ uint64_t peek(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void publish(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kTicketPitch = 32;  // counters a cache line apart

__global__ __launch_bounds__(256) void k_scan_init(uint64_t* __restrict__ words, int64_t n,
                                                   uint32_t* __restrict__ tickets, int64_t chains) {
  const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x, step = int64_t(gridDim.x) * 256;
  for (int64_t i = at; i < n; i += step) words[i] = ~0ull;
  for (int64_t i = at; i < chains; i += step) tickets[i * kTicketPitch] = 0;
}

// What the words of up to `depth` segments j, j - 1, .. of VEC neighbouring chains say about the state behind segment j:
// the composition of their maps, or, once a finished state is met, that state carried through them (A = kDone). The words
// do not depend on each other, so all are read at once. Segments below 0 do not exist: segment 0 always finishes.
constexpr int kLook = 8;
constexpr float kDone = -1.f;
template <int VEC>
__device__ __forceinline__ void look_back(const uint64_t* __restrict__ word, int j, int depth, int64_t stride,
                                          Map (&acc)[VEC]) {
  uint64_t w[kLook][VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) acc[v] = Map{1.f, 0.f};
#pragma unroll
  for (int q = 0; q < kLook; q++) {
    if (q < depth && j - q >= 0) {
#pragma unroll
      for (int v = 0; v < VEC; v++) w[q][v] = peek(word + (j - q) * stride + v);
    }
  }
#pragma unroll
  for (int q = 0; q < kLook; q++) {
    if (q < depth && j - q >= 0) {
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        if (acc[v].A == kDone) continue;
        while (uint32_t(w[q][v] >> 32) == 0xFFFFFFFFu) {
          __builtin_amdgcn_s_sleep(1);
          w[q][v] = peek(word + (j - q) * stride + v);
        }
        const Map m{__uint_as_float(uint32_t(w[q][v] >> 32)), __uint_as_float(uint32_t(w[q][v]))};
        acc[v] = m.A == kDone ? Map{kDone, apply(acc[v], m.H)} : then(m, acc[v]);
        if (acc[v].A == 0.f) acc[v].A = kDone;  // nothing before a reset matters
      }
    }
  }
}

struct ScanPlace {
  int64_t b, d;
  int seg, wave, lane, waves;
};

// Which (sequence, channels, segment) this workgroup has. Neighbouring workgroups are of different chains, so a chain's
// segments start as far apart as the number of chains allows.
template <int VEC>
__device__ __forceinline__ ScanPlace scan_place(const ScanArgs& p, uint32_t* __restrict__ tickets, uint32_t* shared) {
  const uint32_t tiles = uint32_t((p.D + kWave * VEC - 1) / (kWave * VEC)), chains = uint32_t(p.B) * tiles;
  uint32_t seg = 0;
  const uint32_t c = blockIdx.x % chains, b = c / tiles;
  if (tickets != nullptr) {
    if (threadIdx.x == 0) *shared = atomicAdd(tickets + int64_t(c) * kTicketPitch, 1u);
    __syncthreads();
    seg = __builtin_amdgcn_readfirstlane(*shared);
  }
  ScanPlace s;
  s.seg = int(seg);
  s.b = b;
  s.lane = threadIdx.x % kWave;
  s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  s.waves = blockDim.x / kWave;
  s.d = (int64_t(c - b * tiles) * kWave + s.lane) * VEC;
  return s;
}

// Bits of the first cnt (< 32) steps that have a reset; the same in every lane.
__device__ __forceinline__ uint32_t reset_bits(const uint8_t* __restrict__ resets, int64_t at, int lane, int cnt) {
  if (resets == nullptr) return 0;
  return uint32_t(__ballot(lane < cnt && resets[at + lane] != 0));
}

template <typename T, int VEC, int K>
__device__ __forceinline__ void load_rows(const T* __restrict__ p, int64_t stride, int cnt, VecOf<T, VEC> (&r)[K]) {
  if (cnt == K) {
#pragma unroll
    for (int i = 0; i < K; i++) r[i] = *reinterpret_cast<const VecOf<T, VEC>*>(p + i * stride);
  } else {
#pragma unroll
    for (int i = 0; i < K; i++)
      if (i < cnt) r[i] = *reinterpret_cast<const VecOf<T, VEC>*>(p + i * stride);
  }
}

// The state that enters each wave's chunk (`in`), from the waves' compositions and what enters the workgroup, and the
// state behind the workgroup (`last`). The waves look back at different segments at the same time, `depth` each.
template <int VEC>
__device__ __forceinline__ void exchange(const ScanArgs& p, const ScanPlace& s, bool forward, int seg, int nseg, int depth,
                                         const float* __restrict__ start, uint64_t* __restrict__ words,
                                         const Map (&mine)[VEC], float (&in)[VEC], float (&last)[VEC]) {
  __shared__ Map maps[kScanWaves][kWave * VEC];
  __shared__ Map seen[2][kScanWaves][kWave * VEC];
  const bool live = s.d < p.D;
  const int at = s.lane * VEC;
#pragma unroll
  for (int v = 0; v < VEC; v++) maps[s.wave][at + v] = mine[v];
  __syncthreads();
  const int64_t dp = (p.D + 127) / 128 * 128, stride = p.B * dp;
  uint64_t* word = words + s.b * dp + s.d;
  Map all[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    all[v] = Map{1.f, 0.f};
    for (int k = 0; k < s.waves; k++) all[v] = then(all[v], maps[forward ? k : s.waves - 1 - k][at + v]);
  }
  if (seg == 0) {
#pragma unroll
    for (int v = 0; v < VEC; v++) in[v] = live && start ? start[s.b * p.D + s.d + v] : 0.f;
  } else {
    if (s.wave == 0 && live) {
#pragma unroll
      for (int v = 0; v < VEC; v++) publish(word + seg * stride + v, pack(all[v].A, all[v].H));
    }
    Map acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) acc[v] = Map{live ? 1.f : kDone, 0.f};
    // every wave follows the same joined composition, so all leave after the same round
    bool more = true;
    for (int j = seg - 1, round = 0; more; j -= s.waves * depth, round ^= 1) {
      Map found[VEC];
      if (live) look_back<VEC>(word, j - s.wave * depth, depth, stride, found);
#pragma unroll
      for (int v = 0; v < VEC; v++) seen[round][s.wave][at + v] = found[v];
      __syncthreads();
      bool open = false;
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        for (int k = 0; k < s.waves; k++) {
          const Map m = seen[round][k][at + v];
          if (acc[v].A != kDone) {
            acc[v] = m.A == kDone ? Map{kDone, apply(acc[v], m.H)} : then(m, acc[v]);
          }
        }
        open = open || acc[v].A != kDone;
      }
      more = __any(open);
    }
#pragma unroll
    for (int v = 0; v < VEC; v++) in[v] = acc[v].H;
  }
#pragma unroll
  for (int v = 0; v < VEC; v++) last[v] = apply(all[v], in[v]);
  if (nseg > 1 && s.wave == 0 && live) {
#pragma unroll
    for (int v = 0; v < VEC; v++) publish(word + seg * stride + v, pack(kDone, last[v]));
  }
  const int before = forward ? s.wave : s.waves - 1 - s.wave;  // chunks of this workgroup that come before mine
#pragma unroll
  for (int v = 0; v < VEC; v++)
    for (int k = 0; k < before; k++) in[v] = apply(maps[forward ? k : s.waves - 1 - k][at + v], in[v]);
}

// The steps of a chunk: how many lie inside the tensor, how many of them belong to the sequence, which have a reset.
struct Chunk {
  int64_t t0;
  int ck, rows, cnt;
  uint32_t resets;
};

template <int K>
__device__ __forceinline__ Chunk chunk_of(const ScanArgs& p, const ScanPlace& s, int seg) {
  Chunk c;
  c.ck = seg * s.waves + s.wave;
  const int L = int(p.L), t0 = c.ck * K, n = length_of(p.lengths, s.b, L);
  c.t0 = t0;
  c.rows = max(0, min(K, L - t0));
  c.cnt = max(0, min(K, n - t0));
  c.resets = reset_bits(p.resets, s.b * p.L + t0, s.lane, c.cnt);
  return c;
}

// One chunk forward: ca, ch become the composition up to each step, m that of the chunk. PLAIN: all K steps and no reset.
template <bool PLAIN, typename T, int VEC, int K>
__device__ __forceinline__ void compose(const Chunk& c, const VecOf<T, VEC> (&x)[K], const VecOf<T, VEC> (&g)[K],
                                        float (&ca)[K][VEC], float (&ch)[K][VEC], Map (&m)[VEC]) {
#pragma unroll
  for (int i = 0; i < K; i++) {
    const bool drop = !PLAIN && ((c.resets >> i) & 1), dropped = !PLAIN && (c.resets & ((2u << i) - 1)) != 0;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        float z, a;
        gate_of(to_f32(g[i].v[v]), z, a);
        const float u = z * to_f32(x[i].v[v]);
        m[v].H = drop ? u : fmaf(a, m[v].H, u);
        m[v].A = dropped ? 0.f : fmaxf(m[v].A * a, kTiny);
      }
      ca[i][v] = m[v].A;
      ch[i][v] = m[v].H;
    }
  }
}

// s carried through the composition (a, h), which has no reset in it where PLAIN.
template <bool PLAIN>
__device__ __forceinline__ float carry(float a, float h, float s) {
  return PLAIN ? fmaf(a, s, h) : apply(Map{a, h}, s);
}

template <bool PLAIN, typename T, int VEC, int K>
__device__ __forceinline__ void write_states(const Chunk& c, const float (&ca)[K][VEC], const float (&ch)[K][VEC],
                                             const float (&in)[VEC], T* __restrict__ y, int64_t stride) {
#pragma unroll
  for (int i = 0; i < K; i++) {
    if (PLAIN || i < c.rows) {
      float o[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v++) o[v] = PLAIN || i < c.cnt ? carry<PLAIN>(ca[i][v], ch[i][v], in[v]) : 0.f;
      store_vec<T, VEC>(y + i * stride, o);
    }
  }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_scan_fwd(ScanArgs p, const T* __restrict__ x, const T* __restrict__ g,
                                                  T* __restrict__ y, int nseg, int depth, uint64_t* __restrict__ words,
                                                  uint32_t* __restrict__ tickets) {
  constexpr int K = chunk_steps<T>();
  __shared__ uint32_t shared;
  const ScanPlace s = scan_place<VEC>(p, tickets, &shared);
  const bool live = s.d < p.D;
  const Chunk c = chunk_of<K>(p, s, s.seg);
  VecOf<T, VEC> xr[K], gr[K];
  if (live) {
    load_rows<T, VEC, K>(x + s.b * p.xsb + c.t0 * p.xst + s.d, p.xst, c.cnt, xr);
    load_rows<T, VEC, K>(g + s.b * p.gsb + c.t0 * p.gst + s.d, p.gst, c.cnt, gr);
  }
  float ca[K][VEC], ch[K][VEC];
  Map m[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v] = Map{1.f, 0.f};
  const bool plain = c.cnt == K && c.resets == 0;
  if (plain)
    compose<true, T, VEC, K>(c, xr, gr, ca, ch, m);
  else
    compose<false, T, VEC, K>(c, xr, gr, ca, ch, m);
  float in[VEC], last[VEC];
  exchange<VEC>(p, s, true, s.seg, nseg, depth, p.h0, words, m, in, last);
  if (!live) return;
  if (s.wave == 0 && s.seg == nseg - 1) store_vec<float, VEC>(p.h_last + s.b * p.D + s.d, last);
  if (c.rows > 0 && p.ckpt) store_vec<float, VEC>(p.ckpt + (s.b * ((p.L + K - 1) / K) + c.ck) * p.D + s.d, in);
  T* yp = y + (s.b * p.L + c.t0) * p.D + s.d;
  if (plain)
    write_states<true, T, VEC, K>(c, ca, ch, in, yp, p.D);
  else
    write_states<false, T, VEC, K>(c, ca, ch, in, yp, p.D);
}

// One chunk backward: z, the gate's factor dg / dh (cc) and, running against time, the composition of what reaches the
// state behind step i from outside the chunk (aa) and from inside (dh).
template <bool PLAIN, typename T, int VEC, int K>
__device__ __forceinline__ void compose_back(const Chunk& c, const VecOf<T, VEC> (&x)[K], const VecOf<T, VEC> (&g)[K],
                                             const VecOf<T, VEC> (&dy)[K], bool has_dy, float (&h)[VEC],
                                             float (&zz)[K][VEC], float (&cc)[K][VEC], float (&aa)[K][VEC],
                                             float (&dh)[K][VEC], Map (&m)[VEC]) {
#pragma unroll
  for (int i = 0; i < K; i++) {
    const bool drop = !PLAIN && ((c.resets >> i) & 1);
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        gate_of(to_f32(g[i].v[v]), zz[i][v], aa[i][v]);
        const float xv = to_f32(x[i].v[v]), prev = drop ? 0.f : h[v];
        cc[i][v] = (xv - prev) * (zz[i][v] * aa[i][v]);
        h[v] = fmaf(aa[i][v], prev, zz[i][v] * xv);
      }
    }
  }
#pragma unroll
  for (int i = K - 1; i >= 0; i--) {
    const bool drop = !PLAIN && ((c.resets >> i) & 1), dropped = !PLAIN && (c.resets >> i) != 0;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        const float d = has_dy ? m[v].H + to_f32(dy[i].v[v]) : m[v].H, a = aa[i][v];
        dh[i][v] = d;
        aa[i][v] = m[v].A;
        m[v].H = drop ? 0.f : a * d;
        m[v].A = dropped ? 0.f : fmaxf(m[v].A * a, kTiny);
      }
    }
  }
}

template <bool PLAIN, typename T, int VEC, int K>
__device__ __forceinline__ void write_grads(const Chunk& c, const float (&zz)[K][VEC], const float (&cc)[K][VEC],
                                            const float (&aa)[K][VEC], const float (&dh)[K][VEC], const float (&in)[VEC],
                                            T* __restrict__ dx, T* __restrict__ dg, int64_t stride) {
#pragma unroll
  for (int i = 0; i < K; i++) {
    if (PLAIN || i < c.rows) {
      float ox[VEC], og[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        const bool has = PLAIN || i < c.cnt;
        const float d = has ? carry<PLAIN>(aa[i][v], dh[i][v], in[v]) : 0.f;
        ox[v] = has ? d * zz[i][v] : 0.f;
        og[v] = has ? d * cc[i][v] : 0.f;
      }
      store_vec<T, VEC>(dx + i * stride, ox);
      store_vec<T, VEC>(dg + i * stride, og);
    }
  }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_scan_bwd(ScanArgs p, const T* __restrict__ x, const T* __restrict__ g,
                                                  const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ dg,
                                                  int nseg, int depth, uint64_t* __restrict__ words,
                                                  uint32_t* __restrict__ tickets) {
  constexpr int K = chunk_steps<T>();
  __shared__ uint32_t shared;
  const ScanPlace s = scan_place<VEC>(p, tickets, &shared);
  const bool live = s.d < p.D;
  const Chunk c = chunk_of<K>(p, s, nseg - 1 - s.seg);  // time runs backwards along the tickets
  VecOf<T, VEC> xr[K], gr[K], yr[K];
  float h[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) h[v] = 0.f;
  if (live) {
    if (c.rows > 0) load_vec<float, VEC>(p.ckpt + (s.b * ((p.L + K - 1) / K) + c.ck) * p.D + s.d, h);
    load_rows<T, VEC, K>(g + s.b * p.gsb + c.t0 * p.gst + s.d, p.gst, c.cnt, gr);
    load_rows<T, VEC, K>(x + s.b * p.xsb + c.t0 * p.xst + s.d, p.xst, c.cnt, xr);
    if (dy) load_rows<T, VEC, K>(dy + s.b * p.ysb + c.t0 * p.yst + s.d, p.yst, c.cnt, yr);
  }
  float zz[K][VEC], cc[K][VEC], aa[K][VEC], dh[K][VEC];
  Map m[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v] = Map{1.f, 0.f};
  const bool plain = c.cnt == K && c.resets == 0 && dy != nullptr;
  if (plain)
    compose_back<true, T, VEC, K>(c, xr, gr, yr, true, h, zz, cc, aa, dh, m);
  else
    compose_back<false, T, VEC, K>(c, xr, gr, yr, dy != nullptr, h, zz, cc, aa, dh, m);
  float in[VEC], last[VEC];
  exchange<VEC>(p, s, false, s.seg, nseg, depth, p.dh_last, words, m, in, last);
  if (!live) return;
  if (p.dh0 && s.wave == 0 && s.seg == nseg - 1) store_vec<float, VEC>(p.dh0 + s.b * p.D + s.d, last);
  T *xp = dx + s.b * p.dsb + c.t0 * p.dst + s.d, *gp = dg + s.b * p.dsb + c.t0 * p.dst + s.d;
  if (plain)
    write_grads<true, T, VEC, K>(c, zz, cc, aa, dh, in, xp, gp, p.dst);
  else
    write_grads<false, T, VEC, K>(c, zz, cc, aa, dh, in, xp, gp, p.dst);
}

template <typename T>
__global__ __launch_bounds__(256) void k_scan_step(const T* __restrict__ x, int64_t xs, const T* __restrict__ g,
                                                   int64_t gs, const uint8_t* __restrict__ resets, const float* h,
                                                   float* out, T* __restrict__ y, int64_t B, int64_t D) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= B * D) return;
  const int64_t b = i / D, d = i - b * D;
  float z, a;
  gate_of(to_f32(g[b * gs + d]), z, a);
  const float u = z * to_f32(x[b * xs + d]);
  const float hn = resets && resets[b] ? u : fmaf(a, h[i], u);
  out[i] = hn;
  y[i] = from_f32<T>(hn);
}

struct ScanPlan {
  int waves = 1, depth = 1;
  int64_t nseg = 1, chains = 0, blocks = 0;
};

int steps_of(int type) { return type == kF32 ? chunk_steps<float>() : chunk_steps<f16_t>(); }

ScanPlan scan_plan(const ScanArgs& p, int type, int vec, const char* who) {
  ScanPlan s;
  if (p.L >= (int64_t(1) << 31) - 64) throw std::invalid_argument(std::string(who) + ": too many steps");
  const int64_t chunks = std::max<int64_t>(1, (p.L + steps_of(type) - 1) / steps_of(type));
  s.waves = int(std::min<int64_t>(kScanWaves, chunks));
  s.nseg = (chunks + s.waves - 1) / s.waves;
  const int64_t tiles = (p.D + kWave * vec - 1) / (kWave * vec);
  if (p.B > (int64_t(1) << 31) / tiles / s.nseg) throw std::invalid_argument(std::string(who) + ": too many elements");
  s.chains = p.B * tiles;
  s.blocks = s.chains * s.nseg;
  // about 1024 workgroups run at a time, so that many / chains segments of a chain are unfinished
  s.depth = int(std::max<int64_t>(1, std::min<int64_t>(kLook, 1024 / kScanWaves / s.chains)));
  return s;
}

int64_t scan_words(const ScanArgs& p, const ScanPlan& s) { return s.nseg == 1 ? 0 : s.nseg * p.B * ((p.D + 127) / 128 * 128); }

// Two channels a lane where every row of every tensor starts at a multiple of two elements.
template <typename T>
bool pairs(const ScanArgs& p, std::initializer_list<const void*> ptrs) {
  if ((p.D | p.xsb | p.xst | p.gsb | p.gst | p.ysb | p.yst | p.dsb | p.dst) % 2) return false;
  for (const void* q : ptrs)
    if (!vec_aligned<T, 2>(q)) return false;
  return true;
}

// Words not yet written, tickets 0: before a pass whose workgroups hand the state on.
uint32_t* scan_begin(const ScanArgs& p, const ScanPlan& s, const char* who, hipStream_t stream) {
  if (s.nseg == 1) return nullptr;
  if (p.workspace == nullptr) throw std::invalid_argument(std::string(who) + ": no workspace");
  const int64_t n = scan_words(p, s);
  uint64_t* words = static_cast<uint64_t*>(p.workspace);
  uint32_t* tickets = reinterpret_cast<uint32_t*>(words + n);
  hipLaunchKernelGGL(k_scan_init, dim3(uint32_t(std::min<int64_t>((n + 1023) / 1024, 2048))), dim3(256), 0, stream, words,
                     n, tickets, s.chains);
  RMM_HIP_CHECK(hipGetLastError());
  return tickets;
}

}  // namespace

int64_t gated_scan_checkpoints(int64_t L, int type) { return (L + steps_of(type) - 1) / steps_of(type); }

int64_t gated_scan_workspace(int64_t B, int64_t L, int64_t D, int type) {
  ScanArgs p;
  p.B = B, p.L = L, p.D = D;
  if (B <= 0 || D <= 0) return 0;
  const ScanPlan s = scan_plan(p, type, 1, "gated_scan");  // no more words and tickets than with pairs of channels
  const int64_t n = scan_words(p, s);
  return n ? n * int64_t(sizeof(uint64_t)) + s.chains * kTicketPitch * int64_t(sizeof(uint32_t)) : 0;
}

void gated_scan_fwd(const ScanArgs& p, const void* x, const void* g, void* y, int type, hipStream_t stream) {
  if (p.B <= 0 || p.D <= 0) return;
  dispatch_type(type, "gated_scan", [&](auto tag) {
    using T = decltype(tag);
    const bool two = pairs<T>(p, {x, g, y});
    const ScanPlan s = scan_plan(p, type, two ? 2 : 1, "gated_scan");
    uint32_t* tickets = scan_begin(p, s, "gated_scan", stream);
    const dim3 grid(uint32_t(s.blocks)), block(uint32_t(s.waves * kWave));
    const T *xp = static_cast<const T*>(x), *gp = static_cast<const T*>(g);
    T* yp = static_cast<T*>(y);
    uint64_t* words = static_cast<uint64_t*>(p.workspace);
    if (two)
      hipLaunchKernelGGL((k_scan_fwd<T, 2>), grid, block, 0, stream, p, xp, gp, yp, int(s.nseg), s.depth, words, tickets);
    else
      hipLaunchKernelGGL((k_scan_fwd<T, 1>), grid, block, 0, stream, p, xp, gp, yp, int(s.nseg), s.depth, words, tickets);
  });
  RMM_HIP_CHECK(hipGetLastError());
}

void gated_scan_bwd(const ScanArgs& p, const void* x, const void* g, const void* dy, void* dx, void* dg, int type,
                    hipStream_t stream) {
  if (p.B <= 0 || p.D <= 0) return;
  if (p.L > 0 && p.ckpt == nullptr) throw std::invalid_argument("gated_scan backward: no saved states");
  dispatch_type(type, "gated_scan backward", [&](auto tag) {
    using T = decltype(tag);
    const bool two = pairs<T>(p, {x, g, dy, dx, dg});
    const ScanPlan s = scan_plan(p, type, two ? 2 : 1, "gated_scan backward");
    uint32_t* tickets = scan_begin(p, s, "gated_scan backward", stream);
    const dim3 grid(uint32_t(s.blocks)), block(uint32_t(s.waves * kWave));
    const T *xp = static_cast<const T*>(x), *gp = static_cast<const T*>(g), *yp = static_cast<const T*>(dy);
    T *dxp = static_cast<T*>(dx), *dgp = static_cast<T*>(dg);
    uint64_t* words = static_cast<uint64_t*>(p.workspace);
    if (two)
      hipLaunchKernelGGL((k_scan_bwd<T, 2>), grid, block, 0, stream, p, xp, gp, yp, dxp, dgp, int(s.nseg), s.depth, words, tickets);
    else
      hipLaunchKernelGGL((k_scan_bwd<T, 1>), grid, block, 0, stream, p, xp, gp, yp, dxp, dgp, int(s.nseg), s.depth, words, tickets);
  });
  RMM_HIP_CHECK(hipGetLastError());
}

void gated_scan_step(const void* x, int64_t xs, const void* g, int64_t gs, const uint8_t* resets, const float* h,
                     float* out, void* y, int type, int64_t B, int64_t D, hipStream_t stream) {
  if (B <= 0 || D <= 0) return;
  const int64_t blocks = (B * D + 255) / 256;
  if (blocks > (int64_t(1) << 31) - 1) throw std::invalid_argument("gated_scan_step: too many elements");
  dispatch_type(type, "gated_scan_step", [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_scan_step<T>), dim3(uint32_t(blocks)), dim3(256), 0, stream, static_cast<const T*>(x), xs,
                       static_cast<const T*>(g), gs, resets, h, out, static_cast<T*>(y), B, D);
  });
  RMM_HIP_CHECK(hipGetLastError());
}

}  // namespace hip
}  // namespace rmm
