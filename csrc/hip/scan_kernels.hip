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
// up to 8 waves of a workgroup take consecutive chunks, exchange their compositions through LDS, and go on to the next
// tile of chunks with the state behind this one, whose loads they issued before the exchange. With enough chains (one
// sequence's 64 VEC channels) to fill the card, that reads x, g (and dy) once. With fewer, a chain is cut into segments:
// k_scan_maps composes the map of each from a first reading, and the workgroups of the pass itself start from the maps
// before theirs. Rows narrower than half a wave's reach put several chunks into a wave. VEC is 2 at any alignment, 1 for a
// single channel.
//
// Bound by memory, x, g, dy and the outputs crossing the bus once (twice for the inputs where chains are cut): bf16, us and
// TB/s, forward / backward: [1024, 64, 1024] 80 (5.0) / 146 (4.6), [32, 2048, 1024] 87 (4.6) / 149 (4.5),
// [16, 3001, 2048] 112 (5.3) / 203 (4.9), cut: [8, 2048, 1024] 35 / 48, [1, 65536, 1024] 130 / 190 of which the first
// reading is 69 / 63 (4.0); fp32 [64, 1024, 512] 77 (5.2) / 139 (4.8). One step of 512 x 8192 bf16 13 us (4.4). About 20
// instructions a step and channel, two of them at quarter rate, are half of the arithmetic that these times leave room for;
// fp32 tensors have chunks of 8 steps to keep within the registers.
//
// A = 0 stands for a reset alone: what is before it is dropped, not multiplied by zero (it may be infinite or NaN).
// Factors and products that underflow are held at the smallest denormal instead, so an infinite state stays infinite.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "common.h"
#include "kernels.h"
#include "vec_types.h"

namespace rmm {
namespace hip {

namespace {

constexpr int kScanWaves = 8, kScanThreads = kScanWaves * kWave;  // most waves of a workgroup
constexpr float kTiny = 1.4e-45f;

template <typename T>
constexpr int chunk_steps() {
  return sizeof(T) == 4 ? 8 : 16;
}

// z = sigmoid(g) and a = 1 - z from exp(-|g|), which cannot overflow: within about |g| + 8 roundings (the exponent's own
// grows with it). Above 87 the smaller of them is zero, though for a finite gate it is not: the recurrence takes the smallest
// denormal more, at no cost, so that an infinite state or input stays infinite. The gradients' factors do without it.
struct Gate {
  float z, a;
  float dx, dg;  // z and z (1 - z)
};

__device__ __forceinline__ Gate gate_of(float g) {
  const float e = __expf(-fabsf(g));
  const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big, held = fmaf(e, big, kTiny);
  const bool open = g >= 0.f;
  return Gate{open ? big : held, open ? held : big, open ? big : small, big * small};
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

// Which sequence, channels and segment a workgroup has, and where this lane stands. A wave's lanes share a row of
// 1 << lpr lanes (all 64 unless the tensor is narrow); with fewer, the wave has several groups, each at a chunk of its own.
struct ScanPlace {
  int64_t b, d;
  int seg, wave, lane, waves, lpr, group, groups;

  __device__ int column(int vec) const { return (lane & ((1 << lpr) - 1)) * vec; }
};

template <int VEC, bool NARROW>
__device__ __forceinline__ ScanPlace scan_place(const ScanArgs& p, int lpr) {
  if (!NARROW) lpr = 6;
  const uint32_t tiles = uint32_t((p.D + (VEC << lpr) - 1) / (VEC << lpr)), chains = uint32_t(p.B) * tiles;
  const uint32_t seg = blockIdx.x / chains, chain = blockIdx.x - seg * chains, b = chain / tiles;
  ScanPlace s;
  s.seg = int(seg);
  s.b = b;
  s.lane = threadIdx.x % kWave;
  s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  s.waves = blockDim.x / kWave;
  s.lpr = lpr;
  s.group = NARROW ? s.lane >> lpr : 0;
  s.groups = NARROW ? kWave >> lpr : 1;
  // The last pair of an odd row begins one channel earlier: two lanes have that channel and write the same values.
  s.d = (int64_t(chain - b * tiles) << lpr) * VEC + s.column(VEC);
  if (VEC == 2 && s.d == p.D - 1) s.d--;
  return s;
}

// Bits of the first cnt (<= K < 32) steps from `at` on that have a reset, for each group of lanes.
template <bool NARROW, int K>
__device__ __forceinline__ uint32_t reset_bits(const uint8_t* __restrict__ resets, const ScanPlace& s, int64_t at, int cnt) {
  if (resets == nullptr) return 0;
  if (!NARROW) return uint32_t(__ballot(s.lane < cnt && resets[at + s.lane] != 0));
  const int size = 1 << s.lpr, j = s.lane & (size - 1);
  uint32_t bits = 0;
  for (int r = 0; r < K; r += size) {
    const uint64_t m = __ballot(r + j < cnt && resets[at + r + j] != 0);
    bits |= uint32_t((m >> (s.group << s.lpr)) & ((uint64_t(1) << size) - 1)) << r;
  }
  return bits;
}

template <typename T, int VEC, int K>
__device__ __forceinline__ void load_rows(const T* __restrict__ p, int64_t stride, int cnt, RunOf<T, VEC> (&r)[K]) {
  if (cnt == K) {
#pragma unroll
    for (int i = 0; i < K; i++) r[i] = *reinterpret_cast<const RunOf<T, VEC>*>(p + i * stride);
  } else {
#pragma unroll
    for (int i = 0; i < K; i++)
      if (i < cnt) r[i] = *reinterpret_cast<const RunOf<T, VEC>*>(p + i * stride);
  }
}

// The groups' maps composed in the order of the recurrence: m becomes that of all groups up to this one.
template <int VEC>
__device__ __forceinline__ void join_groups(const ScanPlace& s, bool forward, Map (&m)[VEC]) {
  for (int off = 1; off < s.groups; off <<= 1) {
    const bool has = forward ? s.group >= off : s.group + off < s.groups;
    const int from = has ? s.lane + (forward ? -off : off) * (1 << s.lpr) : s.lane;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      const Map o{__shfl(m[v].A, from), __shfl(m[v].H, from)};
      if (has) m[v] = then(o, m[v]);
    }
  }
}

// The state that enters this lane's chunk, from the state before the tile (`carry`, which goes on to that behind it) and
// the compositions of the tile's chunks, in the order of the recurrence. `maps` alternates between two buffers from tile
// to tile, so that one barrier a tile is enough.
template <int VEC, bool NARROW>
__device__ __forceinline__ void exchange(const ScanPlace& s, bool forward, Map (*maps)[kWave * VEC], Map (&mine)[VEC],
                                         float (&carry)[VEC], float (&in)[VEC]) {
  const int at = s.column(VEC);
  if (NARROW) join_groups<VEC>(s, forward, mine);
  if (!NARROW || s.group == (forward ? s.groups - 1 : 0)) {
#pragma unroll
    for (int v = 0; v < VEC; v++) maps[s.wave][at + v] = mine[v];
  }
  __syncthreads();
  for (int k = 0; k < s.waves; k++) {
    const int w = forward ? k : s.waves - 1 - k;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (w == s.wave) in[v] = carry[v];
      carry[v] = apply(maps[w][at + v], carry[v]);
    }
  }
  if (NARROW) {  // through the groups of this wave that come before
    const bool has = forward ? s.group > 0 : s.group + 1 < s.groups;
    const int from = has ? s.lane + (forward ? -1 : 1) * (1 << s.lpr) : s.lane;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      const Map o{__shfl(mine[v].A, from), __shfl(mine[v].H, from)};
      if (has) in[v] = apply(o, in[v]);
    }
  }
}

// The state before segment `seg` in the order of the recurrence: the chain's start carried through the maps of the
// segments before it.
template <int VEC>
__device__ __forceinline__ void start_state(const ScanArgs& p, const ScanPlace& s, int seg, const float* __restrict__ start,
                                            const Map* __restrict__ maps, float (&state)[VEC]) {
  const bool live = s.d < p.D;
#pragma unroll
  for (int v = 0; v < VEC; v++) state[v] = live && start ? start[s.b * p.D + s.d + v] : 0.f;
  if (!live) return;
  const Map* m = maps + s.b * p.D + s.d;
#pragma unroll 8
  for (int k = 0; k < seg; k++) {
#pragma unroll
    for (int v = 0; v < VEC; v++) state[v] = apply(m[k * p.B * p.D + v], state[v]);
  }
}

// The steps of a chunk: how many lie inside the tensor, how many of them belong to the sequence, which have a reset.
struct Chunk {
  int64_t t0;
  int ck, rows, cnt;
  uint32_t resets;
};

template <bool NARROW, int K>
__device__ __forceinline__ Chunk chunk_of(const ScanArgs& p, const ScanPlace& s, int n, int ck) {
  Chunk c;
  c.ck = ck;
  const int L = int(p.L), t0 = ck * K;
  c.t0 = t0;
  c.rows = max(0, min(K, L - t0));
  c.cnt = max(0, min(K, n - t0));
  c.resets = reset_bits<NARROW, K>(p.resets, s, s.b * p.L + t0, c.cnt);
  return c;
}

// Whether the chunk is PLAIN, which has code of its own: all K steps take part, and none has a reset. In a wave of
// several chunks some chunk nearly always has a reset, so that there PLAIN allows them: testing whether each step takes
// part is what costs.
template <bool NARROW, int K>
__device__ __forceinline__ bool is_plain(const Chunk& c) {
  return NARROW ? __all(c.cnt == K) : c.cnt == K && c.resets == 0;
}

template <bool PLAIN, bool NARROW>
__device__ __forceinline__ bool drops(const Chunk& c, int i) {
  return (NARROW || !PLAIN) && ((c.resets >> i) & 1);
}

// The chunk's factor of the state before it, from the plain product of its steps' factors.
__device__ __forceinline__ float chunk_factor(const Chunk& c, float product) {
  return c.resets ? 0.f : fmaxf(product, kTiny);
}

// One chunk forward: 1 - z and z x of each step, and the chunk's map.
template <bool PLAIN, bool NARROW, typename T, int VEC, int K>
__device__ __forceinline__ void compose(const Chunk& c, const RunOf<T, VEC> (&x)[K], const RunOf<T, VEC> (&g)[K],
                                        float (&aa)[K][VEC], float (&uu)[K][VEC], Map (&m)[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v] = Map{1.f, 0.f};
#pragma unroll
  for (int i = 0; i < K; i++) {
    const bool drop = drops<PLAIN, NARROW>(c, i);
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        const Gate q = gate_of(to_f32(g[i].v[v]));
        aa[i][v] = q.a;
        uu[i][v] = q.z * to_f32(x[i].v[v]);
        m[v].H = drop ? uu[i][v] : fmaf(aa[i][v], m[v].H, uu[i][v]);
        m[v].A *= aa[i][v];
      }
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v].A = chunk_factor(c, m[v].A);
}

template <bool PLAIN, bool NARROW, typename T, int VEC, int K>
__device__ __forceinline__ void write_states(const Chunk& c, const float (&aa)[K][VEC], const float (&uu)[K][VEC],
                                             float (&h)[VEC], T* __restrict__ y, int64_t stride) {
#pragma unroll
  for (int i = 0; i < K; i++) {
    if (PLAIN || i < c.rows) {
      const bool drop = drops<PLAIN, NARROW>(c, i), has = PLAIN || i < c.cnt;
      float o[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        if (has) h[v] = drop ? uu[i][v] : fmaf(aa[i][v], h[v], uu[i][v]);
        o[v] = has ? h[v] : 0.f;
      }
      store_run<T, VEC>(y + i * stride, o);
    }
  }
}

// `per` tiles in a segment.
template <typename T, int VEC, bool NARROW>
__global__ __launch_bounds__(kScanThreads, NARROW ? 2 : 4) void k_scan_fwd(ScanArgs p, const T* __restrict__ x,
                                                                            const T* __restrict__ g, T* __restrict__ y,
                                                                            int nseg, int per, int lpr,
                                                                            const Map* __restrict__ seg_maps) {
  constexpr int K = chunk_steps<T>();
  __shared__ Map maps[2][kScanWaves][kWave * VEC];
  const ScanPlace s = scan_place<VEC, NARROW>(p, lpr);
  const bool live = s.d < p.D;
  const int n = length_of(p.lengths, s.b, int(p.L)), nck = int((p.L + K - 1) / K), units = s.waves * s.groups;
  const int unit = s.wave * s.groups + s.group;
  const int first = s.seg * per, last = max(first + 1, min(first + per, (nck + units - 1) / units));
  const T *xp = x + s.b * p.xsb + s.d, *gp = g + s.b * p.gsb + s.d;
  RunOf<T, VEC> xr[K], gr[K];
  Chunk c = chunk_of<NARROW, K>(p, s, n, first * units + unit);
  if (live) {
    load_rows<T, VEC, K>(gp + c.t0 * p.gst, p.gst, c.cnt, gr);
    load_rows<T, VEC, K>(xp + c.t0 * p.xst, p.xst, c.cnt, xr);
  }
  float carry[VEC];
  start_state<VEC>(p, s, s.seg, p.h0, seg_maps, carry);
  for (int tile = first; tile < last; tile++) {
    float aa[K][VEC], uu[K][VEC], in[VEC];
    Map m[VEC];
    const Chunk now = c;
    const bool plain = is_plain<NARROW, K>(now);
    if (plain)
      compose<true, NARROW, T, VEC, K>(now, xr, gr, aa, uu, m);
    else
      compose<false, NARROW, T, VEC, K>(now, xr, gr, aa, uu, m);
    if (tile + 1 < last) {
      c = chunk_of<NARROW, K>(p, s, n, (tile + 1) * units + unit);
      if (live) {
        load_rows<T, VEC, K>(gp + c.t0 * p.gst, p.gst, c.cnt, gr);
        load_rows<T, VEC, K>(xp + c.t0 * p.xst, p.xst, c.cnt, xr);
      }
    }
    exchange<VEC, NARROW>(s, true, maps[tile & 1], m, carry, in);
    if (!live) continue;
    if (now.rows > 0 && p.ckpt) store_run<float, VEC>(p.ckpt + (s.b * nck + now.ck) * p.D + s.d, in);
    T* yp = y + (s.b * p.L + now.t0) * p.D + s.d;
    if (plain)
      write_states<true, NARROW, T, VEC, K>(now, aa, uu, in, yp, p.D);
    else
      write_states<false, NARROW, T, VEC, K>(now, aa, uu, in, yp, p.D);
  }
  if (live && unit == 0 && s.seg == nseg - 1) store_run<float, VEC>(p.h_last + s.b * p.D + s.d, carry);
}

// One chunk backward: z, 1 - z and the gate's factor dg / dh (cc) of each step, and the chunk's map of the state's
// gradient. The gradients themselves follow in write_grads, from what enters the chunk.
template <bool PLAIN, bool NARROW, typename T, int VEC, int K>
__device__ __forceinline__ void compose_back(const Chunk& c, const RunOf<T, VEC> (&x)[K], const RunOf<T, VEC> (&g)[K],
                                             const RunOf<T, VEC> (&dy)[K], bool has_dy, float (&h)[VEC],
                                             float (&zz)[K][VEC], float (&aa)[K][VEC], float (&cc)[K][VEC],
                                             Map (&m)[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v] = Map{1.f, 0.f};
#pragma unroll
  for (int i = 0; i < K; i++) {
    const bool drop = drops<PLAIN, NARROW>(c, i);
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        const Gate q = gate_of(to_f32(g[i].v[v]));
        zz[i][v] = q.dx, aa[i][v] = q.a;
        const float xv = to_f32(x[i].v[v]), prev = drop ? 0.f : h[v];
        cc[i][v] = (xv - prev) * q.dg;
        h[v] = fmaf(q.a, prev, q.z * xv);
      }
    }
  }
#pragma unroll
  for (int i = K - 1; i >= 0; i--) {
    const bool drop = drops<PLAIN, NARROW>(c, i);
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        const float d = has_dy ? m[v].H + to_f32(dy[i].v[v]) : m[v].H;
        m[v].H = drop ? 0.f : aa[i][v] * d;
        m[v].A *= aa[i][v];
      }
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v].A = chunk_factor(c, m[v].A);
}

template <bool PLAIN, bool NARROW, typename T, int VEC, int K>
__device__ __forceinline__ void write_grads(const Chunk& c, const RunOf<T, VEC> (&dy)[K], bool has_dy,
                                            const float (&zz)[K][VEC], const float (&aa)[K][VEC],
                                            const float (&cc)[K][VEC], float (&in)[VEC], T* __restrict__ dx,
                                            T* __restrict__ dg, int64_t stride) {
#pragma unroll
  for (int i = K - 1; i >= 0; i--) {
    if (PLAIN || i < c.rows) {
      const bool drop = drops<PLAIN, NARROW>(c, i), has = PLAIN || i < c.cnt;
      float ox[VEC], og[VEC];
#pragma unroll
      for (int v = 0; v < VEC; v++) {
        const float d = has_dy && has ? in[v] + to_f32(dy[i].v[v]) : in[v];
        ox[v] = has ? d * zz[i][v] : 0.f;
        og[v] = has ? d * cc[i][v] : 0.f;
        if (has) in[v] = drop ? 0.f : d * aa[i][v];
      }
      store_run<T, VEC>(dx + i * stride, ox);
      store_run<T, VEC>(dg + i * stride, og);
    }
  }
}

template <typename T, int VEC, bool NARROW>
__global__ __launch_bounds__(kScanThreads) void k_scan_bwd(ScanArgs p, const T* __restrict__ x, const T* __restrict__ g,
                                                           const T* __restrict__ dy, T* __restrict__ dx,
                                                           T* __restrict__ dg, int nseg, int per, int lpr,
                                                           const Map* __restrict__ seg_maps) {
  constexpr int K = chunk_steps<T>();
  __shared__ Map maps[2][kScanWaves][kWave * VEC];
  const ScanPlace s = scan_place<VEC, NARROW>(p, lpr);  // segment 0 is the last in time, where this pass begins
  const bool live = s.d < p.D;
  const int n = length_of(p.lengths, s.b, int(p.L)), nck = int((p.L + K - 1) / K), units = s.waves * s.groups;
  const int unit = s.wave * s.groups + s.group;
  const int first = (nseg - 1 - s.seg) * per, last = max(first + 1, min(first + per, (nck + units - 1) / units));
  const T *xp = x + s.b * p.xsb + s.d, *gp = g + s.b * p.gsb + s.d, *yp = dy ? dy + s.b * p.ysb + s.d : nullptr;
  RunOf<T, VEC> xr[K], gr[K], yr[K];
  float h[VEC] = {};
  Chunk c;
  const auto load = [&](int tile) {
    c = chunk_of<NARROW, K>(p, s, n, tile * units + unit);
    if (!live) return;
    if (c.cnt > 0) load_run<float, VEC>(p.ckpt + (s.b * nck + c.ck) * p.D + s.d, h);
    load_rows<T, VEC, K>(gp + c.t0 * p.gst, p.gst, c.cnt, gr);
    load_rows<T, VEC, K>(xp + c.t0 * p.xst, p.xst, c.cnt, xr);
    if (dy) load_rows<T, VEC, K>(yp + c.t0 * p.yst, p.yst, c.cnt, yr);
  };
  load(last - 1);
  float carry[VEC];
  start_state<VEC>(p, s, s.seg, p.dh_last, seg_maps, carry);
  for (int tile = last - 1; tile >= first; tile--) {
    float zz[K][VEC], aa[K][VEC], cc[K][VEC], in[VEC];
    RunOf<T, VEC> yn[K];
    Map m[VEC];
    const Chunk now = c;
    const bool plain = is_plain<NARROW, K>(now) && dy != nullptr;
    if (plain)
      compose_back<true, NARROW, T, VEC, K>(now, xr, gr, yr, true, h, zz, aa, cc, m);
    else
      compose_back<false, NARROW, T, VEC, K>(now, xr, gr, yr, dy != nullptr, h, zz, aa, cc, m);
#pragma unroll
    for (int i = 0; i < K; i++) yn[i] = yr[i];
    if (tile > first) load(tile - 1);
    exchange<VEC, NARROW>(s, false, maps[tile & 1], m, carry, in);
    if (!live) continue;
    T *dxp = dx + s.b * p.dsb + now.t0 * p.dst + s.d, *dgp = dg + s.b * p.dsb + now.t0 * p.dst + s.d;
    if (plain)
      write_grads<true, NARROW, T, VEC, K>(now, yn, true, zz, aa, cc, in, dxp, dgp, p.dst);
    else
      write_grads<false, NARROW, T, VEC, K>(now, yn, dy != nullptr, zz, aa, cc, in, dxp, dgp, p.dst);
  }
  if (live && p.dh0 && unit == 0 && s.seg == nseg - 1) store_run<float, VEC>(p.dh0 + s.b * p.D + s.d, carry);
}

// m becomes the chunk's map: forward of (gate, input), backward of (gate, dy).
template <bool FORWARD, bool PLAIN, bool NARROW, typename T, int VEC, int K>
__device__ __forceinline__ void compose_map(const Chunk& c, const RunOf<T, VEC> (&g)[K], const RunOf<T, VEC> (&in)[K],
                                            bool has_in, Map (&m)[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v] = Map{1.f, 0.f};
#pragma unroll
  for (int q = 0; q < K; q++) {
    const int i = FORWARD ? q : K - 1 - q;
    const bool drop = drops<PLAIN, NARROW>(c, i);
#pragma unroll
    for (int v = 0; v < VEC; v++) {
      if (PLAIN || i < c.cnt) {
        const Gate gt = gate_of(to_f32(g[i].v[v]));
        const float iv = PLAIN || has_in ? to_f32(in[i].v[v]) : 0.f;
        if (FORWARD)
          m[v].H = drop ? gt.z * iv : fmaf(gt.a, m[v].H, gt.z * iv);
        else
          m[v].H = drop ? 0.f : gt.a * (m[v].H + iv);
        m[v].A *= gt.a;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v].A = chunk_factor(c, m[v].A);
}

// The maps of all segments but the last, in the order of the recurrence: forward of (gate, input), backward of
// (gate, dy). Each wave composes a run of neighbouring chunks on its own; the runs are joined at the end. `len` chunks
// in a segment. Little is kept from chunk to chunk, so 32 waves a CU hide the loads.
constexpr int kMapWaves = 16;

template <typename T, int VEC, bool NARROW, bool FORWARD>
__global__ __launch_bounds__(kMapWaves* kWave, NARROW || sizeof(T) == 4 ? 4 : 8) void k_scan_maps(
    ScanArgs p, const T* __restrict__ g, const T* __restrict__ in, int nseg, int len, int lpr,
    Map* __restrict__ seg_maps) {
  constexpr int K = chunk_steps<T>();
  __shared__ Map maps[kMapWaves][kWave * VEC];
  const ScanPlace s = scan_place<VEC, NARROW>(p, lpr);
  const bool live = s.d < p.D;
  const int n = length_of(p.lengths, s.b, int(p.L)), nck = int((p.L + K - 1) / K), units = s.waves * s.groups;
  const int begin = (FORWARD ? s.seg : nseg - 1 - s.seg) * len, end = min(begin + len, nck);
  const int each = (len + units - 1) / units, lo = min(begin + (s.wave * s.groups + s.group) * each, end);
  const int hi = min(lo + each, end);
  const int64_t isb = FORWARD ? p.xsb : p.ysb, ist = FORWARD ? p.xst : p.yst;
  const T *gp = g + s.b * p.gsb + s.d, *ip = in ? in + s.b * isb + s.d : nullptr;
  Map m[VEC];
#pragma unroll
  for (int v = 0; v < VEC; v++) m[v] = Map{1.f, 0.f};
  for (int k = 0; k < (NARROW ? each : hi - lo); k++) {  // the same count for all lanes of a wave
    const int ck = FORWARD ? lo + k : hi - 1 - k;
    const Chunk c = chunk_of<NARROW, K>(p, s, NARROW && k >= hi - lo ? 0 : n, ck);
    if (!live || c.cnt == 0) continue;
    RunOf<T, VEC> gr[K], ir[K];
    load_rows<T, VEC, K>(gp + c.t0 * p.gst, p.gst, c.cnt, gr);
    if (in) load_rows<T, VEC, K>(ip + c.t0 * ist, ist, c.cnt, ir);
    Map cm[VEC];
    if (is_plain<NARROW, K>(c) && in)
      compose_map<FORWARD, true, NARROW, T, VEC, K>(c, gr, ir, true, cm);
    else
      compose_map<FORWARD, false, NARROW, T, VEC, K>(c, gr, ir, in != nullptr, cm);
#pragma unroll
    for (int v = 0; v < VEC; v++) m[v] = then(m[v], cm[v]);
  }
  if (NARROW) join_groups<VEC>(s, FORWARD, m);
  const int at = s.column(VEC);
  if (!NARROW || s.group == (FORWARD ? s.groups - 1 : 0)) {
#pragma unroll
    for (int v = 0; v < VEC; v++) maps[s.wave][at + v] = m[v];
  }
  __syncthreads();
  if (s.wave != 0 || s.group != 0 || !live) return;
#pragma unroll
  for (int v = 0; v < VEC; v++) {
    Map all{1.f, 0.f};
    for (int k = 0; k < s.waves; k++) all = then(all, maps[FORWARD ? k : s.waves - 1 - k][at + v]);
    seg_maps[(s.seg * p.B + s.b) * p.D + s.d + v] = all;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_scan_step(const T* __restrict__ x, int64_t xs, const T* __restrict__ g,
                                                   int64_t gs, const uint8_t* __restrict__ resets, const float* h,
                                                   float* out, T* __restrict__ y, int64_t B, int64_t D) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= B * D) return;
  const int64_t b = i / D, d = i - b * D;
  const Gate q = gate_of(to_f32(g[b * gs + d]));
  const float u = q.z * to_f32(x[b * xs + d]);
  const float hn = resets && resets[b] ? u : fmaf(q.a, h[i], u);
  out[i] = hn;
  y[i] = from_f32<T>(hn);
}

struct ScanPlan {
  int waves = 1, per = 1, nseg = 1, lpr = 6, units = 1;
  int64_t chains = 0;
};

int steps_of(int type) { return type == kF32 ? chunk_steps<float>() : chunk_steps<f16_t>(); }

// From kEnoughChains on no chain is cut; with fewer, they are cut into at most kGroups workgroups, one a CU (more would
// leave a second round of the backward pass to few). Measured on bf16 (us, forward / backward): 104 chains of 4096 steps
// 110 / 189 cut and 127 / 211 whole, 136 chains 145 / 261 cut and 129 / 214 whole; 8 chains of 65536 steps 127 / 197 in 256
// segments' workgroups, 127 / 220 in 512, 145 / 250 in 1024.
constexpr int64_t kEnoughChains = 128, kGroups = 256;

ScanPlan scan_plan(const ScanArgs& p, int type, int vec, const char* who) {
  if (p.L >= (int64_t(1) << 31) - 65536) throw std::invalid_argument(std::string(who) + ": too many steps");
  ScanPlan s;
  const int64_t chunks = std::max<int64_t>(1, (p.L + steps_of(type) - 1) / steps_of(type));
  while (s.lpr > 0 && p.D <= (vec << (s.lpr - 1))) s.lpr--;
  const int groups = kWave >> s.lpr;
  s.waves = int(std::min<int64_t>(kScanWaves, (chunks + groups - 1) / groups));
  s.units = s.waves * groups;
  const int64_t tiles = (chunks + s.units - 1) / s.units, cols = (p.D + (vec << s.lpr) - 1) / (vec << s.lpr);
  if (p.B > ((int64_t(1) << 31) - 1) / cols) throw std::invalid_argument(std::string(who) + ": too many sequences");
  s.chains = p.B * cols;
  grid_of(s.chains, s.waves * kWave, who, "sequences");  // fewer than kEnoughChains where they are cut
  int64_t nseg = s.chains >= kEnoughChains ? 1 : std::min(tiles, kGroups / s.chains);
  s.per = int((tiles + nseg - 1) / nseg);
  s.nseg = int((tiles + s.per - 1) / s.per);
  return s;
}

template <typename T, int VEC, bool NARROW, bool FORWARD>
void scan_maps_t(const ScanArgs& p, const ScanPlan& s, const T* g, const T* in, const char* who, hipStream_t stream) {
  if (s.nseg == 1) return;
  if (p.workspace == nullptr) throw std::invalid_argument(std::string(who) + ": no workspace");
  hipLaunchKernelGGL((k_scan_maps<T, VEC, NARROW, FORWARD>), dim3(uint32_t(s.chains * (s.nseg - 1))),
                     dim3(kMapWaves * kWave), 0, stream, p, g, in, s.nseg, s.per * s.units, s.lpr,
                     static_cast<Map*>(p.workspace));
}

template <typename T, int VEC, bool NARROW>
void scan_fwd_t(const ScanArgs& p, const ScanPlan& s, const T* x, const T* g, T* y, hipStream_t stream) {
  scan_maps_t<T, VEC, NARROW, true>(p, s, g, x, "gated_scan", stream);
  hipLaunchKernelGGL((k_scan_fwd<T, VEC, NARROW>), dim3(uint32_t(s.chains * s.nseg)), dim3(uint32_t(s.waves * kWave)), 0,
                     stream, p, x, g, y, s.nseg, s.per, s.lpr, static_cast<const Map*>(p.workspace));
  RMM_HIP_CHECK(hipGetLastError());
}

template <typename T, int VEC, bool NARROW>
void scan_bwd_t(const ScanArgs& p, const ScanPlan& s, const T* x, const T* g, const T* dy, T* dx, T* dg,
                hipStream_t stream) {
  scan_maps_t<T, VEC, NARROW, false>(p, s, g, dy, "gated_scan backward", stream);
  hipLaunchKernelGGL((k_scan_bwd<T, VEC, NARROW>), dim3(uint32_t(s.chains * s.nseg)), dim3(uint32_t(s.waves * kWave)), 0,
                     stream, p, x, g, dy, dx, dg, s.nseg, s.per, s.lpr, static_cast<const Map*>(p.workspace));
  RMM_HIP_CHECK(hipGetLastError());
}

}  // namespace

int64_t gated_scan_checkpoints(int64_t L, int type) { return (L + steps_of(type) - 1) / steps_of(type); }

int64_t gated_scan_workspace(int64_t B, int64_t L, int64_t D, int type) {
  ScanArgs p;
  p.B = B, p.L = L, p.D = D;
  if (B <= 0 || D <= 0) return 0;
  const int nseg = scan_plan(p, type, D > 1 ? 2 : 1, "gated_scan").nseg;
  return nseg == 1 ? 0 : (nseg - 1) * B * D * int64_t(sizeof(Map));
}

void gated_scan_fwd(const ScanArgs& p, const void* x, const void* g, void* y, int type, hipStream_t stream) {
  if (p.B <= 0 || p.D <= 0) return;
  dispatch_type(type, "gated_scan", [&](auto tag) {
    using T = decltype(tag);
    const int vec = p.D > 1 ? 2 : 1;
    const ScanPlan s = scan_plan(p, type, vec, "gated_scan");
    const auto fwd = vec == 1 ? scan_fwd_t<T, 1, true> : s.lpr < 6 ? scan_fwd_t<T, 2, true> : scan_fwd_t<T, 2, false>;
    fwd(p, s, static_cast<const T*>(x), static_cast<const T*>(g), static_cast<T*>(y), stream);
  });
}

void gated_scan_bwd(const ScanArgs& p, const void* x, const void* g, const void* dy, void* dx, void* dg, int type,
                    hipStream_t stream) {
  if (p.B <= 0 || p.D <= 0) return;
  if (p.L > 0 && p.ckpt == nullptr) throw std::invalid_argument("gated_scan backward: no saved states");
  dispatch_type(type, "gated_scan backward", [&](auto tag) {
    using T = decltype(tag);
    const int vec = p.D > 1 ? 2 : 1;
    const ScanPlan s = scan_plan(p, type, vec, "gated_scan backward");
    const auto bwd = vec == 1 ? scan_bwd_t<T, 1, true> : s.lpr < 6 ? scan_bwd_t<T, 2, true> : scan_bwd_t<T, 2, false>;
    bwd(p, s, static_cast<const T*>(x), static_cast<const T*>(g), static_cast<const T*>(dy), static_cast<T*>(dx),
        static_cast<T*>(dg), stream);
  });
}

void gated_scan_step(const void* x, int64_t xs, const void* g, int64_t gs, const uint8_t* resets, const float* h,
                     float* out, void* y, int type, int64_t B, int64_t D, hipStream_t stream) {
  if (B <= 0 || D <= 0) return;
  const int64_t blocks = (B * D + 255) / 256;
  const dim3 grid = grid_of(blocks, 256, "gated_scan_step", "elements");
  dispatch_type(type, "gated_scan_step", [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_scan_step<T>), grid, dim3(256), 0, stream, static_cast<const T*>(x), xs,
                       static_cast<const T*>(g), gs, resets, h, out, static_cast<T*>(y), B, D);
  });
  RMM_HIP_CHECK(hipGetLastError());
}

}  // namespace hip
}  // namespace rmm
