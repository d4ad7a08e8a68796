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
// The forward pass leaves the fp32 state at every kTS-th step, from which the backward pass recomputes h_{t-1}:
// that reads less than a stored h would and keeps the rounding of y out of the gradient.
//
// One lane per (sequence, channel); the loads of kTS steps are issued together.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "common.h"
#include "kernels.h"
#include "vec_types.h"

namespace rmm {
namespace hip {

namespace {

constexpr int kTS = 16;  // steps between saved states

// z = sigmoid(g) and a = 1 - z, both to full relative precision: from exp(-|g|), which cannot overflow.
__device__ __forceinline__ void gate_of(float g, float& z, float& a) {
  const float e = __expf(-fabsf(g));
  const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
  z = g >= 0.f ? big : small;
  a = g >= 0.f ? small : big;
}

__device__ __forceinline__ int64_t length_of(const int64_t* __restrict__ lengths, int64_t b, int64_t L) {
  if (lengths == nullptr) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

template <typename T>
__global__ __launch_bounds__(kWave) void k_scan_fwd(ScanArgs p, const T* __restrict__ x, const T* __restrict__ g,
                                                    T* __restrict__ y) {
  const int64_t d = int64_t(blockIdx.x) * kWave + threadIdx.x, b = blockIdx.y;
  if (d >= p.D) return;
  const int64_t n = length_of(p.lengths, b, p.L), nck = (p.L + kTS - 1) / kTS;
  const T *xp = x + b * p.xsb + d, *gp = g + b * p.gsb + d;
  const uint8_t* rp = p.resets ? p.resets + b * p.L : nullptr;
  float h = p.h0 ? p.h0[b * p.D + d] : 0.f;
  for (int64_t t0 = 0; t0 < p.L; t0 += kTS) {
    if (p.ckpt) p.ckpt[(b * nck + t0 / kTS) * p.D + d] = h;
    float xv[kTS], gv[kTS];
#pragma unroll
    for (int i = 0; i < kTS; i++) {
      if (t0 + i < n) {
        xv[i] = to_f32(xp[(t0 + i) * p.xst]);
        gv[i] = to_f32(gp[(t0 + i) * p.gst]);
      }
    }
#pragma unroll
    for (int i = 0; i < kTS; i++) {
      if (t0 + i < n) {
        float z, a;
        gate_of(gv[i], z, a);
        h = rp && rp[t0 + i] ? z * xv[i] : fmaf(a, h, z * xv[i]);
      }
      if (t0 + i < p.L) y[(b * p.L + t0 + i) * p.D + d] = from_f32<T>(t0 + i < n ? h : 0.f);
    }
  }
  p.h_last[b * p.D + d] = h;
}

template <typename T>
__global__ __launch_bounds__(kWave) void k_scan_bwd(ScanArgs p, const T* __restrict__ x, const T* __restrict__ g,
                                                    const T* __restrict__ dy, T* __restrict__ dx, T* __restrict__ dg) {
  const int64_t d = int64_t(blockIdx.x) * kWave + threadIdx.x, b = blockIdx.y;
  if (d >= p.D) return;
  const int64_t n = length_of(p.lengths, b, p.L), nck = (p.L + kTS - 1) / kTS;
  const T *xp = x + b * p.xsb + d, *gp = g + b * p.gsb + d, *yp = dy ? dy + b * p.ysb + d : nullptr;
  const uint8_t* rp = p.resets ? p.resets + b * p.L : nullptr;
  float dh = p.dh_last ? p.dh_last[b * p.D + d] : 0.f;  // gradient reaching the state behind the step at hand
  for (int64_t k = nck - 1; k >= 0; k--) {
    const int64_t t0 = k * kTS;
    float h = p.ckpt[(b * nck + k) * p.D + d];
    float xv[kTS], gv[kTS], yv[kTS], hp[kTS];
#pragma unroll
    for (int i = 0; i < kTS; i++) {
      if (t0 + i < n) {
        xv[i] = to_f32(xp[(t0 + i) * p.xst]);
        gv[i] = to_f32(gp[(t0 + i) * p.gst]);
        yv[i] = yp ? to_f32(yp[(t0 + i) * p.yst]) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kTS; i++) {
      if (t0 + i < n) {
        float z, a;
        gate_of(gv[i], z, a);
        hp[i] = rp && rp[t0 + i] ? 0.f : h;
        h = fmaf(a, hp[i], z * xv[i]);
      }
    }
#pragma unroll
    for (int i = kTS - 1; i >= 0; i--) {
      if (t0 + i >= p.L) continue;
      float ox = 0.f, og = 0.f;
      if (t0 + i < n) {
        float z, a;
        gate_of(gv[i], z, a);
        dh += yv[i];
        ox = dh * z;
        og = dh * (xv[i] - hp[i]) * z * a;
        dh = rp && rp[t0 + i] ? 0.f : dh * a;
      }
      dx[b * p.dsb + (t0 + i) * p.dst + d] = from_f32<T>(ox);
      dg[b * p.dsb + (t0 + i) * p.dst + d] = from_f32<T>(og);
    }
  }
  if (p.dh0) p.dh0[b * p.D + d] = dh;
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

dim3 scan_grid(const ScanArgs& p, const char* who) {
  const int64_t gx = (p.D + kWave - 1) / kWave;
  if (gx > (int64_t(1) << 31) - 1 || p.B > 65535) throw std::invalid_argument(std::string(who) + ": too many rows");
  return dim3(uint32_t(gx), uint32_t(p.B));
}

}  // namespace

int64_t gated_scan_checkpoints(int64_t L) { return (L + kTS - 1) / kTS; }

void gated_scan_fwd(const ScanArgs& p, const void* x, const void* g, void* y, int type, hipStream_t stream) {
  if (p.B <= 0 || p.D <= 0) return;
  const dim3 grid = scan_grid(p, "gated_scan");
  dispatch_type(type, "gated_scan", [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_scan_fwd<T>), grid, dim3(kWave), 0, stream, p, static_cast<const T*>(x),
                       static_cast<const T*>(g), static_cast<T*>(y));
  });
  RMM_HIP_CHECK(hipGetLastError());
}

void gated_scan_bwd(const ScanArgs& p, const void* x, const void* g, const void* dy, void* dx, void* dg, int type,
                    hipStream_t stream) {
  if (p.B <= 0 || p.D <= 0) return;
  if (p.L > 0 && p.ckpt == nullptr) throw std::invalid_argument("gated_scan backward: no saved states");
  const dim3 grid = scan_grid(p, "gated_scan backward");
  dispatch_type(type, "gated_scan backward", [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((k_scan_bwd<T>), grid, dim3(kWave), 0, stream, p, static_cast<const T*>(x),
                       static_cast<const T*>(g), static_cast<const T*>(dy), static_cast<T*>(dx), static_cast<T*>(dg));
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
