// K23: dropout from a counter-based generator; the mask is never stored.
//
//   out[i] = residual[i] + (u_i >= t ? x[i] * 65536 / (65536 - t) : 0),  t = round(65536 p)
//
// u_i are 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011) with key = seed and counter = (i / 8, offset): one counter gives the bits of 8 consecutive elements,
// the low half of a word before the high one. The backward pass computes the same bits from the same
// (seed, offset). 16 bits an element keep the 20 wide multiplies of a counter below the time of its 8 elements'
// memory traffic; the scale is that of the quantised rate, so the expectation of out is exactly x.
//
// Bound by memory: 32768 x 4097 fp16 88 us (6.1 TB/s), 8192 x 8192 bf16 with a residual 68 us (5.9), 4096 x 4096 fp32
// 24 us (5.6, as the last-level cache holds part of it). 8 elements a thread: one counter, and 16-byte loads of the 16-bit
// types.
#include <hip/hip_runtime.h>

#include <cmath>
#include <stdexcept>

#include "common.h"
#include "kernels.h"
#include "vec_types.h"

namespace rmm {
namespace hip {

namespace {

struct Philox4 {
  uint32_t w[4];
};

__device__ __forceinline__ Philox4 philox10(uint64_t index, uint64_t offset, uint64_t seed) {
  uint32_t a = uint32_t(index), b = uint32_t(index >> 32), c = uint32_t(offset), d = uint32_t(offset >> 32);
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = uint64_t(0xD2511F53u) * a, p1 = uint64_t(0xCD9E8D57u) * c;
    a = uint32_t(p1 >> 32) ^ b ^ k0;
    b = uint32_t(p1);
    c = uint32_t(p0 >> 32) ^ d ^ k1;
    d = uint32_t(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox4{{a, b, c, d}};
}

template <typename T, bool RES>
__global__ __launch_bounds__(256) void k_dropout(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ out,
                                                 int64_t n, uint32_t t, float scale, uint64_t seed, uint64_t offset,
                                                 const int64_t* __restrict__ ctr, int64_t* __restrict__ used) {
  const int64_t q = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const uint64_t off = ctr ? uint64_t(*ctr) : offset;
  if (used && q == 0) *used = int64_t(off);
  const int64_t i = q * 8;
  if (i >= n) return;
  const Philox4 r = philox10(uint64_t(q), off, seed);
  float v[8], s[8];
  const int m = int(n - i < 8 ? n - i : 8);
  if (m == 8) {
    load_run<T, 8>(x + i, v);
    if (RES) load_run<T, 8>(res + i, s);
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      v[k] = k < m ? to_f32(x[i + k]) : 0.f;
      if (RES) s[k] = k < m ? to_f32(res[i + k]) : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const uint32_t u = (k & 1) ? r.w[k >> 1] >> 16 : r.w[k >> 1] & 0xffffu;
    v[k] = u >= t ? v[k] * scale : 0.f;  // a select: what is dropped is zero whatever it held
    if (RES) v[k] += s[k];
  }
  if (m == 8) {
    store_run<T, 8>(out + i, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (k < m) out[i + k] = from_f32<T>(v[k]);
  }
}

}  // namespace

void dropout(const void* x, const void* res, void* out, int type, int64_t n, double p, uint64_t seed, uint64_t offset,
             const int64_t* ctr, int64_t* used, hipStream_t stream) {
  if (!(p >= 0.0 && p <= 1.0)) throw std::invalid_argument("dropout: 0 <= p <= 1");
  if (n <= 0) return;
  const uint32_t t = uint32_t(std::nearbyint(p * 65536.0));
  const float scale = t < 65536u ? float(65536.0 / double(65536u - t)) : 0.f;
  const int64_t blocks = (n + 2047) / 2048;
  const dim3 grid = grid_of(blocks, 256, "dropout", "elements");
  dispatch_type(type, "dropout", [&](auto tag) {
    using T = decltype(tag);
    const auto kernel = res ? k_dropout<T, true> : k_dropout<T, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, static_cast<const T*>(x),
                       static_cast<const T*>(res), static_cast<T*>(out), n, t, scale, seed, offset, ctr, used);
  });
  RMM_HIP_CHECK(hipGetLastError());
}

}  // namespace hip
}  // namespace rmm
