// Element types of the sequence kernels (K22-K24): fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

namespace rmm {
namespace hip {

enum ElemType { kF32 = 0, kBF16 = 1, kF16 = 2 };  // the codes of ops/sequence.py

struct alignas(2) bf16_t {
  uint16_t u;
};
using f16_t = _Float16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16_t v) { return float(v); }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float(uint32_t(v.u) << 16); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ f16_t from_f32<f16_t>(float v) {
  return f16_t(v);  // nearest even, overflow to infinity
}
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
  const __bf16 r = __bf16(v);  // nearest even in one instruction, NaN stays NaN
  return bf16_t{__builtin_bit_cast(uint16_t, r)};
}

// N consecutive elements at any element's address: what gfx950 still reads and writes in one instruction for up to 16
// bytes, whatever the alignment.
template <typename T, int N>
struct RunOf {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, float (&x)[N]) {
  const RunOf<T, N> r = *reinterpret_cast<const RunOf<T, N>*>(p);
#pragma unroll
  for (int k = 0; k < N; k++) x[k] = to_f32(r.v[k]);
}

template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float (&x)[N]) {
  RunOf<T, N> r;
#pragma unroll
  for (int k = 0; k < N; k++) r.v[k] = from_f32<T>(x[k]);
  *reinterpret_cast<RunOf<T, N>*>(p) = r;
}

// A grid of fewer than 2^32 threads, the most that HIP launches.
inline dim3 grid_of(int64_t blocks, int threads, const char* who, const char* what) {
  if (blocks > ((int64_t(1) << 32) - 1) / threads) throw std::invalid_argument(std::string(who) + ": too many " + what);
  return dim3(uint32_t(blocks));
}

// Calls f(T{}) / f(A{}, B{}) for the element types of the codes.
template <typename F>
inline void dispatch_type(int t, const char* who, F&& f) {
  switch (t) {
    case kF32: f(float{}); return;
    case kBF16: f(bf16_t{}); return;
    case kF16: f(f16_t{}); return;
    default: throw std::invalid_argument(std::string(who) + ": element type");
  }
}

template <typename F>
inline void dispatch_types(int a, int b, const char* who, F&& f) {
  dispatch_type(a, who, [&](auto ta) { dispatch_type(b, who, [&](auto tb) { f(ta, tb); }); });
}

}  // namespace hip
}  // namespace rmm
