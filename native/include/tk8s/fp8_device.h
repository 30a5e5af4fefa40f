// Device helpers shared by the 8-bit layer operators (fp8_kernels.hip, matmul_kernels.hip):
// storage types, loads of 8 values at any element alignment, the block scale and the rounding.
#pragma once

#include <cstdint>

#include <hip/hip_runtime.h>

namespace tk8s {
namespace fp8 {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int kScaleBlock = 128;  // values that share a scale, along a row (or a column)

// 8 consecutive values that start at any element: the compiler makes whole-dword loads of it
// (global memory takes them at every address), so an odd row pitch costs no separate kernel.
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };

// v[0..7] = p[0..n-1], zeros behind; n <= 0 reads nothing.
template <class T> __device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  if (n >= 8) {
    const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(e.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? static_cast<float>(p[j]) : 0.f;
  }
}

// p[0..n-1] = v[0..n-1], one rounding to T.
template <class T> __device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    Eight<T> e;
#pragma unroll
    for (int j = 0; j < 8; ++j) e.v[j] = static_cast<T>(v[j]);
    *reinterpret_cast<Eight<T>*>(p) = e;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = static_cast<T>(v[j]);
  }
}

// The float nearest to zero side of v with its last bits standing for "more follows": v cut to 20
// fraction bits, the last one set where anything was cut. Rounding the result once more, to at
// most 18 bits, gives what rounding v itself would -- no second rounding, no false ties.
__device__ __forceinline__ float round_to_odd(double v) {
  const unsigned long long b = __double_as_longlong(v);
  const unsigned lo = static_cast<unsigned>(b);
  const unsigned hi = static_cast<unsigned>(b >> 32) | (lo != 0 ? 1u : 0u);
  return static_cast<float>(__longlong_as_double(static_cast<unsigned long long>(hi) << 32));
}

__device__ __forceinline__ unsigned magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// E8M0 byte of a block whose largest magnitude has these float bits (the bits order as the values
// do, NaN above infinity): the least power of two that brings it to 448 or below; 1 for zeros;
// 255, the type's NaN, where it is not finite.
__device__ __forceinline__ unsigned scale_byte(unsigned amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  if (amax_bits == 0u) return 127u;
  const int b = static_cast<int>(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < 0 ? 0u : static_cast<unsigned>(b);
}

// 1 / scale, exact: at most 2^127, and at least 2^-120 for a finite float's block.
__device__ __forceinline__ float inverse_scale(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// Four e4m3 bytes of v * inv, rounded to nearest even by the conversion instruction; the block's
// scale keeps them within +-448. All NaN where the block's scale is.
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d, unsigned byte) {
  if (byte == 255u) return 0x7f7f7f7fu;
  const float inv = inverse_scale(byte);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true));
}

// The largest over the 16 lanes that hold one block.
__device__ __forceinline__ unsigned max16(unsigned v) {
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) {
    const unsigned o = __shfl_xor(v, off, 64);
    v = o > v ? o : v;
  }
  return v;
}

}  // namespace fp8
}  // namespace tk8s
