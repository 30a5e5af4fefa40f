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

// The same 8 values as they are stored, in whole registers: 16-bit values two to a dword.
template <class T> struct Packed8 { unsigned d[2 * sizeof(T)]; };

template <class T> __device__ __forceinline__ float unpack(const Packed8<T>& p, int j) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(p.d[j]);
  } else if constexpr (__is_same(T, __bf16)) {
    return __uint_as_float(j % 2 ? p.d[j / 2] & 0xffff0000u : p.d[j / 2] << 16);
  } else {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(p.d[j / 2] >> (16 * (j % 2)))));
  }
}

// Two values, rounded to T, into dword i (of 16-bit values), or one into each of two.
template <class T> __device__ __forceinline__ void pack(Packed8<T>& p, int i, float v0, float v1) {
  if constexpr (sizeof(T) == 4) {
    p.d[2 * i] = __float_as_uint(v0);
    p.d[2 * i + 1] = __float_as_uint(v1);
  } else {
    typedef T Two __attribute__((ext_vector_type(2)));
    const Two t = {static_cast<T>(v0), static_cast<T>(v1)};
    p.d[i] = __builtin_bit_cast(unsigned, t);
  }
}

template <int kAlign> struct Dwords;
template <> struct Dwords<2> { typedef unsigned four __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Dwords<4> { typedef unsigned four __attribute__((ext_vector_type(4), aligned(4))); };

// Whole dwords from (to) an address of any element, past the caches: what is streamed is touched once.
template <class T> __device__ __forceinline__ Packed8<T> at_any(const T* p) {
  typedef typename Dwords<sizeof(T)>::four Four;
  Packed8<T> e;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    const Four u = __builtin_nontemporal_load(reinterpret_cast<const Four*>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) e.d[4 * i + j] = u[j];
  }
  return e;
}

template <class T> __device__ __forceinline__ void at_any(T* p, const Packed8<T>& e) {
  typedef typename Dwords<sizeof(T)>::four Four;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    const Four u = {e.d[4 * i], e.d[4 * i + 1], e.d[4 * i + 2], e.d[4 * i + 3]};
    __builtin_nontemporal_store(u, reinterpret_cast<Four*>(p) + i);
  }
}

// n = 1..7 of them. kParts (16-bit values only): in parts of 4, 2 and 1, three loads (stores) where one for each
// value would be seven in a row's last lane, which the others wait for (gradients of 5475 x 438: 15.6 ->
// 13.2 us; 32-bit values are better off with seven: parts made a norm of 1031 x 5003 19 % slower).
template <int kDwords> struct __attribute__((packed, aligned(2))) Dwords2 { unsigned d[kDwords]; };

template <bool kParts, class T> __device__ __forceinline__ Packed8<T> load_tail(const T* p, int n) {
  if constexpr (!kParts) {
    Eight<T> o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = j < n ? p[j] : static_cast<T>(0.f);
    return __builtin_bit_cast(Packed8<T>, o);
  } else {
    Dwords2<2> four = {};
    Dwords2<1> two = {};
    unsigned one = 0;
    if (n & 4) four = *reinterpret_cast<const Dwords2<2>*>(p);
    if (n & 2) two = *reinterpret_cast<const Dwords2<1>*>(p + (n & 4));
    if (n & 1) one = __builtin_bit_cast(unsigned short, p[n & 6]);
    Packed8<T> e = {};
    unsigned rest[2];  // what comes behind the four
    rest[0] = n & 2 ? two.d[0] : one;
    rest[1] = n & 2 ? one : 0u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e.d[i] = n & 4 ? four.d[i] : rest[i];
      e.d[2 + i] = n & 4 ? rest[i] : 0u;
    }
    return e;
  }
}

template <bool kParts, class T> __device__ __forceinline__ void store_tail(T* p, int n, const Packed8<T>& e) {
  if constexpr (!kParts) {
    const Eight<T> o = __builtin_bit_cast(Eight<T>, e);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = o.v[j];
  } else {
    Dwords2<2> four;
    Dwords2<1> two;
    unsigned rest[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      four.d[i] = e.d[i];
      rest[i] = n & 4 ? e.d[2 + i] : e.d[i];
    }
    two.d[0] = rest[0];
    const unsigned one = n & 2 ? rest[1] : rest[0];
    if (n & 4) *reinterpret_cast<Dwords2<2>*>(p) = four;
    if (n & 2) *reinterpret_cast<Dwords2<1>*>(p + (n & 4)) = two;
    if (n & 1) p[n & 6] = __builtin_bit_cast(T, static_cast<unsigned short>(one));
  }
}

// p[0..n-1], zeros behind; n <= 0 reads nothing. kWhole: n is 8 or more, or 0 or less.
template <bool kWhole, class T, bool kParts = sizeof(T) == 2> __device__ __forceinline__ Packed8<T> load_packed(const T* p, int n) {
  Packed8<T> e = {};
  if (kWhole ? n > 0 : n >= 8) e = at_any(p);
  else if (!kWhole && n > 0) e = load_tail<kParts>(p, n);
  return e;
}

template <bool kWhole, class T> __device__ __forceinline__ void store_packed(T* p, int n, const Packed8<T>& e) {
  if (kWhole ? n > 0 : n >= 8) at_any(p, e);
  else if (!kWhole && n > 0) store_tail<sizeof(T) == 2>(p, n, e);
}

// Keeps the compiler from unpacking a loop's constants into twice the registers before it.
template <class T> __device__ __forceinline__ void keep_packed(Packed8<T>& p) {
  if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(p.d[0]), "+v"(p.d[1]), "+v"(p.d[2]), "+v"(p.d[3]));
}

// 8 bytes of e4m3 to where n of them belong.
template <bool kWhole> __device__ __forceinline__ void store_bytes(uint8_t* p, int n, u32x2 v) {
  if (kWhole ? n > 0 : n >= 8) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x2*>(p));
  } else if (!kWhole && n > 0) {  // in parts of 4, 2 and 1, on boundaries of their sizes
    const unsigned rest = n & 4 ? v.y : v.x;
    if (n & 4) *reinterpret_cast<unsigned*>(p) = v.x;
    if (n & 2) *reinterpret_cast<unsigned short*>(p + (n & 4)) = static_cast<unsigned short>(rest);
    if (n & 1) p[n & 6] = static_cast<uint8_t>(rest >> (n & 2 ? 16 : 0));
  }
}

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
template <class T, int N> __device__ __forceinline__ void store_some(T* p, int n, const float (&v)[N]) {
  struct __attribute__((packed, aligned(sizeof(T)))) Some { T v[N]; };
  if (n >= N) {
    Some e;
#pragma unroll
    for (int j = 0; j < N; ++j) e.v[j] = static_cast<T>(v[j]);
    *reinterpret_cast<Some*>(p) = e;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = static_cast<T>(v[j]);
  }
}

// The float on the zero side of v with its last bit standing for "more follows": v cut to 20 fraction bits, the
// last one set where anything was cut. Rounding the result once more, to at most 18 bits, gives what
// rounding v itself would -- no second rounding, no false ties. Below 2^-126 a float has fewer bits: see the next one.
__device__ __forceinline__ unsigned odd_bits(double v) {  // the upper half of the cut v
  const unsigned long long b = __double_as_longlong(v);
  return static_cast<unsigned>(b >> 32) | (static_cast<unsigned>(b) != 0 ? 1u : 0u);
}
__device__ __forceinline__ float round_to_odd(double v) {
  return static_cast<float>(__longlong_as_double(static_cast<unsigned long long>(odd_bits(v)) << 32));
}

// The same of any v: below 2^-126 it is cut to whole multiples of 2^-149, and the result can be rounded once more to
// multiples of 2^-137 and up, which is where the borders between e4m3 values under the least scale lie.
__device__ __forceinline__ float round_tiny_to_odd(double v) {
  if (!(fabs(v) < 0x1p-126)) return round_to_odd(v);
  const double steps = fabs(v) * 0x1p149;  // below 2^23, exact
  const unsigned whole = static_cast<unsigned>(steps);
  return __uint_as_float((odd_bits(v) & 0x80000000u) | whole | (steps != static_cast<double>(whole) ? 1u : 0u));
}

// 1 / sqrt(x) to the last bits of 64: the instruction's first 2^-25 or so, then one step of third order.
// 0 and infinity keep what the instruction says.
__device__ __forceinline__ double inverse_sqrt(double x) {
  const double r = __builtin_amdgcn_rsq(x);
  const double e = fma(-x * r, r, 1.0);
  const double better = fma(r * e, fma(0.375, e, 0.5), r);
  return x > 0.0 && x < __builtin_inf() ? better : r;
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

// Whether a 32-bit value that may be kSlack units in its last place off could round to another e4m3
// value than the exact one, or its block get another scale: the borders between e4m3 values are
// numbers whose low 19 fraction bits are 0 (those between scales, 448 2^e, too).
constexpr unsigned kSlack = 4;
__device__ __forceinline__ unsigned from_border(float v) { return (__float_as_uint(v) + kSlack) & 0x7ffffu; }
__device__ __forceinline__ bool near_border(unsigned least) { return least <= 2 * kSlack; }

// Magnitudes of 8 stored values, compared as they are stored: 16-bit ones two to a dword (their bits,
// sign off, order as the values do, NaN above infinity).
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <class T> __device__ __forceinline__ Packed8<T> magnitudes(const Packed8<T>& v) {
  Packed8<T> m;
#pragma unroll
  for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) m.d[i] = v.d[i] & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu);
  return m;
}

template <class T> __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {  // of one dword
  if constexpr (sizeof(T) == 2)
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
  else
    return max(a, b);
}

template <class T> __device__ __forceinline__ Packed8<T> larger(const Packed8<T>& a, const Packed8<T>& b) {
  Packed8<T> m;
#pragma unroll
  for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) m.d[i] = larger<T>(a.d[i], b.d[i]);
  return m;
}

// The bits, as a float's, of magnitude j; of the largest of the 8.
template <class T> __device__ __forceinline__ unsigned magnitude_of(const Packed8<T>& m, int j) { return __float_as_uint(unpack(m, j)); }

template <class T> __device__ __forceinline__ unsigned largest_of(const Packed8<T>& m) {
  unsigned v = m.d[0];
#pragma unroll
  for (int i = 1; i < 2 * static_cast<int>(sizeof(T)); ++i) v = larger<T>(v, m.d[i]);
  if constexpr (sizeof(T) == 2) {
    const unsigned top = max(v & 0xffffu, v >> 16);
    if constexpr (__is_same(T, __bf16)) return top << 16;
    else return __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(top))));
  } else {
    return v;
  }
}

// Four e4m3 bytes of values 4 i .. 4 i + 3 under one block's scale. 16-bit values go through the conversion
// that takes the scale's exponent along; its ends (2^-127 and NaN) go the long way.
template <class T> __device__ __forceinline__ unsigned pack_four(const Packed8<T>& v, int i, unsigned byte) {
  if constexpr (sizeof(T) == 2) {
    if (byte - 1u < 254u) {
      typedef short Old __attribute__((ext_vector_type(2)));
      typedef T Two __attribute__((ext_vector_type(2)));
      const float scale = __uint_as_float(byte << 23);
      Old r = {0, 0};
      if constexpr (__is_same(T, __bf16)) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(Two, v.d[2 * i]), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(Two, v.d[2 * i + 1]), scale, true);
      } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(Two, v.d[2 * i]), scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(Two, v.d[2 * i + 1]), scale, true);
      }
      return __builtin_bit_cast(unsigned, r);
    }
  }
  return pack4(unpack(v, 4 * i), unpack(v, 4 * i + 1), unpack(v, 4 * i + 2), unpack(v, 4 * i + 3), byte);
}

// Column j of 8 rows of 8 values, as 8 stored values.
template <class T> __device__ __forceinline__ Packed8<T> column(const Packed8<T> (&v)[8], int j) {
  Packed8<T> c;
#pragma unroll
  for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) {
    if constexpr (sizeof(T) == 2) c.d[i] = __builtin_amdgcn_perm(v[2 * i + 1].d[j / 2], v[2 * i].d[j / 2], j % 2 ? 0x07060302u : 0x05040100u);
    else c.d[i] = v[i].d[j];
  }
  return c;
}

// v of the lane kBy places on within its 16, on the vector unit's own crossbar.
template <int kBy> __device__ __forceinline__ unsigned rotate16(unsigned v) {
  return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x120 + kBy, 0xf, 0xf, false));
}

// The largest over the 16 lanes that hold one block.
__device__ __forceinline__ unsigned max16(unsigned v) {
  v = max(v, rotate16<8>(v));
  v = max(v, rotate16<4>(v));
  v = max(v, rotate16<2>(v));
  return max(v, rotate16<1>(v));
}

template <int kBy> __device__ __forceinline__ float rotate16(float v) { return __uint_as_float(rotate16<kBy>(__float_as_uint(v))); }
template <int kBy> __device__ __forceinline__ double rotate16(double v) {
  const unsigned long long b = __double_as_longlong(v);
  const unsigned long long lo = rotate16<kBy>(static_cast<unsigned>(b)), hi = rotate16<kBy>(static_cast<unsigned>(b >> 32));
  return __longlong_as_double(hi << 32 | lo);
}

// The sum over kLanes (16, 32 or 64) neighbouring lanes, the same in all of them and in every call.
template <int kLanes, class V> __device__ __forceinline__ V sum_lanes(V v) {
  v += rotate16<8>(v);
  v += rotate16<4>(v);
  v += rotate16<2>(v);
  v += rotate16<1>(v);
  if constexpr (kLanes >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (kLanes >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

}  // namespace fp8
}  // namespace tk8s
