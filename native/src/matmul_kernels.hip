// The product of two matrices in 8 bits with a scale for each block of 128 values, for gfx950.
//
//   C[m, n] = sum over blocks b of 2^(sa[m, b] + sb[n, b]) * sum over k in b of A[m, k] B[n, k]
//
// Two arithmetics, by the type of C:
//  * 16 bits: CDNA4's scaled matrix instruction (16 x 16 x 128). It takes exactly one block per step,
//    e4m3 values and an E8M0 byte for every 32 of them (here the same byte four times), and adds
//    the scaled products to 32-bit sums; no scale is multiplied in by the vector units. Inside, it
//    lines the products of 8 neighbouring k up at the largest and drops what is below 2^-13 of it
//    (measured with products of known size): 1.5e-5 of a sum of random values, a hundredth of the
//    rounding to bf16 and a tenth of that to fp16 that follow.
//  * 32 bits: there that would be what limits the result. The values are widened to bf16 (exact: 4
//    significant bits; the conversion instruction multiplies the scale in) and multiplied by the
//    16 x 16 x 32 instruction, whose sums are good to 2^-24, at half the rate.
//
// Which 32 of a block's 128 values a group of lanes holds does not matter to a sum as long as both
// operands do the same: lane group g takes bytes 16 g .. and 64 + 16 g .., two 16-byte pieces.
// The instructions' first operand is B, the second A: a lane then holds neighbouring columns of C.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "tk8s/common.h"
#include "tk8s/fp8_device.h"
#include "tk8s/kernels.h"

namespace tk8s {

using namespace fp8;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A lane's 32 values of 16 rows x 128: row lane % 16.
union Fragment {
  i32x8 v;
  u32x4 half[2];
  int word[8];
};

// The same values widened: four operands of the 16 x 16 x 32 instruction.
union Wide {
  bf16x8 v[4];
  bf16x2 pair[16];
};

__device__ __forceinline__ Wide widen(const Fragment& f, float scale) {
  Wide w;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w.pair[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.word[i], scale, false);
    w.pair[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.word[i], scale, true);
  }
  return w;
}

__device__ __forceinline__ f32x4 multiply(const Wide& b, const Wide& a, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[i], a.v[i], acc, 0, 0, 0);
  return acc;
}

__device__ __forceinline__ float scale_value(unsigned byte) { return __uint_as_float(byte << 23); }

// Scales that widened values can carry: products of two such, and 448 times one, are 32-bit numbers
// (or beyond what a 32-bit C could hold). Others, and NaN, take the way through ldexp.
__device__ __forceinline__ bool far_scale(unsigned byte) { return byte - 27u > 200u; }

// part * 2^(sa + sb - 254), NaN for a NaN scale.
__device__ __forceinline__ float scaled(float part, unsigned sa, unsigned sb) {
  if (sa == 255u || sb == 255u) return __uint_as_float(0x7fc00000u);
  return ldexpf(part, static_cast<int>(sa + sb) - 254);
}

// 16 bytes of a row at k, zeros from k_end on; reads no byte behind k_end.
__device__ __forceinline__ u32x4 load16(const uint8_t* row, size_t k, size_t k_end) {
  if (k + 16 <= k_end) return *reinterpret_cast<const u32x4*>(row + k);
  u32x4 r = {0, 0, 0, 0};
  for (int j = 0; k + j < k_end; ++j) r[j / 4] |= static_cast<unsigned>(row[k + j]) << (8 * (j % 4));
  return r;
}

// ------------------------------------------------------------------------------------------
// Few rows of A
// ------------------------------------------------------------------------------------------
// The weights are read once and nothing else matters. A block makes 16 columns of C; its waves share
// them along k, wave w the blocks w, w + WAVES, ..., so the block reads whole rows in order, and join
// their sums in LDS in the order of the waves. B and A go from memory to registers directly (A
// is small and stays in L2), kAhead steps requested at a time.
template <class O, bool kExact, int MT, int WAVES, int kAhead>
__global__ __launch_bounds__(WAVES * 64) void matmul_rows_kernel(MatmulArgs a) {
  __shared__ float part[WAVES][MT * 256];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, group = lane / 16;
  const size_t n0 = static_cast<size_t>(blockIdx.x) * 16, m0 = static_cast<size_t>(blockIdx.y) * (16 * MT);
  const size_t nb = (a.k + kScaleBlock - 1) / kScaleBlock;
  const size_t whole = a.k / kScaleBlock;  // blocks with all their values
  const size_t n = std::min(n0 + lane % 16, a.n - 1);  // what is behind the last row is computed, not stored
  const uint8_t* const brow = a.b.values + n * a.b.ld + 16 * group;
  const uint8_t* const bscale = a.b.scales + (a.b_tiles ? n / kScaleBlock : n);
  const uint8_t* arow[MT];
  const uint8_t* ascale[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const size_t m = std::min(m0 + 16 * i + lane % 16, a.m - 1);
    arow[i] = a.a.values + m * a.a.ld + 16 * group;
    ascale[i] = a.a.scales + m;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto step = [&](const Fragment& fb, const Fragment (&fa)[MT], unsigned sb, const unsigned (&sa)[MT]) {
    if constexpr (!kExact) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb.v, fa[i].v, acc[i], 0, 0, 0, static_cast<int>(sb), 0,
                                                                 static_cast<int>(sa[i]));
    } else {
      bool far = far_scale(sb);
#pragma unroll
      for (int i = 0; i < MT; ++i) far |= far_scale(sa[i]);
      if (__builtin_amdgcn_ballot_w64(far) == 0) {
        const Wide wb = widen(fb, scale_value(sb));
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = multiply(wb, widen(fa[i], scale_value(sa[i])), acc[i]);
      } else {
        const Wide wb = widen(fb, 1.f);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const f32x4 p = multiply(wb, widen(fa[i], 1.f), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][r] += scaled(p[r], sa[i], __shfl(sb, 4 * group + r, 64));
        }
      }
    }
  };

  size_t b = wave;
  for (; b + (kAhead - 1) * WAVES < whole; b += kAhead * WAVES) {
    Fragment fb[kAhead], fa[kAhead][MT];
    unsigned sb[kAhead], sa[kAhead][MT];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const size_t at = b + u * WAVES;
      fb[u].half[0] = *reinterpret_cast<const u32x4*>(brow + at * kScaleBlock);
      fb[u].half[1] = *reinterpret_cast<const u32x4*>(brow + at * kScaleBlock + 64);
      sb[u] = bscale[at * a.b.ld_scales];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        fa[u][i].half[0] = *reinterpret_cast<const u32x4*>(arow[i] + at * kScaleBlock);
        fa[u][i].half[1] = *reinterpret_cast<const u32x4*>(arow[i] + at * kScaleBlock + 64);
        sa[u][i] = ascale[i][at * a.a.ld_scales];
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) step(fb[u], fa[u], sb[u], sa[u]);
  }
  for (; b < nb; b += WAVES) {  // what is left, the block cut off by the end of the rows included
    Fragment fb, fa[MT];
    unsigned sa[MT];
    const size_t k = b * kScaleBlock + 16 * group;
    fb.half[0] = load16(brow - 16 * group, k, a.k);
    fb.half[1] = load16(brow - 16 * group, k + 64, a.k);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      fa[i].half[0] = load16(arow[i] - 16 * group, k, a.k);
      fa[i].half[1] = load16(arow[i] - 16 * group, k + 64, a.k);
      sa[i] = ascale[i][b * a.a.ld_scales];
    }
    step(fb, fa, bscale[b * a.b.ld_scales], sa);
  }

  // lane: row lane % 16 of A, columns 4 * group .. + 3
#pragma unroll
  for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(&part[wave][i * 256 + (lane % 16) * 16 + 4 * group]) = acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 256; e += WAVES * 64) {
    float s = part[0][e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += part[w][e];
    const size_t row = m0 + e / 16, col = n0 + e % 16;
    if (row < a.m && col < a.n) static_cast<O*>(a.c)[row * a.ldc + col] = static_cast<O>(s);
  }
}

void check(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

template <class O, bool kExact> void launch(const MatmulArgs& a, hipStream_t stream) {
  const unsigned gx = static_cast<unsigned>((a.n + 15) / 16);
  if (a.m <= 16)
    hipLaunchKernelGGL((matmul_rows_kernel<O, kExact, 1, 8, 4>), dim3(gx, 1), dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((matmul_rows_kernel<O, kExact, 2, 8, 2>), dim3(gx, static_cast<unsigned>((a.m + 31) / 32)), dim3(512), 0, stream, a);
}

}  // namespace

void fp8_matmul(const MatmulArgs& a, LayerType out, hipStream_t stream) {
  if (a.m == 0 || a.n == 0) return;
  check(a.c != nullptr, "fp8_matmul: c is needed");
  check(a.k == 0 || (a.a.values && a.a.scales && a.b.values && a.b.scales), "fp8_matmul: a pointer is missing");
  check(reinterpret_cast<uintptr_t>(a.a.values) % 16 == 0 && reinterpret_cast<uintptr_t>(a.b.values) % 16 == 0 &&
            a.a.ld % 16 == 0 && a.b.ld % 16 == 0,
        "fp8: the rows of 8-bit values must start on 16-byte boundaries");
  check(reinterpret_cast<uintptr_t>(a.a.scales) % 4 == 0 && a.a.ld_scales % 4 == 0 &&
            (a.b_tiles || (reinterpret_cast<uintptr_t>(a.b.scales) % 4 == 0 && a.b.ld_scales % 4 == 0)),
        "fp8: the scales of a block must start on a 4-byte boundary");
  check(a.m <= (1u << 20) && a.n <= (1u << 24), "fp8_matmul: at most 2^20 rows and 2^24 columns of C");
  switch (out) {
    case LayerType::kF32: launch<float, true>(a, stream); break;
    case LayerType::kBF16: launch<__bf16, false>(a, stream); break;
    case LayerType::kF16: launch<_Float16, false>(a, stream); break;
  }
  TK8S_HIP_CHECK(hipGetLastError());
}

}  // namespace tk8s
