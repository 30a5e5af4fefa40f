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
#include <cmath>

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

template <int OB, int OA>
__device__ __forceinline__ f32x4 mfma_scaled(const Fragment& b, const Fragment& a, f32x4 acc, unsigned sb, unsigned sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, acc, 0, 0, OB, static_cast<int>(sb), OA,
                                                          static_cast<int>(sa));
}

__device__ __forceinline__ float scale_value(unsigned byte) { return __uint_as_float(byte << 23); }

// Scales that widened values can carry: products of two such, and 448 times one, are 32-bit numbers
// (or beyond what a 32-bit C could hold). Others, and NaN, take the way through ldexp.
__device__ __forceinline__ bool far_scale(unsigned byte) { return byte - 27u > 200u; }

// Of the four scales of a dword those of rows below count, the first being row `first`; 2^0 for the others,
// whose bytes are anything: they must not decide which way the sums go.
__device__ __forceinline__ unsigned own_scales(unsigned scales, size_t first, size_t count) {
  const size_t n = first < count ? count - first : 0;
  const unsigned keep = n >= 4 ? ~0u : (1u << (8 * n)) - 1;
  return (scales & keep) | (0x7f7f7f7fu & ~keep);
}

// part * 2^(sa + sb - 254), NaN for a NaN scale.
__device__ __forceinline__ float scaled(float part, unsigned sa, unsigned sb) {
  if (sa == 255u || sb == 255u) return __uint_as_float(0x7fc00000u);
  return ldexpf(part, static_cast<int>(sa + sb) - 254);
}

// 16 bytes of a row at k, zeros from k_end on. Rows start on 16 bytes and so does k: the 16 bytes that hold
// the row's last value lie in one page with it, and what is read behind it is masked off.
__device__ __forceinline__ u32x4 load16(const uint8_t* row, size_t k, size_t k_end) {
  u32x4 r = *reinterpret_cast<const u32x4*>(row + std::min(k, (k_end - 1) / 16 * 16));
  const int n = k < k_end ? static_cast<int>(std::min<size_t>(k_end - k, 16)) : 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] &= n >= 4 * j + 4 ? ~0u : n <= 4 * j ? 0u : (1u << (8 * (n - 4 * j))) - 1;
  return r;
}

// ------------------------------------------------------------------------------------------
// Few rows of A
// ------------------------------------------------------------------------------------------
// Up to 16. The weights are read once and that is what it should take. A block makes 16 columns of C; its
// waves share them along k, wave w the blocks w, w + kRowWaves, ..., so the block reads whole rows in
// order, and join their sums in LDS in the order of the waves. B and A go from memory to registers
// directly; kAhead of a wave's blocks are on their way at any time. One row by 4096 x 4096: 5.3 us, 3.2 TB/s
// of weights; the latency of one round of loads and of the join is what is left.
constexpr int kRowWaves = 8, kAhead = 4;

template <class O, bool kExact>
__global__ __launch_bounds__(kRowWaves * 64) void matmul_rows_kernel(MatmulArgs a) {
  __shared__ float part[kRowWaves][256];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, group = lane / 16;
  const size_t n0 = static_cast<size_t>(blockIdx.x) * 16;
  const size_t nb = (a.k + kScaleBlock - 1) / kScaleBlock;
  const size_t whole = a.k / kScaleBlock;  // blocks with all their values
  // what is behind the last row of either is computed, not stored
  const size_t n = std::min(n0 + lane % 16, a.n - 1), m = std::min<size_t>(lane % 16, a.m - 1);
  const uint8_t* const brow = a.b.values + n * a.b.ld;
  const uint8_t* const arow = a.a.values + m * a.a.ld;
  const uint8_t* const bscale = a.b.scales + (a.b_tiles ? n / kScaleBlock : n);
  const uint8_t* const ascale = a.a.scales + m;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};

  auto step = [&](const Fragment& fb, const Fragment& fa, unsigned sb, unsigned sa) {
    if constexpr (!kExact) {
      acc = mfma_scaled<0, 0>(fb, fa, acc, sb, sa);
    } else if (__builtin_amdgcn_ballot_w64(far_scale(sb) || far_scale(sa)) == 0) {
      acc = multiply(widen(fb, scale_value(sb)), widen(fa, scale_value(sa)), acc);
    } else {
      const f32x4 p = multiply(widen(fb, 1.f), widen(fa, 1.f), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] += scaled(p[r], sa, __shfl(sb, 4 * group + r, 64));
    }
  };

  // This wave's whole blocks: wave, wave + kRowWaves, ..., from a place of the block's own on and round, so that
  // the blocks do not all ask the same channel of L2 for the same piece of A.
  // Loads come back in the order of their requests, so A's are made as early as B's, though A is near.
  const unsigned steps = whole > static_cast<size_t>(wave) ? static_cast<unsigned>((whole - wave + kRowWaves - 1) / kRowWaves) : 0;
  Fragment fb[kAhead], fa[kAhead];
  unsigned sb[kAhead], sa[kAhead];
  const unsigned turn = steps ? blockIdx.x & ((1u << (31 - __builtin_clz(steps))) - 1) : 0;
  auto request = [&](unsigned s, int u) {
    unsigned q = (s < steps ? s : steps - 1) + turn;
    q = q >= steps ? q - steps : q;
    const size_t at = wave + static_cast<size_t>(q) * kRowWaves, k = at * kScaleBlock + 16 * group;
    fb[u].half[0] = *reinterpret_cast<const u32x4*>(brow + k);
    fb[u].half[1] = *reinterpret_cast<const u32x4*>(brow + k + 64);
    sb[u] = bscale[at * a.b.ld_scales];
    fa[u].half[0] = *reinterpret_cast<const u32x4*>(arow + k);
    fa[u].half[1] = *reinterpret_cast<const u32x4*>(arow + k + 64);
    sa[u] = ascale[at * a.a.ld_scales];
  };
  if (steps) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) request(u, u);
    for (unsigned s = 0; s < steps; s += kAhead) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u && s + u >= steps) break;
        step(fb[u], fa[u], sb[u], sa[u]);
        if (s + u + kAhead < steps) request(s + u + kAhead, u);
      }
    }
  }
  const size_t b = wave + static_cast<size_t>(steps) * kRowWaves;
  if (b < nb) {  // the block cut off by the end of the rows, if it is this wave's
    const size_t k = b * kScaleBlock + 16 * group;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fb[0].half[h] = load16(brow, k + 64 * h, a.k);
      fa[0].half[h] = load16(arow, k + 64 * h, a.k);
    }
    step(fb[0], fa[0], bscale[b * a.b.ld_scales], ascale[b * a.a.ld_scales]);
  }

  // lane: row lane % 16 of A, columns 4 * group .. + 3
  *reinterpret_cast<f32x4*>(&part[wave][lane % 16 * 16 + 4 * group]) = acc;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  float sum = part[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) sum += part[w][threadIdx.x];
  const size_t row = threadIdx.x / 16, col = n0 + threadIdx.x % 16;
  if (row < a.m && col < a.n) static_cast<O*>(a.c)[row * a.ldc + col] = static_cast<O>(sum);
}

// ------------------------------------------------------------------------------------------
// Tiles
// ------------------------------------------------------------------------------------------
// A step is one block of 128 k from LDS. Rows of 128 bytes lie in LDS as 8 pieces, piece p of row r at
// p ^ (r / 4 % 8): of the 16 rows 4 j + i that a fragment's lanes read at once, 8 hit 8 different pieces,
// and slot_row() puts the other 8 into the other banks.
// Tile i of 64 rows holds the rows 4 j + i (j = 0..15): one dword of scales then serves four tiles,
// a byte each (the instruction picks it), and a lane ends with 16 neighbouring columns of C.
// The row that lies at place p of a group of 64 in LDS (and the place of row p): neighbours change places
// in the upper 32, so that of a fragment's rows 4 j + i those with j < 8 and j >= 8 lie in different
// halves of the 64 banks.
__device__ __forceinline__ int slot_row(int p) { return p ^ (p / 32 % 2); }

constexpr int kXcds = 8;   // dies with an L2 of their own; blocks go to them in turn
constexpr int kPanel = 8;  // tiles of A that a die's neighbouring blocks share

// Block -> tile: blocks b, b + 8, ... run on one die; they take neighbouring tiles, column after
// column of panels kPanel tiles high, so that a die's running blocks share rows of both operands.
__device__ __forceinline__ void tile_of(unsigned block, unsigned tiles_m, unsigned tiles_n, unsigned& tm, unsigned& tn) {
  const unsigned total = tiles_m * tiles_n, die = block % kXcds, per = total / kXcds, more = total % kXcds;
  const unsigned t = die * per + (die < more ? die : more) + block / kXcds;
  const unsigned panel = t / (kPanel * tiles_n), first = panel * kPanel;
  const unsigned high = tiles_m - first < kPanel ? tiles_m - first : kPanel;
  const unsigned in_panel = t - panel * kPanel * tiles_n;
  tm = first + in_panel % high;
  tn = in_panel / high;
}

__device__ __forceinline__ unsigned lds_address(const void* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

// 16 (4) bytes for each lane from base + offset to LDS at `to` + 16 (4) * lane. Written as assembly
// so that the compiler does not wait for all of them before it next reads LDS; no register is written.
__device__ __forceinline__ void load_lds16(unsigned to, const uint8_t* base, unsigned offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void load_lds4(unsigned to, const uint8_t* base, unsigned offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(base) : "m0", "memory");
}

// Waits until at most kLeft of this wave's loads are on their way, then for the other waves.
template <int kLeft> __device__ __forceinline__ void wait_and_meet() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// Lanes change values: the upper 32 of x with the lower 32 of y; odd 16 of x with the even 16 of y behind which they lie.
__device__ __forceinline__ void swap32(float& x, float& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  x = __uint_as_float(r[0]);
  y = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap16(float& x, float& y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  x = __uint_as_float(r[0]);
  y = __uint_as_float(r[1]);
}

// 64 columns of C from c on, of `left` there are: a lane has 16 neighbouring ones of its row, 16 group + 4 r + j
// in sums[j][r]. They change lanes first, so that the four lanes of a row write 64 neighbouring bytes with
// every store instead of 16 here and there (8192 x 8192 x 1024, 16-bit: 117 -> 104 us; 2048 x 4096 x 4096,
// 32-bit: 84 -> 75).
template <class O> __device__ __forceinline__ void store_row(O* c, bool inside, int left, const f32x4 (&sums)[4], int group) {
  constexpr int kPer = 16 / sizeof(O), kStores = 16 / kPer;
  float v[kStores][kPer];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e / kPer][e % kPer] = sums[e % 4][e / 4];
#pragma unroll
  for (int s = 0; s < kStores / 2; ++s)
#pragma unroll
    for (int e = 0; e < kPer; ++e) swap32(v[s][e], v[s + kStores / 2][e]);
  if constexpr (kStores == 4) {
#pragma unroll
    for (int s = 0; s < 4; s += 2)
#pragma unroll
      for (int e = 0; e < kPer; ++e) swap16(v[s][e], v[s + 1][e]);
  }
  if (!inside) return;
  const int at = kPer * (kStores == 4 ? group : group % 2 * 2 + group / 2);
#pragma unroll
  for (int s = 0; s < kStores; ++s) store_some(c + 4 * kPer * s + at, left - 4 * kPer * s - at, v[s]);
}

// What a wave multiplies in one step: four tiles of 16 rows of each operand and their scales.
struct Operands {
  Fragment b[4], a[4];
  unsigned sb, sa;
};

// acc += a step's 64 x 64 x 128; between(0) .. between(15) are issued one by one in the shadow of the
// matrix instructions.
template <class F>
__device__ __forceinline__ void multiply_step(const Operands& f, f32x4 (&acc)[4][4], F between) {
  auto pin = [&](int i) {
    __builtin_amdgcn_sched_barrier(0);
    between(i);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto four = [&](auto tag) {
    constexpr int i = decltype(tag)::value;
    acc[i][0] = mfma_scaled<0, i>(f.b[0], f.a[i], acc[i][0], f.sb, f.sa);
    pin(4 * i);
    acc[i][1] = mfma_scaled<1, i>(f.b[1], f.a[i], acc[i][1], f.sb, f.sa);
    pin(4 * i + 1);
    acc[i][2] = mfma_scaled<2, i>(f.b[2], f.a[i], acc[i][2], f.sb, f.sa);
    pin(4 * i + 2);
    acc[i][3] = mfma_scaled<3, i>(f.b[3], f.a[i], acc[i][3], f.sb, f.sa);
    pin(4 * i + 3);
  };
  four(std::integral_constant<int, 0>{});
  four(std::integral_constant<int, 1>{});
  four(std::integral_constant<int, 2>{});
  four(std::integral_constant<int, 3>{});
}

// The same with 32-bit sums, in two halves: B widened, then A tile by tile while it is multiplied. The
// widening multiplies the scales in, if they are near; else they are left for scaled_sums().
__device__ __forceinline__ void widen_b(const Operands& f, unsigned scales, Wide (&wb)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) wb[j] = widen(f.b[j], scale_value(scales >> (8 * j) & 255u));
}

__device__ __forceinline__ void multiply_wide(const Operands& f, const Wide (&wb)[4], f32x4 (&acc)[4][4]) {
  Wide wa[2];
  wa[0] = widen(f.a[0], scale_value(f.sa & 255u));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float scale = i < 3 ? scale_value(f.sa >> (8 * i + 8) & 255u) : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[i][j] = multiply(wb[j], wa[i % 2], acc[i][j]);
      if (i < 3) {  // a quarter of the next tile is widened in the shadow of these four
#pragma unroll
        for (int h = 2 * j; h < 2 * j + 2; ++h) {
          wa[1 - i % 2].pair[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.a[i + 1].word[h], scale, false);
          wa[1 - i % 2].pair[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.a[i + 1].word[h], scale, true);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

__device__ __forceinline__ void scaled_sums(const Operands& f, const Wide (&wb)[4], f32x4 (&acc)[4][4], int group) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Wide wa = widen(f.a[i], 1.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 p = multiply(wb[j], wa, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[i][j][r] += scaled(p[r], f.sa >> (8 * i) & 255u, __shfl(f.sb, 4 * group + r, 64) >> (8 * j) & 255u);
      __builtin_amdgcn_sched_barrier(0);  // one pair at a time: this way is rare, its registers are not free
    }
  }
}

// A block of (TM / 64) x (TN / 64) waves makes TM x TN of C, each wave 64 x 64. kStages steps of LDS go
// round: while a step is multiplied from registers, the next one is read from LDS and the bytes
// of the step kStages ahead are requested (straight into LDS, no registers). One barrier a step
// says both that the next step has arrived and that the slot to be refilled has been read. What
// bounds it is the time a request takes against kStages - 1 steps: LDS is as full of bytes on
// their way as it can be. 1024 x 4096 x 4096, 16-bit: 24.2 us, 1420 TFLOP/s (128 x 128); 2048 rows: 39.2, 1750
// (256 x 128). 32-bit sums, 4096 x 4096 x 10007: 281 - 301 us, 1120 - 1200 TFLOP/s, the matrix units busy half of the
// time and the vector units with the widening.
template <class O, bool kExact, int TM, int TN, int kStages>
__global__ __launch_bounds__(TM / 64 * (TN / 64) * 64) void matmul_stage_kernel(MatmulArgs a, unsigned tiles_m, unsigned tiles_n) {
  constexpr int WM = TM / 64, WN = TN / 64, kWaves = WM * WN;
  constexpr int kRows = (TM + TN) / 8;                       // loads of 8 rows x 128 bytes in a step
  constexpr int kLoads = (kRows + kWaves - 1) / kWaves + 1;  // by each wave, the scales' one included
  constexpr int kScales = (TM + TN) * 128, kSlot = kScales + 512;
  static_assert(kWaves >= 2 && kLoads <= 16 && kStages >= 3 && kStages * kSlot <= 160 * 1024, "tile shape");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * kSlot];
  const int lane = threadIdx.x % 64, group = lane / 16, j16 = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wm = wave / WN, wn = wave % WN;
  const unsigned lds0 = lds_address(lds);
  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const size_t m0 = static_cast<size_t>(tm) * TM, n0 = static_cast<size_t>(tn) * TN;
  const unsigned whole = static_cast<unsigned>(a.k / kScaleBlock);

  // Load c of this wave: 8 of the slot's rows, A's TM, then B's TN; pitches are below 2^23, so offsets
  // from the tile's first row fit 32 bits. Rows behind the last one are that one again.
  const uint8_t* const abase = a.a.values + m0 * a.a.ld;
  const uint8_t* const bbase = a.b.values + n0 * a.b.ld;
  unsigned off[kLoads - 1];
#pragma unroll
  for (int c = 0; c < kLoads - 1; ++c) {
    const int q = std::min(wave + c * kWaves, kRows - 1);  // where they do not come out even, the last ones twice
    const int r = slot_row(8 * q + lane / 8);
    const unsigned piece = 16u * ((lane % 8) ^ (r / 4 % 8));
    off[c] = r < TM ? static_cast<unsigned>(std::min<size_t>(r, a.m - 1 - m0)) * static_cast<unsigned>(a.a.ld) + piece
                    : static_cast<unsigned>(std::min<size_t>(r - TM, a.n - 1 - n0)) * static_cast<unsigned>(a.b.ld) + piece;
  }
  // scales: a dword a lane of A's rows (even waves) or B's (odd waves); for 128 x 128 tiles of B the
  // dword with those of this tile in every lane
  const uint8_t* sbase;
  unsigned off_s;
  if (wave % 2 == 0) {
    sbase = a.a.scales + m0;
    off_s = static_cast<unsigned>(std::min<size_t>(4 * lane, (a.m - 1) / 4 * 4 - m0));
  } else if (a.b_tiles) {
    sbase = a.b.scales + n0 / kScaleBlock / 4 * 4;
    off_s = 4 * (lane % 2) <= (a.n - 1) / kScaleBlock / 4 * 4 - n0 / kScaleBlock / 4 * 4 ? 4 * (lane % 2) : 0;
  } else {
    sbase = a.b.scales + n0;
    off_s = static_cast<unsigned>(std::min<size_t>(4 * lane, (a.n - 1) / 4 * 4 - n0));
  }
  const size_t s_step = wave % 2 == 0 ? a.a.ld_scales : a.b.ld_scales;
  // Behind the last step it is read once more, into a slot nobody reads again: the counts stay true.
  auto load = [&](unsigned step, unsigned slot, int c) {
    const size_t b = step < whole ? step : whole - 1;
    if (c == 0) {
      load_lds4(lds0 + slot * kSlot + kScales + (wave % 2) * 256, sbase + b * s_step, off_s);
    } else {
      const int q = std::min(wave + (c - 1) * kWaves, kRows - 1);
      load_lds16(lds0 + slot * kSlot + q * 1024, (8 * q < TM ? abase : bbase) + b * kScaleBlock, off[c - 1]);
    }
  };

  unsigned lane_at[2][2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      lane_at[odd][h] = lds0 + 512u * j16 + 128u * (odd ^ (j16 / 8)) + 16u * ((4 * h + group) ^ (j16 % 8));
  const size_t tile_n = (n0 + wn * 64) / kScaleBlock;
  const unsigned pick = a.b_tiles ? static_cast<unsigned>(tile_n % 4) * 0x01010101u : 0x03020100u;
  const int at_sb = 64 + (a.b_tiles ? static_cast<int>(tile_n / 4 - n0 / kScaleBlock / 4) : wn * 16 + j16);
  auto read_scales = [&](unsigned slot, Operands& f) {
    const unsigned* const scales = reinterpret_cast<const unsigned*>(lds + slot * kSlot + kScales);
    f.sa = scales[wm * 16 + j16];
    f.sb = __builtin_amdgcn_perm(0, scales[at_sb], pick);
  };
  auto read_piece = [&](unsigned slot, Operands& f, int c) {  // piece c of the 16: B's, then A's
    typedef const __attribute__((address_space(3))) u32x4* lds16;
    const int i = c / 2 % 4, h = c % 2;
    if (c < 8) f.b[i].half[h] = *reinterpret_cast<lds16>(lane_at[i % 2][h] + (slot * kSlot + TM * 128 + wn * 8192) + i / 2 * 256);
    else f.a[i].half[h] = *reinterpret_cast<lds16>(lane_at[i % 2][h] + (slot * kSlot + wm * 8192) + i / 2 * 256);
  };
  auto read_step = [&](unsigned slot, Operands& f) {
    read_scales(slot, f);
#pragma unroll
    for (int c = 0; c < 16; ++c) read_piece(slot, f, c);
  };

  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Operands f[2];

  // A step loaded with zeros behind the end of the rows, everything waited for.
  auto load_slowly = [&](unsigned b) {
#pragma unroll 2
    for (int q = wave; q < kRows; q += kWaves) {
      const int r = slot_row(8 * q + lane / 8);
      const size_t k = static_cast<size_t>(b) * kScaleBlock + 16 * ((lane % 8) ^ (r / 4 % 8));
      const uint8_t* const src = r < TM ? a.a.values + std::min(m0 + r, a.m - 1) * a.a.ld : a.b.values + std::min(n0 + r - TM, a.n - 1) * a.b.ld;
      *reinterpret_cast<u32x4*>(lds + q * 1024 + lane * 16) = load16(src, k, a.k);
    }
    load_lds4(lds0 + kScales + (wave % 2) * 256, sbase + b * s_step, off_s);
    wait_and_meet<0>();
  };

  auto store = [&](const f32x4 (&sums)[4][4]) {
    // lane: row 4 * j16 + i, columns 16 * group + 4 r + j
    const size_t mw = m0 + wm * 64, col = n0 + wn * 64;
    const int left = col < a.n ? static_cast<int>(std::min<size_t>(a.n - col, 64)) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t row = mw + 4 * j16 + i;
      store_row(static_cast<O*>(a.c) + row * a.ldc + col, row < a.m, left, sums[i], group);
    }
  };

  if constexpr (!kExact) {
    if (a.k % kScaleBlock) {  // first the block that the end of the rows cuts off
      load_slowly(whole);
      read_step(0, f[0]);
      multiply_step(f[0], acc, [](int) {});
      wait_and_meet<0>();
    }
    if (whole) {
#pragma unroll
      for (int s = 0; s < kStages; ++s)
#pragma unroll
        for (int c = 0; c < kLoads; ++c) load(s, s, c);
      unsigned slot = 0;
      wait_and_meet<(kStages - 1) * kLoads>();
      read_step(0, f[0]);
      auto step = [&](unsigned b, const Operands& now, Operands& then) {
        wait_and_meet<(kStages - 2) * kLoads>();  // step b is in everyone's registers, step b + 1 in LDS
        const unsigned next = slot + 1 == kStages ? 0 : slot + 1;
        read_scales(next, then);
        multiply_step(now, acc, [&](int c) {
          read_piece(next, then, c);
          if (c < kLoads) load(b + kStages, slot, c);
        });
        slot = next;
      };
      for (unsigned b = 0; b < whole; b += 2) {
        step(b, f[0], f[1]);
        if (b + 1 < whole) step(b + 1, f[1], f[0]);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may still be on its way to LDS when the block ends
    }
  } else {
    // Two groups of waves take turns, one phase apart: while one reads a step and widens B, the other
    // multiplies. A slot is refilled when the later group has read it. All waves look at all scales
    // of a step, so they give up together when one is far and make the tile again the slow way.
    static_assert(kStages == 3 && kWaves == 8 && TN == kScaleBlock, "two groups, one tile of B's scales");
    auto all_near = [&](unsigned slot) {
      const unsigned* const scales = reinterpret_cast<const unsigned*>(lds + slot * kSlot + kScales);
      const unsigned va = own_scales(scales[lane % (TM / 4)], m0 + 4 * (lane % (TM / 4)), a.m);
      const unsigned vb = a.b_tiles ? __builtin_amdgcn_perm(0, scales[64], pick) : own_scales(scales[64 + lane % (TN / 4)], n0 + 4 * (lane % (TN / 4)), a.n);
      bool far = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) far = far || far_scale(va >> (8 * i) & 255u) || far_scale(vb >> (8 * i) & 255u);
      return __builtin_amdgcn_ballot_w64(far) == 0;
    };
    bool near = true;
    if (a.k % kScaleBlock) {
      Wide wb[4];
      load_slowly(whole);
      read_step(0, f[0]);
      near = all_near(0);
      widen_b(f[0], f[0].sb, wb);
      multiply_wide(f[0], wb, acc);
      wait_and_meet<0>();
    }
    if (whole && near) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < kLoads; ++c) load(s, s, c);
      unsigned slot = 0;
      wait_and_meet<0>();
      if (wave >= kWaves / 2) wait_and_meet<0>();
      for (unsigned b = 0; b < whole; ++b) {
        near = all_near(slot);
        if (!near) break;
        Wide wb[4];
        const unsigned before = slot == 0 ? kStages - 1 : slot - 1;
        // changed as far as the compiler knows: it would otherwise keep every address of the loop in a
        // register of its own, and sums in scratch memory
        asm volatile("" : "+v"(lane_at[0][0]), "+v"(lane_at[0][1]), "+v"(lane_at[1][0]), "+v"(lane_at[1][1]));
#pragma unroll
        for (int c = 0; c < kLoads; ++c) load(b + 2, before, c);
        read_scales(slot, f[0]);
#pragma unroll
        for (int c = 0; c < 16; ++c) read_piece(slot, f[0], c);
        __builtin_amdgcn_sched_barrier(0);
        widen_b(f[0], f[0].sb, wb);
        wait_and_meet<kLoads>();  // the next step is in LDS
        multiply_wide(f[0], wb, acc);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        slot = slot + 1 == kStages ? 0 : slot + 1;
      }
      if (wave < kWaves / 2) wait_and_meet<0>();
      wait_and_meet<0>();
    }
    if (!near) {
      f32x4 sums[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (unsigned b = 0; b * static_cast<size_t>(kScaleBlock) < a.k; ++b) {
        Wide wb[4];
        load_slowly(b);
        read_step(0, f[0]);
        widen_b(f[0], 0x7f7f7f7fu, wb);
        scaled_sums(f[0], wb, sums, group);
        wait_and_meet<0>();
      }
      store(sums);
      return;
    }
  }
  store(acc);
}

// ------------------------------------------------------------------------------------------
// Small tiles, shared along k
// ------------------------------------------------------------------------------------------
// Where larger tiles would leave most of the chip idle (100 x 8192 x 8192: 17.4 us, 128 x 128 31.8): a block makes
// 64 x 64 of C, and each of its WAVES waves takes every WAVES-th step of 128 k for itself -- its own slots in LDS,
// eight in all, waited for by count, no barrier -- with the sums joined in LDS at the end, in
// order. Four waves keep two steps each on their way; eight (32-bit results) one, and two to a SIMD.
constexpr int kSplitSlot = 128 * 128 + 256;  // 64 rows of A, 64 of B, 16 dwords of scales of each (and room)
constexpr int kSplitPitch = 68;              // floats of a row of partial sums

// A dword for each lane from its own address to LDS.
__device__ __forceinline__ void load_lds4_each(unsigned to, const uint8_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "m0", "memory");
}

template <class O, bool kExact, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void matmul_split_kernel(MatmulArgs a, unsigned tiles_m, unsigned tiles_n) {
  constexpr int kSlots = 8 / WAVES;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[8 * kSplitSlot];
  static_assert(4 * 64 * kSplitPitch * 4 <= sizeof(lds), "four waves' sums go where the steps were");
  const int lane = threadIdx.x % 64, group = lane / 16, j16 = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const size_t m0 = static_cast<size_t>(tm) * 64, n0 = static_cast<size_t>(tn) * 64;
  const unsigned whole = static_cast<unsigned>(a.k / kScaleBlock);
  const unsigned steps = whole > static_cast<unsigned>(wave) ? (whole - wave + WAVES - 1) / WAVES : 0;
  uint8_t* const mine = lds + wave * kSlots * kSplitSlot;
  const unsigned lds0 = lds_address(mine);

  const uint8_t* const abase = a.a.values + m0 * a.a.ld;
  const uint8_t* const bbase = a.b.values + n0 * a.b.ld;
  unsigned off_a[8], off_b[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int r = slot_row(8 * c + lane / 8);
    const unsigned piece = 16u * ((lane % 8) ^ (r / 4 % 8));
    off_a[c] = static_cast<unsigned>(std::min<size_t>(r, a.m - 1 - m0)) * static_cast<unsigned>(a.a.ld) + piece;
    off_b[c] = static_cast<unsigned>(std::min<size_t>(r, a.n - 1 - n0)) * static_cast<unsigned>(a.b.ld) + piece;
  }
  // scales: lanes 0-15 a dword of A's rows each, 16-31 of B's (for 128 x 128 tiles of B the same one, with
  // this tile's byte in it); the others repeat them
  const bool of_b = lane / 16 % 2;
  const size_t tile_n = n0 / kScaleBlock;
  const uint8_t* const scales = !of_b       ? a.a.scales + std::min(m0 + 4 * j16, (a.m - 1) / 4 * 4)
                                : a.b_tiles ? a.b.scales + tile_n / 4 * 4
                                            : a.b.scales + std::min(n0 + 4 * j16, (a.n - 1) / 4 * 4);
  const size_t scale_step = of_b ? a.b.ld_scales : a.a.ld_scales;
  const unsigned pick = a.b_tiles ? static_cast<unsigned>(tile_n % 4) * 0x01010101u : 0x03020100u;

  constexpr int kLoads = 17;
  auto load = [&](unsigned s, unsigned slot, int c) {  // behind the last step it is read once more, for the counts
    const size_t b = static_cast<size_t>(s < steps ? s : steps - 1) * WAVES + wave;
    const unsigned to = lds0 + slot * kSplitSlot;
    if (c == 0) load_lds4_each(to + 128 * 128, scales + b * scale_step);
    else if (c < 9) load_lds16(to + (c - 1) * 1024, abase + b * kScaleBlock, off_a[c - 1]);
    else load_lds16(to + (c - 1) * 1024, bbase + b * kScaleBlock, off_b[c - 9]);
  };
  unsigned lane_at[2][2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      lane_at[odd][h] = lds0 + 512u * j16 + 128u * (odd ^ (j16 / 8)) + 16u * ((4 * h + group) ^ (j16 % 8));
  auto read_scales = [&](unsigned slot, Operands& f) {
    const unsigned* const at = reinterpret_cast<const unsigned*>(mine + slot * kSplitSlot + 128 * 128);
    f.sa = own_scales(at[j16], m0 + 4 * j16, a.m);
    f.sb = __builtin_amdgcn_perm(0, at[16 + j16], pick);
    if (!a.b_tiles) f.sb = own_scales(f.sb, n0 + 4 * j16, a.n);
  };
  auto read_piece = [&](unsigned slot, Operands& f, int c) {  // piece c of the 16: B's, then A's
    typedef const __attribute__((address_space(3))) u32x4* lds16;
    const int i = c / 2 % 4, h = c % 2;
    if (c < 8) f.b[i].half[h] = *reinterpret_cast<lds16>(lane_at[i % 2][h] + slot * kSplitSlot + 8192 + i / 2 * 256);
    else f.a[i].half[h] = *reinterpret_cast<lds16>(lane_at[i % 2][h] + slot * kSplitSlot + i / 2 * 256);
  };
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Operands f[kSlots];
  auto read = [&](unsigned slot, Operands& o) {
    read_scales(slot, o);
#pragma unroll
    for (int c = 0; c < 16; ++c) read_piece(slot, o, c);
  };
  auto far_step = [&](const Operands& o) {
    bool far = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) far = far || far_scale(o.sb >> (8 * i) & 255u) || far_scale(o.sa >> (8 * i) & 255u);
    return __builtin_amdgcn_ballot_w64(far) != 0;
  };
  bool far = false;
  // the block cut off by the end of the rows, zeros behind it
  const bool cut = a.k % kScaleBlock && whole % WAVES == static_cast<unsigned>(wave);
  auto load_cut = [&] {
    const size_t k = static_cast<size_t>(whole) * kScaleBlock;
#pragma unroll 8
    for (int c = 0; c < 16; ++c) {
      const int r = slot_row(8 * (c % 8) + lane / 8);
      const size_t piece = 16 * ((lane % 8) ^ (r / 4 % 8));
      const uint8_t* const src = c < 8 ? a.a.values + std::min(m0 + r, a.m - 1) * a.a.ld : a.b.values + std::min(n0 + r, a.n - 1) * a.b.ld;
      *reinterpret_cast<u32x4*>(mine + c * 1024 + lane * 16) = load16(src, k + piece, a.k);
    }
    load_lds4_each(lds0 + 128 * 128, scales + whole * scale_step);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    read(0, f[0]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  if (cut) {
    load_cut();
    if constexpr (kExact) {
      far = far_step(f[0]);
      Wide wb[4];
      widen_b(f[0], f[0].sb, wb);
      multiply_wide(f[0], wb, acc);
    } else {
      multiply_step(f[0], acc, [](int) {});
    }
  }
  if (steps && !far) {
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
#pragma unroll
      for (int c = 0; c < kLoads; ++c) load(s, s, c);
    if constexpr (kSlots == 2) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
      read(0, f[0]);
      auto step = [&](unsigned s, const Operands& now, Operands& then) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // step s is in registers: its slot is free
#pragma unroll
        for (int c = 0; c < kLoads; ++c) load(s + 2, s % 2, c);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");  // step s + 1 is in LDS
        read_scales((s + 1) % 2, then);
        multiply_step(now, acc, [&](int c) { read_piece((s + 1) % 2, then, c); });
      };
      for (unsigned s = 0; s < steps; s += 2) {
        step(s, f[0], f[1]);
        if (s + 1 < steps) step(s + 1, f[1], f[0]);
      }
    } else {
      for (unsigned s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        read(0, f[0]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // step s is in registers: its slot is free
#pragma unroll
        for (int c = 0; c < kLoads; ++c) load(s + 1, 0, c);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kExact) {
          far = far_step(f[0]);
          if (far) break;
          Wide wb[4];
          widen_b(f[0], f[0].sb, wb);
          multiply_wide(f[0], wb, acc);
        } else {
          multiply_step(f[0], acc, [](int) {});
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
  if constexpr (kExact) {
    if (far) {  // all of this wave's steps again, the slow way
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      for (unsigned s = 0; s < steps + cut; ++s) {
        if (s < steps) {
#pragma unroll
          for (int c = 0; c < kLoads; ++c) load(s, 0, c);
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          read(0, f[0]);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
          load_cut();
        }
        Wide wb[4];
        widen_b(f[0], 0x7f7f7f7fu, wb);
        scaled_sums(f[0], wb, acc, group);
      }
    }
  }

  // The waves' sums, joined: with eight, the upper four hand theirs over first.
  float* const part = reinterpret_cast<float*>(lds) + wave % 4 * 64 * kSplitPitch;
  auto hand_over = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(part + (4 * j16 + i) * kSplitPitch + 16 * group + 4 * r) =
            f32x4{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
  };
  __syncthreads();  // everyone has read its last step
  if constexpr (WAVES == 8) {
    if (wave >= 4) hand_over();
    __syncthreads();
    if (wave < 4)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 more = *reinterpret_cast<const f32x4*>(part + (4 * j16 + i) * kSplitPitch + 16 * group + 4 * r);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j][r] += more[j];
        }
  }
  if (wave < 4) hand_over();  // where it read
  __syncthreads();
  constexpr int kPer = 16 / sizeof(O), kRows = WAVES * kPer;  // columns of a thread, rows that all of them store at once
  const int col = threadIdx.x % (64 / kPer) * kPer;
  const int left = a.n > n0 + col ? static_cast<int>(std::min<size_t>(a.n - n0 - col, kPer)) : 0;
#pragma unroll
  for (int row = threadIdx.x / (64 / kPer); row < 64; row += kRows) {
    if (m0 + row >= a.m) return;
    const float* const sums = reinterpret_cast<const float*>(lds) + row * kSplitPitch + col;
    float v[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      v[e] = sums[e];
#pragma unroll
      for (int w = 1; w < 4; ++w) v[e] += sums[w * 64 * kSplitPitch + e];
    }
    store_some(static_cast<O*>(a.c) + (m0 + row) * a.ldc + n0 + col, left, v);
  }
}

// The same at 32 x 32, for few rows or few tiles (27 rows by 8192 x 8192: 13.3 us, 5.0 TB/s of weights): 32 rows
// of A and 32 of B lie in LDS as the 64 rows of a tile would, rows 2 j and 2 j + 1 of A at places 4 j and
// 4 j + 1, those of B behind them. 16 steps of 8 KB are on their way for a CU, shared by its waves.
constexpr int kSmallSlot = 64 * 128 + 256;
constexpr int kSmallPitch = 36;  // floats of a row of partial sums

__device__ __forceinline__ void load_lds16_each(unsigned to, const uint8_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0", "memory");
}

template <class O, bool kExact, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void matmul_small_kernel(MatmulArgs a, unsigned tiles_m, unsigned tiles_n) {
  constexpr int kSlots = 16 / WAVES;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * kSlots * kSmallSlot];
  static_assert(WAVES * 32 * kSmallPitch * 4 <= sizeof(lds), "the partial sums go where the steps were");
  const int lane = threadIdx.x % 64, group = lane / 16, j16 = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const size_t m0 = static_cast<size_t>(tm) * 32, n0 = static_cast<size_t>(tn) * 32;
  const unsigned whole = static_cast<unsigned>(a.k / kScaleBlock);
  const unsigned steps = whole > static_cast<unsigned>(wave) ? (whole - wave + WAVES - 1) / WAVES : 0;
  uint8_t* const mine = lds + wave * kSlots * kSmallSlot;
  const unsigned lds0 = lds_address(mine);

  // where this lane's part of place 8 c + lane / 8 comes from, from k = 0 on
  const uint8_t* from[8];
  unsigned piece[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int r = slot_row(8 * c + lane / 8), of_tile = 2 * (r / 4) + r % 2;
    piece[c] = 16u * ((lane % 8) ^ (r / 4 % 8));
    from[c] = r % 4 < 2 ? a.a.values + std::min(m0 + of_tile, a.m - 1) * a.a.ld : a.b.values + std::min(n0 + of_tile, a.n - 1) * a.b.ld;
  }
  // scales: lanes 0-7 a dword of A's rows each, 8-15 of B's (or the one with the tile's byte); the others repeat them
  const bool of_b = lane / 8 % 2;
  const size_t tile_n = n0 / kScaleBlock;
  const uint8_t* const scales = !of_b       ? a.a.scales + std::min(m0 + 4 * (lane % 8), (a.m - 1) / 4 * 4)
                                : a.b_tiles ? a.b.scales + tile_n / 4 * 4
                                            : a.b.scales + std::min(n0 + 4 * (lane % 8), (a.n - 1) / 4 * 4);
  const size_t scale_step = of_b ? a.b.ld_scales : a.a.ld_scales;

  constexpr int kLoads = 9;
  auto load = [&](unsigned s, unsigned slot) {  // behind the last step it is read once more, for the counts
    const size_t b = static_cast<size_t>(s < steps ? s : steps - 1) * WAVES + wave;
    const unsigned to = lds0 + slot * kSmallSlot;
    load_lds4_each(to + 64 * 128, scales + b * scale_step);
#pragma unroll
    for (int c = 0; c < 8; ++c) load_lds16_each(to + c * 1024, from[c] + piece[c] + b * kScaleBlock);
  };
  unsigned lane_at[2][2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      lane_at[odd][h] = lds0 + 512u * j16 + 128u * (odd ^ (j16 / 8)) + 16u * ((4 * h + group) ^ (j16 % 8));
  struct Step {
    Fragment a[2], b[2];
    unsigned sa, sb;  // bytes 0 and 1
  };
  const size_t row2 = m0 + 2 * j16, col2 = n0 + 2 * j16;
  const unsigned pick = a.b_tiles ? static_cast<unsigned>(tile_n % 4) * 0x0101u : j16 % 2 ? 0x0302u : 0x0100u;
  auto read = [&](unsigned slot, Step& f) {
    typedef const __attribute__((address_space(3))) u32x4* lds16;
    const unsigned* const at = reinterpret_cast<const unsigned*>(mine + slot * kSmallSlot + 64 * 128);
    f.sa = __builtin_amdgcn_perm(0, at[j16 / 2], j16 % 2 ? 0x0302u : 0x0100u);
    f.sb = __builtin_amdgcn_perm(0, at[8 + j16 / 2], pick);
    if constexpr (kExact) {
      f.sa = own_scales(f.sa, row2, a.m);
      if (!a.b_tiles) f.sb = own_scales(f.sb, col2, a.n);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f.a[i].half[h] = *reinterpret_cast<lds16>(lane_at[i][h] + slot * kSmallSlot);
        f.b[i].half[h] = *reinterpret_cast<lds16>(lane_at[i][h] + slot * kSmallSlot + 256);
      }
  };
  f32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply_all = [&](const Step& f) {
    if constexpr (!kExact) {
      acc[0][0] = mfma_scaled<0, 0>(f.b[0], f.a[0], acc[0][0], f.sb, f.sa);
      acc[0][1] = mfma_scaled<1, 0>(f.b[1], f.a[0], acc[0][1], f.sb, f.sa);
      acc[1][0] = mfma_scaled<0, 1>(f.b[0], f.a[1], acc[1][0], f.sb, f.sa);
      acc[1][1] = mfma_scaled<1, 1>(f.b[1], f.a[1], acc[1][1], f.sb, f.sa);
    } else {
      const bool far = far_scale(f.sa & 255u) || far_scale(f.sa >> 8 & 255u) || far_scale(f.sb & 255u) || far_scale(f.sb >> 8 & 255u);
      const bool near = __builtin_amdgcn_ballot_w64(far) == 0;
      Wide wb[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) wb[j] = widen(f.b[j], near ? scale_value(f.sb >> (8 * j) & 255u) : 1.f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Wide wa = widen(f.a[i], near ? scale_value(f.sa >> (8 * i) & 255u) : 1.f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (near) {
            acc[i][j] = multiply(wb[j], wa, acc[i][j]);
          } else {
            const f32x4 p = multiply(wb[j], wa, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[i][j][r] += scaled(p[r], f.sa >> (8 * i) & 255u, __shfl(f.sb, 4 * group + r, 64) >> (8 * j) & 255u);
          }
        }
      }
    }
  };

  Step f[2];
  if (steps) {
#pragma unroll
    for (int s = 0; s < kSlots; ++s) load(s, s);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kSlots - 1) * kLoads) : "memory");
    read(0, f[0]);
    auto step = [&](unsigned s, const Step& now, Step& then) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // step s is in registers: its slot is free
      load(s + kSlots, s % kSlots);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kSlots - 1) * kLoads) : "memory");  // step s + 1 is in LDS
      read((s + 1) % kSlots, then);
      __builtin_amdgcn_sched_barrier(0);
      multiply_all(now);
    };
    for (unsigned s = 0; s < steps; s += 2) {
      step(s, f[0], f[1]);
      if (s + 1 < steps) step(s + 1, f[1], f[0]);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
  if (a.k % kScaleBlock && whole % WAVES == static_cast<unsigned>(wave)) {  // the block cut off by the end of the rows
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<u32x4*>(mine + c * 1024 + lane * 16) = load16(from[c], static_cast<size_t>(whole) * kScaleBlock + piece[c], a.k);
    load_lds4_each(lds0 + 64 * 128, scales + whole * scale_step);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    read(0, f[0]);
    multiply_all(f[0]);
  }

  __syncthreads();  // everyone has read its last step
  float* const part = reinterpret_cast<float*>(lds) + wave * 32 * kSmallPitch;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h)  // lane: row 2 j16 + i, columns 8 group + 2 r + j
      *reinterpret_cast<f32x4*>(part + (2 * j16 + i) * kSmallPitch + 8 * group + 4 * h) =
          f32x4{acc[i][0][2 * h], acc[i][1][2 * h], acc[i][0][2 * h + 1], acc[i][1][2 * h + 1]};
  __syncthreads();
  constexpr int kPer = 16 / sizeof(O);  // columns of a thread
  const int row = threadIdx.x / (32 / kPer), col = threadIdx.x % (32 / kPer) * kPer;
  if (row >= 32 || m0 + row >= a.m) return;
  const float* const sums = reinterpret_cast<const float*>(lds) + row * kSmallPitch + col;
  float v[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    v[e] = sums[e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v[e] += sums[w * 32 * kSmallPitch + e];
  }
  store_some(static_cast<O*>(a.c) + (m0 + row) * a.ldc + n0 + col, a.n > n0 + col ? static_cast<int>(std::min<size_t>(a.n - n0 - col, kPer)) : 0, v);
}

// ------------------------------------------------------------------------------------------
// Large tiles: 256 x 256 of C, eight waves in two groups that take turns
// ------------------------------------------------------------------------------------------
// Four waves (one on each SIMD unit) make the upper 128 rows, four the lower ones, each 128 x 64. A
// step of 128 k is four phases, a barrier after each: read B and half of A from LDS | 16 matrix
// instructions | read the other half of A | 16 matrix instructions. The lower group runs one phase
// behind, so on every SIMD one wave multiplies while the other reads.
// LDS holds two steps. A slot is refilled once both groups have read it -- B and the first half of A in
// the second multiplying phase of a step, the second half in the first one of the next -- and waits
// count the loads that may still be on their way instead of draining them: a step's bytes have
// about four phases to arrive. Every wave issues the same nine loads a step between its matrix
// instructions (256 bytes of scales, four pieces of 1 KiB of B, two of A's first half; two of A's
// second half), which makes the counts the same for all.
// 8192 x 8192 x 8192: 428 - 452 us, 2430 - 2570 TFLOP/s at the 2.0 GHz that power leaves; no access to LDS conflicts.
// LDS: two slots each of B's 256 rows, of A's first and of its second halves (128 rows each) and of the
// scales, so that both slots lie within the reach of one address.
constexpr int kBigB = 0, kBigA = 2 * 256 * 128, kBigHalf = 128 * 128, kBigScales = 2 * 512 * 128;
constexpr int kBigLds = kBigScales + 2 * 512;

// End of a reading phase: what this wave read has arrived, of its loads at most kLeft are on their way.
template <int kLeft> __device__ __forceinline__ void read_end() {
  static_assert(kLeft == 0 || kLeft == 2 || kLeft == 7, "waits");
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (kLeft == 7) asm volatile("s_waitcnt vmcnt(7) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  else if constexpr (kLeft == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// End of a multiplying phase (or a phase a group sits out).
__device__ __forceinline__ void phase_end() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <class O>
__global__ __launch_bounds__(512, 2) void matmul_big_kernel(MatmulArgs a, unsigned tiles_m, unsigned tiles_n) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kBigLds];
  const int lane = threadIdx.x % 64, group = lane / 16, j16 = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wm = wave / 4, wn = wave % 4;
  const unsigned lds0 = lds_address(lds);

  unsigned tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const size_t m0 = static_cast<size_t>(tm) * 256, n0 = static_cast<size_t>(tn) * 256;
  const unsigned whole = static_cast<unsigned>(a.k / kScaleBlock);  // 1 at least

  // A lane loads 16 bytes at row r of each 64 rows (pitches below 2^23: the offsets from the tile's
  // first row fit 32 bits); rows behind the last one are that one again. Slots hold of A the rows
  // 0-63 and 128-191 (first halves), 64-127 and 192-255 (second halves).
  const unsigned r = static_cast<unsigned>(slot_row(8 * wave + lane / 8));
  const unsigned piece = 16u * ((lane % 8) ^ (r / 4 % 8));
  const unsigned lda = static_cast<unsigned>(a.a.ld), ldb = static_cast<unsigned>(a.b.ld);
  unsigned row_a = r * lda, row_b = r * ldb;
  const unsigned last_a = static_cast<unsigned>(std::min<size_t>(255, a.m - 1 - m0)) * lda;
  const unsigned last_b = static_cast<unsigned>(std::min<size_t>(255, a.n - 1 - n0)) * ldb;
  const uint8_t* const abase = a.a.values + m0 * a.a.ld;
  const uint8_t* const bbase = a.b.values + n0 * a.b.ld;
  // scales: the tile's 256 rows of A (even waves load them) or of B (odd waves), a dword a lane; for
  // 128 x 128 tiles of B the dword that holds the two of this tile, in every lane
  const uint8_t* sbase;
  unsigned off_s;
  if (wave % 2 == 0) {
    sbase = a.a.scales + m0;
    off_s = static_cast<unsigned>(std::min<size_t>(4 * lane, (a.m - 1) / 4 * 4 - m0));
  } else if (a.b_tiles) {
    sbase = a.b.scales + n0 / kScaleBlock / 4 * 4;
    off_s = 0;
  } else {
    sbase = a.b.scales + n0;
    off_s = static_cast<unsigned>(std::min<size_t>(4 * lane, (a.n - 1) / 4 * 4 - n0));
  }
  const size_t s_step = wave % 2 == 0 ? a.a.ld_scales : a.b.ld_scales;

  // Load c of the nine of step b: 0 the scales, 1-4 B, 5-6 A's first halves; 7-8 its second halves.
  // Behind the last step it is read once more, into a slot nobody reads again: the counts stay true.
  auto load = [&](unsigned step, int c, int slot) {
    const size_t b = step < whole ? step : whole - 1;
    if (c == 0) load_lds4(lds0 + kBigScales + slot * 512 + (wave % 2) * 256, sbase + b * s_step, off_s);
    else if (c < 5)
      load_lds16(lds0 + kBigB + slot * 32768 + (wave + 8 * (c - 1)) * 1024, bbase + b * kScaleBlock,
                 std::min(row_b + (c - 1) * 64 * ldb, last_b) + piece);
    else
      load_lds16(lds0 + kBigA + (2 * ((c - 5) / 2) + slot) * kBigHalf + (wave + 8 * ((c - 5) % 2)) * 1024,
                 abase + b * kScaleBlock, std::min(row_a + ((c - 5) % 2 * 128 + (c - 5) / 2 * 64) * lda, last_a) + piece);
  };

  f32x4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Fragment fb[4], fa[4];
  unsigned sa[2], sb = 0;
  sa[0] = sa[1] = 0;

  // Where in 64 rows of LDS this lane finds its two pieces of an even and of an odd tile's row: all
  // other offsets are constants of the read instructions.
  unsigned lane_at[2][2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      lane_at[odd][h] = lds0 + 512u * j16 + 128u * (odd ^ (j16 / 8)) + 16u * ((4 * h + group) ^ (j16 % 8));
  auto fragment = [&](unsigned offset, int i, int fixed) {
    typedef const __attribute__((address_space(3))) u32x4* lds16;
    Fragment f;
    f.half[0] = *reinterpret_cast<lds16>(lane_at[i % 2][0] + offset + (fixed + i / 2 * 256));
    f.half[1] = *reinterpret_cast<lds16>(lane_at[i % 2][1] + offset + (fixed + i / 2 * 256));
    return f;
  };
  // 16 matrix instructions; issue(i) after each four of them, in their shadow.
  auto multiply_half = [&](auto half, auto issue) {
    constexpr int g = decltype(half)::value;
    auto four = [&](auto tag) {
      constexpr int i = decltype(tag)::value;
      f32x4(&c)[4] = acc[g * 4 + i];
      c[0] = mfma_scaled<0, i>(fb[0], fa[i], c[0], sb, sa[g]);
      c[1] = mfma_scaled<1, i>(fb[1], fa[i], c[1], sb, sa[g]);
      c[2] = mfma_scaled<2, i>(fb[2], fa[i], c[2], sb, sa[g]);
      c[3] = mfma_scaled<3, i>(fb[3], fa[i], c[3], sb, sa[g]);
      __builtin_amdgcn_sched_barrier(0);
      issue(i);
      __builtin_amdgcn_sched_barrier(0);
    };
    four(std::integral_constant<int, 0>{});
    four(std::integral_constant<int, 1>{});
    four(std::integral_constant<int, 2>{});
    four(std::integral_constant<int, 3>{});
  };
  constexpr auto kHalf0 = std::integral_constant<int, 0>{};
  constexpr auto kHalf1 = std::integral_constant<int, 1>{};
  const auto nothing = [](int) {};

  const unsigned pick = a.b_tiles ? static_cast<unsigned>((n0 / kScaleBlock + wn / 2) % 4) * 0x01010101u : 0x03020100u;
  const int at_sb = 64 + (a.b_tiles ? 0 : wn * 16 + j16);
  // B, the first two of this wave's four tiles in A's first half, the scales; then the other two
  auto read_first = [&](int slot) {
#pragma unroll
    for (int j = 0; j < 4; ++j) fb[j] = fragment(kBigB + wn * 8192, j, slot * 32768);
#pragma unroll
    for (int i = 0; i < 2; ++i) fa[i] = fragment(kBigA + wm * 8192, i, slot * kBigHalf);
    const unsigned* const scales = reinterpret_cast<const unsigned*>(lds + kBigScales + slot * 512);
    sa[0] = scales[wm * 32 + j16];
    sa[1] = scales[wm * 32 + 16 + j16];
    sb = __builtin_amdgcn_perm(0, scales[at_sb], pick);
  };
  auto read_more = [&](int slot) {
#pragma unroll
    for (int i = 2; i < 4; ++i) fa[i] = fragment(kBigA + wm * 8192, i, slot * kBigHalf);
  };
  auto read_second = [&](int slot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[i] = fragment(kBigA + wm * 8192, i, (2 + slot) * kBigHalf);
  };

  if (a.k % kScaleBlock) {  // first the block that the end of the rows cuts off, zeros behind it
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int row = static_cast<int>(r) + (c < 4 ? 64 * c : (c - 4) % 2 * 128 + (c - 4) / 2 * 64);
      const uint8_t* const src = c < 4 ? a.b.values + std::min(n0 + row, a.n - 1) * a.b.ld : a.a.values + std::min(m0 + row, a.m - 1) * a.a.ld;
      uint8_t* const to = lds + (c < 4 ? kBigB + c * 8192 : kBigA + (c - 4) / 2 * 2 * kBigHalf + (c - 4) % 2 * 8192) + wave * 1024 + lane * 16;
      *reinterpret_cast<u32x4*>(to) = load16(src, static_cast<size_t>(whole) * kScaleBlock + piece, a.k);
    }
    load_lds4(lds0 + kBigScales + (wave % 2) * 256, sbase + whole * s_step, off_s);
    read_end<0>();
    read_first(0);
    read_more(0);
    multiply_half(kHalf0, nothing);
    read_second(0);
    multiply_half(kHalf1, nothing);
    __syncthreads();
  }

#pragma unroll
  for (int c = 0; c < 9; ++c) load(0, c, 0);
#pragma unroll
  for (int c = 0; c < 7; ++c) load(1, c, 1);
  read_end<0>();
  if (wm == 1) phase_end();  // the lower group runs one phase behind
  auto step = [&](unsigned b, auto parity) {
    constexpr int slot = decltype(parity)::value;
    // changed as far as the compiler knows: it would otherwise keep every offset of the loop, and the
    // sums that belong in these registers in scratch memory
    asm volatile("" : "+v"(row_a), "+v"(row_b), "+v"(lane_at[0][0]), "+v"(lane_at[0][1]), "+v"(lane_at[1][0]), "+v"(lane_at[1][1]));
    read_first(slot);
    read_end<7>();  // this step's second halves, requested a step ago, are there
    read_more(slot);
    multiply_half(kHalf0, [&](int i) { if (i < 2) load(b + 1, 7 + i, 1 - slot); });
    phase_end();
    read_second(slot);
    read_end<2>();  // the next step's first seven are there
    multiply_half(kHalf1, [&](int i) { load(b + 2, 2 * i, slot); if (i < 3) load(b + 2, 2 * i + 1, slot); });
    phase_end();
  };
  for (unsigned b = 0; b + 1 < whole; b += 2) {
    step(b, kHalf0);
    step(b + 1, kHalf1);
  }
  if (whole % 2) step(whole - 1, kHalf0);
  if (wm == 0) phase_end();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may still be on its way to LDS when the block ends
  const size_t mw = m0 + wm * 128, col = n0 + wn * 64;
  const int left = col < a.n ? static_cast<int>(std::min<size_t>(a.n - col, 64)) : 0;
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t row = mw + 64 * g + 4 * j16 + i;
      store_row(static_cast<O*>(a.c) + row * a.ldc + col, row < a.m, left, acc[g * 4 + i], group);
    }
}

void check(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

template <class O, bool kExact, int TM, int TN, int kStages> void launch_stage(const MatmulArgs& a, hipStream_t stream) {
  const size_t tm = (a.m + TM - 1) / TM, tn = (a.n + TN - 1) / TN;
  hipLaunchKernelGGL((matmul_stage_kernel<O, kExact, TM, TN, kStages>), dim3(static_cast<unsigned>(tm * tn)), dim3(TM / 64 * (TN / 64) * 64),
                     0, stream, a, static_cast<unsigned>(tm), static_cast<unsigned>(tn));
}

template <class O, bool kExact> void launch_rows(const MatmulArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((matmul_rows_kernel<O, kExact>), dim3(static_cast<unsigned>((a.n + 15) / 16)), dim3(kRowWaves * 64), 0, stream, a);
}

// Which tile makes a product: each kernel has one block on a CU at a time, so it takes ceil(tiles / 256) rounds,
// each of a start and an end and a time for every 128 k (for every 512 where four waves share k, 1024 for eight). The
// figures in launch() are microseconds, fitted to these (those in brackets are not chosen). 16-bit:
//
//     m x n x k            32 x 32   64 x 64   128 x 128   192 x 128   256 x 128   256 x 256
//     32 x 8192 x 8192      14.2     (15.8)
//     24 x 4096 x 4096       6.4     (9.2)                                                    (rows 8.1)
//     16 x 1024 x 8192       8.0     (12.3)                                                   (rows 10.4)
//     500 x 500 x 8000      10.3     (17.9)     (33.1)
//     27 x 14336 x 4096    (14.9)     13.5                                                    (rows 23.4)
//     100 x 8192 x 8192    (33.1)     17.3      (31.5)
//     256 x 4096 x 4096    (23.7)     12.8      (20.1)      (27.3)      (29.6)      (50.7)
//     512 x 4096 x 4096               21.4      (21.3)      (28.6)      (31.4)      (51.6)
//     2000 x 2000 x 2000             (34.1)      20.3       (23.7)      (26.6)      (36.6)
//     1024 x 4096 x 4096             (41.0)      24.2       (31.3)      (33.9)      (52.8)
//     607 x 12416 x 256              (33.4)      16.6       (21.3)      (21.5)      (20.1)
//     777 x 5003 x 4432              (56.5)     (47.9)       34.9       (38.6)      (58.2)
//     2521 x 2176 x 128              (24.5)     (15.0)       12.1       (13.4)      (18.0)
//     2048 x 4096 x 4096             (78.8)     (46.9)      (58.8)       39.2       (56.4)
//     8192 x 1024 x 8192             (130.9)    (91.8)      (98.2)       68.3       (96.4)
//     3000 x 8192 x 2048             (156.4)    (86.5)      (79.3)       70.8       (71.3)
//     4096 x 4096 x 512              (76.8)     (32.9)      (33.5)      (29.3)       23.2
//     4096 x 4096 x 4096             (150.5)   (100.7)      (93.9)      (76.1)       65.1
//     8192 x 8192 x 1024             (316.4)   (149.3)     (141.6)     (123.4)       98.0
//
// float32, where eight waves share k: two on a SIMD, one widens while the other multiplies (with four, one
// to a SIMD: 64 x 64 19.3, 30.2, 36.4 and 78.3 us in rows 1, 2, 4 and 5; 32 x 32 11.4, 16.6 in rows 1 and 2):
//
//     m x n x k            32 x 32   64 x 64   256 x 128
//     64 x 4096 x 4096       9.7     (13.7)     (50.2)
//     100 x 1024 x 8192     11.6     (19.3)     (93.0)     (rows of 16 columns 21.5)
//     100 x 8192 x 1024    (18.8)      9.8      (19.3)     (rows of 16 columns 11.9)
//     1000 x 1000 x 8000   (49.6)     24.9     (101.2)
//     1024 x 4096 x 4096  (113.5)     58.3      (61.6)
//     2394 x 1408 x 2048   (70.2)    (40.9)      38.1
//     2521 x 2176 x 128    (62.6)    (36.4)      16.5
//     2048 x 4096 x 4096            (112.8)      70.6
struct Tiles {
  unsigned m, n;
  Tiles(const MatmulArgs& a, size_t tm, size_t tn) : m(static_cast<unsigned>((a.m + tm - 1) / tm)), n(static_cast<unsigned>((a.n + tn - 1) / tn)) {}
  dim3 grid() const { return dim3(m * n); }
  // a launch has fewer than 2^32 threads
  bool fit(size_t threads) const { return static_cast<size_t>(m) * n * threads >> 32 == 0; }
  double time(size_t threads, double ends, double step, size_t steps) const {
    if (!fit(threads)) return HUGE_VAL;
    const size_t rounds = (static_cast<size_t>(m) * n + 255) / 256;
    return static_cast<double>(rounds) * (ends + step * static_cast<double>(steps));
  }
};

template <class O, bool kExact> void launch(const MatmulArgs& a, hipStream_t stream) {
  const Tiles small(a, 32, 32), split(a, 64, 64), mid(a, 128, 128), high(a, 192, 128), tall(a, 256, 128), big(a, 256, 256);
  constexpr int kWaves = kExact ? 8 : 4;  // that share k in the smaller tiles
  const size_t steps = (a.k + kScaleBlock - 1) / kScaleBlock, shared = (steps + kWaves - 1) / kWaves;
  auto by_small = [&] { hipLaunchKernelGGL((matmul_small_kernel<O, kExact, kWaves>), small.grid(), dim3(kWaves * 64), 0, stream, a, small.m, small.n); };
  auto by_split = [&] { hipLaunchKernelGGL((matmul_split_kernel<O, kExact, kWaves>), split.grid(), dim3(kWaves * 64), 0, stream, a, split.m, split.n); };
  // rows too long for the larger tiles' 32-bit offsets
  if (a.a.ld >= (1u << 23) || a.b.ld >= (1u << 23)) {
    check(small.fit(kWaves * 64), "fp8_matmul: too many values of C for rows 2^23 bytes apart");
    return by_small();
  }
  if constexpr (kExact) {
    // One row of A or a few, for which 16 columns to a block leave fewer CUs without one: 1 x 4096 x 4096 6.3 us
    // and 8.0 (32 x 32), 16 x 4096 x 4096 7.4 and 8.1, 16 x 8192 x 1024 11.1 and 5.7.
    if (a.m <= 16 && a.n <= 6144) return launch_rows<O, true>(a, stream);
    const double smalls = small.time(512, 3.8, 0.95, shared), splits = split.time(512, 6.5, 1.95, shared);
    const double talls = tall.time(512, 10.0, 1.75, steps);
    if (smalls <= std::min(splits, talls)) by_small();
    else if (splits <= talls) by_split();
    else launch_stage<O, true, 256, 128, 3>(a, stream);
  } else {
    // One token or so: 16 columns to a block put 1024 < n <= 4096 on twice as many CUs (4096 x 4096: 5.6 us and
    // 6.2; 1024 x 8192: 7.8 both; 1000 x 1024: 5.7 and 5.2; 8192 x 1024: 7.5 and 5.3). From 8 rows on they
    // are no faster.
    if (a.m <= 4 && a.n > 1024 && a.n <= 4096) return launch_rows<O, false>(a, stream);
    const double smalls = small.time(256, 2.7, 0.45, shared), splits = split.time(256, 4.5, 0.75, shared), mids = mid.time(256, 6.0, 0.55, steps);
    const double highs = high.time(384, 8.5, 0.78, steps), talls = tall.time(512, 10.0, 0.95, steps);
    const double bigs = a.k >= kScaleBlock ? big.time(512, 13.0, 1.6, steps) : HUGE_VAL;  // it takes at least one whole block
    const double least = std::min({smalls, splits, mids, highs, talls, bigs});
    if (least == smalls) by_small();
    else if (least == splits) by_split();
    else if (least == mids) launch_stage<O, false, 128, 128, 4>(a, stream);
    else if (least == highs) launch_stage<O, false, 192, 128, 3>(a, stream);
    else if (least == talls) launch_stage<O, false, 256, 128, 3>(a, stream);
    else hipLaunchKernelGGL(matmul_big_kernel<O>, big.grid(), dim3(512), 0, stream, a, big.m, big.n);
  }
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
            reinterpret_cast<uintptr_t>(a.b.scales) % 4 == 0 && a.b.ld_scales % 4 == 0,
        "fp8: the scales of a block must start on a 4-byte boundary");
  check(a.m <= (size_t(1) << 32) && a.n <= (size_t(1) << 32) && (a.m + 63) / 64 * ((a.n + 63) / 64) <= (size_t(1) << 22),
        "fp8_matmul: at most 2^32 rows and columns of C, and 2^34 values");
  switch (out) {
    case LayerType::kF32: launch<float, true>(a, stream); break;
    case LayerType::kBF16: launch<__bf16, false>(a, stream); break;
    case LayerType::kF16: launch<_Float16, false>(a, stream); break;
  }
  TK8S_HIP_CHECK(hipGetLastError());
}

}  // namespace tk8s
