// Row operators of the 8-bit layer for gfx950: RMS norm with the residual's addition and an 8-bit
// output, its backward pass, and the rounding of a tensor to 8 bits. All of them stream: every
// value is read once, kept in registers, and written once, so HBM bounds them.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "tk8s/common.h"
#include "tk8s/fp8_device.h"
#include "tk8s/kernels.h"

namespace tk8s {

using namespace fp8;

namespace {

// Sum over the TPR threads of a row (consecutive ones; 16, 32 or whole waves). `slot`: one value per wave.
// Every thread of the block calls it when TPR > 64.
template <int TPR, class V>
__device__ __forceinline__ V row_sum(V v, V* slot) {
  v = sum_lanes<(TPR < 64 ? TPR : 64)>(v);
  if constexpr (TPR > 64) {
    constexpr int kWaves = TPR / 64;
    if (threadIdx.x % 64 == 0) slot[threadIdx.x / 64] = v;
    __syncthreads();
    v = V(0);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += slot[w];
    __syncthreads();  // the slots are free for the next sum
  }
  return v;
}

// ------------------------------------------------------------------------------------------
// RMS norm: h = x + residual rounded to T; y = h * rstd * w; the block's scale and e4m3 values
// ------------------------------------------------------------------------------------------
// y and its 8-bit form of 8 columns from h and the weight. y is in 32 bits, at most 3 units in the last
// place off (v w, rstd and their product are rounded once each) where all three are normal numbers. Where
// one of a wave's 512 values is near enough to a border between two e4m3 values for that to matter --
// one time in a hundred, and wherever there is a zero: in a padded row, in lanes behind a row's end -- or
// where a lane's values are so small that one of the three may not be normal (`low`), the wave makes
// them again in 64 bits, so that every value falls where the formula puts it.
//
// A value counts in its block if it is above 2^-10 of the block's scale, 2^-19 of the block's largest. Its v w
// is below 2^-126 only if it is below 2^-126 rstd, so blocks whose largest is 2^-107 rstd or more
// hold none such that count; those of 2^-107 or more none whose y is below 2^-126.
__device__ __forceinline__ unsigned low_below(float rstd32) {  // bits of the least largest magnitude that is not low
  return __float_as_uint(rstd32 < 0x1p-126f ? __builtin_inff() : 0x1p-107f * fmaxf(rstd32, 1.f));
}

template <bool kWhole, class T, class W>
__device__ __forceinline__ void norm_eight(const NormArgs& a, size_t row, int col, int n, const Packed8<T>& h, const Packed8<W>& w,
                                           double rstd, float rstd32, unsigned low) {
  float y[8];
  unsigned least = ~0u, top = 0;  // columns behind the end are zeros
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    y[j] = unpack(h, j) * unpack(w, j) * rstd32;
    least = min(least, from_border(y[j]));
    top = max(top, magnitude_bits(y[j]));
  }
  const bool small = top < low;
  if (__builtin_amdgcn_ballot_w64(near_border(least) || small) != 0 || a.y) {
    Packed8<T> o;
    float y32[8];
    unsigned any = 0;
    auto y64 = [&](int j) { return static_cast<double>(unpack(h, j)) * rstd * static_cast<double>(unpack(w, j)); };
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double v = y64(j);
      y[j] = round_to_odd(v);
      y32[j] = sizeof(T) == 4 ? static_cast<float>(v) : y[j];
      any |= odd_bits(v);
    }
    if (__builtin_amdgcn_ballot_w64(small && any << 1 != 0) != 0) {  // some are not 0, and below 2^-126 perhaps
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = round_tiny_to_odd(y64(j));
        if (sizeof(T) == 2) y32[j] = y[j];
      }
    }
    top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(y[j]));
    if (a.y) {
#pragma unroll
      for (int j = 0; j < 4; ++j) pack(o, j, y32[2 * j], y32[2 * j + 1]);
      store_packed<kWhole>(static_cast<T*>(a.y) + row * a.ldy + col, n, o);
    }
  }
  if (!a.q) return;
  const unsigned byte = scale_byte(max16(top));
  store_bytes<kWhole>(a.q + row * a.ldq + col, n,
                      u32x2{pack4(y[0], y[1], y[2], y[3], byte), pack4(y[4], y[5], y[6], y[7], byte)});
  if (n > 0 && col % kScaleBlock == 0) a.scales[static_cast<size_t>(col / kScaleBlock) * a.lds + row] = static_cast<uint8_t>(byte);
}

// 8 values of h = x + residual, rounded once.
template <class T> __device__ __forceinline__ Packed8<T> add_eight(const Packed8<T>& x, const Packed8<T>& r) {
  Packed8<T> h;
#pragma unroll
  for (int j = 0; j < 4; ++j) pack(h, j, unpack(x, 2 * j) + unpack(r, 2 * j), unpack(x, 2 * j + 1) + unpack(r, 2 * j + 1));
  return h;
}

template <class T> __device__ __forceinline__ double add_squares(const Packed8<T>& h, double sum) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const double v = static_cast<double>(unpack(h, j));
    sum = fma(v, v, sum);
  }
  return sum;
}

// A row belongs to TPR threads; thread t holds chunks c of 8 values at (c * TPR + t) * 8, so 16
// neighbouring lanes hold exactly one block of 128. The sum of squares and rstd are in 64 bits. A block
// walks rows a grid apart: the weight stays in its registers, and the next row is requested before the
// sum of this one is waited for. kWhole: rows are a whole number of chunks. 16384 x 8192, 16-bit, with a
// residual: 163 us, 5.8 TB/s, which HBM bounds; 1031 x 5003 without: 9.1 us, 1.7 TB/s, the time of a row and, for
// seven of the 1024 blocks, which are all there at once, of a second one (in 32 bits 11.4, from HBM, where 512 blocks
// make a third pass for seven rows); one row of 4096: 3.3 us, the latency of its loads and of its sum.
template <class T, class W, int TPR, int NCH, bool kWhole>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(NormArgs a) {
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
  __shared__ double slot[TPR < 64 ? 1 : TPR / 64 * kRows];
  const int t = threadIdx.x % TPR;
  const T* const x = static_cast<const T*>(a.x);
  const T* const res = static_cast<const T*>(a.residual);
  const W* const weight = static_cast<const W*>(a.weight);
  const int cols = static_cast<int>(a.cols);
  const double per_col = 1.0 / cols;
  const size_t step = static_cast<size_t>(gridDim.x) * kRows;
  size_t row = static_cast<size_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  Packed8<T> h[NCH], r[NCH];
  Packed8<W> w[NCH];
  auto request = [&](size_t from) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * 8, n = from < a.rows ? cols - col : 0;
      h[c] = load_packed<kWhole>(x + from * a.ldx + col, n);
      if (res) r[c] = load_packed<kWhole>(res + from * a.ldr + col, n);
    }
  };
  // whether chunk c of the whole wave lies behind the end of the rows
  const int first = __builtin_amdgcn_readfirstlane(t);
  auto behind = [&](int c) { return NCH > 1 && (c * TPR + first) * 8 >= cols; };
  request(row);
#pragma unroll
  for (int c = 0; c < NCH; ++c) w[c] = load_packed<kWhole>(weight + (c * TPR + t) * 8, cols - (c * TPR + t) * 8);
  for (size_t row0 = static_cast<size_t>(blockIdx.x) * kRows; row0 < a.rows; row0 += step, row += step) {
    const bool live = row < a.rows;
    Packed8<T> sums[NCH];
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * 8;
      sums[c] = h[c];
      if (behind(c)) continue;
      if (res) {
        sums[c] = add_eight(h[c], r[c]);
        store_packed<kWhole>(static_cast<T*>(a.h) + row * a.ldh + col, live ? cols - col : 0, sums[c]);
      }
      sum = add_squares(sums[c], sum);
    }
    if (row0 + step < a.rows) request(row + step);
    sum = row_sum<TPR>(sum, slot);
    const double rstd = inverse_sqrt(sum * per_col + a.eps);
    const float rstd32 = static_cast<float>(rstd);
    const unsigned low = low_below(rstd32);
    if (live && t == 0 && a.rstd) a.rstd[row] = rstd32;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * 8;
      if (behind(c)) continue;
      keep_packed(sums[c]);
      keep_packed(w[c]);
      norm_eight<kWhole>(a, row, col, live ? cols - col : 0, sums[c], w[c], rstd, rstd32, low);
    }
  }
}

// Rows longer than the registers of a block hold: h is read again for y.
template <class T, class W>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(NormArgs a) {
  __shared__ double slot[16];
  const T* const res = static_cast<const T*>(a.residual);
  const int cols = static_cast<int>(a.cols);
  const double per_col = 1.0 / cols;
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const xr = static_cast<const T*>(a.x) + row * a.ldx;
    T* const hr = static_cast<T*>(a.h) + row * a.ldh;
    double sum = 0.0;
    for (int col = threadIdx.x * 8; col < cols; col += 8192) {
      Packed8<T> h = load_packed<false>(xr + col, cols - col);
      if (res) {
        h = add_eight(h, load_packed<false>(res + row * a.ldr + col, cols - col));
        store_packed<false>(hr + col, cols - col, h);
      }
      sum = add_squares(h, sum);
    }
    sum = row_sum<1024>(sum, slot);
    const double rstd = inverse_sqrt(sum * per_col + a.eps);
    const float rstd32 = static_cast<float>(rstd);
    const unsigned low = low_below(rstd32);
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd32;
    const int end = (cols + 8191) / 8192 * 8192;  // whole waves: a block's lanes look at each other
    for (int col = threadIdx.x * 8; col < end; col += 8192) {
      const Packed8<T> h = load_packed<false>((res ? static_cast<const T*>(hr) : xr) + col, cols - col);
      const Packed8<W> w = load_packed<false>(static_cast<const W*>(a.weight) + col, cols - col);
      norm_eight<false>(a, row, col, cols - col, h, w, rstd, rstd32, low);
    }
  }
}

template <class T, class W, bool kWhole> void launch_norm(const NormArgs& a, hipStream_t stream) {
  // per_cu: blocks a CU holds. More of them would hide more, but each loads the weight for fewer rows: 4 of 256
  // threads against 8 take 10.3 us and 11.8 for 1031 x 5003 (16-bit, no residual), 24.2 and 25.4 for
  // 4096 x 4096. Rows of 8192 over 256 threads are too long a chain when there are few of them (1031 rows
  // 16.9 us, over 1024 threads 14.4; 16384 rows 172.9 and 172.1), those of 16384 over 512 threads likewise
  // (30.5 and 28.9; 4096 rows 88.1 and 85.5).
  auto go = [&](auto kernel, int threads, int rows_per_block, int per_cu) {
    const size_t blocks = (a.rows + rows_per_block - 1) / rows_per_block;
    const size_t cap = static_cast<size_t>(streaming_grid(per_cu));
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min(blocks, cap))), dim3(threads), 0, stream, a);
  };
  if (a.cols <= 128) go(rms_norm_kernel<T, W, 16, 1, kWhole>, 256, 16, 8);
  else if (a.cols <= 256) go(rms_norm_kernel<T, W, 32, 1, kWhole>, 256, 8, 8);
  else if (a.cols <= 512) go(rms_norm_kernel<T, W, 64, 1, kWhole>, 256, 4, 8);
  else if (a.cols <= 1024) go(rms_norm_kernel<T, W, 64, 2, kWhole>, 256, 4, 4);
  else if constexpr (sizeof(T) == 2) {
    if (a.cols <= 2048) go(rms_norm_kernel<T, W, 64, 4, kWhole>, 256, 4, 4);
    else if (a.cols <= 4096) go(rms_norm_kernel<T, W, 256, 2, kWhole>, 256, 1, 4);
    else if (a.cols <= 6144) go(rms_norm_kernel<T, W, 256, 3, kWhole>, 256, 1, 4);
    else if (a.cols <= 8192) go(rms_norm_kernel<T, W, 1024, 1, kWhole>, 1024, 1, 2);
    else if (a.cols <= 16384) go(rms_norm_kernel<T, W, 1024, 2, kWhole>, 1024, 1, 1);
    else go(rms_norm_long_kernel<T, W>, 1024, 1, 2);
  } else {
    if (a.cols <= 2048) go(rms_norm_kernel<T, W, 256, 1, kWhole>, 256, 1, 4);
    else if (a.cols <= 4096) go(rms_norm_kernel<T, W, 512, 1, kWhole>, 512, 1, 2);
    else if (a.cols <= 8192) go(rms_norm_kernel<T, W, 512, 2, kWhole>, 512, 1, 2);
    else if (a.cols <= 16384) go(rms_norm_kernel<T, W, 1024, 2, kWhole>, 1024, 1, 1);
    else go(rms_norm_long_kernel<T, W>, 1024, 1, 2);
  }
  TK8S_HIP_CHECK(hipGetLastError());
}

template <class T, class W> void launch_norm(const NormArgs& a, hipStream_t stream) {
  a.cols % 8 == 0 ? launch_norm<T, W, true>(a, stream) : launch_norm<T, W, false>(a, stream);
}

// ------------------------------------------------------------------------------------------
// Backward: xh = h * rstd, g = dy * w, c = mean(g * xh); dx = rstd * (g - xh * c) + dh;
// dw = sum over rows of dy * xh
// ------------------------------------------------------------------------------------------
// dx of 8 columns.
template <bool kWhole, class T, class W>
__device__ __forceinline__ void store_dx(const NormBackwardArgs& a, size_t row, int col, int n, const Packed8<T>& dy, const Packed8<T>& h,
                                         const Packed8<W>& w, const Packed8<T>& dh, float rstd, float mean) {
  float d[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = rstd * fmaf(-(unpack(h, j) * rstd), mean, unpack(dy, j) * unpack(w, j));
    d[j] = a.dh ? unpack(dh, j) + v : v;
  }
  Packed8<T> o;
#pragma unroll
  for (int j = 0; j < 4; ++j) pack(o, j, d[2 * j], d[2 * j + 1]);
  store_packed<kWhole>(static_cast<T*>(a.dx) + row * a.lddx + col, n, o);
}

// Threads of a block whose rows take `threads` each: short rows share one, so that a CU makes one partial row.
constexpr int backward_block(int threads) { return threads <= 64 ? 512 : threads; }

// A block walks rows b, b + G, ...; a thread owns the same columns in all of them and sums its part of
// dw in registers, so dw costs G partial rows instead of a second pass over dy and h. The next row is
// requested before the sum over this one is waited for. 16384 x 8192, 16-bit, with dh: 177 us with the sum
// of the partial rows (5), 6.1 TB/s, which HBM bounds.
template <class T, class W, int TPR, int NCH, bool kWhole>
__global__ __launch_bounds__(backward_block(TPR)) void rms_norm_backward_kernel(NormBackwardArgs a) {
  constexpr int kThreads = backward_block(TPR), kRows = kThreads / TPR;
  __shared__ float slot[kThreads / 64];
  const int t = threadIdx.x % TPR;
  const size_t step = static_cast<size_t>(gridDim.x) * kRows, row0 = static_cast<size_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  const int cols = static_cast<int>(a.cols);
  const float per_col = 1.f / cols;
  Packed8<W> w[NCH];
  Packed8<T> dy[NCH], h[NCH], dh[NCH];
  float dw[NCH][8], rstd = 0.f;
  const int first = __builtin_amdgcn_readfirstlane(t);
  auto behind = [&](int c) { return NCH > 1 && (c * TPR + first) * 8 >= cols; };
  auto request = [&](size_t row) {
    if (row >= a.rows) return;
    rstd = a.rstd[row];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * 8, n = cols - col;
      dy[c] = load_packed<kWhole>(static_cast<const T*>(a.dy) + row * a.lddy + col, n);
      h[c] = load_packed<kWhole>(static_cast<const T*>(a.h) + row * a.ldh + col, n);
      if (a.dh) dh[c] = load_packed<kWhole>(static_cast<const T*>(a.dh) + row * a.lddh + col, n);
    }
  };
  constexpr bool kAhead = sizeof(T) * NCH <= 4;  // more would not fit the registers
  if (kAhead) request(row0);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    w[c] = load_packed<kWhole>(static_cast<const W*>(a.weight) + (c * TPR + t) * 8, cols - (c * TPR + t) * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[c][j] = 0.f;
  }
  for (size_t row = row0; row < a.rows; row += step) {
    if (!kAhead) request(row);
    Packed8<T> dy0[NCH], h0[NCH], dh0[NCH];
    const float rstd0 = rstd;
    float inner = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      dy0[c] = dy[c];
      h0[c] = h[c];
      dh0[c] = dh[c];
      if (behind(c)) continue;
      keep_packed(w[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float g = unpack(dy0[c], j), xh = unpack(h0[c], j) * rstd0;
        dw[c][j] = fmaf(g, xh, dw[c][j]);
        inner = fmaf(g * unpack(w[c], j), xh, inner);
      }
    }
    if (kAhead) request(row + step);
    const float mean = row_sum<TPR>(inner, slot) * per_col;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + t) * 8;
      if (behind(c)) continue;
      keep_packed(dy0[c]);
      keep_packed(h0[c]);
      keep_packed(w[c]);
      store_dx<kWhole>(a, row, col, cols - col, dy0[c], h0[c], w[c], dh0[c], rstd0, mean);
    }
  }
  float* const part = a.workspace + static_cast<size_t>(blockIdx.x) * a.cols;
  if constexpr (kRows > 1) {  // one partial row for the block's rows, added in order
    __shared__ float rows[kRows][TPR * NCH * 8];
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) rows[threadIdx.x / TPR][(c * TPR + t) * 8 + j] = dw[c][j];
    __syncthreads();
    for (int col = threadIdx.x; col < cols; col += kThreads) {
      float sum = rows[0][col];
#pragma unroll
      for (int i = 1; i < kRows; ++i) sum += rows[i][col];
      part[col] = sum;
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) store_some(part + (c * TPR + t) * 8, cols - (c * TPR + t) * 8, dw[c]);
}

// Rows longer than the registers of a block hold: dy and h are read again for dx, and the partial sums
// of dw stay in the block's own row of the workspace.
template <class T, class W>
__global__ __launch_bounds__(1024) void rms_norm_backward_long_kernel(NormBackwardArgs a) {
  __shared__ float slot[16];
  const int cols = static_cast<int>(a.cols);
  float* const part = a.workspace + static_cast<size_t>(blockIdx.x) * a.cols;
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const dyr = static_cast<const T*>(a.dy) + row * a.lddy;
    const T* const hr = static_cast<const T*>(a.h) + row * a.ldh;
    const float rstd = a.rstd[row];
    float inner = 0.f;
    for (int col = threadIdx.x * 8; col < cols; col += 8192) {
      const Packed8<T> dy = load_packed<false>(dyr + col, cols - col), h = load_packed<false>(hr + col, cols - col);
      const Packed8<W> w = load_packed<false>(static_cast<const W*>(a.weight) + col, cols - col);
      float dw[8];
      load8(part + col, row == blockIdx.x ? 0 : cols - col, dw);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xh = unpack(h, j) * rstd;
        dw[j] = fmaf(unpack(dy, j), xh, dw[j]);
        inner = fmaf(unpack(dy, j) * unpack(w, j), xh, inner);
      }
      store_some(part + col, cols - col, dw);
    }
    const float mean = row_sum<1024>(inner, slot) / cols;
    for (int col = threadIdx.x * 8; col < cols; col += 8192) {
      const int n = cols - col;
      Packed8<T> dh = {};
      if (a.dh) dh = load_packed<false>(static_cast<const T*>(a.dh) + row * a.lddh + col, n);
      store_dx<false>(a, row, col, n, load_packed<false>(dyr + col, n), load_packed<false>(hr + col, n),
                      load_packed<false>(static_cast<const W*>(a.weight) + col, n), dh, rstd, mean);
    }
  }
}

// Sums kSumCols columns over `rows` rows in 32 interleaved slices, then the slices in order: the same bits on
// every run. value(row, col) is what is summed; out(col, sum) takes the result.
constexpr int kSumCols = 32, kSlices = 1024 / kSumCols;
template <class F, class O> __device__ __forceinline__ void sum_columns(size_t rows, size_t cols, size_t col0, F value, O out) {
  __shared__ float slices[kSlices][kSumCols];
  const int at = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
  const size_t col = col0 + at;
  float s = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (size_t r = slice; r < rows; r += kSlices) s += value(r, col);
  }
  slices[slice][at] = s;
  __syncthreads();
  if (slice == 0 && col < cols) {
    s = slices[0][at];
#pragma unroll
    for (int i = 1; i < kSlices; ++i) s += slices[i][at];
    out(col, s);
  }
}

constexpr size_t kSumBlocks = size_t(1) << 20;  // at most: a launch has fewer than 2^32 threads

__global__ __launch_bounds__(1024) void column_sum_kernel(const float* part, size_t rows, size_t cols, float* dw) {
  for (size_t col0 = static_cast<size_t>(blockIdx.x) * kSumCols; col0 < cols; col0 += static_cast<size_t>(gridDim.x) * kSumCols) {
    sum_columns(rows, cols, col0, [&](size_t r, size_t c) { return part[r * cols + c]; }, [&](size_t c, float s) { dw[c] = s; });
    __syncthreads();  // the slices have been read
  }
}

// Few rows: one launch. The first blocks make dx, a row each; the others dw, kSumCols columns each, from dy and
// h themselves (they are in the caches). 37 x 4096, 32-bit: 5.9 us a call, 9.6 with a second launch for dw.
template <class T, class W>
__global__ __launch_bounds__(1024) void rms_norm_backward_few_kernel(NormBackwardArgs a) {
  if (blockIdx.x >= a.rows) {
    const T* const dy = static_cast<const T*>(a.dy);
    const T* const h = static_cast<const T*>(a.h);
    sum_columns(a.rows, a.cols, (blockIdx.x - a.rows) * kSumCols,
                [&](size_t r, size_t c) {
                  return static_cast<float>(dy[r * a.lddy + c]) * (static_cast<float>(h[r * a.ldh + c]) * a.rstd[r]);
                },
                [&](size_t c, float s) { a.dw[c] = s; });
    return;
  }
  __shared__ float slot[16];
  const size_t row = blockIdx.x;
  const int cols = static_cast<int>(a.cols), col0 = threadIdx.x * 8;
  const float rstd = a.rstd[row];
  Packed8<T> dy[2], h[2], dh[2];
  Packed8<W> w[2];
  float inner = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = col0 + c * 8192, n = cols - col;
    dy[c] = load_packed<false>(static_cast<const T*>(a.dy) + row * a.lddy + col, n);
    h[c] = load_packed<false>(static_cast<const T*>(a.h) + row * a.ldh + col, n);
    w[c] = load_packed<false>(static_cast<const W*>(a.weight) + col, n);
    if (a.dh) dh[c] = load_packed<false>(static_cast<const T*>(a.dh) + row * a.lddh + col, n);
#pragma unroll
    for (int j = 0; j < 8; ++j) inner = fmaf(unpack(dy[c], j) * unpack(w[c], j), unpack(h[c], j) * rstd, inner);
  }
  const float mean = row_sum<1024>(inner, slot) / cols;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = col0 + c * 8192;
    store_dx<false>(a, row, col, cols - col, dy[c], h[c], w[c], dh[c], rstd, mean);
  }
}

constexpr size_t kFewRows = 512, kFewCols = 16384;
bool few(size_t rows, size_t cols) { return rows <= kFewRows && cols <= kFewCols; }

// Threads of a row.
int backward_threads(size_t cols) { return cols <= 128 ? 16 : cols <= 256 ? 32 : cols <= 1024 ? 64 : cols <= 2048 ? 256 : cols <= 2560 ? 320 : cols <= 4096 ? 512 : 1024; }
// Blocks: enough for the loads of two rows a CU of the widest to be on their way, of narrower ones more, and few
// enough for the weight, the partial rows and their sum to cost little next to dy and h (600 x 8192: 512 blocks
// 22.6 us, 256 15.8; 16384 x 8192: 177 and 183; 11638 x 4096, 32-bit: 727 blocks 154, 640 165, 364 180; 20000 x
// 2048, 16-bit: 512 blocks 59, 640 65; 5000 x 5000: 312 blocks 58, 256 43).
size_t backward_grid(size_t rows, size_t cols) {
  const int threads = backward_threads(cols);
  const size_t at_once = static_cast<size_t>(backward_block(threads) / threads), sets = (rows + at_once - 1) / at_once;
  const size_t most = at_once > 1   ? 512
                      : cols > 4096 ? (sets / 32 >= 512 ? 512 : 256)
                                    : std::clamp<size_t>(sets / 16, 256, threads > 256 ? 768 : 512);
  return std::min(sets, most);
}

template <class T, class W, bool kWhole> void launch_backward_rows(const NormBackwardArgs& a, unsigned grid, hipStream_t stream) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(backward_block(backward_threads(a.cols))), 0, stream, a);
  };
  if (a.cols <= 128) go(rms_norm_backward_kernel<T, W, 16, 1, kWhole>);
  else if (a.cols <= 256) go(rms_norm_backward_kernel<T, W, 32, 1, kWhole>);
  else if (a.cols <= 512) go(rms_norm_backward_kernel<T, W, 64, 1, kWhole>);
  else if (a.cols <= 1024) go(rms_norm_backward_kernel<T, W, 64, 2, kWhole>);
  else if (a.cols <= 2048) go(rms_norm_backward_kernel<T, W, 256, 1, kWhole>);
  else if (a.cols <= 2560) go(rms_norm_backward_kernel<T, W, 320, 1, kWhole>);
  else if (a.cols <= 4096) go(rms_norm_backward_kernel<T, W, 512, 1, kWhole>);
  else if (a.cols <= 8192) go(rms_norm_backward_kernel<T, W, 1024, 1, kWhole>);
  else if (a.cols <= 16384) go(rms_norm_backward_kernel<T, W, 1024, 2, kWhole>);
  else go(rms_norm_backward_long_kernel<T, W>);
}

template <class T, class W> void launch_backward(const NormBackwardArgs& a, hipStream_t stream) {
  const size_t sums = (a.cols + kSumCols - 1) / kSumCols;
  if (few(a.rows, a.cols)) {
    hipLaunchKernelGGL((rms_norm_backward_few_kernel<T, W>), dim3(static_cast<unsigned>(a.rows + sums)), dim3(1024), 0, stream, a);
  } else {
    const unsigned grid = static_cast<unsigned>(backward_grid(a.rows, a.cols));
    if (a.cols % 8 == 0) launch_backward_rows<T, W, true>(a, grid, stream);
    else launch_backward_rows<T, W, false>(a, grid, stream);
    TK8S_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(column_sum_kernel, dim3(static_cast<unsigned>(std::min(sums, kSumBlocks))), dim3(1024), 0, stream, a.workspace,
                       static_cast<size_t>(grid), a.cols, a.dw);
  }
  TK8S_HIP_CHECK(hipGetLastError());
}

// ------------------------------------------------------------------------------------------
// Rounding to 8 bits
// ------------------------------------------------------------------------------------------
// One layout, a scale for 128 columns of a row: 16 lanes hold a block, 8 columns each. One row of 8192: 2.6 us,
// latency; 9864 x 1536, 16-bit: 10.0 us, 4.5 TB/s, HBM.
template <class T, bool kWhole>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
  const unsigned blocks = static_cast<unsigned>((a.cols + kScaleBlock - 1) / kScaleBlock);
  const size_t items = a.rows * blocks, step = static_cast<size_t>(gridDim.x) * 16;
  const int c = threadIdx.x % 16 * 8;
  for (size_t first = static_cast<size_t>(blockIdx.x) * 16; first < items; first += step) {  // a block's lanes stay together
    const size_t item = first + threadIdx.x / 16;
    const size_t row = items >> 32 ? item / blocks : static_cast<unsigned>(item) / blocks;
    const size_t block = item - row * blocks, col = block * kScaleBlock + c;
    const int n = item < items && a.cols > col ? static_cast<int>(std::min<size_t>(a.cols - col, 8)) : 0;
    const Packed8<T> v = load_packed<kWhole, T, false>(static_cast<const T*>(a.x) + row * a.ldx + col, n);
    const unsigned byte = scale_byte(max16(largest_of(magnitudes(v))));
    store_bytes<kWhole>(a.rows_out.values + row * a.rows_out.ld + col, n, u32x2{pack_four(v, 0, byte), pack_four(v, 1, byte)});
    if (n > 0 && c == 0) a.rows_out.scales[block * a.rows_out.ld_scales + row] = static_cast<uint8_t>(byte);
  }
}

// n bytes, one of each of v[0..7]'s low bytes, to where they belong.
__device__ __forceinline__ void store_scales(uint8_t* p, int n, const unsigned (&v)[8]) {
  struct __attribute__((packed, aligned(1))) Any { u32x2 v; };
  const u32x2 b = {v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24, v[4] | v[5] << 8 | v[6] << 16 | v[7] << 24};
  if (n >= 8) {
    reinterpret_cast<Any*>(p)->v = b;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = static_cast<uint8_t>(v[j]);
  }
}

// All layouts from one read: a block of 256 threads holds a 128 x 128 tile in registers as it is stored,
// thread t the columns 8 (t % 16) .. + 7 of rows 8 (t / 16) .. + 7. A row's largest magnitude is over 16
// lanes, a column's over the thread's 8 rows, the wave's 4 groups of lanes and the 4 waves. The
// transposed bytes, 8 rows of a column at a time, go through LDS so that both writes are whole
// lines; piece p of a transposed row lies at p ^ (row / 8), which spreads a wave's writes over the banks.
// 10007 x 8192, 16-bit, both layouts: 59 us, 5.5 TB/s, HBM.
constexpr int kTile = 128;

template <class T, bool kWhole>
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a) {
  __shared__ unsigned col_top[4][16][2 * sizeof(T)];
  __shared__ unsigned tile_top[4];
  __shared__ __attribute__((aligned(16))) u32x2 turned[kTile][16];
  const int t = threadIdx.x, lane = t % 64, wave = t / 64, c = t % 16 * 8, r = t / 16 * 8;
  const size_t tiles_c = (a.cols + kTile - 1) / kTile, tiles_r = (a.rows + kTile - 1) / kTile;
  for (size_t tile = blockIdx.x; tile < tiles_c * tiles_r; tile += gridDim.x) {
    const size_t tile_r = (tiles_c * tiles_r) >> 32 ? tile / tiles_c : static_cast<unsigned>(tile) / static_cast<unsigned>(tiles_c);
    const size_t r0 = tile_r * kTile, c0 = (tile - tile_r * tiles_c) * kTile;
    const int n = a.cols > c0 + c ? static_cast<int>(std::min<size_t>(a.cols - c0 - c, 8)) : 0;
    const int m = a.rows > r0 + r ? static_cast<int>(std::min<size_t>(a.rows - r0 - r, 8)) : 0;
    const T* const x = static_cast<const T*>(a.x) + (r0 + r) * a.ldx + c0 + c;
    Packed8<T> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_packed<kWhole, T, false>(x + i * a.ldx, i < m ? n : 0);
    if (a.rows_out.values) {
      unsigned bytes[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bytes[i] = scale_byte(max16(largest_of(magnitudes(v[i]))));
        store_bytes<kWhole>(a.rows_out.values + (r0 + r + i) * a.rows_out.ld + c0 + c, i < m ? n : 0,
                            u32x2{pack_four(v[i], 0, bytes[i]), pack_four(v[i], 1, bytes[i])});
      }
      if (c == 0) store_scales(a.rows_out.scales + c0 / kScaleBlock * a.rows_out.ld_scales + r0 + r, m, bytes);
    }
    Packed8<T> top = magnitudes(v[0]);  // the largest of each of the thread's columns
#pragma unroll
    for (int i = 1; i < 8; ++i) top = larger(top, magnitudes(v[i]));
    if (a.tiles_out.values) {
      unsigned all = max16(largest_of(top));
      all = max(all, static_cast<unsigned>(__shfl_xor(all, 16, 64)));
      all = max(all, static_cast<unsigned>(__shfl_xor(all, 32, 64)));
      if (lane == 0) tile_top[wave] = all;
      __syncthreads();
      const unsigned byte = scale_byte(max(max(tile_top[0], tile_top[1]), max(tile_top[2], tile_top[3])));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        store_bytes<kWhole>(a.tiles_out.values + (r0 + r + i) * a.tiles_out.ld + c0 + c, i < m ? n : 0,
                            u32x2{pack_four(v[i], 0, byte), pack_four(v[i], 1, byte)});
      if (t == 0) a.tiles_out.scales[c0 / kTile * a.tiles_out.ld_scales + r0 / kTile] = static_cast<uint8_t>(byte);
    }
    if (a.cols_out.values) {
#pragma unroll
      for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) {
        top.d[i] = larger<T>(top.d[i], __shfl_xor(top.d[i], 16, 64));
        top.d[i] = larger<T>(top.d[i], __shfl_xor(top.d[i], 32, 64));
        if (lane < 16) col_top[wave][lane][i] = top.d[i];
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) top.d[i] = larger<T>(top.d[i], col_top[w][t % 16][i]);
      unsigned bytes[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bytes[j] = scale_byte(magnitude_of(top, j));
        const Packed8<T> col = column(v, j);
        turned[c + j][(r / 8) ^ (c / 8)] = u32x2{pack_four(col, 0, bytes[j]), pack_four(col, 1, bytes[j])};
      }
      if (r == 0) store_scales(a.cols_out.scales + r0 / kScaleBlock * a.cols_out.ld_scales + c0 + c, n, bytes);
      __syncthreads();
      // thread t: bytes 16 (t % 8) .. + 15 of transposed rows t / 8 + 32 i
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tr = t / 8 + 32 * i, p = t % 8 * 2;
        if (c0 + tr >= a.cols || r0 + 8 * p >= a.rows) continue;
        const u32x2 low = turned[tr][p ^ (tr / 8)], high = turned[tr][(p + 1) ^ (tr / 8)];
        uint8_t* const q = a.cols_out.values + (c0 + tr) * a.cols_out.ld + r0 + 8 * p;
        const int left = static_cast<int>(std::min<size_t>(a.rows - r0 - 8 * p, 16));
        if (left == 16) {
          *reinterpret_cast<u32x4*>(q) = u32x4{low.x, low.y, high.x, high.y};
        } else {
          store_bytes<false>(q, left, low);
          store_bytes<false>(q + 8, left - 8, high);
        }
      }
    }
    __syncthreads();  // the tile's shared memory is free for the next one
  }
}

template <class T> void launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  const bool whole = a.cols % 8 == 0;
  auto go = [&](auto kernel, size_t blocks, size_t cap) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min(blocks, cap))), dim3(256), 0, stream, a);
  };
  if (!a.cols_out.values && !a.tiles_out.values) {
    if (!a.rows_out.values) return;
    const size_t blocks = (a.rows * ((a.cols + kScaleBlock - 1) / kScaleBlock) + 15) / 16, cap = size_t(1) << 22;
    whole ? go(quantize_rows_kernel<T, true>, blocks, cap) : go(quantize_rows_kernel<T, false>, blocks, cap);
  } else {
    const size_t tiles = (a.rows + kTile - 1) / kTile * ((a.cols + kTile - 1) / kTile), cap = size_t(1) << 22;
    whole ? go(quantize_kernel<T, true>, tiles, cap) : go(quantize_kernel<T, false>, tiles, cap);
  }
  TK8S_HIP_CHECK(hipGetLastError());
}

// 8 values a thread, each of 8 bits of a 64-bit mix of their number (splitmix64's finaliser, by S. Vigna).
__global__ __launch_bounds__(256) void layer_fill_kernel(uint4* dst, size_t eights, uint64_t seed) {
  for (size_t i = blockIdx.x * size_t(256) + threadIdx.x; i < eights; i += static_cast<size_t>(gridDim.x) * 256) {
    uint64_t z = (seed + 1) * 0x9e3779b97f4a7c15ull + i * 0xd1342543de82ef95ull;
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    z ^= z >> 31;
    unsigned v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = static_cast<float>(static_cast<int>(z >> (16 * j) & 255u) - 128) * (1.f / 32);
      const float hi = static_cast<float>(static_cast<int>(z >> (16 * j + 8) & 255u) - 128) * (1.f / 32);
      v[j] = __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xffff0000u);  // 8 significant bits: exact
    }
    dst[i] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

void check(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

void check_out(const Fp8Matrix& m, const char* what) {
  if (!m.values) return;
  check(m.scales != nullptr, what);
  check(aligned(m.values, 16) && m.ld % 16 == 0, "fp8: the rows of 8-bit values must start on 16-byte boundaries");
}

}  // namespace

void rms_norm_fp8(const NormArgs& a, LayerType type, LayerType weight_type, hipStream_t stream) {
  check(a.cols <= (1u << 30), "rms_norm_fp8: at most 2^30 columns");
  check(weight_type == type || weight_type == LayerType::kF32, "rms_norm_fp8: the weight is of x's type or float32");
  if (a.rows == 0 || (a.cols == 0 && !a.rstd)) return;  // rows of no columns: their rstd is NaN
  check(a.cols == 0 || (a.x && a.weight), "rms_norm_fp8: x and weight are needed");
  check(!a.residual || a.h || a.cols == 0, "rms_norm_fp8: a residual needs h, where the sum is stored");
  check(!a.q || a.scales, "rms_norm_fp8: 8-bit values need scales");
  check(!a.q || (aligned(a.q, 16) && a.ldq % 16 == 0), "fp8: the rows of 8-bit values must start on 16-byte boundaries");
  const bool wide = weight_type == LayerType::kF32;
  switch (type) {
    case LayerType::kF32: return launch_norm<float, float>(a, stream);
    case LayerType::kBF16: return wide ? launch_norm<__bf16, float>(a, stream) : launch_norm<__bf16, __bf16>(a, stream);
    case LayerType::kF16: return wide ? launch_norm<_Float16, float>(a, stream) : launch_norm<_Float16, _Float16>(a, stream);
  }
}

size_t rms_norm_backward_workspace(size_t rows, size_t cols) {
  return few(rows, cols) ? 0 : backward_grid(rows, cols) * cols * sizeof(float);
}

void rms_norm_backward(const NormBackwardArgs& a, LayerType type, LayerType weight_type, hipStream_t stream) {
  check(a.cols <= (1u << 30), "rms_norm_backward: at most 2^30 columns");
  check(weight_type == type || weight_type == LayerType::kF32, "rms_norm_backward: the weight is of h's type or float32");
  check(a.rows > 0, "rms_norm_backward: no rows");
  if (a.cols == 0) return;
  check(a.dy && a.h && a.weight && a.rstd && a.dx && a.dw && (a.workspace || few(a.rows, a.cols)),
        "rms_norm_backward: a pointer is missing");
  const bool wide = weight_type == LayerType::kF32;
  switch (type) {
    case LayerType::kF32: return launch_backward<float, float>(a, stream);
    case LayerType::kBF16: return wide ? launch_backward<__bf16, float>(a, stream) : launch_backward<__bf16, __bf16>(a, stream);
    case LayerType::kF16: return wide ? launch_backward<_Float16, float>(a, stream) : launch_backward<_Float16, _Float16>(a, stream);
  }
}

void fp8_quantize(const QuantizeArgs& a, LayerType type, hipStream_t stream) {
  check_out(a.rows_out, "fp8_quantize: row-scaled values need scales");
  check_out(a.cols_out, "fp8_quantize: column-scaled values need scales");
  check_out(a.tiles_out, "fp8_quantize: tile-scaled values need scales");
  if (a.rows == 0 || a.cols == 0) return;
  check(a.x != nullptr, "fp8_quantize: x is needed");
  switch (type) {
    case LayerType::kF32: return launch_quantize<float>(a, stream);
    case LayerType::kBF16: return launch_quantize<__bf16>(a, stream);
    case LayerType::kF16: return launch_quantize<_Float16>(a, stream);
  }
}

void layer_fill(void* dst, size_t count, uint64_t seed, hipStream_t stream) {
  check(count % 8 == 0, "layer_fill: the number of values must be a multiple of 8");
  if (count == 0) return;
  const size_t blocks = (count / 8 + 255) / 256;
  hipLaunchKernelGGL(layer_fill_kernel, dim3(static_cast<unsigned>(std::min<size_t>(blocks, static_cast<size_t>(streaming_grid())))), dim3(256), 0,
                     stream, static_cast<uint4*>(dst), count / 8, seed);
  TK8S_HIP_CHECK(hipGetLastError());
}

}  // namespace tk8s
