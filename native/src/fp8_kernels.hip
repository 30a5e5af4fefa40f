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

// Sum over the TPR threads of a row (TPR consecutive threads; whole waves). `slot`: one double per
// wave. Every thread of the block calls it when TPR > 64.
template <int TPR, class V>
__device__ __forceinline__ V row_sum(V v, V* slot) {
#pragma unroll
  for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (TPR > 64) {
    constexpr int kWaves = TPR / 64;
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) slot[wave] = v;
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
// A row belongs to TPR threads; thread t holds chunks c of 8 values at (c * TPR + t) * 8, so 16
// neighbouring lanes hold exactly one block of 128. Sum of squares, rstd and y are in 64 bits: a
// value next to the border of two e4m3 ones then falls where the formula puts it (the vector
// units run 64-bit FMAs at the rate of 32-bit ones), and the result is rounded once.
// NCH = 0: rows of any length; the values are read again instead of held.
template <class T, class W, int TPR, int NCH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(NormArgs a) {
  constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
  __shared__ double slot[TPR < 64 ? 1 : TPR / 64 * kRows];
  const int t = threadIdx.x % TPR;
  const T* const x = static_cast<const T*>(a.x);
  const T* const res = static_cast<const T*>(a.residual);
  const W* const weight = static_cast<const W*>(a.weight);
  const int cols = static_cast<int>(a.cols);
  const int chunks = NCH ? NCH : (cols + TPR * 8 - 1) / (TPR * 8);
  for (size_t row0 = static_cast<size_t>(blockIdx.x) * kRows; row0 < a.rows; row0 += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const T* const xr = x + row * a.ldx;
    const T* const rr = res + row * a.ldr;
    T* const hr = static_cast<T*>(a.h) + row * a.ldh;
    float h[NCH ? NCH : 1][8];
    double sum = 0.0;
    for (int c = 0; c < chunks; ++c) {
      float(&v)[8] = h[NCH ? c : 0];
      const int col = (c * TPR + t) * 8;
      const int n = live ? cols - col : 0;
      load8(xr + col, n, v);
      if (res) {
        float r[8];
        load8(rr + col, n, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<T>(v[j] + r[j]));
        store8(hr + col, n, v);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma(static_cast<double>(v[j]), static_cast<double>(v[j]), sum);
    }
    sum = row_sum<TPR>(sum, slot);
    const double rstd = 1.0 / sqrt(sum / cols + a.eps);
    if (live && t == 0 && a.rstd) a.rstd[row] = static_cast<float>(rstd);
    for (int c = 0; c < chunks; ++c) {
      float(&v)[8] = h[NCH ? c : 0];
      const int col = (c * TPR + t) * 8;
      const int n = live ? cols - col : 0;
      if (!NCH) {  // the stored sum, or x itself
        if (res) load8(static_cast<const T*>(hr) + col, n, v);
        else load8(xr + col, n, v);
      }
      float w[8], y[8];
      load8(weight + col, n, w);
      unsigned top = 0;
      double y64[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y64[j] = static_cast<double>(v[j]) * rstd * static_cast<double>(w[j]);
        y[j] = round_to_odd(y64[j]);
        const unsigned m = j < n ? magnitude_bits(y[j]) : 0u;
        top = m > top ? m : top;
      }
      if (a.y) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = sizeof(T) == 4 ? static_cast<float>(y64[j]) : y[j];
        store8(static_cast<T*>(a.y) + row * a.ldy + col, n, o);
      }
      if (a.q) {
        top = max16(top);
        const unsigned byte = scale_byte(top);
        const u32x2 p = {pack4(y[0], y[1], y[2], y[3], byte), pack4(y[4], y[5], y[6], y[7], byte)};
        uint8_t* const qr = a.q + row * a.ldq + col;
        if (n >= 8) {
          *reinterpret_cast<u32x2*>(qr) = p;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < n) qr[j] = static_cast<uint8_t>((j < 4 ? p.x : p.y) >> (8 * (j & 3)));
        }
        if (n > 0 && t % 16 == 0) a.scales[static_cast<size_t>(col / kScaleBlock) * a.lds + row] = static_cast<uint8_t>(byte);
      }
    }
  }
}

template <class T, class W> void launch_norm(const NormArgs& a, hipStream_t stream) {
  auto go = [&](auto kernel, int threads, int rows_per_block) {
    const size_t blocks = (a.rows + rows_per_block - 1) / rows_per_block;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<size_t>(blocks, 1u << 20))), dim3(threads), 0, stream, a);
  };
  if (a.cols <= 512) go(rms_norm_kernel<T, W, 64, 1>, 256, 4);
  else if (a.cols <= 1024) go(rms_norm_kernel<T, W, 64, 2>, 256, 4);
  else if (a.cols <= 2048) go(rms_norm_kernel<T, W, 256, 1>, 256, 1);
  else if (a.cols <= 4096) go(rms_norm_kernel<T, W, 256, 2>, 256, 1);
  else if (a.cols <= 8192) go(rms_norm_kernel<T, W, 256, 4>, 256, 1);
  else if (a.cols <= 16384) go(rms_norm_kernel<T, W, 512, 4>, 512, 1);
  else go(rms_norm_kernel<T, W, 512, 0>, 512, 1);
  TK8S_HIP_CHECK(hipGetLastError());
}

// ------------------------------------------------------------------------------------------
// Backward: xh = h * rstd, g = dy * w, c = mean(g * xh); dx = rstd * (g - xh * c) + dh;
// dw = sum over rows of dy * xh
// ------------------------------------------------------------------------------------------
// A block walks rows b, b + G, ...; a thread owns the same columns in all of them and sums its
// part of dw in registers, so dw costs G partial rows instead of a second pass over dy and h.
// NCH = 0: rows of any length, the partial sums kept in the block's own row of the workspace.
template <class T, class W, int TPR, int NCH>
__global__ __launch_bounds__(TPR) void rms_norm_backward_kernel(NormBackwardArgs a) {
  __shared__ float slot[TPR / 64];
  const int t = threadIdx.x;
  const int cols = static_cast<int>(a.cols);
  const int chunks = NCH ? NCH : (cols + TPR * 8 - 1) / (TPR * 8);
  const W* const weight = static_cast<const W*>(a.weight);
  float* const part = a.workspace + static_cast<size_t>(blockIdx.x) * a.cols;
  float w[NCH ? NCH : 1][8], dw[NCH ? NCH : 1][8];
  if (NCH) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      load8(weight + (c * TPR + t) * 8, cols - (c * TPR + t) * 8, w[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) dw[c][j] = 0.f;
    }
  }
  bool first = true;
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const dyr = static_cast<const T*>(a.dy) + row * a.lddy;
    const T* const hr = static_cast<const T*>(a.h) + row * a.ldh;
    const T* const dhr = static_cast<const T*>(a.dh) + row * a.lddh;
    T* const dxr = static_cast<T*>(a.dx) + row * a.lddx;
    const float rstd = a.rstd[row];
    float dy[NCH ? NCH : 1][8], xh[NCH ? NCH : 1][8];
    float inner = 0.f;
    for (int c = 0; c < chunks; ++c) {
      const int k = NCH ? c : 0, col = (c * TPR + t) * 8, n = cols - col;
      load8(dyr + col, n, dy[k]);
      load8(hr + col, n, xh[k]);
      if (!NCH) {
        load8(weight + col, n, w[0]);
        load8(part + col, first ? 0 : n, dw[0]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[k][j] *= rstd;
        dw[k][j] = fmaf(dy[k][j], xh[k][j], dw[k][j]);
        inner = fmaf(dy[k][j] * w[k][j], xh[k][j], inner);
      }
      if (!NCH) store8(part + col, n, dw[0]);
    }
    first = false;
    const float mean = row_sum<TPR>(inner, slot) / cols;
    for (int c = 0; c < chunks; ++c) {
      const int k = NCH ? c : 0, col = (c * TPR + t) * 8, n = cols - col;
      if (!NCH) {
        load8(dyr + col, n, dy[0]);
        load8(hr + col, n, xh[0]);
        load8(weight + col, n, w[0]);
#pragma unroll
        for (int j = 0; j < 8; ++j) xh[0][j] *= rstd;
      }
      float d[8];
      if (a.dh) load8(dhr + col, n, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = rstd * fmaf(-xh[k][j], mean, dy[k][j] * w[k][j]);
        d[j] = a.dh ? d[j] + v : v;
      }
      store8(dxr + col, n, d);
    }
  }
  if (NCH) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) store8(part + (c * TPR + t) * 8, cols - (c * TPR + t) * 8, dw[c]);
  }
}

// dw[col] = sum of the partial rows, in order: the same bits on every run.
__global__ __launch_bounds__(256) void column_sum_kernel(const float* part, size_t rows, size_t cols, float* out) {
  const size_t col = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (col >= cols) return;
  float s = 0.f;
  for (size_t r = 0; r < rows; ++r) s += part[r * cols + col];
  out[col] = s;
}

size_t backward_grid(size_t rows) { return std::min<size_t>(rows, 512); }

template <class T, class W> void launch_backward(const NormBackwardArgs& a, hipStream_t stream) {
  const unsigned grid = static_cast<unsigned>(backward_grid(a.rows));
  auto go = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, stream, a); };
  if (a.cols <= 2048) go(rms_norm_backward_kernel<T, W, 256, 1>, 256);
  else if (a.cols <= 4096) go(rms_norm_backward_kernel<T, W, 256, 2>, 256);
  else if (a.cols <= 8192) go(rms_norm_backward_kernel<T, W, 256, 4>, 256);
  else if (a.cols <= 16384) go(rms_norm_backward_kernel<T, W, 512, 4>, 512);
  else go(rms_norm_backward_kernel<T, W, 512, 0>, 512);
  TK8S_HIP_CHECK(hipGetLastError());
  hipLaunchKernelGGL(column_sum_kernel, dim3(static_cast<unsigned>((a.cols + 255) / 256)), dim3(256), 0, stream, a.workspace,
                     static_cast<size_t>(grid), a.cols, a.dw);
  TK8S_HIP_CHECK(hipGetLastError());
}

// ------------------------------------------------------------------------------------------
// Rounding to 8 bits
// ------------------------------------------------------------------------------------------
// A block of 256 threads holds a 128 x 128 tile in registers: thread t the columns 8 * (t % 16) ..
// + 7 of rows t / 16 + 16 i. A row's largest magnitude is then over 16 lanes, a column's over the
// thread's own 8 rows, the 4 lane groups of the wave and the 4 waves, and all layouts come from
// one read. The transposed bytes go through LDS so that both writes are whole lines.
constexpr int kTile = 128;
constexpr int kPitch = kTile + 16;  // bytes of a transposed row in LDS

template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a) {
  __shared__ unsigned col_top[4][kTile];
  __shared__ unsigned tile_top[4];
  __shared__ __attribute__((aligned(16))) uint8_t turned[kTile * kPitch];
  const int t = threadIdx.x, lane = t % 64, wave = t / 64;
  const size_t tiles_c = (a.cols + kTile - 1) / kTile, tiles_r = (a.rows + kTile - 1) / kTile;
  for (size_t tile = blockIdx.x; tile < tiles_c * tiles_r; tile += gridDim.x) {
    const size_t r0 = tile / tiles_c * kTile, c0 = tile % tiles_c * kTile;
    const int c = (t % 16) * 8;
    const int n = a.cols - c0 > static_cast<size_t>(c) ? static_cast<int>(std::min<size_t>(a.cols - c0 - c, 8)) : 0;
    float v[8][8];
    unsigned row_top[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const size_t r = r0 + t / 16 + 16 * i;
      load8(static_cast<const T*>(a.x) + r * a.ldx + c0 + c, r < a.rows ? n : 0, v[i]);
      row_top[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) row_top[i] = max(row_top[i], magnitude_bits(v[i][j]));
    }
    if (a.rows_out.values) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const size_t r = r0 + t / 16 + 16 * i;
        const unsigned byte = scale_byte(max16(row_top[i]));
        const u32x2 p = {pack4(v[i][0], v[i][1], v[i][2], v[i][3], byte), pack4(v[i][4], v[i][5], v[i][6], v[i][7], byte)};
        if (r < a.rows) {
          uint8_t* const q = a.rows_out.values + r * a.rows_out.ld + c0 + c;
          if (n == 8) {
            *reinterpret_cast<u32x2*>(q) = p;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j < n) q[j] = static_cast<uint8_t>((j < 4 ? p.x : p.y) >> (8 * (j & 3)));
          }
          if (c == 0) a.rows_out.scales[c0 / kScaleBlock * a.rows_out.ld_scales + r] = static_cast<uint8_t>(byte);
        }
      }
    }
    if (a.tiles_out.values) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, row_top[i]);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) top = max(top, static_cast<unsigned>(__shfl_xor(top, off, 64)));
      if (lane == 0) tile_top[wave] = top;
      __syncthreads();
      const unsigned byte = scale_byte(max(max(tile_top[0], tile_top[1]), max(tile_top[2], tile_top[3])));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const size_t r = r0 + t / 16 + 16 * i;
        const u32x2 p = {pack4(v[i][0], v[i][1], v[i][2], v[i][3], byte), pack4(v[i][4], v[i][5], v[i][6], v[i][7], byte)};
        if (r < a.rows) {
          uint8_t* const q = a.tiles_out.values + r * a.tiles_out.ld + c0 + c;
          if (n == 8) {
            *reinterpret_cast<u32x2*>(q) = p;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j < n) q[j] = static_cast<uint8_t>((j < 4 ? p.x : p.y) >> (8 * (j & 3)));
          }
        }
      }
      if (t == 0) a.tiles_out.scales[c0 / kTile * a.tiles_out.ld_scales + r0 / kTile] = static_cast<uint8_t>(byte);
    }
    if (a.cols_out.values) {
      unsigned top[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top[j] = max(top[j], magnitude_bits(v[i][j]));
        top[j] = max(top[j], static_cast<unsigned>(__shfl_xor(top[j], 16, 64)));
        top[j] = max(top[j], static_cast<unsigned>(__shfl_xor(top[j], 32, 64)));
        if (lane < 16) col_top[wave][c + j] = top[j];
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned byte = scale_byte(max(max(col_top[0][c + j], col_top[1][c + j]), max(col_top[2][c + j], col_top[3][c + j])));
#pragma unroll
        for (int i = 0; i < 8; ++i)
          turned[(c + j) * kPitch + t / 16 + 16 * i] = static_cast<uint8_t>(pack4(v[i][j], 0.f, 0.f, 0.f, byte));
        if (t < 16 && j < n) a.cols_out.scales[r0 / kScaleBlock * a.cols_out.ld_scales + c0 + c + j] = static_cast<uint8_t>(byte);
      }
      __syncthreads();
      // thread t: bytes 16 * (t % 8) .. + 15 of transposed rows t / 8 + 32 i
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tr = t / 8 + 32 * i, b = (t % 8) * 16;
        if (c0 + tr >= a.cols || r0 + b >= a.rows) continue;
        uint8_t* const q = a.cols_out.values + (c0 + tr) * a.cols_out.ld + r0 + b;
        const uint8_t* const s = turned + tr * kPitch + b;
        if (r0 + b + 16 <= a.rows) {
          *reinterpret_cast<u32x4*>(q) = *reinterpret_cast<const u32x4*>(s);
        } else {
          for (int j = 0; r0 + b + j < a.rows; ++j) q[j] = s[j];
        }
      }
    }
    __syncthreads();  // the tile's shared memory is free for the next one
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
  if (a.rows == 0 || a.cols == 0) return;
  check(a.x && a.weight, "rms_norm_fp8: x and weight are needed");
  check(!a.residual || a.h, "rms_norm_fp8: a residual needs h, where the sum is stored");
  check(!a.q || a.scales, "rms_norm_fp8: 8-bit values need scales");
  check(!a.q || (aligned(a.q, 16) && a.ldq % 16 == 0), "fp8: the rows of 8-bit values must start on 16-byte boundaries");
  const bool wide = weight_type == LayerType::kF32;
  switch (type) {
    case LayerType::kF32: return launch_norm<float, float>(a, stream);
    case LayerType::kBF16: return wide ? launch_norm<__bf16, float>(a, stream) : launch_norm<__bf16, __bf16>(a, stream);
    case LayerType::kF16: return wide ? launch_norm<_Float16, float>(a, stream) : launch_norm<_Float16, _Float16>(a, stream);
  }
}

size_t rms_norm_backward_workspace(size_t rows, size_t cols) { return backward_grid(rows) * cols * sizeof(float); }

void rms_norm_backward(const NormBackwardArgs& a, LayerType type, LayerType weight_type, hipStream_t stream) {
  check(a.cols <= (1u << 30), "rms_norm_backward: at most 2^30 columns");
  check(weight_type == type || weight_type == LayerType::kF32, "rms_norm_backward: the weight is of h's type or float32");
  check(a.rows > 0, "rms_norm_backward: no rows");
  if (a.cols == 0) return;
  check(a.dy && a.h && a.weight && a.rstd && a.dx && a.dw && a.workspace, "rms_norm_backward: a pointer is missing");
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
  const size_t tiles = (a.rows + kTile - 1) / kTile * ((a.cols + kTile - 1) / kTile);
  const dim3 grid(static_cast<unsigned>(std::min<size_t>(tiles, 1u << 20))), block(256);
  switch (type) {
    case LayerType::kF32: hipLaunchKernelGGL(quantize_kernel<float>, grid, block, 0, stream, a); break;
    case LayerType::kBF16: hipLaunchKernelGGL(quantize_kernel<__bf16>, grid, block, 0, stream, a); break;
    case LayerType::kF16: hipLaunchKernelGGL(quantize_kernel<_Float16>, grid, block, 0, stream, a); break;
  }
  TK8S_HIP_CHECK(hipGetLastError());
}

}  // namespace tk8s
