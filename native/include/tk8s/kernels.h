// Host-side launch API for the tk8s validation kernels (gfx950 / CDNA4).
//
// Kernel inventory:
//   N4  hbm_fill          — HBM write-bandwidth probe (GPU analogue of docs/benchmarks.md:8-9,
//                           "pipes a gigabyte of zeros").
//   N5  philox_fill +     — on-device random data + chunked MD5 tree hash (GPU analogue of
//       md5_tree            docs/benchmarks.md:11-12, "fetches random numbers and md5 hashes them").
//   N6  ar_fill/ar_check  — all-reduce pattern generator + max-abs-error checker.
//   N7  stream_copy       — device copy kernel used for local and xGMI peer-pull bandwidth probes.
//   8-bit layer           — what the matrix cores are validated with: an RMS norm with 8-bit output,
//       rms_norm_fp8,       its gradient, rounding to e4m3 with a power-of-two scale for each block
//       fp8_quantize,       of 128 values, and the product of two such matrices
//       fp8_matmul          (fp8_kernels.hip, matmul_kernels.hip).
//
// All launchers are asynchronous on `stream` and never allocate, synchronise or free, so a
// caller may capture them into a hipGraph.
#pragma once

#include <cstddef>
#include <cstdint>

#include <hip/hip_runtime.h>

namespace tk8s {

enum class StoreMode : int { kNonTemporal = 0, kPlain = 1 };
enum class DType : int { kF32 = 0, kBF16 = 1 };

// Number of workgroups for a grid-stride streaming kernel on the current device
// (CU count x blocks_per_cu, cached per device).
int streaming_grid(int blocks_per_cu = 8);

// N4: write `nbytes` (multiple of 16) of the 32-bit pattern `value` to dst.
void hbm_fill(void* dst, size_t nbytes, uint32_t value, StoreMode mode, hipStream_t stream);

// Counts 32-bit words in src (nbytes multiple of 16) that differ from `value`; *bad_words must
// point to device memory that the caller zeroed.
void verify_fill(const void* src, size_t nbytes, uint32_t value, unsigned long long* bad_words,
                 hipStream_t stream);

// N5: fill dst with Philox4x32-10 output (counter = 16-byte block index, key = seed).
// nbytes must be a multiple of 16.
void philox_fill(void* dst, size_t nbytes, uint64_t seed, hipStream_t stream);

// N5: one level of the MD5 tree: digest of every `chunk_bytes` chunk of src (last chunk may be
// partial) into `digests` (16 bytes each). chunk_bytes must be a multiple of 64.
void md5_chunks(const void* src, size_t nbytes, uint32_t chunk_bytes, void* digests,
                hipStream_t stream);

// Number of digest bytes needed as workspace by md5_tree for `nbytes` input (two ping-pong
// buffers of this size).
size_t md5_tree_workspace(size_t nbytes, uint32_t chunk_bytes);

// N5: MD5 tree hash. Level 0 hashes chunks of src; each next level hashes the concatenated
// digests of the previous one, until one digest remains. Writes 16 bytes to out16 (device).
// ws_a/ws_b: device workspaces of md5_tree_workspace() bytes each.
void md5_tree(const void* src, size_t nbytes, uint32_t chunk_bytes, void* ws_a, void* ws_b,
              void* out16, hipStream_t stream);

// N6: buf[i] = (rank + 1) + (i % 7) in dtype.
void ar_fill(void* buf, size_t count, int rank, DType dtype, hipStream_t stream);

// N6: compares buf (after a sum all-reduce over nranks ranks filled by ar_fill) with the exact
// expected value nranks*(nranks+1)/2 + nranks*(i % 7). Writes max |err| as float bits into
// *max_err_bits (device, caller-zeroed) and the number of elements with |err| > tol into
// *bad (device, caller-zeroed).
void ar_check(const void* buf, size_t count, int nranks, DType dtype, float tol,
              unsigned int* max_err_bits, unsigned long long* bad, hipStream_t stream);

// N7: dst[i] = src[i] for nbytes (multiple of 16). src may live on a peer GPU (xGMI pull).
void stream_copy(void* dst, const void* src, size_t nbytes, hipStream_t stream);

// Fault injection (TK8S_FAULTS "...hang@<phase>" on a GPU phase, failfast.h): enqueue on `stream`
// a one-wave kernel that spins until gpu_stall_release() (common.h) is called or `max_s` seconds
// of GPU wall clock pass -- so a stalled queue always drains, whoever forgets to release it.
// Everything queued behind it on `stream` waits: a hung collective or pull, made on purpose.
void gpu_stall(hipStream_t stream, double max_s);

// ---- 8-bit layer ----------------------------------------------------------------------------
// Values are e4m3 (OCP), scales E8M0 bytes: 2^(byte - 127), 255 = NaN. Strides are in elements.

enum class LayerType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// rows x cols values in 8 bits; row r starts at values + r * ld (16-byte boundaries). Scales lie
// block by block: that of block b (128 columns) of row r at scales[b * ld_scales + r]; for 128 x 128
// tiles, r counts tiles of rows. values == nullptr: not asked for. fp8_matmul reads scales four rows at a
// time: they start on 4-byte boundaries, ld_scales is a multiple of 4, and the rows up to the next
// multiple of 4 can be read (their values do not matter).
struct Fp8Matrix {
  uint8_t* values;
  size_t ld;
  uint8_t* scales;
  size_t ld_scales;
};

// h = x + residual, rounded to the type (no residual: h = x, nothing is stored);
// rstd = 1 / sqrt(mean(h^2) + eps); y = h * rstd * weight. q/scales: y in 8 bits with a scale for
// each 128 columns of a row; y itself and rstd are stored where their pointers are given. Sums and rstd are in 64
// bits; y and its 8-bit values are those of y in 64 bits, rounded once (it is computed in 32 where that gives the same 8
// bits). y beyond the range of 32 bits is an infinity. A block that holds a NaN or an infinity is NaN.
struct NormArgs {
  const void* x;
  size_t ldx;
  const void* residual;  // or nullptr
  size_t ldr;
  const void* weight;
  void* h;  // needed with a residual; may be x or residual itself
  size_t ldh;
  uint8_t* q;  // or nullptr
  size_t ldq;
  uint8_t* scales;
  size_t lds;
  void* y;  // or nullptr
  size_t ldy;
  float* rstd;  // or nullptr
  size_t rows, cols;
  double eps;
};
void rms_norm_fp8(const NormArgs& a, LayerType type, LayerType weight_type, hipStream_t stream);

// Gradients of rms_norm_fp8's y through to x (and the residual, whose gradient is the same) and
// the weight; dh, if given, is what else flows into h. dw is in 32 bits. workspace: device memory of
// rms_norm_backward_workspace() bytes that no other call uses at the same time.
struct NormBackwardArgs {
  const void* dy;
  size_t lddy;
  const void* h;
  size_t ldh;
  const void* weight;
  const float* rstd;
  const void* dh;  // or nullptr
  size_t lddh;
  void* dx;
  size_t lddx;
  float* dw;
  float* workspace;
  size_t rows, cols;
};
size_t rms_norm_backward_workspace(size_t rows, size_t cols);
void rms_norm_backward(const NormBackwardArgs& a, LayerType type, LayerType weight_type, hipStream_t stream);

// x in 8 bits, in any of three layouts from one read: a scale for each 128 columns of a row; the
// transpose (cols x rows) with a scale for each 128 rows of a column; a scale for each 128 x 128.
struct QuantizeArgs {
  const void* x;
  size_t ldx, rows, cols;
  Fp8Matrix rows_out, cols_out, tiles_out;
};
void fp8_quantize(const QuantizeArgs& a, LayerType type, hipStream_t stream);

// C[m, n] = A B^T with A m x k and B n x k in 8 bits; A has a scale for each 128 columns of a row,
// B the same or one for each 128 x 128 (b_tiles). 32-bit sums, one rounding to the type of C.
struct MatmulArgs {
  Fp8Matrix a, b;
  bool b_tiles;
  void* c;
  size_t ldc, m, n, k;
};
void fp8_matmul(const MatmulArgs& a, LayerType out, hipStream_t stream);

// dst[i], 16-bit (kBF16): a multiple of 1/32 in [-4, 4) that depends on the seed and i alone (count a
// multiple of 8): what the layer probe works on.
void layer_fill(void* dst, size_t count, uint64_t seed, hipStream_t stream);

}  // namespace tk8s
