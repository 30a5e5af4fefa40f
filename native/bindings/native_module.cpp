// pybind11 module `_tk8s_native`: HIP kernels, node probes and the RCCL validator for gfx950.
//
// Two levels of API:
//  * probes (*_probe, gpuinfo_json, rccl_allreduce): self-contained, allocate their own
//    buffers, return a JSON string — what the node agent / validation pods use.
//  * raw launchers (hbm_fill, philox_fill, md5_tree, ar_fill, ar_check, stream_copy): take
//    device pointers and a hipStream_t as integers (e.g. torch tensor.data_ptr() and
//    torch.cuda.current_stream().cuda_stream) — what the numerics tests use.
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include "tk8s/kernels.h"
#include "tk8s/probes.h"
#include "tk8s/rccl_bench.h"

namespace py = pybind11;
using tk8s::DType;
using tk8s::StoreMode;

namespace {

template <class T> T* ptr(uintptr_t p) { return reinterpret_cast<T*>(p); }
hipStream_t stream_of(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }

StoreMode mode_of(const std::string& m) {
  if (m == "nontemporal" || m == "nt") return StoreMode::kNonTemporal;
  if (m == "plain") return StoreMode::kPlain;
  throw std::invalid_argument("mode must be 'nontemporal' or 'plain'");
}

DType dtype_of(const std::string& d) {
  if (d == "float32" || d == "f32" || d == "fp32") return DType::kF32;
  if (d == "bfloat16" || d == "bf16") return DType::kBF16;
  throw std::invalid_argument("dtype must be 'float32' or 'bfloat16'");
}

tk8s::LayerType layer_type_of(int t) {
  if (t < 0 || t > 2) throw std::invalid_argument("type must be 0 (float32), 1 (bfloat16) or 2 (float16)");
  return static_cast<tk8s::LayerType>(t);
}

template <class T> using Array = py::array_t<T, py::array::c_style | py::array::forcecast>;

// (values, row pitch, scales, scale pitch); zeros: not asked for
using Fp8Tuple = std::tuple<uintptr_t, size_t, uintptr_t, size_t>;
tk8s::Fp8Matrix fp8_of(const Fp8Tuple& t) {
  return {ptr<uint8_t>(std::get<0>(t)), std::get<1>(t), ptr<uint8_t>(std::get<2>(t)), std::get<3>(t)};
}

}  // namespace

PYBIND11_MODULE(_tk8s_native, m) {
  m.doc() = "tk8s gfx950 validation kernels (HIP) and RCCL all-reduce validator";
  using G = py::call_guard<py::gil_scoped_release>;

  m.def("gpuinfo_json", &tk8s::gpuinfo_json, py::arg("with_links") = true, G());
  m.def(
      "hbm_write_probe",
      [](size_t bytes, int iters, const std::string& mode, int device, uint32_t value) {
        return tk8s::hbm_write_probe(bytes, iters, mode_of(mode), device, value);
      },
      py::arg("bytes"), py::arg("iters") = 10, py::arg("mode") = "nontemporal",
      py::arg("device") = 0, py::arg("value") = 0, G());
  m.def("md5_probe", &tk8s::md5_probe, py::arg("bytes"), py::arg("chunk_bytes") = 1024,
        py::arg("seed") = 0, py::arg("iters") = 10, py::arg("device") = 0, G());
  m.def("copy_probe", &tk8s::copy_probe, py::arg("src_device"), py::arg("dst_device"),
        py::arg("bytes"), py::arg("iters") = 10, py::arg("dma") = true, G());
  m.def("layer_probe", &tk8s::layer_probe, py::arg("rows") = 4096, py::arg("width") = 4096, py::arg("seed") = 0,
        py::arg("iters") = 3, py::arg("device") = 0, G());
  // the layer probe's host checks on numpy arrays (bf16 as uint16)
  m.def(
      "layer_rounding_error",
      [](const Array<uint16_t>& source, const Array<uint8_t>& values, uint8_t scale) {
        if (source.size() != values.size()) throw std::invalid_argument("as many values as were rounded");
        return tk8s::layer_rounding_error(source.data(), values.data(), static_cast<size_t>(source.size()), scale);
      },
      py::arg("source"), py::arg("values"), py::arg("scale"));
  m.def(
      "layer_weight_sum_error",
      [](float got, const Array<uint16_t>& dy, const Array<uint16_t>& h, const Array<float>& rstd) {
        if (dy.size() != h.size() || dy.size() != rstd.size()) throw std::invalid_argument("dy, h and rstd must have as many rows");
        return tk8s::layer_weight_sum_error(got, dy.data(), h.data(), rstd.data(), static_cast<size_t>(dy.size()));
      },
      py::arg("got"), py::arg("dy"), py::arg("h"), py::arg("rstd"));
  m.def(
      "rccl_allreduce",
      [](const std::vector<int>& devices, size_t min_bytes, size_t max_bytes, int factor,
         int iters, int warmup, const std::string& dtype, bool check) {
        tk8s::AllReduceConfig c;
        c.min_bytes = min_bytes;
        c.max_bytes = max_bytes;
        c.factor = factor;
        c.iters = iters;
        c.warmup = warmup;
        c.dtypes = {dtype_of(dtype)};
        c.check = check;
        return tk8s::allreduce_single_process(devices, c);
      },
      py::arg("devices"), py::arg("min_bytes") = 8, py::arg("max_bytes") = size_t(1) << 26,
      py::arg("factor") = 4, py::arg("iters") = 10, py::arg("warmup") = 2,
      py::arg("dtype") = "float32", py::arg("check") = true, G());
  m.def("rccl_version", &tk8s::rccl_version);
  m.def("allreduce_busbw", &tk8s::allreduce_busbw, py::arg("algbw_gbps"), py::arg("nranks"),
        "busbw of a ring all-reduce: algbw * 2(n-1)/n, 0 at n <= 1 (SURVEY.md N3)");
  m.def("release_probe_scratch", &tk8s::release_probe_scratch, G());

  // ---- raw launchers --------------------------------------------------------------------
  m.def("streaming_grid", &tk8s::streaming_grid, py::arg("blocks_per_cu") = 8);
  m.def(
      "hbm_fill",
      [](uintptr_t dst, size_t nbytes, uint32_t value, const std::string& mode, uintptr_t s) {
        tk8s::hbm_fill(ptr<void>(dst), nbytes, value, mode_of(mode), stream_of(s));
      },
      py::arg("dst"), py::arg("nbytes"), py::arg("value"), py::arg("mode") = "nontemporal",
      py::arg("stream") = 0);
  m.def(
      "verify_fill",
      [](uintptr_t src, size_t nbytes, uint32_t value, uintptr_t bad, uintptr_t s) {
        tk8s::verify_fill(ptr<const void>(src), nbytes, value, ptr<unsigned long long>(bad),
                          stream_of(s));
      },
      py::arg("src"), py::arg("nbytes"), py::arg("value"), py::arg("bad_words"),
      py::arg("stream") = 0);
  m.def(
      "philox_fill",
      [](uintptr_t dst, size_t nbytes, uint64_t seed, uintptr_t s) {
        tk8s::philox_fill(ptr<void>(dst), nbytes, seed, stream_of(s));
      },
      py::arg("dst"), py::arg("nbytes"), py::arg("seed"), py::arg("stream") = 0);
  m.def(
      "layer_fill",
      [](uintptr_t dst, size_t count, uint64_t seed, uintptr_t s) { tk8s::layer_fill(ptr<void>(dst), count, seed, stream_of(s)); },
      py::arg("dst"), py::arg("count"), py::arg("seed"), py::arg("stream") = 0);
  m.def("md5_tree_workspace", &tk8s::md5_tree_workspace, py::arg("nbytes"),
        py::arg("chunk_bytes") = 1024);
  m.def(
      "md5_chunks",
      [](uintptr_t src, size_t nbytes, uint32_t chunk, uintptr_t digests, uintptr_t s) {
        tk8s::md5_chunks(ptr<const void>(src), nbytes, chunk, ptr<void>(digests), stream_of(s));
      },
      py::arg("src"), py::arg("nbytes"), py::arg("chunk_bytes"), py::arg("digests"),
      py::arg("stream") = 0);
  m.def(
      "md5_tree",
      [](uintptr_t src, size_t nbytes, uint32_t chunk, uintptr_t ws_a, uintptr_t ws_b,
         uintptr_t out16, uintptr_t s) {
        tk8s::md5_tree(ptr<const void>(src), nbytes, chunk, ptr<void>(ws_a), ptr<void>(ws_b),
                       ptr<void>(out16), stream_of(s));
      },
      py::arg("src"), py::arg("nbytes"), py::arg("chunk_bytes"), py::arg("ws_a"), py::arg("ws_b"),
      py::arg("out16"), py::arg("stream") = 0);
  m.def(
      "ar_fill",
      [](uintptr_t buf, size_t count, int rank, const std::string& dtype, uintptr_t s) {
        tk8s::ar_fill(ptr<void>(buf), count, rank, dtype_of(dtype), stream_of(s));
      },
      py::arg("buf"), py::arg("count"), py::arg("rank"), py::arg("dtype") = "float32",
      py::arg("stream") = 0);
  m.def(
      "ar_check",
      [](uintptr_t buf, size_t count, int nranks, const std::string& dtype, float tol,
         uintptr_t max_err_bits, uintptr_t bad, uintptr_t s) {
        tk8s::ar_check(ptr<const void>(buf), count, nranks, dtype_of(dtype), tol,
                       ptr<unsigned>(max_err_bits), ptr<unsigned long long>(bad), stream_of(s));
      },
      py::arg("buf"), py::arg("count"), py::arg("nranks"), py::arg("dtype") = "float32",
      py::arg("tol") = 0.0f, py::arg("max_err_bits") = 0, py::arg("bad") = 0,
      py::arg("stream") = 0);
  m.def(
      "stream_copy",
      [](uintptr_t dst, uintptr_t src, size_t nbytes, uintptr_t s) {
        tk8s::stream_copy(ptr<void>(dst), ptr<const void>(src), nbytes, stream_of(s));
      },
      py::arg("dst"), py::arg("src"), py::arg("nbytes"), py::arg("stream") = 0);

  // ---- 8-bit layer (tritonk8ssupervisor_amd/ops/fp8.py checks tensors and calls these) ----------
  m.def(
      "rms_norm_fp8",
      [](uintptr_t x, size_t ldx, uintptr_t residual, size_t ldr, uintptr_t weight, uintptr_t h, size_t ldh,
         const Fp8Tuple& q, uintptr_t y, size_t ldy, uintptr_t rstd, size_t rows, size_t cols, double eps, int type,
         int weight_type, uintptr_t s) {
        const tk8s::Fp8Matrix o = fp8_of(q);
        tk8s::rms_norm_fp8({ptr<const void>(x), ldx, ptr<const void>(residual), ldr, ptr<const void>(weight),
                            ptr<void>(h), ldh, o.values, o.ld, o.scales, o.ld_scales, ptr<void>(y), ldy,
                            ptr<float>(rstd), rows, cols, eps},
                           layer_type_of(type), layer_type_of(weight_type), stream_of(s));
      },
      py::arg("x"), py::arg("ldx"), py::arg("residual"), py::arg("ldr"), py::arg("weight"), py::arg("h"),
      py::arg("ldh"), py::arg("q"), py::arg("y"), py::arg("ldy"), py::arg("rstd"), py::arg("rows"), py::arg("cols"),
      py::arg("eps"), py::arg("type"), py::arg("weight_type"), py::arg("stream") = 0);
  m.def("rms_norm_backward_workspace", &tk8s::rms_norm_backward_workspace, py::arg("rows"), py::arg("cols"));
  m.def(
      "rms_norm_backward",
      [](uintptr_t dy, size_t lddy, uintptr_t h, size_t ldh, uintptr_t weight, uintptr_t rstd, uintptr_t dh,
         size_t lddh, uintptr_t dx, size_t lddx, uintptr_t dw, uintptr_t workspace, size_t rows, size_t cols, int type,
         int weight_type, uintptr_t s) {
        tk8s::rms_norm_backward({ptr<const void>(dy), lddy, ptr<const void>(h), ldh, ptr<const void>(weight),
                                 ptr<const float>(rstd), ptr<const void>(dh), lddh, ptr<void>(dx), lddx,
                                 ptr<float>(dw), ptr<float>(workspace), rows, cols},
                                layer_type_of(type), layer_type_of(weight_type), stream_of(s));
      },
      py::arg("dy"), py::arg("lddy"), py::arg("h"), py::arg("ldh"), py::arg("weight"), py::arg("rstd"), py::arg("dh"),
      py::arg("lddh"), py::arg("dx"), py::arg("lddx"), py::arg("dw"), py::arg("workspace"), py::arg("rows"),
      py::arg("cols"), py::arg("type"), py::arg("weight_type"), py::arg("stream") = 0);
  m.def(
      "fp8_quantize",
      [](uintptr_t x, size_t ldx, size_t rows, size_t cols, int type, const Fp8Tuple& by_rows, const Fp8Tuple& by_cols,
         const Fp8Tuple& by_tiles, uintptr_t s) {
        tk8s::fp8_quantize({ptr<const void>(x), ldx, rows, cols, fp8_of(by_rows), fp8_of(by_cols), fp8_of(by_tiles)},
                           layer_type_of(type), stream_of(s));
      },
      py::arg("x"), py::arg("ldx"), py::arg("rows"), py::arg("cols"), py::arg("type"), py::arg("by_rows"),
      py::arg("by_cols"), py::arg("by_tiles"), py::arg("stream") = 0);
  m.def(
      "fp8_matmul",
      [](const Fp8Tuple& a, const Fp8Tuple& b, bool b_tiles, uintptr_t c, size_t ldc, size_t rows, size_t cols,
         size_t k, int out, uintptr_t s) {
        tk8s::fp8_matmul({fp8_of(a), fp8_of(b), b_tiles, ptr<void>(c), ldc, rows, cols, k}, layer_type_of(out),
                         stream_of(s));
      },
      py::arg("a"), py::arg("b"), py::arg("b_tiles"), py::arg("c"), py::arg("ldc"), py::arg("rows"), py::arg("cols"),
      py::arg("k"), py::arg("out"), py::arg("stream") = 0);
}
