// pybind11 / libtorch module `mixedgemm_ops`: the 8-bit operators and the fused norms for torch tensors, and
// the mixed product that follows the norm (mixedgemm_b200/api.py documents and re-exports them).  Checks,
// allocation and launch in one compiled call: at one token the kernels take 2 to 9 us, and the same steps in
// Python took 9 (quantize_int8), 10 (matmul_int8), 14 (rms_norm_int8), 24 (matmul) and 31 us
// (rms_norm_reorder_quantize_x) of host time.
//
// torch owns the memory and names the current stream; all work goes through the C ABI (mixedgemm_c.h).
// Nothing is kept from one call to the next.  Inputs that a call does not take raise RuntimeError
// before anything is launched; what the C ABI refuses is the package's MixedGemmError with the status, as on the
// ctypes route.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <string>
#include <tuple>
#include <vector>

#include "mixedgemm_c.h"

namespace {

using at::ScalarType;
using at::Tensor;
using std::optional;

void check(int status, const char* what) {
  if (status != MG_OK) py::module_::import("mixedgemm_b200._capi").attr("check")(status, what);  // raises
}

int element(ScalarType t, const char* what, const char* name) {
  switch (t) {
    case ScalarType::BFloat16: return MG_BF16;
    case ScalarType::Half: return MG_FP16;
    case ScalarType::Float: return MG_FP32;
    default: TORCH_CHECK(false, what, ": ", name, " must be bfloat16, float16 or float32, not ", t);
  }
}

int as_int(int64_t v, const char* what) {
  TORCH_CHECK(v >= 0 && v <= 0x7fffffff, what, ": a size of ", v, " is out of range");
  return (int)v;
}

// Row pitch (elements) of a 2-D tensor whose rows are dense and do not overlap.
size_t rows(const Tensor& t, const char* what, const char* name, at::Device dev, ScalarType type) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == type && t.dim() == 2, what, ": ", name, " must be a 2-D ", type,
              " tensor on ", dev, ", not ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  const int64_t M = t.size(0), K = t.size(1);
  TORCH_CHECK((K <= 1 || t.stride(1) == 1) && (M <= 1 || t.stride(0) >= K), what, ": the rows of ", name,
              " must have unit stride and must not overlap (strides ", t.strides(), ")");
  return (size_t)(M > 1 ? t.stride(0) : K);
}

size_t rows_of(const Tensor& t, const char* what, const char* name, int64_t M, int64_t K, at::Device dev, ScalarType type) {
  TORCH_CHECK(t.dim() == 2 && t.size(0) == M && t.size(1) == K, what, ": ", name, " has shape ", t.sizes(), " where [", M, ", ",
              K, "] is expected");
  return rows(t, what, name, dev, type);
}

void vector_of(const Tensor& t, const char* what, const char* name, int64_t n, at::Device dev, ScalarType type) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == type && t.numel() == n && t.is_contiguous(), what, ": ", name,
              " must be a contiguous ", type, " tensor of ", n, " elements on ", dev, ", not ", t.scalar_type(), " ", t.sizes(),
              " on ", t.device());
}

Tensor new_rows(int64_t M, int64_t K, int64_t pitch, ScalarType type, at::Device dev) {
  return at::detail::empty_strided_cuda({M, K}, {pitch, 1}, type, dev);
}
Tensor new_vector(int64_t n, ScalarType type, at::Device dev) { return at::detail::empty_strided_cuda({n}, {1}, type, dev); }

// Rows of bytes, or a vector of K (M < 0), inside a block that other tensors share.  (Asking the allocator for each
// of the six buffers of a quantised activation, and giving them back, takes 3 us of host time more than one block.
// The two of the 8-bit quantisers are not worth it: 4.2 and 4.3 us.)
Tensor part_of(const c10::Storage& block, int64_t offset, int64_t M, int64_t K, int64_t pitch) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(block), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                      caffe2::TypeMeta::Make<uint8_t>());
  const int64_t sizes[2] = {M, K}, strides[2] = {pitch, 1};
  const int first = M < 0;
  t.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef(sizes + first, 2 - first),
                                                 c10::IntArrayRef(strides + first, 2 - first), offset);
  return t;
}

// The activation that a call starts with.
struct Activation {
  at::Device dev;
  ScalarType type;
  int element, M, K;
  size_t pitch;

  Activation(const Tensor& X, const char* what)
      : dev(X.device()), type(X.scalar_type()), element(0), M(0), K(0), pitch(0) {
    TORCH_CHECK(X.is_cuda(), what, ": X must be a CUDA tensor");
    element = ::element(type, what, "X");
    pitch = rows(X, what, "X", dev, type);
    M = as_int(X.size(0), what);
    K = as_int(X.size(1), what);
  }
};

// The weight, the residual and the stream of a fused norm.
struct Norm {
  Tensor stream;
  size_t ldr = 0, ldu = 0;
  const void* R = nullptr;
  void* U = nullptr;

  Norm(const Activation& x, const Tensor& weight, const optional<Tensor>& residual, const optional<Tensor>& residual_out,
       const char* what) {
    vector_of(weight, what, "the norm's weight", x.K, x.dev, x.type);
    TORCH_CHECK(residual || !residual_out, what, ": residual_out without a residual");
    if (!residual) return;
    ldr = rows_of(*residual, what, "the residual", x.M, x.K, x.dev, x.type);
    if (residual_out) {
      stream = *residual_out;
      ldu = rows_of(stream, what, "residual_out", x.M, x.K, x.dev, x.type);
    } else {
      stream = new_rows(x.M, x.K, x.K, x.type, x.dev);
      ldu = (size_t)x.K;
    }
    R = residual->data_ptr();
    U = stream.data_ptr();
  }
};

using Codes = std::tuple<Tensor, Tensor>;

// (codes, scale): the caller's, or new ones whose rows matmul_int8 can read in place.
Codes int8_outputs(const Activation& x, const optional<Codes>& out, size_t* ldq, const char* what) {
  if (!out) {
    const int64_t pitch = ((int64_t)x.K + 15) / 16 * 16;
    *ldq = (size_t)pitch;
    return {new_rows(x.M, x.K, pitch, ScalarType::Char, x.dev), new_vector(x.M, ScalarType::Float, x.dev)};
  }
  *ldq = rows_of(std::get<0>(*out), what, "the codes", x.M, x.K, x.dev, ScalarType::Char);
  vector_of(std::get<1>(*out), what, "the scale", x.M, x.dev, ScalarType::Float);
  return *out;
}

void* stream_of(at::Device dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

Codes quantize_int8(const Tensor& X, const optional<Codes>& out) {
  const char* what = "quantize_int8";
  const Activation x(X, what);
  size_t ldq;
  const Codes o = int8_outputs(x, out, &ldq, what);
  const c10::cuda::CUDAGuard guard(x.dev);
  check(mg_quantize_int8(X.data_ptr(), x.element, x.M, x.K, x.pitch, static_cast<int8_t*>(std::get<0>(o).data_ptr()), ldq,
                         static_cast<float*>(std::get<1>(o).data_ptr()), stream_of(x.dev)),
        what);
  return o;
}

py::tuple rms_norm_int8(const Tensor& X, const Tensor& weight, double eps, const optional<Tensor>& residual,
                        const optional<Tensor>& residual_out, const optional<Codes>& out) {
  const char* what = "rms_norm_int8";
  const Activation x(X, what);
  const Norm n(x, weight, residual, residual_out, what);
  size_t ldq;
  const Codes o = int8_outputs(x, out, &ldq, what);
  const c10::cuda::CUDAGuard guard(x.dev);
  check(mg_rms_norm_int8(X.data_ptr(), n.R, weight.data_ptr(), (float)eps, x.element, x.M, x.K, x.pitch, n.ldr, n.U, n.ldu,
                         static_cast<int8_t*>(std::get<0>(o).data_ptr()), ldq, static_cast<float*>(std::get<1>(o).data_ptr()),
                         stream_of(x.dev)),
        what);
  if (!residual) return py::make_tuple(std::get<0>(o), std::get<1>(o));
  return py::make_tuple(std::get<0>(o), std::get<1>(o), n.stream);
}

Tensor matmul_int8(const Tensor& A, const Tensor& B, const Tensor& scale_a, const Tensor& scale_b,
                   const optional<Tensor>& bias, const optional<Tensor>& out, const optional<ScalarType>& out_dtype) {
  const char* what = "matmul_int8";
  TORCH_CHECK(A.is_cuda(), what, ": A must be a CUDA tensor");
  const at::Device dev = A.device();
  const size_t lda = rows(A, what, "A", dev, ScalarType::Char), ldb = rows(B, what, "B", dev, ScalarType::Char);
  const int M = as_int(A.size(0), what), K = as_int(A.size(1), what), N = as_int(B.size(0), what);
  TORCH_CHECK(B.size(1) == K, what, ": A has rows of ", K, " elements, B of ", B.size(1));
  vector_of(scale_a, what, "scale_a", M, dev, ScalarType::Float);
  vector_of(scale_b, what, "scale_b", N, dev, ScalarType::Float);
  if (bias) vector_of(*bias, what, "the bias", N, dev, ScalarType::Float);
  const ScalarType type = out_dtype ? *out_dtype : out ? out->scalar_type() : ScalarType::BFloat16;
  const int e = element(type, what, "the result");
  const size_t ldd = out ? rows_of(*out, what, "out", M, N, dev, type) : (size_t)N;
  const Tensor D = out ? *out : new_rows(M, N, N, type, dev);
  const c10::cuda::CUDAGuard guard(dev);
  check(mg_matmul_int8(static_cast<const int8_t*>(A.data_ptr()), lda, static_cast<const int8_t*>(B.data_ptr()), ldb,
                       static_cast<const float*>(scale_a.data_ptr()), static_cast<const float*>(scale_b.data_ptr()),
                       bias ? static_cast<const float*>(bias->data_ptr()) : nullptr, M, N, K, D.data_ptr(), e, ldd,
                       stream_of(dev)),
        what);
  return D;
}

uint8_t* bytes(const Tensor& t) { return t.numel() ? static_cast<uint8_t*>(t.data_ptr()) : nullptr; }

py::tuple rms_norm_reorder_quantize_x(const Tensor& X, const Tensor& weight, const Tensor& reorder_index, int KN, int KS,
                                      int KO, double eps, const optional<Tensor>& residual,
                                      const optional<Tensor>& residual_out, const optional<std::vector<Tensor>>& out) {
  const char* what = "rms_norm_reorder_quantize_x";
  const Activation x(X, what);
  TORCH_CHECK(x.type == ScalarType::BFloat16, what, ": X must be bfloat16, not ", x.type);
  TORCH_CHECK(KN >= 0 && KS >= 0 && KO >= 0 && (int64_t)KN + KS + KO == x.K, what, ": K = ", x.K, " does not match KN+KS+KO");
  const Norm n(x, weight, residual, residual_out, what);
  vector_of(reorder_index, what, "reorder_index", x.K, x.dev, ScalarType::Short);
  const int k[3] = {KN, KS, KO};
  const int64_t logical[3] = {KN / 2, (int64_t)KS / 4 * 3, KO};
  std::vector<Tensor> o;
  size_t pitch[3];
  if (out) {
    o = *out;
    TORCH_CHECK(o.size() == 6, what, ": out must be six tensors");
    for (int i = 0; i < 3; ++i) {
      pitch[i] = rows_of(o[i], what, "a code buffer", x.M, logical[i], x.dev, ScalarType::Byte);
      const Tensor& s = o[3 + i];
      TORCH_CHECK(s.device() == x.dev && s.scalar_type() == ScalarType::Byte && s.is_contiguous() &&
                      (size_t)s.numel() >= mg_sf_bytes(x.M, k[i]),
                  what, ": a scale buffer is too small, on another device or not of bytes");
    }
  } else {  // as alloc_quantized_x does: rows padded to what the product reads in place
    int64_t at[6], size[6], end = 0;
    for (int i = 0; i < 6; ++i) {
      if (i < 3) {
        pitch[i] = mg_code_pitch(0, i, k[i]);
        size[i] = x.M * (int64_t)pitch[i];
      } else {
        size[i] = std::max<int64_t>((int64_t)mg_sf_bytes(x.M, k[i - 3]), ((int64_t)x.M / 128 + 1) * 128 * k[i - 3] / 32);
      }
      at[i] = end;
      end += (size[i] + 511) / 512 * 512;  // what an allocation is rounded to
    }
    const Tensor block = new_vector(end, ScalarType::Byte, x.dev);
    o.resize(6);
    for (int i = 0; i < 3; ++i) {
      o[i] = part_of(block.storage(), at[i], x.M, logical[i], (int64_t)pitch[i]);
      o[3 + i] = part_of(block.storage(), at[3 + i], -1, size[3 + i], 0);
    }
  }
  const c10::cuda::CUDAGuard guard(x.dev);
  check(mg_rms_norm_reorder_quantize(X.data_ptr(), x.pitch, n.R, n.ldr, weight.data_ptr(), (float)eps, n.U, n.ldu, x.M, x.K,
                                     static_cast<const int16_t*>(reorder_index.data_ptr()), KN, KS, KO, bytes(o[0]), bytes(o[1]),
                                     bytes(o[2]), pitch, bytes(o[3]), bytes(o[4]), bytes(o[5]), stream_of(x.dev)),
        what);
  if (!residual) return py::make_tuple(o[0], o[1], o[2], o[3], o[4], o[5]);
  return py::make_tuple(o[0], o[1], o[2], o[3], o[4], o[5], n.stream);
}

// The mixed product over the tensors of the two quantisers, in the order of the reference's binding.
// `workspace(device, bytes)` hands out scratch as (address, bytes); it is asked only when scratch is needed.
Tensor matmul(const Tensor& AN, const Tensor& BN, const Tensor& AS, const Tensor& BS, const Tensor& AO, const Tensor& BO,
              const Tensor& SFAN, const Tensor& SFBN, const Tensor& SFAS, const Tensor& SFBS, const Tensor& SFAO,
              const Tensor& SFBO, const optional<Tensor>& out, const optional<Tensor>& C,
              const optional<ScalarType>& out_dtype, const py::function& workspace) {
  const char* what = "matmul";
  const Tensor* codes[6] = {&AN, &BN, &AS, &BS, &AO, &BO};
  const Tensor* scales[6] = {&SFAN, &SFBN, &SFAS, &SFBS, &SFAO, &SFBO};
  const at::Device dev = AN.device();
  size_t pitches[6];
  for (int i = 0; i < 6; ++i) {
    const Tensor& t = *codes[i];
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == ScalarType::Byte && t.dim() == 2 && (t.size(1) == 0 || t.stride(1) == 1), what,
                ": code tensors must be 2-D CUDA uint8 with unit column stride");
    TORCH_CHECK(t.size(0) == codes[i & 1]->size(0), what, ": the three code tensors of an operand must have the same row count");
    pitches[i] = t.size(1) ? (size_t)t.stride(0) : 0;
  }
  const int M = as_int(AN.size(0), what), N = as_int(BN.size(0), what);
  const int KN = as_int(AN.size(1) * 2, what), KS = as_int(AS.size(1) * 4 / 3, what), KO = as_int(AO.size(1), what);
  TORCH_CHECK(AS.size(1) * 4 == (int64_t)KS * 3 && BN.size(1) * 2 == KN && BS.size(1) * 2 == KS && BO.size(1) * 2 == KO, what,
              ": code widths of the two operands do not describe the same K split");
  const int k[3] = {KN, KS, KO};
  for (int i = 0; i < 6; ++i) {
    const Tensor& t = *scales[i];
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == ScalarType::Byte && t.is_contiguous(), what,
                ": scale tensors must be contiguous CUDA uint8 tensors");
    const size_t need = mg_sf_bytes(i & 1 ? N : M, k[i >> 1]);
    TORCH_CHECK((size_t)t.numel() >= need, what, ": a scale tensor holds ", t.numel(), " bytes, ", need,
                " are read (whole 512-byte atoms)");
    TORCH_CHECK(t.device() == dev && codes[i]->device() == dev, what, ": all operands must be on one device");
  }
  const ScalarType type = out ? out->scalar_type() : out_dtype ? *out_dtype : ScalarType::BFloat16;
  TORCH_CHECK(type == ScalarType::BFloat16 || type == ScalarType::Float, what, ": output dtype must be bfloat16 or float32");
  const Tensor D = out ? *out : new_rows(M, N, N, type, dev);
  TORCH_CHECK(D.dim() == 2 && D.size(0) == M && D.size(1) == N && D.stride(1) == 1 && D.device() == dev, what,
              ": out must be [M,N] on the operands' device with unit column stride");
  TORCH_CHECK(!C || (C->scalar_type() == ScalarType::BFloat16 && C->dim() == 2 && C->size(0) == M && C->size(1) == N &&
                     C->device() == dev && C->stride(1) == 1 && C->stride(0) == D.stride(0)),
              what, ": C must be bf16 [M,N] on the operands' device with out's row pitch");
  const c10::cuda::CUDAGuard guard(dev);
  const size_t need = mg_matmul_pitched_workspace_bytes(M, N, KN, KS, KO, pitches);
  void* ws = nullptr;
  size_t ws_bytes = 0;
  if (need) {
    const py::tuple got = workspace(dev, need);
    ws = reinterpret_cast<void*>(got[0].cast<uintptr_t>());
    ws_bytes = got[1].cast<size_t>();
  }
  check(mg_matmul_pitched(bytes(AN), bytes(BN), bytes(AS), bytes(BS), bytes(AO), bytes(BO), pitches, type == ScalarType::Float, M, N,
                          KN, KS, KO, C ? C->data_ptr() : nullptr, D.numel() ? D.data_ptr() : nullptr, as_int(D.stride(0), what),
                          bytes(SFAN), bytes(SFBN), bytes(SFAS), bytes(SFBS), bytes(SFAO), bytes(SFBO), ws, ws_bytes,
                          stream_of(dev)),
        what);
  return D;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("quantize_int8", &quantize_int8, py::arg("X"), py::arg("out") = py::none());
  m.def("rms_norm_int8", &rms_norm_int8, py::arg("X"), py::arg("weight"), py::arg("eps"), py::arg("residual") = py::none(),
        py::arg("residual_out") = py::none(), py::arg("out") = py::none());
  m.def("matmul_int8", &matmul_int8, py::arg("A"), py::arg("B"), py::arg("scale_a"), py::arg("scale_b"),
        py::arg("bias") = py::none(), py::arg("out") = py::none(), py::arg("out_dtype") = py::none());
  m.def("rms_norm_reorder_quantize_x", &rms_norm_reorder_quantize_x, py::arg("X"), py::arg("weight"), py::arg("reorder_index"),
        py::arg("KN"), py::arg("KS"), py::arg("KO"), py::arg("eps"), py::arg("residual") = py::none(),
        py::arg("residual_out") = py::none(), py::arg("out") = py::none());
  m.def("matmul", &matmul);
}
