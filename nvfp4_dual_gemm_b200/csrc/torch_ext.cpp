// torch_ext.cpp — the thin torch extension between the reference-compatible
// Python entry points and the C ABI of libnvfp4dg.so.
//
// The reference binds its kernel with load_inline/pybind as
// cuda_nvfp4_dual_gemm(A, B1, B2, SFA, SFB1, SFB2, C) (submission.py:17-20,
// nvfp4_dual_gemm.cu:381-446) and calls it from custom_kernel(data)
// (submission.py:1153-1157).  This module exposes the same two functions
// plus dual_gemm (flags, caller workspace).  It checks the tensors (shape,
// strides, dtype, device: the same rules and messages as the Python checks
// in api.py), takes the current CUDA stream of C's device, and calls
// nvfp4_dual_gemm_run / nvfp4_dual_gemm_run_ws.  All of that costs a few
// microseconds per call, against tens for the same checks in Python plus a
// ctypes call, which matters when a caller launches one call at a time.
// Invalid arguments raise ValueError; CUDA and device failures RuntimeError.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <vector>

#include "nvfp4_dual_gemm.h"

namespace {

namespace py = pybind11;

[[noreturn]] void bad(const std::string& msg) { throw py::value_error(msg); }

std::string dims(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (i) s += ", ";
    s += std::to_string(t.size(i));
  }
  return s + (t.dim() == 1 ? ",)" : ")");
}

unsigned flag_bits(int64_t flags) {
  if (flags < 0 || flags > int64_t{UINT32_MAX})
    bad("flags must be 32 bits, got " + std::to_string(flags));
  return static_cast<unsigned>(flags);
}

void check_bytes(const char* name, const at::Tensor& t) {
  if (t.element_size() != 1)
    bad(std::string(name) +
        " must hold 1-byte elements (fp4x2 / fp8 / uint8), got " +
        std::string(c10::toString(t.scalar_type())));
  if (!t.is_cuda()) bad(std::string(name) + " must be a CUDA tensor");
}

int64_t batches(const at::Tensor& t) { return t.dim() == 3 ? t.size(2) : 1; }

// [rows, row_bytes] or [rows, row_bytes, L], rows dense and K-major, a batch
// stored batch after batch (api._rows_dense).
void rows_dense(const char* name, const at::Tensor& t, int64_t rows,
                int64_t row_bytes, int64_t L) {
  if (t.dim() != 2 && t.dim() != 3)
    bad(std::string(name) + " must be [rows, K/2] or [rows, K/2, L]");
  if (batches(t) != L)
    bad(std::string(name) + " holds " + std::to_string(batches(t)) +
        " batches, A holds " + std::to_string(L));
  if (t.size(0) != rows || t.size(1) != row_bytes)
    bad(std::string(name) + " has shape " + dims(t) + ", expected [" +
        std::to_string(rows) + ", " + std::to_string(row_bytes) + "(, " +
        std::to_string(L) + ")]");
  if (rows > 1 && row_bytes > 0 && t.stride(0) != row_bytes)
    bad(std::string(name) + " rows must be dense (stride(0) == K/2)");
  if (row_bytes > 1 && t.stride(1) != 1)
    bad(std::string(name) + " must be K-major (stride(1) == 1)");
  if (L > 1 && rows * row_bytes > 0 && t.stride(2) != rows * row_bytes)
    bad(std::string(name) + ": the batches must follow one another "
        "(stride(2) == " + std::to_string(rows * row_bytes) + ")");
}

int64_t blocked_bytes(int64_t rows, int64_t k) {
  return ((rows + 127) / 128) * (k / 64) * 512;
}

bool batch_major(const at::Tensor& t, int64_t L) {
  return t.is_contiguous() ||
         (L > 1 && t.dim() >= 2 && t.size(-1) == L &&
          t.movedim(-1, 0).is_contiguous());
}

void check_blocked(const char* name, const at::Tensor& t, int64_t rows,
                   int64_t k, int64_t L) {
  check_bytes(name, t);
  const int64_t need = blocked_bytes(rows, k);
  if (!batch_major(t, L))
    bad(std::string(name) + " must be contiguous (batch after batch)");
  if (L > 1 && !t.is_contiguous() && t.numel() != L * need)
    bad(std::string(name) + " holds " + std::to_string(t.numel()) +
        " bytes, " + std::to_string(L) +
        " batches of the blocked layout need " + std::to_string(L * need));
  if (t.numel() < L * need)
    bad(std::string(name) + " holds " + std::to_string(t.numel()) +
        " bytes, the blocked layout needs " + std::to_string(L * need));
}

struct Problem {
  int64_t M, N, K, L;
};

Problem check_problem(const at::Tensor& A, const at::Tensor& B1,
                      const at::Tensor& B2, const at::Tensor& SFA,
                      const at::Tensor& SFB1, const at::Tensor& SFB2,
                      const at::Tensor& C) {
  check_bytes("A", A);
  check_bytes("B1", B1);
  check_bytes("B2", B2);
  Problem p;
  p.M = A.size(0);
  p.N = B1.size(0);
  p.K = A.dim() >= 2 ? 2 * A.size(1) : 0;
  p.L = batches(A);
  if (p.L < 1) bad("L must be >= 1");
  rows_dense("A", A, p.M, p.K / 2, p.L);
  rows_dense("B1", B1, p.N, p.K / 2, p.L);
  rows_dense("B2", B2, p.N, p.K / 2, p.L);
  if (p.N % 64 != 0)
    bad("N = " + std::to_string(p.N) + " must be a multiple of 64");
  if (p.K % 256 != 0)
    bad("K = " + std::to_string(p.K) + " must be a multiple of 256");
  check_blocked("SFA", SFA, p.M, p.K, p.L);
  check_blocked("SFB1", SFB1, p.N, p.K, p.L);
  check_blocked("SFB2", SFB2, p.N, p.K, p.L);
  if (C.scalar_type() != at::kHalf)
    bad("C must be float16, got " +
        std::string(c10::toString(C.scalar_type())));
  if (!C.is_cuda() || !batch_major(C, p.L))
    bad("C must be a contiguous CUDA tensor (batch after batch)");
  if (C.numel() != p.L * p.M * p.N || C.size(0) != p.M ||
      (C.dim() == 3 && C.size(2) != p.L))
    bad("C has shape " + dims(C) + ", expected [" + std::to_string(p.M) +
        ", " + std::to_string(p.N) + "(, " + std::to_string(p.L) + ")]");
  if (p.L > 1 && C.dim() != 3)
    bad("C must be [" + std::to_string(p.M) + ", " + std::to_string(p.N) +
        ", " + std::to_string(p.L) + "] for a batch");
  const at::Device dev = C.device();
  const char* names[6] = {"A", "B1", "B2", "SFA", "SFB1", "SFB2"};
  const at::Tensor* ts[6] = {&A, &B1, &B2, &SFA, &SFB1, &SFB2};
  for (int i = 0; i < 6; ++i)
    if (ts[i]->device() != dev)
      bad(std::string(names[i]) + " is on " + ts[i]->device().str() +
          ", C on " + dev.str());
  return p;
}

void check_status(int rc, const char* what) {
  if (rc == NVFP4DG_OK) return;
  const char* m = nvfp4_dual_gemm_last_error();
  const std::string msg = std::string(what) + " failed (status " +
                          std::to_string(rc) + "): " + (m ? m : "");
  if (rc == NVFP4DG_ERR_INVALID || rc == NVFP4DG_ERR_ALIGN ||
      rc == NVFP4DG_ERR_WORKSPACE)
    throw py::value_error(msg);
  throw std::runtime_error(msg);
}

// A caller's tensor was written in place: autograd's check of the tensors it
// saved goes by their version.  (Inference tensors have none.)
void wrote(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor run(const at::Tensor& A, const at::Tensor& B1, const at::Tensor& B2,
               const at::Tensor& SFA, const at::Tensor& SFB1,
               const at::Tensor& SFB2, const at::Tensor& C, int64_t flags,
               const at::Tensor* ws) {
  const Problem p = check_problem(A, B1, B2, SFA, SFB1, SFB2, C);
  const c10::cuda::CUDAGuard guard(C.device());
  void* stream = at::cuda::getCurrentCUDAStream(C.device().index()).stream();
  int rc;
  if (ws == nullptr) {
    rc = nvfp4_dual_gemm_run(A.data_ptr(), B1.data_ptr(), B2.data_ptr(),
                             SFA.data_ptr(), SFB1.data_ptr(), SFB2.data_ptr(),
                             C.data_ptr(), static_cast<int>(p.M),
                             static_cast<int>(p.N), static_cast<int>(p.K),
                             static_cast<int>(p.L),
                             flag_bits(flags), stream);
  } else {
    if (ws->device() != C.device() || !ws->is_contiguous())
      bad("workspace must be a contiguous tensor on C's device");
    rc = nvfp4_dual_gemm_run_ws(
        A.data_ptr(), B1.data_ptr(), B2.data_ptr(), SFA.data_ptr(),
        SFB1.data_ptr(), SFB2.data_ptr(), C.data_ptr(), static_cast<int>(p.M),
        static_cast<int>(p.N), static_cast<int>(p.K), static_cast<int>(p.L),
        flag_bits(flags), ws->data_ptr(),
        static_cast<size_t>(ws->numel()) * ws->element_size(), stream);
  }
  check_status(rc, "nvfp4_dual_gemm_run");
  wrote(C);
  return C;
}

// The reference's torch-extension function: packed A/B1/B2, blocked
// SFA/SFB1/SFB2, preallocated fp16 C; returns C.
at::Tensor cuda_nvfp4_dual_gemm(const at::Tensor& A, const at::Tensor& B1,
                                const at::Tensor& B2, const at::Tensor& SFA,
                                const at::Tensor& SFB1, const at::Tensor& SFB2,
                                const at::Tensor& C) {
  return run(A, B1, B2, SFA, SFB1, SFB2, C, 0, nullptr);
}

// custom_kernel(data): data = (a, b1, b2, sfa, sfb1, sfb2, sfa_blocked,
// sfb1_blocked, sfb2_blocked, c), a tuple or any sequence of 10 tensors; the
// plain scales are not read.  The tensors are taken straight from the
// sequence's items (no per-item conversion objects).
at::Tensor custom_kernel(const py::object& data) {
  PyObject* seq = PySequence_Fast(data.ptr(), "data must be a sequence");
  if (seq == nullptr) throw py::error_already_set();
  const py::object keep = py::reinterpret_steal<py::object>(seq);
  if (PySequence_Fast_GET_SIZE(seq) != 10)
    bad("data must be the 10-tuple (a, b1, b2, sfa, sfb1, sfb2, "
        "sfa_blocked, sfb1_blocked, sfb2_blocked, c)");
  PyObject** items = PySequence_Fast_ITEMS(seq);
  auto t = [&](int i) -> const at::Tensor& {
    if (!THPVariable_Check(items[i]))
      throw py::type_error("data[" + std::to_string(i) +
                           "] must be a torch.Tensor");
    return THPVariable_Unpack(items[i]);
  };
  return run(t(0), t(1), t(2), t(6), t(7), t(8), t(9), 0, nullptr);
}

at::Tensor dual_gemm(const at::Tensor& A, const at::Tensor& B1,
                     const at::Tensor& B2, const at::Tensor& SFA,
                     const at::Tensor& SFB1, const at::Tensor& SFB2,
                     const at::Tensor& C, int64_t flags,
                     const c10::optional<at::Tensor>& workspace) {
  return run(A, B1, B2, SFA, SFB1, SFB2, C, flags,
             workspace.has_value() ? &workspace.value() : nullptr);
}

// ---------------------------------------------------------------------------
// linear / linear_grouped
// ---------------------------------------------------------------------------
using OptTensor = c10::optional<at::Tensor>;

// These operators have no gradient: rather than cut one silently, they refuse
// inputs that ask for it, by a backward pass or by a forward-mode tangent.
void no_grad_input(const char* name, const at::Tensor& t) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    bad(std::string(name) + " requires grad; this operator is inference only "
        "(use torch.no_grad())");
  if (t._fw_grad(/*level=*/0).defined() &&
      c10::AutogradState::get_tls_state().get_fw_grad_mode())
    bad(std::string(name) + " has a forward-mode tangent; this operator is "
        "inference only (use torch.autograd.forward_ad.unpack_dual)");
}

void on_device(const char* name, const at::Tensor& t, const at::Device& dev) {
  if (t.device() != dev)
    bad(std::string(name) + " is on " + t.device().str() + ", A on " +
        dev.str());
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NVFP4DG_DTYPE_F32;
    case at::kHalf: return NVFP4DG_DTYPE_F16;
    case at::kBFloat16: return NVFP4DG_DTYPE_BF16;
    default: return -1;
  }
}

int activation_code(const c10::optional<std::string>& name) {
  if (!name.has_value()) return NVFP4DG_ACT_NONE;
  const std::string& s = *name;
  if (s == "relu") return NVFP4DG_ACT_RELU;
  if (s == "silu") return NVFP4DG_ACT_SILU;
  if (s == "gelu_tanh") return NVFP4DG_ACT_GELU_TANH;
  if (s == "gelu") return NVFP4DG_ACT_GELU;
  bad("activation must be None, 'relu', 'silu', 'gelu_tanh' or 'gelu', got '" +
      s + "'");
}

int dim32(const char* name, int64_t v) {
  if (v > (int64_t{1} << 30)) bad(std::string(name) + " is too large");
  return static_cast<int>(v);
}

// [rows, N], rows dense inside, any row pitch
void check_matrix(const char* name, const at::Tensor& t, int64_t rows,
                  int64_t n, const at::Device& dev) {
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) != n)
    bad(std::string(name) + " has shape " + dims(t) + ", expected [" +
        std::to_string(rows) + ", " + std::to_string(n) + "]");
  if (n > 1 && t.stride(1) != 1)
    bad(std::string(name) + " must be row-major (stride(1) == 1)");
  on_device(name, t, dev);
}

int64_t pitch(const at::Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// at::empty without its dispatch.
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType t,
                      const at::Device& dev) {
  return at::detail::empty_cuda(sizes, t, dev, c10::nullopt);
}

// What linear and linear_grouped share: everything but the groups.
nvfp4_linear_args linear_args(const at::Tensor& A, const at::Tensor& B,
                              const at::Tensor& SFA, const at::Tensor& SFB,
                              const at::Tensor& C, const OptTensor& bias,
                              const c10::optional<std::string>& activation,
                              const OptTensor& residual,
                              const OptTensor& row_scale, double alpha,
                              int64_t flags, int64_t rows, int64_t groups) {
  const at::Device dev = A.device();
  const int64_t N = B.size(0), K = 2 * A.size(1), L = groups ? groups : 1;
  if (N % 8 != 0) bad("N = " + std::to_string(N) + " must be a multiple of 8");
  if (K == 0 || K % 64 != 0)
    bad("K = " + std::to_string(K) + " must be a positive multiple of 64");
  check_blocked("SFA", SFA, A.size(0), K, 1);
  check_blocked("SFB", SFB, N, K, L);
  no_grad_input("SFA", SFA);
  no_grad_input("SFB", SFB);
  on_device("B", B, dev);
  on_device("SFA", SFA, dev);
  on_device("SFB", SFB, dev);
  on_device("C", C, dev);
  nvfp4_linear_args a = {};
  a.A = A.data_ptr();
  a.B = B.data_ptr();
  a.SFA = SFA.data_ptr();
  a.SFB = SFB.data_ptr();
  a.C = C.data_ptr();
  a.M = dim32("M", rows);
  a.N = dim32("N", N);
  a.K = dim32("K", K);
  a.ldc = pitch(C);
  a.c_dtype = dtype_code(C.scalar_type());
  if (a.c_dtype < 0 || a.c_dtype == NVFP4DG_DTYPE_F32)
    bad("C must be float16 or bfloat16, got " +
        std::string(c10::toString(C.scalar_type())));
  if (bias.has_value()) {
    const at::Tensor& b = *bias;
    no_grad_input("bias", b);
    on_device("bias", b, dev);
    const bool fits = groups ? b.dim() == 2 && b.size(0) == groups &&
                                   b.size(1) == N
                             : b.dim() == 1 && b.size(0) == N;
    if (!fits || !b.is_contiguous())
      bad("bias has shape " + dims(b) + ", expected a contiguous [" +
          (groups ? std::to_string(groups) + ", " : std::string()) +
          std::to_string(N) + "]");
    a.bias_dtype = dtype_code(b.scalar_type());
    if (a.bias_dtype != NVFP4DG_DTYPE_F32 && a.bias_dtype != a.c_dtype)
      bad("bias must be float32 or of C's type");
    a.bias = b.data_ptr();
  }
  if (residual.has_value()) {
    no_grad_input("residual", *residual);
    check_matrix("residual", *residual, rows, N, dev);
    if (residual->scalar_type() != C.scalar_type())
      bad("residual must be of C's type");
    a.residual = residual->data_ptr();
    a.ldr = pitch(*residual);
  }
  if (row_scale.has_value()) {
    const at::Tensor& r = *row_scale;
    no_grad_input("row_scale", r);
    on_device("row_scale", r, dev);
    if (r.scalar_type() != at::kFloat || !r.is_contiguous() || r.dim() != 1 ||
        r.size(0) < rows || (groups == 0 && r.size(0) != rows))
      bad("row_scale must be a contiguous float32 [" + std::to_string(rows) +
          "] tensor");
    a.row_scale = r.data_ptr<float>();
  }
  a.activation = activation_code(activation);
  a.alpha = static_cast<float>(alpha);
  a.flags = flag_bits(flags);
  return a;
}

void check_operands(const at::Tensor& A, const at::Tensor& B, int64_t L) {
  check_bytes("A", A);
  check_bytes("B", B);
  if (A.dim() < 2 || B.dim() < 2) bad("A and B must be [rows, K/2]");
  no_grad_input("A", A);
  no_grad_input("B", B);
  rows_dense("A", A, A.size(0), A.size(1), 1);
  if (batches(B) != L)
    bad("B holds " + std::to_string(batches(B)) + " matrices, expected " +
        std::to_string(L));
  rows_dense("B", B, B.size(0), A.size(1), L);
}

at::Tensor linear(const at::Tensor& A, const at::Tensor& B,
                  const at::Tensor& SFA, const at::Tensor& SFB,
                  const OptTensor& C_in, const OptTensor& bias,
                  const c10::optional<std::string>& activation,
                  const OptTensor& residual, const OptTensor& row_scale,
                  double alpha, const c10::optional<at::ScalarType>& dtype,
                  int64_t flags) {
  check_operands(A, B, 1);
  const int64_t M = A.size(0), N = B.size(0);
  const c10::cuda::CUDAGuard guard(A.device());
  at::Tensor C;
  if (C_in.has_value()) {
    C = *C_in;
    no_grad_input("C", C);
    check_matrix("C", C, M, N, A.device());
    if (dtype.has_value() && *dtype != C.scalar_type())
      bad("dtype does not match C's");
  } else {
    const at::ScalarType t = dtype.has_value()      ? *dtype
                             : residual.has_value() ? residual->scalar_type()
                                                    : at::kHalf;
    C = new_tensor({M, N}, t, A.device());
  }
  const nvfp4_linear_args a =
      linear_args(A, B, SFA, SFB, C, bias, activation, residual, row_scale,
                  alpha, flags, M, 0);
  check_status(
      nvfp4_linear_run(
          &a, at::cuda::getCurrentCUDAStream(A.device().index()).stream()),
      "nvfp4_linear_run");
  if (C_in.has_value()) wrote(C);
  return C;
}

// A sequence of integers, or a CPU tensor of them, as ints.
std::vector<int> host_ints(const char* name, const py::object& o) {
  std::vector<int> v;
  const py::object seq = py::hasattr(o, "tolist") ? o.attr("tolist")() : o;
  for (const py::handle h : seq) {
    int64_t x;
    try {
      x = py::cast<int64_t>(h);
    } catch (const py::cast_error&) {
      bad(std::string(name) + " must hold integers of 32 bits");
    }
    if (x < INT32_MIN || x > INT32_MAX)
      bad(std::string(name) + " does not fit 32 bits");
    v.push_back(static_cast<int>(x));
  }
  return v;
}

const at::Tensor& device_ints(const char* name, const at::Tensor& t,
                              int64_t n, const at::Device& dev) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || !t.is_contiguous())
    bad(std::string(name) + " on the device must be a contiguous int32 [" +
        (n < 0 ? std::string("groups") : std::to_string(n)) + "] tensor");
  if (n >= 0 && t.size(0) != n)
    bad(std::string(name) + " needs one entry per group");
  on_device(name, t, dev);
  return t;
}

at::Tensor linear_grouped(const at::Tensor& A, const at::Tensor& B,
                          const at::Tensor& SFA, const at::Tensor& SFB,
                          const at::Tensor& C, const py::object& group_rows,
                          const py::object& group_row0, const OptTensor& bias,
                          const c10::optional<std::string>& activation,
                          const OptTensor& row_scale, double alpha,
                          int64_t flags) {
  const at::Tensor* dev_rows = nullptr;
  const at::Tensor* dev_row0 = nullptr;
  std::vector<int> rows, row0;
  auto cuda_tensor = [](const py::object& o) -> const at::Tensor* {
    if (!THPVariable_Check(o.ptr())) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o.ptr());
    return t.is_cuda() ? &t : nullptr;
  };
  dev_rows = cuda_tensor(group_rows);
  const bool on_dev = dev_rows != nullptr;
  int64_t G;
  if (on_dev) {
    device_ints("group_rows", *dev_rows, -1, A.device());
    G = dev_rows->size(0);
    if (!group_row0.is_none()) {
      dev_row0 = cuda_tensor(group_row0);
      if (dev_row0 == nullptr)
        bad("group_row0 must be on the device as group_rows is");
      device_ints("group_row0", *dev_row0, G, A.device());
    }
  } else {
    rows = host_ints("group_rows", group_rows);
    G = static_cast<int64_t>(rows.size());
    if (!group_row0.is_none()) {
      if (cuda_tensor(group_row0))
        bad("group_row0 must be on the host as group_rows is");
      row0 = host_ints("group_row0", group_row0);
      if (row0.size() != rows.size())
        bad("group_row0 needs one entry per group");
    }
  }
  check_operands(A, B, G);
  no_grad_input("C", C);
  const int64_t R = std::min(A.size(0), C.dim() == 2 ? C.size(0) : 0);
  if (C.dim() != 2 || C.size(1) != B.size(0) ||
      (C.size(1) > 1 && C.stride(1) != 1))
    bad("C has shape " + dims(C) + ", expected row-major [rows, " +
        std::to_string(B.size(0)) + "]");
  const c10::cuda::CUDAGuard guard(A.device());
  const nvfp4_linear_args a =
      linear_args(A, B, SFA, SFB, C, bias, activation, c10::nullopt,
                  row_scale, alpha, flags, R, G);
  check_status(
      nvfp4_linear_run_grouped(
          &a, on_dev ? dev_rows->data_ptr<int>() : rows.data(),
          on_dev ? (dev_row0 ? dev_row0->data_ptr<int>() : nullptr)
                 : (group_row0.is_none() ? nullptr : row0.data()),
          dim32("groups", G), on_dev ? 1 : 0,
          at::cuda::getCurrentCUDAStream(A.device().index()).stream()),
      "nvfp4_linear_run_grouped");
  wrote(C);
  return C;
}

// ---------------------------------------------------------------------------
// block_norm / block_norm_nvfp4
// ---------------------------------------------------------------------------
// [..., D] as rows: two dimensions with any row pitch, else contiguous.
at::Tensor as_rows(const char* name, const at::Tensor& t) {
  if (t.dim() < 1) bad(std::string(name) + " must be [..., D]");
  if (t.dim() == 2) {
    if (t.size(1) > 1 && t.stride(1) != 1)
      bad(std::string(name) + " must be row-major (stride(-1) == 1)");
    return t;
  }
  if (!t.is_contiguous())
    bad(std::string(name) + " must be contiguous, or [rows, D]");
  return t.reshape({t.size(-1) ? t.numel() / t.size(-1) : 0, t.size(-1)});
}

struct NormOut {
  at::Tensor R, Z, codes, sf;
};

NormOut norm(const at::Tensor& x_in, const OptTensor& y_in,
             const OptTensor& weight, const OptTensor& bias,
             const OptTensor& post_weight, const OptTensor& post_bias,
             const OptTensor& gate, double scale, const std::string& kind,
             double eps, bool post, bool pre, const OptTensor& R_in,
             const OptTensor& Z_in, bool nvfp4, int64_t flags) {
  if (!x_in.is_cuda()) bad("x must be a CUDA tensor");
  no_grad_input("x", x_in);
  nvfp4_block_norm_args a = {};
  a.dtype = dtype_code(x_in.scalar_type());
  if (a.dtype < 0)
    bad("x must be float32, float16 or bfloat16, got " +
        std::string(c10::toString(x_in.scalar_type())));
  const at::Tensor x = as_rows("x", x_in);
  const at::Device dev = x.device();
  const int64_t rows = x.size(0), D = x.size(1);
  a.rows = dim32("rows", rows);
  a.D = dim32("D", D);
  if (D % 8 != 0 || D < 8 || D > 32768)
    bad("D = " + std::to_string(D) +
        " must be a multiple of 8 between 8 and 32768");
  if (nvfp4 && D % 64 != 0)
    bad("D = " + std::to_string(D) +
        " must be a multiple of 64 for NVFP4 output");
  auto same = [&](const char* name, const at::Tensor& t) {
    no_grad_input(name, t);
    if (t.device() != dev)
      bad(std::string(name) + " is on " + t.device().str() + ", x on " +
          dev.str());
    if (t.scalar_type() != x.scalar_type())
      bad(std::string(name) + " must be of x's type");
    if (t.sizes() != x_in.sizes())
      bad(std::string(name) + " has shape " + dims(t) + ", x " + dims(x_in));
    return as_rows(name, t);
  };
  const c10::cuda::CUDAGuard guard(dev);
  NormOut out;
  a.x = x.data_ptr();
  a.ldx = pitch(x);
  a.w_dtype = NVFP4DG_DTYPE_F32;
  bool w_seen = false;
  auto param = [&](const char* name, const OptTensor& t) -> const void* {
    if (!t.has_value()) return nullptr;
    no_grad_input(name, *t);
    if (t->device() != dev)
      bad(std::string(name) + " is on " + t->device().str() + ", x on " +
          dev.str());
    if (t->dim() != 1 || t->size(0) != D || !t->is_contiguous())
      bad(std::string(name) + " has shape " + dims(*t) +
          ", expected a contiguous [" + std::to_string(D) + "]");
    const int c = dtype_code(t->scalar_type());
    if (c != NVFP4DG_DTYPE_F32 && c != a.dtype)
      bad(std::string(name) + " must be float32 or of x's type");
    if (w_seen && c != a.w_dtype)
      bad("weights and biases must share one type");
    a.w_dtype = c;
    w_seen = true;
    return t->data_ptr();
  };
  if (!pre && (weight.has_value() || bias.has_value()))
    bad("weight and bias need pre");
  a.weight = param("weight", weight);
  a.bias = param("bias", bias);
  a.post_weight = param("post_weight", post_weight);
  a.post_bias = param("post_bias", post_bias);
  a.post = post || a.post_weight != nullptr || a.post_bias != nullptr;
  if (kind == "rms")
    a.kind = NVFP4DG_NORM_RMS;
  else if (kind == "layer")
    a.kind = NVFP4DG_NORM_LAYER;
  else
    bad("kind must be 'rms' or 'layer', got '" + kind + "'");
  if (!(eps >= 0)) bad("eps must not be negative");
  a.eps = static_cast<float>(eps);
  a.scale = static_cast<float>(scale);
  a.flags = flag_bits(flags);
  at::Tensor y, g, r, z;
  if (y_in.has_value()) {
    y = same("y", *y_in);
    a.y = y.data_ptr();
    a.ldy = pitch(y);
    out.R = R_in.has_value()
                ? *R_in
                : new_tensor(x_in.sizes(), x.scalar_type(), dev);
    r = same("R", out.R);
    a.R = r.data_ptr();
    a.ldr = pitch(r);
  } else {
    if (a.post || gate.has_value() || R_in.has_value())
      bad("post, gate and R need y");
    out.R = x_in;
  }
  if (gate.has_value()) {
    no_grad_input("gate", *gate);
    if (gate->device() != dev)
      bad("gate is on " + gate->device().str() + ", x on " + dev.str());
    if (gate->scalar_type() != x.scalar_type())
      bad("gate must be of x's type");
    if (gate->dim() < 1 || gate->size(-1) != D || !gate->is_contiguous() ||
        (rows > 0 && (gate->numel() == 0 || rows % (gate->numel() / D) != 0)))
      bad("gate has shape " + dims(*gate) + ", expected a contiguous [G, " +
          std::to_string(D) + "] with G dividing the " +
          std::to_string(rows) + " rows");
    a.gate = gate->data_ptr();
    a.gate_rows = static_cast<int>(gate->numel() / D);
  }
  if (pre && nvfp4) {
    if (Z_in.has_value()) bad("Z is for block_norm");
    out.codes = new_tensor({rows, D / 2}, at::kByte, dev);
    out.sf = new_tensor({blocked_bytes(rows, D)}, at::kByte, dev);
    a.codes = out.codes.data_ptr();
    a.sf = out.sf.data_ptr();
  } else if (pre) {
    out.Z = Z_in.has_value()
                ? *Z_in
                : new_tensor(x_in.sizes(), x.scalar_type(), dev);
    z = same("Z", out.Z);
    a.Z = z.data_ptr();
    a.ldz = pitch(z);
  } else if (Z_in.has_value()) {
    bad("Z needs pre");
  }
  check_status(nvfp4_block_norm_run(
                   &a, at::cuda::getCurrentCUDAStream(dev.index()).stream()),
               "nvfp4_block_norm_run");
  if (R_in.has_value()) wrote(out.R);
  if (Z_in.has_value()) wrote(out.Z);
  return out;
}

py::tuple block_norm(const at::Tensor& x, const OptTensor& y,
                     const OptTensor& weight, const OptTensor& bias,
                     const OptTensor& post_weight, const OptTensor& post_bias,
                     const OptTensor& gate, double scale,
                     const std::string& kind, double eps, bool post, bool pre,
                     const OptTensor& R, const OptTensor& Z, int64_t flags) {
  const NormOut o = norm(x, y, weight, bias, post_weight, post_bias, gate,
                         scale, kind, eps, post, pre, R, Z, false, flags);
  return py::make_tuple(o.R, pre ? py::cast(o.Z) : py::none());
}

py::tuple block_norm_nvfp4(const at::Tensor& x, const OptTensor& y,
                           const OptTensor& weight, const OptTensor& bias,
                           const OptTensor& post_weight,
                           const OptTensor& post_bias, const OptTensor& gate,
                           double scale, const std::string& kind, double eps,
                           bool post, const OptTensor& R, int64_t flags) {
  const NormOut o = norm(x, y, weight, bias, post_weight, post_bias, gate,
                         scale, kind, eps, post, true, R, c10::nullopt, true,
                         flags);
  return py::make_tuple(o.R, o.codes, o.sf);
}

}  // namespace

PYBIND11_MODULE(_C, m) {
  m.doc() = "torch binding of the NVFP4 dual GEMM C ABI (libnvfp4dg.so)";
  m.def("custom_kernel", &custom_kernel, py::arg("data"));
  m.def("cuda_nvfp4_dual_gemm", &cuda_nvfp4_dual_gemm, py::arg("A"),
        py::arg("B1"), py::arg("B2"), py::arg("SFA"), py::arg("SFB1"),
        py::arg("SFB2"), py::arg("C"));
  m.def("dual_gemm", &dual_gemm, py::arg("A"), py::arg("B1"), py::arg("B2"),
        py::arg("SFA"), py::arg("SFB1"), py::arg("SFB2"), py::arg("C"),
        py::arg("flags") = 0, py::arg("workspace") = py::none());
  // (called with positional arguments: api.py holds the names and defaults,
  // and keywords cost about a microsecond a call here)
  m.def("linear", &linear);
  m.def("linear_grouped", &linear_grouped);
  m.def("block_norm", &block_norm);
  m.def("block_norm_nvfp4", &block_norm_nvfp4);
}
