// Helpers shared by the three op-registration libraries (_C, _moe_C, _xpu_C).
// They translate torch tensors into the plain pointers of the C ABI
// (include/b200moe.h), pick the current CUDA stream and turn a non-zero status
// into the RuntimeError a TORCH_CHECK raises.  No kernel lives here.
#pragma once

#include <Python.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/types.h>

#include <algorithm>
#include <optional>

#include "../../../include/b200moe.h"

#define B200_REGISTER_EXTENSION(NAME)                                        \
  PyMODINIT_FUNC PyInit_##NAME() {                                           \
    static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, #NAME,       \
                                        nullptr, 0, nullptr, nullptr,       \
                                        nullptr, nullptr, nullptr};         \
    return PyModule_Create(&module);                                         \
  }

// The same with a table of module functions.
#define B200_REGISTER_EXTENSION_METHODS(NAME, METHODS)                       \
  PyMODINIT_FUNC PyInit_##NAME() {                                           \
    static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, #NAME,       \
                                        nullptr, 0, METHODS, nullptr,       \
                                        nullptr, nullptr, nullptr};         \
    return PyModule_Create(&module);                                         \
  }

namespace b200shim {

inline b200moe_stream current_stream() {
  return (b200moe_stream)at::cuda::getCurrentCUDAStream().stream();
}

inline void check_status(int rc) {
  TORCH_CHECK(rc == B200MOE_OK, b200moe_last_error(), " [", b200moe_status_string(rc), "]");
}

inline b200moe_dtype float_dtype(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return B200MOE_F32;
    case at::kHalf: return B200MOE_F16;
    case at::kBFloat16: return B200MOE_BF16;
    default: TORCH_CHECK(false, what, ": only float32, float16 and bfloat16 are supported");
  }
  return B200MOE_F32;
}

inline b200moe_dtype index_dtype(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kInt: return B200MOE_I32;
    case at::kUInt32: return B200MOE_U32;
    case at::kLong: return B200MOE_I64;
    default: return B200MOE_U8;  // rejected by the callee
  }
}

inline void check_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
}

// Rows [..., n] whose last dimension is dense and whose rows are evenly spaced: the row stride in elements.
inline int64_t row_stride(const at::Tensor& t, const char* op, const char* name) {
  const int64_t n = t.size(-1);
  if (t.numel() == 0) return n;
  TORCH_CHECK(n == 1 || t.stride(-1) == 1, op, ": the last dimension of ", name, " must be contiguous");
  if (t.dim() == 1) return n;
  int64_t at = t.dim() - 2;
  while (at > 0 && t.size(at) == 1) --at;       // (the stride of a single row says nothing)
  const int64_t stride = t.size(at) == 1 ? n : t.stride(at);
  int64_t next = stride * t.size(at);
  for (int64_t d = at - 1; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    TORCH_CHECK(t.stride(d) == next, op, ": the rows of ", name, " must be evenly spaced");
    next *= t.size(d);
  }
  return stride;
}

// Memory as `n` pieces of `length` bytes, `stride` bytes apart.
struct Pieces {
  const char* at;
  int64_t n, stride, length;
  const char* end() const { return at + (n - 1) * stride + length; }
};
inline Pieces pieces_of_rows(const at::Tensor& t, int64_t row_stride) {
  const int64_t hidden = t.size(-1), rows = hidden ? t.numel() / hidden : 0, size = t.element_size();
  return {(const char*)t.data_ptr(), row_stride == 0 ? std::min<int64_t>(rows, 1) : rows, row_stride * size, hidden * size};
}
// Whether a and b share bytes.  (Pieces of different strides whose spans overlap are taken to.)
inline bool overlap(const Pieces& a, const Pieces& b) {
  if (a.n == 0 || b.n == 0 || a.length == 0 || b.length == 0 || a.at >= b.end() || b.at >= a.end()) return false;
  if (a.n > 1 && b.n > 1 && a.stride != b.stride) return true;
  // columns of one buffer: where b's pieces are, modulo the stride
  const int64_t stride = a.n > 1 ? a.stride : b.stride;
  if ((a.n == 1 && b.n == 1) || stride <= 0) return true;
  const int64_t d = ((b.at - a.at) % stride + stride) % stride;
  return d < a.length || d + b.length > stride;
}

// Scratch for the multi-block sort path; empty when the single-block path runs.
inline at::Tensor sort_workspace(const at::Tensor& like, int64_t numel, int64_t buckets) {
  const size_t bytes = b200moe_sort_workspace_bytes(numel, (int)buckets);
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

}  // namespace b200shim
