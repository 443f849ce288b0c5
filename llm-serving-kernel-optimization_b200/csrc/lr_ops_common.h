// lr_ops_common.h -- argument checks shared by the torch custom-op sources.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "../../include/lightning_router.h"

namespace lr_ops {

inline void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == LR_OK, "lightning_router.", what, " failed: ", lr_status_string(rc), " (",
              rc, ")");
}

inline lr_stream_t cur_stream() {
  return reinterpret_cast<lr_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

inline void check_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// A size as the C interface's int.
inline int as_int(int64_t n) {
  TORCH_CHECK(n >= 0 && n <= 0x7fffffff, "lightning_router: a size of ", n, " is out of range");
  return static_cast<int>(n);
}

inline int32_t* err_ptr(const c10::optional<at::Tensor>& err) {
  if (!err.has_value() || !err->defined()) return nullptr;
  TORCH_CHECK(err->is_cuda() && err->scalar_type() == at::kInt && err->numel() >= 1,
              "err must be a CUDA int32 tensor");
  return err->data_ptr<int32_t>();
}

inline at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes < 16 ? 16 : bytes)},
                   like.options().dtype(at::kByte));
}

// Kernels write through raw pointers: a graph that saved `t` learns of it here.
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace lr_ops
