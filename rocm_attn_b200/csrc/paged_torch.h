// What the PyTorch bindings of the paged key-value cache operators share
// (paged_torch.cpp, branches_torch.cpp): the checks of their tensors, the
// AttnPagedCache of a call, workspaces and streams.
#pragma once

#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <optional>
#include <tuple>

#include "attn_kernel.h"

namespace py = pybind11;
using torch::Tensor;
using OptTensor = std::optional<Tensor>;

const char* status_text(int s);

namespace {

void check_launch(int st, const char* what) {
  TORCH_CHECK(st == ATTN_OK, what, ": ", status_text(st), " (status ", st, ")");
}

void check_cuda(const Tensor& t, const char* name) { TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor"); }

void check_float(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kFloat16 ||
                  t.scalar_type() == torch::kBFloat16,
              name, " must be float32, float16, or bfloat16");
}

// A device tensor of 32-bit integers that belongs to the cache on `dev`.
Tensor int_tensor(const Tensor& t, const char* name, int64_t dim, const c10::Device& dev) {
  check_cuda(t, name);
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == dim, name, " must be ", dim, "D");
  TORCH_CHECK(t.device() == dev, name, " must be on the same device as the cache");
  return t;
}

void check_unit_inner(const Tensor& t, const char* name) {
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have a contiguous last dim");
}

// Tensors a kernel writes to: no two of their elements in one place.
void check_written(const Tensor& t, const char* name) {
  TORCH_CHECK(at::has_internal_overlap(t) != at::MemOverlap::Yes, name, " must not be an expanded tensor");
}

// Element strides over the n dims from `first`; a dim of size 1 may carry any
// stride in torch and gets one of the contiguous layout.
void strides_of(const Tensor& t, int first, int n, long long* s) {
  long long next = t.size(-1);
  for (int64_t d = t.dim() - 2; d >= first + n; --d) next *= t.size(d);
  for (int i = n - 1; i >= 0; --i) {
    s[i] = t.size(first + i) <= 1 ? next : t.stride(first + i);
    next = s[i] * (t.size(first + i) > 0 ? t.size(first + i) : 1);
  }
}

AttnDType dtype_of(const Tensor& t) {
  return t.scalar_type() == torch::kFloat16 ? ATTN_F16 : t.scalar_type() == torch::kBFloat16 ? ATTN_BF16 : ATTN_F32;
}

// The AttnPagedCache of a call, and the tensors it points into.
struct Cache {
  AttnPagedCache c = {};
  Tensor table, lens;
  c10::Device device;

  // k, v: [num_pages, Hkv, page_size, D]; either may be absent (no tensor),
  // then the shape is set by the caller.
  Cache(const Tensor* k, const Tensor* v, const Tensor& block_table, const Tensor& seq_lens, const c10::Device& dev)
      : device(dev) {
    table = int_tensor(block_table, "block_table", 2, dev);
    if (table.size(1) > 1 && table.stride(1) != 1) table = table.contiguous();
    lens = int_tensor(seq_lens, "seq_lens", 1, dev).contiguous();
    TORCH_CHECK(table.size(0) == lens.size(0), "block_table and seq_lens must have the same batch size");
    TORCH_CHECK(table.size(0) <= INT32_MAX && table.size(1) <= INT32_MAX, "sizes must fit in 32-bit integers");
    c.block_table = table.data_ptr<int>();
    c.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
    c.table_width = static_cast<int>(table.size(1));
    c.seq_lens = lens.data_ptr<int>();
    c.B = static_cast<int>(lens.size(0));
    if (k) {
      shape(k->size(0), k->size(1), k->size(2), k->size(3), *k);
      c.k = k->data_ptr();
      strides_of(*k, 0, 3, c.k_strides);
    }
    if (v) {
      TORCH_CHECK(v->sizes() == k->sizes(), "k_cache and v_cache must have the same shape");
      TORCH_CHECK(v->scalar_type() == k->scalar_type(), "k_cache and v_cache must have the same dtype");
      TORCH_CHECK(v->device() == dev, "k_cache and v_cache must be on the same device");
      check_unit_inner(*v, "v_cache");
      c.v = v->data_ptr();
      strides_of(*v, 0, 3, c.v_strides);
    }
  }

  void shape(int64_t pages, int64_t heads, int64_t page_size, int64_t D, const Tensor& like) {
    TORCH_CHECK(pages <= INT32_MAX && heads <= INT32_MAX && page_size <= INT32_MAX && D <= INT32_MAX,
                "sizes must fit in 32-bit integers");
    TORCH_CHECK(heads >= 1 && page_size >= 1 && D >= 1, "heads, page size and head dim must be at least 1");
    TORCH_CHECK(page_size * c.table_width <= 0x7fffffffLL - 65536,
                "the block table names too many tokens: W * page_size must be at most 2^31 - 65537");
    c.num_pages = static_cast<int>(pages);
    c.heads = static_cast<int>(heads);
    c.page_size = static_cast<int>(page_size);
    c.D = static_cast<int>(D);
    c.dtype = dtype_of(like);
  }
};

void check_cache_tensor(const Tensor& t, const char* name) {
  check_cuda(t, name);
  check_float(t, name);
  TORCH_CHECK(t.dim() == 4, name, " must be 4D [num_pages, Hkv, page_size, D]");
  check_unit_inner(t, name);
}

// bounds [num_pages, Hkv, 2, D] like the cache's keys.
void check_bounds(const Tensor& b, int64_t pages, int64_t heads, int64_t D, const Tensor& like, long long* strides) {
  check_cuda(b, "bounds");
  TORCH_CHECK(b.dim() == 4 && b.size(0) == pages && b.size(1) == heads && b.size(2) == 2 && b.size(3) == D,
              "bounds must be [num_pages, Hkv, 2, D]");
  TORCH_CHECK(b.scalar_type() == like.scalar_type(), "bounds must have the cache's dtype");
  TORCH_CHECK(b.device() == like.device(), "bounds must be on the same device as the cache");
  check_unit_inner(b, "bounds");
  strides_of(b, 0, 3, strides);
}

Tensor workspace(size_t bytes, const c10::Device& dev) {
  return torch::empty({static_cast<int64_t>(bytes > 0 ? bytes : 16)}, torch::dtype(torch::kUInt8).device(dev));
}

cudaStream_t stream_of(const c10::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

}  // namespace
