// PyTorch binding of the operators for drafted tokens and shared pages on the
// paged key-value cache, part of the module `rocm_attn_ext` (attn_torch.cpp).
#include "paged_torch.h"

namespace {

// An int32 vector of n entries of the cache's device, read by a kernel.
Tensor int_vector(const Tensor& t, const char* name, int64_t n, const char* like, const c10::Device& dev) {
  Tensor x = int_tensor(t, name, 1, dev).contiguous();
  TORCH_CHECK(x.size(0) == n, name, " must have the batch size of ", like);
  return x;
}

// One that a kernel changes in place.
void check_changed(const Tensor& t, const char* name, int64_t n, const c10::Device& dev) {
  int_tensor(t, name, 1, dev);
  TORCH_CHECK(n < 0 || t.size(0) == n, name, " must have the batch size of block_table");
  TORCH_CHECK(t.is_contiguous(), name, " is changed in place and must be contiguous");
}

// Rows of int32, contiguous or copied; the entries from one row to the next.
Tensor int_rows(const Tensor& t, const char* name, int64_t rows, const c10::Device& dev, long long* stride) {
  Tensor x = int_tensor(t, name, 2, dev);
  TORCH_CHECK(x.size(0) == rows, name, " must have the batch size of block_table");
  if (x.size(1) > 1 && x.stride(1) != 1) x = x.contiguous();
  *stride = x.size(0) > 1 ? x.stride(0) : x.size(1);
  return x;
}

Tensor attn_tree(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                 const Tensor& seq_lens, const OptTensor& parents, const OptTensor& new_lens, double scale) {
  check_cuda(q, "q");
  check_cache_tensor(k_cache, "k_cache");
  check_cache_tensor(v_cache, "v_cache");
  const c10::Device dev = k_cache.device();
  TORCH_CHECK(q.device() == dev, "q and the cache must be on the same device");
  TORCH_CHECK(q.scalar_type() == k_cache.scalar_type(), "q and the cache must have the same dtype");
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, &v_cache, block_table, seq_lens, dev);
  TORCH_CHECK(q.dim() == 4, "q must be 4D [B, Hq, S, D]");
  TORCH_CHECK(q.size(0) == c.c.B, "q's batch size must match seq_lens");
  TORCH_CHECK(q.size(3) == c.c.D, "q's head dim must match the cache");
  TORCH_CHECK(q.size(1) <= INT32_MAX && q.size(1) % c.c.heads == 0,
              "q's heads must be a multiple of the cache's heads");
  TORCH_CHECK(q.size(2) <= 1024, "at most 1024 drafted tokens per sequence");
  const int Hq = static_cast<int>(q.size(1)), S = static_cast<int>(q.size(2));
  Tensor x = q.size(3) > 1 && q.stride(3) != 1 ? q.contiguous() : q;
  long long qs[3], tree_stride = 0;
  strides_of(x, 0, 3, qs);
  // a copy of a q whose rows are not 16-byte aligned costs less than the kernel that could read it
  const int64_t vec = 16 / x.element_size();
  if (c.c.D % vec == 0 && (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || qs[0] % vec || qs[1] % vec || qs[2] % vec)) {
    x = x.clone(at::MemoryFormat::Contiguous);
    strides_of(x, 0, 3, qs);
  }
  Tensor tree, n;
  if (parents) {
    tree = int_rows(*parents, "parents", c.c.B, dev, &tree_stride);
    TORCH_CHECK(tree.size(1) == S, "parents must be [B, S]");
  }
  if (new_lens) n = int_vector(*new_lens, "new_lens", c.c.B, "seq_lens", dev);
  Tensor out = torch::empty({q.size(0), q.size(1), q.size(2), q.size(3)}, q.options());
  if (out.numel() == 0) return out;
  size_t bytes = 0;
  check_launch(attn_tree_workspace_bytes(&c.c, Hq, S, &bytes), "attn_tree_workspace_bytes");
  const Tensor space = workspace(bytes, dev);
  check_launch(launch_attn_tree(&c.c, x.data_ptr(), qs, out.data_ptr(), Hq, S, static_cast<float>(scale),
                                parents ? tree.data_ptr<int>() : nullptr, tree_stride,
                                new_lens ? n.data_ptr<int>() : nullptr, space.data_ptr(), bytes, stream_of(dev)),
               "launch_attn_tree");
  return out;
}

Tensor kv_compact(const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& seq_lens,
                  const Tensor& kept, const Tensor& new_lens, const OptTensor& bounds) {
  check_cache_tensor(k_cache, "k_cache");
  check_cache_tensor(v_cache, "v_cache");
  check_written(k_cache, "k_cache");
  check_written(v_cache, "v_cache");
  const c10::Device dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, &v_cache, block_table, seq_lens, dev);
  long long stride;
  const Tensor list = int_rows(kept, "kept", c.c.B, dev, &stride);
  TORCH_CHECK(list.size(1) <= INT32_MAX, "sizes must fit in 32-bit integers");
  const Tensor n = int_vector(new_lens, "new_lens", c.c.B, "seq_lens", dev);
  long long bs[3] = {0, 0, 0};
  if (bounds) {
    check_bounds(*bounds, c.c.num_pages, c.c.heads, c.c.D, k_cache, bs);
    check_written(*bounds, "bounds");
  }
  Tensor lens = torch::empty({c.c.B}, torch::dtype(torch::kInt32).device(dev));
  if (c.c.B > 0)
    check_launch(launch_kv_compact_bounds(&c.c, n.data_ptr<int>(), list.data_ptr<int>(), stride,
                                          static_cast<int>(list.size(1)), lens.data_ptr<int>(),
                                          bounds ? bounds->data_ptr() : nullptr, bs, stream_of(dev)),
                 "launch_kv_compact");
  return lens;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> kv_fork(const Tensor& k_cache, const Tensor& v_cache,
                                                   const Tensor& block_table, const Tensor& held,
                                                   const Tensor& seq_lens, const Tensor& refs, const Tensor& parents,
                                                   const OptTensor& bounds) {
  check_cache_tensor(k_cache, "k_cache");
  check_cache_tensor(v_cache, "v_cache");
  check_written(k_cache, "k_cache");
  check_written(v_cache, "v_cache");
  const c10::Device dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, &v_cache, block_table, seq_lens, dev);
  const Tensor have = int_vector(held, "held", c.c.B, "block_table", dev);
  check_changed(refs, "refs", -1, dev);
  TORCH_CHECK(refs.size(0) == c.c.num_pages, "refs must have an entry for each page of the cache");
  const Tensor from = int_tensor(parents, "parents", 1, dev).contiguous();
  TORCH_CHECK(from.size(0) <= INT32_MAX, "sizes must fit in 32-bit integers");
  const int n = static_cast<int>(from.size(0));
  long long bs[3] = {0, 0, 0};
  if (bounds) {
    check_bounds(*bounds, c.c.num_pages, c.c.heads, c.c.D, k_cache, bs);
    check_written(*bounds, "bounds");
  }
  const auto ints = torch::dtype(torch::kInt32).device(dev);
  Tensor new_table = torch::empty({n, c.c.table_width}, ints), new_held = torch::empty({n}, ints),
         new_lens = torch::empty({n}, ints), missing = torch::empty({1}, ints);
  size_t bytes = 0;
  check_launch(kv_fork_workspace_bytes(&c.c, n, &bytes), "kv_fork_workspace_bytes");
  const Tensor space = workspace(bytes, dev);
  check_launch(launch_kv_fork_bounds(&c.c, have.data_ptr<int>(), refs.data_ptr<int>(), from.data_ptr<int>(), n,
                                     new_table.data_ptr<int>(), new_held.data_ptr<int>(), new_lens.data_ptr<int>(),
                                     missing.data_ptr<int>(), bounds ? bounds->data_ptr() : nullptr, bs,
                                     space.data_ptr(), bytes, stream_of(dev)),
               "launch_kv_fork");
  return {new_table, new_held, new_lens, missing};
}

Tensor kv_resize(const Tensor& block_table, const Tensor& held, const Tensor& seq_lens, const Tensor& refs,
                 int64_t page_size) {
  check_cuda(block_table, "block_table");
  const c10::Device dev = block_table.device();
  const c10::cuda::CUDAGuard guard(dev);
  check_written(block_table, "block_table");
  TORCH_CHECK(block_table.dim() != 2 || block_table.size(1) <= 1 || block_table.stride(1) == 1,
              "block_table is changed in place and must have contiguous rows");
  Cache c(nullptr, nullptr, block_table, seq_lens, dev);
  check_changed(held, "held", c.c.B, dev);
  check_changed(refs, "refs", -1, dev);
  c.shape(refs.size(0), 1, page_size, 1, refs);
  Tensor missing = torch::empty({c.c.B}, torch::dtype(torch::kInt32).device(dev));
  if (c.c.B == 0) return missing;
  size_t bytes = 0;
  check_launch(kv_resize_workspace_bytes(&c.c, &bytes), "kv_resize_workspace_bytes");
  const Tensor space = workspace(bytes, dev);
  check_launch(launch_kv_resize(&c.c, c.table.data_ptr<int>(), held.data_ptr<int>(), refs.data_ptr<int>(),
                                missing.data_ptr<int>(), space.data_ptr(), bytes, stream_of(dev)),
               "launch_kv_resize");
  return missing;
}

}  // namespace

void bind_branches(py::module& m) {
  m.def("attn_tree", &attn_tree, "Attention of drafted tokens over a paged cache", py::arg("q"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"), py::arg("parents") = py::none(),
        py::arg("new_lens") = py::none(), py::arg("scale") = -1.0);
  m.def("kv_compact", &kv_compact, "Move accepted drafted tokens to their places", py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"), py::arg("kept"), py::arg("new_lens"),
        py::arg("bounds") = py::none());
  m.def("kv_fork", &kv_fork, "Sequences that continue others, full pages shared", py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("held"), py::arg("seq_lens"), py::arg("refs"),
        py::arg("parents"), py::arg("bounds") = py::none());
  m.def("kv_resize", &kv_resize, "Hold the pages that lengths need", py::arg("block_table"), py::arg("held"),
        py::arg("seq_lens"), py::arg("refs"), py::arg("page_size"));
}
