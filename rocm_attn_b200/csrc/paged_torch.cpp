// PyTorch binding of the paged key-value cache operators, part of the module
// `rocm_attn_ext` (attn_torch.cpp).  Checks the tensors, allocates outputs and
// workspaces with the caching allocator (each call its own workspace, so calls
// on other streams and captured graphs share none) and queues the work on the
// current stream of the tensors' device.
#include "paged_torch.h"

namespace {

// q [B, Hq, 1, D] of the cache's type; strides over (batch, head).
Tensor check_q(const Tensor& q, const Cache& c, long long* strides) {
  TORCH_CHECK(q.dim() == 4, "q must be 4D [B, Hq, 1, D]");
  TORCH_CHECK(q.size(2) == 1, "q must have one token per sequence: [B, Hq, 1, D]");
  TORCH_CHECK(q.size(0) == c.c.B, "q's batch size must match seq_lens");
  TORCH_CHECK(q.size(3) == c.c.D, "q's head dim must match the cache");
  TORCH_CHECK(q.size(1) <= INT32_MAX && q.size(1) % c.c.heads == 0,
              "q's heads must be a multiple of the cache's heads");
  Tensor x = q.size(3) > 1 && q.stride(3) != 1 ? q.contiguous() : q;
  strides[1] = x.size(1) > 1 ? x.stride(1) : x.size(3);
  strides[0] = x.size(0) > 1 ? x.stride(0) : strides[1] * x.size(1);
  return x;
}

// weights [B, heads, >= W * page_size] fp32; strides over (batch, head).
void check_weights(const Tensor& w, const Cache& c, long long* strides) {
  check_cuda(w, "weights");
  TORCH_CHECK(w.scalar_type() == torch::kFloat32, "weights must be float32");
  TORCH_CHECK(w.dim() == 3 && w.size(0) == c.c.B && w.size(1) == c.c.heads, "weights must be 3D [B, Hkv, n]");
  TORCH_CHECK(w.size(2) >= static_cast<int64_t>(c.c.table_width) * c.c.page_size,
              "weights must have room for W * page_size tokens");
  TORCH_CHECK(w.device() == c.device, "weights must be on the same device as the cache");
  check_unit_inner(w, "weights");
  strides_of(w, 0, 2, strides);
}

Tensor attn_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                   const Tensor& seq_lens, double scale, const OptTensor& pages, const OptTensor& weights) {
  check_cuda(q, "q");
  check_cache_tensor(k_cache, "k_cache");
  check_cache_tensor(v_cache, "v_cache");
  const c10::Device dev = k_cache.device();
  TORCH_CHECK(q.device() == dev, "q and the cache must be on the same device");
  TORCH_CHECK(q.scalar_type() == k_cache.scalar_type(), "q and the cache must have the same dtype");
  TORCH_CHECK(!(pages && weights), "pages and weights cannot be given together");
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, &v_cache, block_table, seq_lens, dev);
  long long qs[2], ws[2] = {0, 0};
  const Tensor x = check_q(q, c, qs);
  const int Hq = static_cast<int>(q.size(1));
  Tensor list;
  int n_pages = 0;
  if (pages) {
    list = int_tensor(*pages, "pages", 3, dev).contiguous();
    TORCH_CHECK(list.size(0) == c.c.B && list.size(1) == c.c.heads, "pages must be [B, Hkv, n]");
    TORCH_CHECK(list.size(2) * c.c.page_size <= 0x7fffffffLL - 65536, "pages names too many tokens");
    n_pages = static_cast<int>(list.size(2));
  }
  if (weights) {
    check_weights(*weights, c, ws);
    check_written(*weights, "weights");
  }
  Tensor out = torch::empty({q.size(0), q.size(1), 1, q.size(3)}, q.options());
  if (out.numel() == 0) return out;
  size_t bytes = 0;
  check_launch(attn_decode_workspace_bytes(&c.c, Hq, pages.has_value(), n_pages, weights.has_value(), &bytes),
               "attn_decode_workspace_bytes");
  const Tensor space = bytes > 0 ? workspace(bytes, dev) : out;  // nothing is written to an empty workspace
  // an empty list has no data, but is a list all the same
  static const int none = 0;
  const int* list_ptr = !pages ? nullptr : n_pages > 0 ? list.data_ptr<int>() : &none;
  check_launch(launch_attn_decode(&c.c, x.data_ptr(), qs, out.data_ptr(), Hq, static_cast<float>(scale), list_ptr,
                                  n_pages, weights ? weights->data_ptr<float>() : nullptr, weights ? ws : nullptr,
                                  space.data_ptr(), bytes, stream_of(dev)),
               "launch_attn_decode");
  return out;
}

void kv_append(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache,
               const Tensor& block_table, const Tensor& seq_lens, const OptTensor& new_lens, const OptTensor& bounds) {
  check_cache_tensor(k_cache, "k_cache");
  check_cache_tensor(v_cache, "v_cache");
  check_written(k_cache, "k_cache");
  check_written(v_cache, "v_cache");
  const c10::Device dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, &v_cache, block_table, seq_lens, dev);
  auto rows = [&](const Tensor& t, const char* name, long long* s) {
    check_cuda(t, name);
    TORCH_CHECK(t.device() == dev, name, " and the cache must be on the same device");
    TORCH_CHECK(t.scalar_type() == k_cache.scalar_type(), name, " and the cache must have the same dtype");
    TORCH_CHECK(t.dim() == 4 && t.size(0) == c.c.B && t.size(1) == c.c.heads && t.size(3) == c.c.D, name,
                " must be [B, Hkv, S, D] with the cache's heads and head dim");
    Tensor x = t.size(3) > 1 && t.stride(3) != 1 ? t.contiguous() : t;
    strides_of(x, 0, 3, s);
    return x;
  };
  long long ks[3], vs[3], bs[3] = {0, 0, 0};
  const Tensor x = rows(k, "k", ks), y = rows(v, "v", vs);
  TORCH_CHECK(x.size(2) == y.size(2), "k and v must have the same number of tokens");
  TORCH_CHECK(x.size(2) <= INT32_MAX, "sizes must fit in 32-bit integers");
  Tensor n;
  if (new_lens) {
    n = int_tensor(*new_lens, "new_lens", 1, dev).contiguous();
    TORCH_CHECK(n.size(0) == c.c.B, "new_lens must have the batch size of seq_lens");
  }
  if (bounds) {
    check_bounds(*bounds, c.c.num_pages, c.c.heads, c.c.D, k_cache, bs);
    check_written(*bounds, "bounds");
  }
  if (x.numel() == 0) return;
  check_launch(launch_kv_append(&c.c, x.data_ptr(), ks, y.data_ptr(), vs, static_cast<int>(x.size(2)),
                                new_lens ? n.data_ptr<int>() : nullptr, bounds ? bounds->data_ptr() : nullptr,
                                bounds ? bs : nullptr, stream_of(dev)),
               "launch_kv_append");
}

Tensor kv_page_bounds(const Tensor& k_cache, const Tensor& block_table, const Tensor& seq_lens,
                      const OptTensor& bounds) {
  check_cache_tensor(k_cache, "k_cache");
  const c10::Device dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, nullptr, block_table, seq_lens, dev);
  Tensor out;
  long long bs[3];
  if (bounds) {
    out = *bounds;
    check_bounds(out, c.c.num_pages, c.c.heads, c.c.D, k_cache, bs);
    check_written(out, "bounds");
  } else {
    out = torch::zeros({c.c.num_pages, c.c.heads, 2, c.c.D}, k_cache.options());
    strides_of(out, 0, 3, bs);
  }
  if (c.c.B == 0) return out;
  check_launch(launch_kv_page_bounds(&c.c, out.data_ptr(), bs, stream_of(dev)), "launch_kv_page_bounds");
  return out;
}

Tensor kv_select_pages(const Tensor& q, const Tensor& bounds, const Tensor& block_table, const Tensor& seq_lens,
                       int64_t page_size, int64_t top) {
  check_cuda(q, "q");
  check_cuda(bounds, "bounds");
  check_float(bounds, "bounds");
  TORCH_CHECK(bounds.dim() == 4 && bounds.size(2) == 2, "bounds must be [num_pages, Hkv, 2, D]");
  TORCH_CHECK(q.device() == bounds.device(), "q and bounds must be on the same device");
  TORCH_CHECK(q.scalar_type() == bounds.scalar_type(), "q and bounds must have the same dtype");
  TORCH_CHECK(top >= 1 && top <= INT32_MAX, "top must be at least 1");
  const c10::Device dev = bounds.device();
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(nullptr, nullptr, block_table, seq_lens, dev);
  c.shape(bounds.size(0), bounds.size(1), page_size, bounds.size(3), bounds);
  long long bs[3], qs[2];
  check_bounds(bounds, bounds.size(0), bounds.size(1), bounds.size(3), bounds, bs);
  const Tensor x = check_q(q, c, qs);
  Tensor pages = torch::empty({c.c.B, c.c.heads, top}, torch::dtype(torch::kInt32).device(dev));
  if (c.c.B == 0) return pages;
  size_t bytes = 0;
  check_launch(kv_select_pages_workspace_bytes(&c.c, &bytes), "kv_select_pages_workspace_bytes");
  const Tensor space = workspace(bytes, dev);
  check_launch(launch_kv_select_pages(&c.c, x.data_ptr(), qs, static_cast<int>(q.size(1)), bounds.data_ptr(), bs,
                                      static_cast<int>(top), pages.data_ptr<int>(), space.data_ptr(), bytes,
                                      stream_of(dev)),
               "launch_kv_select_pages");
  return pages;
}

std::tuple<Tensor, Tensor, Tensor> kv_evict(const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table,
                                            const Tensor& seq_lens, const Tensor& weights,
                                            const Tensor& new_block_table, int64_t budget, int64_t recent) {
  check_cache_tensor(k_cache, "k_cache");
  check_cache_tensor(v_cache, "v_cache");
  check_written(k_cache, "k_cache");
  check_written(v_cache, "v_cache");
  const c10::Device dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  Cache c(&k_cache, &v_cache, block_table, seq_lens, dev);
  long long ws[2];
  check_weights(weights, c, ws);
  Tensor to = int_tensor(new_block_table, "new_block_table", 2, dev);
  if (to.size(1) > 1 && to.stride(1) != 1) to = to.contiguous();
  TORCH_CHECK(to.size(0) == c.c.B, "new_block_table must have the batch size of block_table");
  const int64_t width = to.size(1), room = width * c.c.page_size;
  TORCH_CHECK(width <= INT32_MAX && room <= 0x7fffffffLL - 65536, "new_block_table names too many tokens");
  TORCH_CHECK(budget >= 1 && budget <= room, "budget must be between 1 and the tokens new_block_table has room for");
  TORCH_CHECK(recent >= 0 && recent <= budget, "recent must be between 0 and budget");
  const auto ints = torch::dtype(torch::kInt32).device(dev);
  Tensor new_lens = torch::empty({c.c.B}, ints);
  Tensor new_weights = torch::empty({c.c.B, c.c.heads, room}, weights.options());
  Tensor kept = torch::empty({c.c.B, c.c.heads, budget}, ints);
  if (c.c.B > 0)
    check_launch(launch_kv_evict(&c.c, weights.data_ptr<float>(), ws, to.data_ptr<int>(),
                                 to.size(0) > 1 ? to.stride(0) : width, static_cast<int>(width),
                                 static_cast<int>(budget), static_cast<int>(recent), new_weights.data_ptr<float>(),
                                 kept.data_ptr<int>(), new_lens.data_ptr<int>(), stream_of(dev)),
                 "launch_kv_evict");
  return {new_lens, new_weights, kept};
}

}  // namespace

void bind_paged(py::module& m) {
  m.def("attn_decode", &attn_decode, "Attention of one new token per sequence over a paged cache", py::arg("q"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"), py::arg("scale") = -1.0,
        py::arg("pages") = py::none(), py::arg("weights") = py::none());
  m.def("kv_append", &kv_append, "Write new tokens to a paged cache", py::arg("k"), py::arg("v"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"), py::arg("new_lens") = py::none(),
        py::arg("bounds") = py::none());
  m.def("kv_page_bounds", &kv_page_bounds, "Elementwise bounds of the keys of each page", py::arg("k_cache"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("bounds") = py::none());
  m.def("kv_select_pages", &kv_select_pages, "Pages of largest score for a new token", py::arg("q"), py::arg("bounds"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("page_size"), py::arg("top"));
  m.def("kv_evict", &kv_evict, "Keep the tokens of largest accumulated weight", py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("weights"), py::arg("new_block_table"), py::arg("budget"),
        py::arg("recent") = 0);
}
