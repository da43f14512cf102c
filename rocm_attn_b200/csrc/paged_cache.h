// Internal view of a paged key-value cache, shared by the kernels that read
// and write it (attn_decode.cu, kv_cache.cu) and by their host-side checks.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_kernel.h"

namespace ra {

// What a kernel needs of an AttnPagedCache.  Strides are elements over (page,
// head, row); the head dim is contiguous.
struct PagedView {
  void *k, *v;
  long long ks[3], vs[3];
  const int* table;
  long long table_stride;
  const int* lens;
  int table_width, num_pages, heads, page_size, D, B;

  // Token positions the block table can name; the host checks that it fits an
  // int with room for one tile behind it.
  __host__ __device__ int capacity() const { return table_width * page_size; }
};

// Largest capacity (table_width * page_size) the kernels take: positions,
// rounded up by a tile, stay within an int.
constexpr long long kMaxCapacity = 0x7fffffffLL - 65536;

// Checks an AttnPagedCache (everything but the device) and fills *view.
// tensors: which of k and v the call uses.  Returns ATTN_OK or the status the
// entry point reports.
constexpr int kCacheK = 1, kCacheV = 2;
int check_paged_cache(const AttnPagedCache* c, int tensors, PagedView* view);

// Compute capability 10.0 check of the current device (attn_kernel.cu), and
// its multiprocessor count (0 if it cannot be read).
int check_device();
int sm_count();
unsigned long long wait_limit_ns();  // the setting of attn_set_wait_limit_ns
int drop_arrival_requested();        // watchdog test build only

// Faults a kernel records: a page or length out of range, a wait that ran out.
constexpr int kFaultPage = 1, kFaultWait = 2;

// Copies of the fault words of the translation units into *host and resets,
// queued on `stream` (see attn_get_status).
int page_word_read_clear_decode(cudaStream_t stream, int* host);
int page_word_read_clear_cache(cudaStream_t stream, int* host);
int page_word_read_clear_pages(cudaStream_t stream, int* host);
int page_word_read_clear_tree(cudaStream_t stream, int* host);

// Attention of drafted tokens on the kernel of attn_decode.cu, whose query
// heads are then the rows (query head, token) of a kv head: whether it takes
// the call (few rows, 16-bit types, 16-byte rows), its workspace, and the
// launch, for a q of rows q_row elements apart and out as for launch_attn_tree.
bool decode_rows_plan(const AttnPagedCache* c, int Hq, int S, int sms, size_t* bytes);
bool launch_decode_rows(const AttnPagedCache* c, const PagedView& view, const void* q, long long q_b, long long q_row,
                        void* out, int Hq, int S, float scale, const int* parents, long long parents_stride,
                        const int* new_lens, void* workspace, cudaStream_t stream);

inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

#ifdef __CUDACC__
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that waits itself for the work before it in the stream
// (every thread calls grid_dependency_wait before it touches memory), so that
// its launch overlaps that work.  The wait ends when the grid before has
// completed, and so, as that grid waited too, everything before it.  Back to
// back this hides about a microsecond per kernel.  `cluster` CTAs per cluster
// (1 or 0: none); `ahead` false launches after the work before it: clusters
// that need more than half of the GPU, since eight CTAs' room at once is hard to
// find beside that work (attention of 32 units in 256 CTAs, calls in a row,
// behind / ahead, us: 16 tiles 10.3 / 11.9, 32 tiles 14.4 / 15.4; 8 tiles, which
// take 128 CTAs instead, 10.3 / 9.9).
template <typename... Params, typename... Args>
bool launch_after(void (*kern)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int cluster,
                  bool ahead, const Args&... args) {
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (ahead) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess) return true;
  cudaGetLastError();  // reported by the caller's status
  return false;
}

// (Loads of what other kernels write, lengths and tables among it, are plain
// ones throughout: a kernel launched ahead may not take the read-only path to
// memory that is still being written when it starts.)

// The length of sequence b as the kernels use it: negative lengths are empty,
// and lengths beyond the block table's capacity end there, with the fault
// recorded.
__device__ __forceinline__ int paged_len(const PagedView& c, int b, int* fault) {
  const int n = *(c.lens + b);
  if (n > c.capacity()) {
    *fault |= kFaultPage;
    return c.capacity();
  }
  return n > 0 ? n : 0;
}

// The physical page of logical page lp of sequence b, or -1, with the fault
// recorded, when the table names a page outside the cache.
__device__ __forceinline__ int paged_page(const PagedView& c, int b, int lp, int* fault) {
  const int p = *(c.table + static_cast<long long>(b) * c.table_stride + lp);
  if (static_cast<unsigned>(p) < static_cast<unsigned>(c.num_pages)) return p;
  *fault |= kFaultPage;
  return -1;
}
#endif

}  // namespace ra
