// Pages of a paged key-value cache changing hands: the move of accepted drafted
// tokens to their places (launch_kv_compact), the pages that lengths need
// (launch_kv_resize) and sequences that continue others (launch_kv_fork).
//
// All of them are short: a few thousand table entries, the counts of the
// pages, and for a fork the rows of a partly filled page per copy.  The time
// of small calls is that of their dependent loads (a length, a table entry, a
// count, each half a microsecond), so these are kept few and in parallel.
//
// A free page is one whose count is 0 at the start of the call; pages are
// given out from the lowest on, in the order of the sequences, so results do
// not depend on timing.  Finding them is one pass over the counts by a cluster
// of CTAs: each warp counts its stretch and keeps its bits, the cluster's prefix
// sum gives each stretch the rank of its first free page, and the pages of the
// ranks that were asked for are written to a list.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <type_traits>

#include "key_bounds.cuh"
#include "paged_cache.h"
#include "sm100_ptx.cuh"

namespace ra {

namespace {

__device__ int g_page_fault = 0;

constexpr int kFindMost = 8;  // CTAs that look for free pages, one cluster: the grid
constexpr int kFindWarps = 32;
constexpr int kFindThreads = kFindWarps * 32;
constexpr int kStep = 256;  // pages a warp looks at in one turn
constexpr int kTurnsKept = 8;  // turns whose bits are kept (half a million pages); others are looked at again
constexpr int kCopyAhead = 4;  // rows a thread copies in one turn

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_load(const int* p, int rank) {
  uint32_t at;
  int x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
  return x;
}

// ---------------------------------------------------------------------------
// Free pages
// ---------------------------------------------------------------------------

struct FindSmem {
  int warp_count[kFindWarps];
  int total;  // free pages of this CTA's stretch, read by the cluster
  long long warp_sum[kFindWarps];
  unsigned bits[kFindWarps][kTurnsKept][kStep / 32];
};

// The stretch of pages of this warp, a multiple of kStep long but for the last.
struct Stretch {
  long long lo, hi;
};
__device__ __forceinline__ Stretch stretch(int num_pages) {
  const int w = blockIdx.x * kFindWarps + (threadIdx.x >> 5);
  const long long warps = static_cast<long long>(gridDim.x) * kFindWarps;
  const long long per = ((num_pages + warps - 1) / warps + kStep - 1) / kStep * kStep;
  Stretch s{w * per, (w + 1) * per};
  if (s.lo > num_pages) s.lo = num_pages;
  if (s.hi > num_pages) s.hi = num_pages;
  return s;
}

// Which of the kStep pages from p on are free: lane i gets the bits of pages p +
// 32 i and following (lanes behind kStep / 32 nothing).
__device__ __forceinline__ unsigned free_bits(const int* refs, long long p, long long hi) {
  const int lane = threadIdx.x & 31;
  int r[kStep / 32];
#pragma unroll
  for (int i = 0; i < kStep / 32; ++i) {
    const long long at = p + i * 32 + lane;
    r[i] = at < hi ? *(refs + at) : 1;
  }
  unsigned mine = 0;
#pragma unroll
  for (int i = 0; i < kStep / 32; ++i) {
    const unsigned b = __ballot_sync(0xffffffffu, r[i] == 0);
    if (lane == i) mine = b;
  }
  return mine;
}

// Free pages of the warp's stretch.
__device__ __forceinline__ int count_free(FindSmem& sm, const int* refs, const Stretch& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n = 0, turn = 0;
#pragma unroll 2
  for (long long p = s.lo; p < s.hi; p += kStep, ++turn) {
    const unsigned b = free_bits(refs, p, s.hi);
    if (turn < kTurnsKept && lane < kStep / 32) sm.bits[warp][turn][lane] = b;
    n += __reduce_add_sync(0xffffffffu, __popc(b));
  }
  __syncwarp();
  return n;
}

// After count_free by every warp: the rank of the first free page of this
// warp's stretch, and the free pages of all.  Holds one cluster barrier.
__device__ __forceinline__ long long first_rank(FindSmem& s, int count, long long* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) s.warp_count[warp] = count;
  __syncthreads();
  if (warp == 0) {
    const int sum = __reduce_add_sync(0xffffffffu, s.warp_count[lane]);
    if (lane == 0) s.total = sum;
  }
  cluster_sync();
  long long rank = 0;
  *all = 0;
  for (int c = 0; c < static_cast<int>(gridDim.x); ++c) {
    const int x = cluster_load(&s.total, c);
    if (c < static_cast<int>(blockIdx.x)) rank += x;
    *all += x;
  }
  for (int w = 0; w < warp; ++w) rank += s.warp_count[w];
  return rank;
}

// Writes the stretch's free pages of rank below `wanted` to their places in `order`.
__device__ __forceinline__ void list_free(const FindSmem& sm, const int* refs, const Stretch& s, long long rank,
                                          long long wanted, int* order) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int turn = 0;
  for (long long p = s.lo; p < s.hi && rank < wanted; p += kStep, ++turn) {
    const unsigned mine = turn < kTurnsKept ? (lane < kStep / 32 ? sm.bits[warp][turn][lane] : 0u)
                                            : free_bits(refs, p, s.hi);
#pragma unroll 4
    for (int i = 0; i < kStep / 32; ++i) {
      const unsigned free = __shfl_sync(0xffffffffu, mine, i);
      const long long at = rank + __popc(free & ((1u << lane) - 1u));
      if ((free >> lane & 1u) && at < wanted) order[at] = static_cast<int>(p + i * 32 + lane);
      rank += __popc(free);
    }
  }
}

// Sum of `x` over the threads of the CTA before this one, and of all.
__device__ __forceinline__ long long cta_prefix(FindSmem& s, int x, long long* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long upto = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  __syncthreads();  // the sums of the turn before have been read
  if (lane == 31) s.warp_sum[warp] = upto;
  __syncthreads();
  long long before = upto - x;
  *all = 0;
#pragma unroll 8
  for (int w = 0; w < kFindWarps; ++w) {
    const long long y = s.warp_sum[w];
    if (w < warp) before += y;
    *all += y;
  }
  return before;
}

// What the table's row b holds: held[b], or the nearest count that its width allows.
__device__ __forceinline__ int held_pages(const PagedView& c, const int* held, int b, int* fault) {
  const int n = *(held + b);
  if (n >= 0 && n <= c.table_width) return n;
  *fault |= kFaultPage;
  return n < 0 ? 0 : c.table_width;
}

// Changes the counts of the pages that row[first], row[first + step], ... below
// `end` name by by_of(index) (0: none): kBatch entries, then as many counts, on
// their way at once, as each takes the better part of a microsecond.
constexpr int kBatch = 8;
template <typename By>
__device__ __forceinline__ void change_refs(const PagedView& c, int* refs, const int* row, long long first,
                                            long long end, int step, By by_of, int* fault) {
  for (long long j = first; j < end; j += static_cast<long long>(kBatch) * step) {
    int page[kBatch], by[kBatch], was[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const long long at = j + static_cast<long long>(k) * step;
      by[k] = at < end ? by_of(at) : 0;
      page[k] = by[k] != 0 ? row[at] : 0;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      was[k] = 0;
      if (by[k] == 0) continue;
      if (static_cast<unsigned>(page[k]) >= static_cast<unsigned>(c.num_pages)) {
        *fault |= kFaultPage;
        by[k] = 0;
      } else {
        was[k] = atomicAdd(refs + page[k], by[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (was[k] + by[k] < 0) *fault |= kFaultPage;
  }
}

// ---------------------------------------------------------------------------
// The pages that lengths need
// ---------------------------------------------------------------------------

struct ResizeArgs {
  PagedView c;
  int *table, *held, *refs, *missing;
  int *have, *start;  // [B] workspace (rows from kFindThreads on): held pages, rank of the first page taken
  int* order;         // workspace: free pages by rank
};

__global__ void __launch_bounds__(kFindThreads) kv_resize_kernel(const __grid_constant__ ResizeArgs a) {
  __shared__ FindSmem s;
  __shared__ int s_have[kFindThreads], s_start[kFindThreads];
  launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int fault = 0;
  auto want_of = [&](int b) {
    const int len = paged_len(a.c, b, &fault);
    return static_cast<int>((static_cast<long long>(len) + a.c.page_size - 1) / a.c.page_size);
  };
  // What each sequence lacks, and the sum of it over those before: all of it
  // in every CTA, which saves a barrier.
  long long wanted = 0;
  for (long long b0 = 0; b0 < a.c.B; b0 += kFindThreads) {
    const long long b = b0 + threadIdx.x;
    int have = 0, need = 0;
    if (b < a.c.B) {
      have = held_pages(a.c, a.held, b, &fault);
      need = max(0, want_of(b) - have);
    }
    long long all;
    const long long at = wanted + cta_prefix(s, need, &all);
    const int start = static_cast<int>(at < INT_MAX ? at : INT_MAX);
    if (b0 == 0) {
      s_have[threadIdx.x] = have;
      s_start[threadIdx.x] = start;
    } else if (b < a.c.B && blockIdx.x == 0) {
      a.have[b] = have;
      a.start[b] = start;
    }
    wanted += all;
  }
  long long free = 0;
  if (wanted > 0) {
    const Stretch mine = stretch(a.c.num_pages);
    const long long rank = first_rank(s, count_free(s, a.refs, mine), &free);
    list_free(s, a.refs, mine, rank, wanted, a.order);
  }
  cluster_sync();
  // Several warps to a sequence where there are few.
  const int all_warps = gridDim.x * kFindWarps, split = a.c.B < all_warps ? all_warps / a.c.B : 1;
  const long long w = static_cast<long long>(blockIdx.x) * kFindWarps + warp;
  for (long long u = w; u < static_cast<long long>(a.c.B) * split; u += all_warps) {
    const int b = static_cast<int>(u / split), part = static_cast<int>(u % split);
    const int have = b < kFindThreads ? s_have[b] : a.have[b], start = b < kFindThreads ? s_start[b] : a.start[b];
    const int want = want_of(b);
    int* row = a.table + b * a.c.table_stride;
    const bool granted = want <= have || static_cast<long long>(start) + (want - have) <= free;
    if (granted) {
#pragma unroll 8
      for (long long j = static_cast<long long>(have) + part * 32 + lane; j < want; j += split * 32) {
        const int page = *(a.order + start + (j - have));
        row[j] = page;
        a.refs[page] = 1;
      }
    }
    change_refs(a.c, a.refs, row, static_cast<long long>(want) + part * 32 + lane, have, split * 32,
                [](long long) { return -1; }, &fault);
    if (part == 0 && lane == 0) {
      a.held[b] = granted ? want : have;
      a.missing[b] = granted ? 0 : want - have;
    }
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Sequences that continue others
// ---------------------------------------------------------------------------

struct ForkArgs {
  PagedView c;
  const int *held, *parents;
  int* refs;
  int n;
  int *new_table, *new_held, *new_lens, *missing;
  int *first, *kids;  // [B] workspace: the first sequence that continues this one, and how many do
  int4* copy;         // [n] workspace, of the new sequence: parent, tokens, page to copy (or none), rank of the free page
  int2* list;         // [n] workspace, by rank of the free page: page to copy and its rows
  int* copies;        // workspace: how many
  int* order;         // workspace: free pages by rank
  int cols;           // 16-byte (or element) columns of a row
  int chunks;         // CTAs per head's K (or V) rows of a copied page
  void* bounds;             // page bounds, or null: a copied page's go with it
  long long b_p, b_h, b_m;  // their strides over (page, head, min/max)
};

// A new sequence's parent and what it takes from it: len tokens in `full` full
// pages and `rest` rows of another.
struct Branch {
  int parent, len, full, rest;
};
__device__ __forceinline__ Branch branch_of_parent(const ForkArgs& a, int parent, int* fault) {
  const int have = held_pages(a.c, a.held, parent, fault), room = have * a.c.page_size;
  int len = paged_len(a.c, parent, fault);
  if (len > room) {
    *fault |= kFaultPage;
    len = room;
  }
  const int full = len / a.c.page_size;
  return Branch{parent, len, full, len - full * a.c.page_size};
}
__device__ __forceinline__ Branch branch_of(const ForkArgs& a, int i, int* fault) {
  const int parent = *(a.parents + i);
  if (parent >= 0 && parent < a.c.B) return branch_of_parent(a, parent, fault);
  if (parent != -1) *fault |= kFaultPage;
  return Branch{-1, 0, 0, 0};
}

// Which new sequences copy their last page, and where to: one cluster.
__global__ void __launch_bounds__(kFindThreads) kv_fork_plan_kernel(const __grid_constant__ ForkArgs a) {
  __shared__ FindSmem s;
  launch_dependents();
  grid_dependency_wait();
  int fault = 0;
  const long long id = static_cast<long long>(blockIdx.x) * kFindThreads + threadIdx.x;
  for (long long b = id; b < a.c.B; b += gridDim.x * kFindThreads) {
    a.first[b] = INT_MAX;
    a.kids[b] = 0;
  }
  // A new sequence, its partly filled page (-1: none) and whether others hold that too.
  struct Want {
    Branch br;
    int page;
    bool shared;
  };
  auto look = [&](long long i) {
    Want w{{-1, 0, 0, 0}, -1, false};
    if (i < a.n) {
      w.br = branch_of(a, static_cast<int>(i), &fault);
      if (w.br.rest > 0) w.page = paged_page(a.c, w.br.parent, w.br.full, &fault);
      if (w.page >= 0) w.shared = *(a.refs + w.page) != 1;
    }
    return w;
  };
  Want want = look(threadIdx.x);  // ahead of the barriers: four loads that wait for one another
  cluster_sync();
  for (long long i = id; i < a.n; i += gridDim.x * kFindThreads) {
    const int parent = *(a.parents + i);
    if (parent >= 0 && parent < a.c.B) {
      atomicMin(a.first + parent, static_cast<int>(i));
      atomicAdd(a.kids + parent, 1);
    }
  }
  const Stretch mine = stretch(a.c.num_pages);
  long long free;
  const long long rank = first_rank(s, count_free(s, a.refs, mine), &free);  // a cluster barrier: first is complete
  long long wanted = 0;
  for (long long i0 = 0; i0 < a.n; i0 += kFindThreads) {
    const long long i = i0 + threadIdx.x;
    if (i0 > 0) want = look(i);
    const bool copies = want.page >= 0 && (want.shared || a.first[want.br.parent] != i);
    long long all;
    const long long at = wanted + cta_prefix(s, copies ? 1 : 0, &all);
    if (i < a.n && blockIdx.x == 0) {
      a.copy[i] = make_int4(want.br.parent, want.br.len, copies ? want.page : -1, static_cast<int>(at));
      if (copies) a.list[at] = make_int2(want.page, want.br.rest);
    }
    wanted += all;
  }
  if (wanted <= free) list_free(s, a.refs, mine, rank, wanted, a.order);
  if (id == 0) {
    *a.missing = static_cast<int>(wanted > free ? wanted - free : 0);
    *a.copies = wanted > free ? 0 : static_cast<int>(wanted);
  }
  if (fault) atomicOr(&g_page_fault, fault);
  cluster_sync();  // no CTA leaves while its count may be read
}

// The tables and counts, and the copies, dealt out to a grid that fills the GPU
// once: first row i of the tables, then the K or V rows of one head of a page.
template <typename E, int kVec>
__global__ void __launch_bounds__(256) kv_fork_copy_kernel(const __grid_constant__ ForkArgs a) {
  using V = Vec<E, kVec>;
  launch_dependents();
  grid_dependency_wait();
  int fault = 0;
  const bool fits = *a.missing == 0;
  const int copies = *a.copies;
  const int rows = max(a.n, a.c.B), each = 2 * a.c.heads * a.chunks;
  for (long long item = blockIdx.x; item < rows + static_cast<long long>(copies) * each; item += gridDim.x) {
    if (item < rows) {
      const int i = static_cast<int>(item);
      if (i < a.n) {
        const int4 plan = a.copy[i];
        const int full = plan.y / a.c.page_size, rest = plan.y - full * a.c.page_size;
        const int count = fits ? full + (rest > 0) : 0;
        int* row = a.new_table + static_cast<long long>(i) * a.c.table_width;
        for (int j = threadIdx.x; j < a.c.table_width; j += 256) {
          int page = -1;
          if (j < count) {
            const bool copied = plan.z >= 0 && j == full;
            page = copied ? a.order[plan.w] : *(a.c.table + static_cast<long long>(plan.x) * a.c.table_stride + j);
            if (copied) a.refs[page] = 1;
          }
          row[j] = page;
        }
        if (threadIdx.x == 0) {
          a.new_held[i] = count;
          a.new_lens[i] = fits ? plan.y : 0;
        }
      }
      if (fits && i < a.c.B) {
        // One holder less, and as many more as continue it.
        const Branch br = branch_of_parent(a, i, &fault);
        const int have = held_pages(a.c, a.held, i, &fault), kids = a.kids[i];
        const bool keeps = kids > 0 && br.rest > 0 && a.copy[a.first[i]].z < 0;
        change_refs(a.c, a.refs, a.c.table + i * a.c.table_stride, threadIdx.x, have, 256,
                    [&](long long j) { return (j < br.full ? kids : j == br.full && keeps ? 1 : 0) - 1; }, &fault);
      }
      continue;
    }
    const long long at = item - rows;
    const int k = static_cast<int>(at / each), hc = static_cast<int>(at - static_cast<long long>(k) * each);
    const int2 what = a.list[k];
    const long long from = what.x, to = a.order[k];
    const int hv = hc / a.chunks, chunk = hc - hv * a.chunks;
    const bool is_v = hv >= a.c.heads;
    const int h = is_v ? hv - a.c.heads : hv;
    const long long* st = is_v ? a.c.vs : a.c.ks;
    const int in = threadIdx.x / a.cols, at_once = 256 / a.cols;
    E* x = static_cast<E*>(is_v ? a.c.v : a.c.k) + h * st[1] + static_cast<long long>(threadIdx.x - in * a.cols) * kVec;
    if (in < at_once) {
      const long long step = static_cast<long long>(a.chunks) * at_once;
      for (long long r0 = chunk * at_once + in; r0 < what.y; r0 += kCopyAhead * step) {
        V row[kCopyAhead];
#pragma unroll
        for (int p = 0; p < kCopyAhead; ++p)
          if (r0 + p * step < what.y)
            row[p] = *reinterpret_cast<const V*>(x + from * st[0] + (r0 + p * step) * st[2]);
#pragma unroll
        for (int p = 0; p < kCopyAhead; ++p)
          if (r0 + p * step < what.y) *reinterpret_cast<V*>(x + to * st[0] + (r0 + p * step) * st[2]) = row[p];
      }
    }
    if (a.bounds && !is_v && chunk == 0) {
      E* y = static_cast<E*>(a.bounds) + h * a.b_h;
      for (int e = threadIdx.x; e < 2 * a.cols; e += 256) {
        const int m = e >= a.cols;
        const long long off = m * a.b_m + static_cast<long long>(e - m * a.cols) * kVec;
        *reinterpret_cast<V*>(y + to * a.b_p + off) = *reinterpret_cast<const V*>(y + from * a.b_p + off);
      }
    }
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Accepted tokens to their places
// ---------------------------------------------------------------------------

struct CompactArgs {
  PagedView c;
  const int *new_lens, *kept;
  long long kept_stride;
  int n;
  int* lens;
  int cols;  // 16-byte (or element) columns of a row
};
// (Apart, as a launch takes longer with them: 4.9 us from the host instead of 4.4.)
struct CompactBoundsArgs : CompactArgs {
  void* bounds;             // page bounds
  long long b_p, b_h, b_m;  // their strides over (page, head, min/max)
};
template <bool kBounds>
using CompactArgsOf = typename std::conditional<kBounds, CompactBoundsArgs, CompactArgs>::type;

// Warp (b, head), lane a column of K or V: a kept token's place is never behind
// it, and the places of the tokens of one turn never among the sources of a later one, so
// each lane moves its column by itself, the rows of a turn read before any of
// them is written.  kBounds: keys that change pages are folded into the bounds
// of the page they come to, which has been appended to from its row 0 on and so
// has bounds, by the lane that moves them (those that stay in a page are in its
// bounds already).  E: the cache's type, or any of its size without bounds.
constexpr int kMoveWarps = 4, kMoveAhead = 16;

template <typename E, int kVec, bool kBounds>
__global__ void __launch_bounds__(kMoveWarps * 32) kv_compact_kernel(const __grid_constant__ CompactArgsOf<kBounds> a) {
  using V = Vec<E, kVec>;
  launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long task = static_cast<long long>(blockIdx.x) * kMoveWarps + (threadIdx.x >> 5);
  const int b = static_cast<int>(task / a.c.heads), h = static_cast<int>(task - static_cast<long long>(b) * a.c.heads);
  if (b >= a.c.B) return;
  int fault = 0;
  const int* list = a.kept + b * a.kept_stride;
  int kept = lane < a.n ? list[lane] : -1;
  const long long len = *(a.c.lens + b);
  const int drafted = *(a.new_lens + b);
  const long long base = len - (drafted > 0 ? drafted : 0);
  const int cap = a.c.capacity();
  if (len > cap) fault |= kFaultPage;
  long long count = 0;
  int last = -1;  // the kept token before this turn's
  for (int i0 = 0; i0 < a.n; i0 += 32) {
    if (i0 > 0) kept = i0 + lane < a.n ? list[i0 + lane] : -1;
    int before = __shfl_up_sync(0xffffffffu, kept, 1);
    if (lane == 0) before = last;
    last = __shfl_sync(0xffffffffu, kept, 31);
    const bool ok = kept > before && kept < drafted;
    const unsigned bad = __ballot_sync(0xffffffffu, !ok);
    const int here = bad ? __ffs(bad) - 1 : 32;
    if (here < 32 && i0 + here < a.n && __shfl_sync(0xffffffffu, kept, here) != -1) fault |= kFaultPage;
    // Where this lane's token comes from and goes to; one that stays, or lies
    // in no page, is not moved.
    int from_page = -1, to_page = -1, from_row = 0, to_row = 0;
    const long long from = base + kept, to = base + i0 + lane;
    if (lane < here && from != to && to >= 0 && from < cap) {
      const int fp = static_cast<int>(from) / a.c.page_size, tp = static_cast<int>(to) / a.c.page_size;
      from_row = static_cast<int>(from) - fp * a.c.page_size;
      to_row = static_cast<int>(to) - tp * a.c.page_size;
      from_page = paged_page(a.c, b, fp, &fault);
      to_page = paged_page(a.c, b, tp, &fault);
    }
    const unsigned moves = __ballot_sync(0xffffffffu, from_page >= 0 && to_page >= 0);
    unsigned crosses = 0;  // those of them that change pages
    if constexpr (kBounds)
      crosses = __ballot_sync(0xffffffffu, from_page >= 0 && to_page >= 0 && from_page != to_page);
    for (int half = 0; half < 32; half += kMoveAhead) {
      if ((moves >> half & (0xffffffffu >> (32 - kMoveAhead))) == 0) continue;
      for (int c0 = 0; c0 < 2 * a.cols; c0 += 32) {
        const int c = c0 + lane;
        const bool is_v = c >= a.cols, live = c < 2 * a.cols;
        const long long* st = is_v ? a.c.vs : a.c.ks;
        E* x = static_cast<E*>(is_v ? a.c.v : a.c.k) + h * st[1] + static_cast<long long>(is_v ? c - a.cols : c) * kVec;
        V row[kMoveAhead];
#pragma unroll
        for (int p = 0; p < kMoveAhead; ++p) {
          const long long pg = __shfl_sync(0xffffffffu, from_page, half + p);
          const int in = __shfl_sync(0xffffffffu, from_row, half + p);
          if (live && (moves >> (half + p) & 1u)) row[p] = *reinterpret_cast<const V*>(x + pg * st[0] + in * st[2]);
        }
        long long open = -1;  // the page whose bounds are to take in lo and hi
        V lo = {}, hi = {};
        auto close = [&] {
          if constexpr (kBounds) {
            if (open < 0) return;
            E* to = static_cast<E*>(a.bounds) + open * a.b_p + h * a.b_h + static_cast<long long>(c) * kVec;
            V *to_lo = reinterpret_cast<V*>(to), *to_hi = reinterpret_cast<V*>(to + a.b_m);
            fold(lo, hi, *to_lo, *to_hi);
            *to_lo = lo;
            *to_hi = hi;
          }
        };
#pragma unroll
        for (int p = 0; p < kMoveAhead; ++p) {
          const long long pg = __shfl_sync(0xffffffffu, to_page, half + p);
          const int in = __shfl_sync(0xffffffffu, to_row, half + p);
          if (live && (moves >> (half + p) & 1u)) *reinterpret_cast<V*>(x + pg * st[0] + in * st[2]) = row[p];
          if constexpr (kBounds) {
            if (!live || is_v || !(crosses >> (half + p) & 1u)) continue;
            if (pg == open) {
              fold(lo, hi, row[p], row[p]);
            } else {
              close();
              open = pg;
              lo = hi = row[p];
            }
          }
        }
        if constexpr (kBounds) close();
      }
    }
    count += here;
    if (here < 32) break;
  }
  if (h == 0 && lane == 0) {
    const long long now = base + count;
    a.lens[b] = static_cast<int>(now > 0 ? now : 0);
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

size_t round_up(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// CTAs that look for free pages: as many as take one turn each, since a barrier
// of several costs about what a turn does (384 sequences forked in a pool of
// 5000 pages: 16.6 us with one CTA, 17.7 with eight).
int find_ctas(int num_pages) {
  int n = 1;
  while (n < kFindMost && static_cast<long long>(n) * kFindWarps * kStep < num_pages) n *= 2;
  return n;
}

// Places of a call's arrays in its workspace.
struct ResizePlan {
  size_t have_at, start_at, order_at, bytes;
};
ResizePlan resize_plan(const AttnPagedCache* c) {
  const size_t rows = round_up(sizeof(int) * static_cast<size_t>(c->B));
  const long long most = static_cast<long long>(c->B) * c->table_width;
  const size_t listed = static_cast<size_t>(most < c->num_pages ? most : c->num_pages);
  return ResizePlan{0, rows, 2 * rows, 2 * rows + round_up(sizeof(int) * listed)};
}
struct ForkPlan {
  size_t first_at, kids_at, copy_at, list_at, copies_at, order_at, bytes;
};
ForkPlan fork_plan(const AttnPagedCache* c, int n) {
  const size_t old = round_up(sizeof(int) * static_cast<size_t>(c->B)), now = round_up(sizeof(int) * static_cast<size_t>(n));
  const size_t listed = static_cast<size_t>(n < c->num_pages ? n : c->num_pages);
  const size_t copy = 2 * old, list = copy + 4 * now, copies = list + 2 * now, order = copies + 256;
  return ForkPlan{0, old, copy, list, copies, order, order + round_up(sizeof(int) * listed)};
}

// Elements per access: 16 bytes where rows, strides and addresses of K and V,
// and of the page bounds if there are any, allow them, else one.
int access_width(const AttnPagedCache* c, const void* bounds, const long long* bounds_strides) {
  const int vec = c->dtype == ATTN_F32 ? 4 : 8;
  bool fits = c->D % vec == 0 && aligned_to(c->k, 16) && aligned_to(c->v, 16) && aligned_to(bounds, 16);
  for (int i = 0; i < 3; ++i)
    fits = fits && c->k_strides[i] % vec == 0 && c->v_strides[i] % vec == 0 &&
           (!bounds || bounds_strides[i] % vec == 0);
  return fits ? vec : 1;
}

// The checks of page bounds (none: null) that need no device.
int check_bounds(const AttnPagedCache* c, const void* bounds, const long long* strides) {
  if (!bounds) return ATTN_OK;
  if (!strides || strides[0] < 0 || strides[1] < 0 || strides[2] < 0) return ATTN_ERR_INVALID_ARGUMENT;
  return aligned_to(bounds, c->dtype == ATTN_F32 ? 4 : 2) ? ATTN_OK : ATTN_ERR_MISALIGNED;
}

template <typename E, int kVec, bool kBounds>
bool launch_compact(const CompactBoundsArgs& args, cudaStream_t stream) {
  const CompactArgsOf<kBounds>& a = args;
  const long long warps = static_cast<long long>(a.c.B) * a.c.heads;
  return launch_after(kv_compact_kernel<E, kVec, kBounds>, dim3(static_cast<unsigned>((warps + kMoveWarps - 1) / kMoveWarps)),
                      dim3(kMoveWarps * 32), 0, stream, 1, true, a);
}

}  // namespace

int page_word_read_clear_pages(cudaStream_t stream, int* host) {
  static const int zero = 0;
  return cudaMemcpyFromSymbolAsync(host, g_page_fault, sizeof(int), 0, cudaMemcpyDeviceToHost, stream) ==
                     cudaSuccess &&
                 cudaMemcpyToSymbolAsync(g_page_fault, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream) ==
                     cudaSuccess
             ? 0
             : -1;
}

}  // namespace ra

extern "C" int launch_kv_compact(const AttnPagedCache* cache, const int* new_lens, const int* kept,
                                 long long kept_stride, int n, int* lens, cudaStream_t stream) {
  return launch_kv_compact_bounds(cache, new_lens, kept, kept_stride, n, lens, nullptr, nullptr, stream);
}

extern "C" int launch_kv_compact_bounds(const AttnPagedCache* cache, const int* new_lens, const int* kept,
                                        long long kept_stride, int n, int* lens, void* bounds,
                                        const long long* bounds_strides, cudaStream_t stream) {
  using namespace ra;
  CompactBoundsArgs a;
  int st = check_paged_cache(cache, kCacheK | kCacheV, &a.c);
  if (st != ATTN_OK) return st;
  if (n < 0 || kept_stride < 0) return ATTN_ERR_INVALID_ARGUMENT;
  if (cache->B == 0) return ATTN_OK;
  if (!new_lens || (n > 0 && !kept) || !lens) return ATTN_ERR_INVALID_ARGUMENT;
  if (!aligned_to(new_lens, 4) || !aligned_to(kept, 4) || !aligned_to(lens, 4)) return ATTN_ERR_MISALIGNED;
  st = check_bounds(cache, bounds, bounds_strides);
  if (st != ATTN_OK) return st;
  const long long blocks = (static_cast<long long>(cache->B) * cache->heads + kMoveWarps - 1) / kMoveWarps;
  if (blocks > 0x7fffffffLL) return ATTN_ERR_INVALID_ARGUMENT;
  st = check_device();
  if (st != ATTN_OK) return st;
  a.new_lens = new_lens;
  a.kept = kept;
  a.kept_stride = kept_stride;
  a.n = n;
  a.lens = lens;
  a.bounds = bounds;
  a.b_p = a.b_h = a.b_m = 0;
  if (bounds) a.b_p = bounds_strides[0], a.b_h = bounds_strides[1], a.b_m = bounds_strides[2];
  const int vec = access_width(cache, bounds, bounds_strides);
  a.cols = cache->D / vec;
  bool ok;
  if (!bounds && cache->dtype == ATTN_F32)
    ok = vec == 4 ? launch_compact<uint32_t, 4, false>(a, stream) : launch_compact<uint32_t, 1, false>(a, stream);
  else if (!bounds)
    ok = vec == 8 ? launch_compact<uint16_t, 8, false>(a, stream) : launch_compact<uint16_t, 1, false>(a, stream);
  else if (cache->dtype == ATTN_F32)
    ok = vec == 4 ? launch_compact<float, 4, true>(a, stream) : launch_compact<float, 1, true>(a, stream);
  else if (cache->dtype == ATTN_F16)
    ok = vec == 8 ? launch_compact<__half, 8, true>(a, stream) : launch_compact<__half, 1, true>(a, stream);
  else
    ok = vec == 8 ? launch_compact<__nv_bfloat16, 8, true>(a, stream) : launch_compact<__nv_bfloat16, 1, true>(a, stream);
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}

extern "C" int kv_resize_workspace_bytes(const AttnPagedCache* cache, size_t* bytes) {
  using namespace ra;
  if (!bytes) return ATTN_ERR_INVALID_ARGUMENT;
  PagedView view;
  const int st = check_paged_cache(cache, 0, &view);
  if (st != ATTN_OK) return st;
  *bytes = resize_plan(cache).bytes;
  return ATTN_OK;
}

extern "C" int launch_kv_resize(const AttnPagedCache* cache, int* table, int* held, int* refs, int* missing,
                                void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using namespace ra;
  ResizeArgs a;
  int st = check_paged_cache(cache, 0, &a.c);
  if (st != ATTN_OK) return st;
  if (cache->B == 0) return ATTN_OK;
  if (table != cache->block_table || !held || (cache->num_pages > 0 && !refs) || !missing || !workspace)
    return ATTN_ERR_INVALID_ARGUMENT;
  if (!aligned_to(held, 4) || !aligned_to(refs, 4) || !aligned_to(missing, 4) || !aligned_to(workspace, 16))
    return ATTN_ERR_MISALIGNED;
  const ResizePlan p = resize_plan(cache);
  if (workspace_bytes < p.bytes) return ATTN_ERR_INVALID_ARGUMENT;
  st = check_device();
  if (st != ATTN_OK) return st;
  char* ws = static_cast<char*>(workspace);
  a.table = table;
  a.held = held;
  a.refs = refs;
  a.missing = missing;
  a.have = reinterpret_cast<int*>(ws + p.have_at);
  a.start = reinterpret_cast<int*>(ws + p.start_at);
  a.order = reinterpret_cast<int*>(ws + p.order_at);
  const int ctas = find_ctas(cache->num_pages);
  return launch_after(kv_resize_kernel, dim3(ctas), dim3(kFindThreads), 0, stream, ctas, true, a)
             ? ATTN_OK
             : ATTN_ERR_LAUNCH;
}

extern "C" int kv_fork_workspace_bytes(const AttnPagedCache* cache, int n, size_t* bytes) {
  using namespace ra;
  if (!bytes || n < 0) return ATTN_ERR_INVALID_ARGUMENT;
  PagedView view;
  const int st = check_paged_cache(cache, kCacheK | kCacheV, &view);
  if (st != ATTN_OK) return st;
  *bytes = fork_plan(cache, n).bytes;
  return ATTN_OK;
}

extern "C" int launch_kv_fork(const AttnPagedCache* cache, const int* held, int* refs, const int* parents, int n,
                              int* new_table, int* new_held, int* new_lens, int* missing, void* workspace,
                              size_t workspace_bytes, cudaStream_t stream) {
  return launch_kv_fork_bounds(cache, held, refs, parents, n, new_table, new_held, new_lens, missing, nullptr, nullptr,
                               workspace, workspace_bytes, stream);
}

extern "C" int launch_kv_fork_bounds(const AttnPagedCache* cache, const int* held, int* refs, const int* parents, int n,
                                     int* new_table, int* new_held, int* new_lens, int* missing, void* bounds,
                                     const long long* bounds_strides, void* workspace, size_t workspace_bytes,
                                     cudaStream_t stream) {
  using namespace ra;
  ForkArgs a;
  int st = check_paged_cache(cache, kCacheK | kCacheV, &a.c);
  if (st != ATTN_OK) return st;
  if (n < 0) return ATTN_ERR_INVALID_ARGUMENT;
  if ((cache->B > 0 && !held) || (cache->num_pages > 0 && !refs) || !missing || !workspace ||
      (n > 0 && (!parents || (cache->table_width > 0 && !new_table) || !new_held || !new_lens)))
    return ATTN_ERR_INVALID_ARGUMENT;
  for (const void* p : {static_cast<const void*>(held), static_cast<const void*>(refs), static_cast<const void*>(parents),
                        static_cast<const void*>(new_table), static_cast<const void*>(new_held),
                        static_cast<const void*>(new_lens), static_cast<const void*>(missing)})
    if (!aligned_to(p, 4)) return ATTN_ERR_MISALIGNED;
  if (!aligned_to(workspace, 16)) return ATTN_ERR_MISALIGNED;
  st = check_bounds(cache, bounds, bounds_strides);
  if (st != ATTN_OK) return st;
  const ForkPlan p = fork_plan(cache, n);
  const int vec = access_width(cache, bounds, bounds_strides);
  a.cols = cache->D / vec;
  // Rows per thread: up to two turns of kCopyAhead, in large pages more.
  const long long per = 2LL * kCopyAhead * (256 / a.cols), chunks = (cache->page_size + per - 1) / per;
  a.chunks = static_cast<int>(chunks < 64 ? chunks : 64);
  if (workspace_bytes < p.bytes || 2LL * cache->heads * a.chunks > 0x7fffffffLL) return ATTN_ERR_INVALID_ARGUMENT;
  st = check_device();
  if (st != ATTN_OK) return st;
  char* ws = static_cast<char*>(workspace);
  a.held = held;
  a.parents = parents;
  a.refs = refs;
  a.n = n;
  a.bounds = bounds;
  a.b_p = a.b_h = a.b_m = 0;
  if (bounds) a.b_p = bounds_strides[0], a.b_h = bounds_strides[1], a.b_m = bounds_strides[2];
  a.new_table = new_table;
  a.new_held = new_held;
  a.new_lens = new_lens;
  a.missing = missing;
  a.first = reinterpret_cast<int*>(ws + p.first_at);
  a.kids = reinterpret_cast<int*>(ws + p.kids_at);
  a.copy = reinterpret_cast<int4*>(ws + p.copy_at);
  a.list = reinterpret_cast<int2*>(ws + p.list_at);
  a.copies = reinterpret_cast<int*>(ws + p.copies_at);
  a.order = reinterpret_cast<int*>(ws + p.order_at);
  const int ctas = find_ctas(cache->num_pages);
  if (!launch_after(kv_fork_plan_kernel, dim3(ctas), dim3(kFindThreads), 0, stream, ctas, true, a))
    return ATTN_ERR_LAUNCH;
  const int rows = n > cache->B ? n : cache->B;
  if (rows == 0) return ATTN_OK;
  const long long items = rows + static_cast<long long>(n) * 2 * cache->heads * a.chunks, fill = 8LL * sm_count();
  const dim3 grid(static_cast<unsigned>(items < fill ? items : fill)), block(256);
  const auto kern = cache->dtype == ATTN_F32
                        ? (vec == 4 ? kv_fork_copy_kernel<uint32_t, 4> : kv_fork_copy_kernel<uint32_t, 1>)
                        : (vec == 8 ? kv_fork_copy_kernel<uint16_t, 8> : kv_fork_copy_kernel<uint16_t, 1>);
  return launch_after(kern, grid, block, 0, stream, 1, true, a) ? ATTN_OK : ATTN_ERR_LAUNCH;
}
