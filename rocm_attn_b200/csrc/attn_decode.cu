// Attention of one new token per sequence over a paged key-value cache
// (launch_attn_decode).
//
// For sequence b, query head i of the g heads that read kv head h, and the
// tokens t of the sequence (all of them, or those of the listed pages):
//   x_t = scale * log2(e) * (q_i . k_t),  M = max x_t,  L = sum 2^(x_t - M),
//   o_i = sum 2^(x_t - M) v_t / L,  and 0 where there is no token
//   (where there are tokens and every x_t is -inf, 0 / 0: NaN, as the formula),
//   weights[b, h, t] += sum_i 2^(x_t - M_i - log2 L_i)   when asked for.
//
// Every K and V element is used by the g query heads of one token only, so up
// to about 64 query heads per kv head the floor is the time to read the cache
// once.  What that asks for:
//   * The work is cut by tokens, not by sequences.  A unit is one (sequence,
//     kv head, tile of query heads); its tokens are cut in tiles, and the tiles
//     of all units in a row are dealt out in equal runs to a grid that fills
//     the GPU once.  Each CTA works out its own run from seq_lens (a sum over
//     the batch), so the host needs no lengths, a captured call follows
//     lengths that change, and a ragged batch loads every SM alike.
//   * A unit inside one run is finished by its CTA.  A unit cut by the ends of
//     runs leaves its parts (M, L and the unscaled O, fp32) in the workspace,
//     and a second small kernel joins them in the order of the tokens, so
//     results do not depend on timing.  It is launched early and waits on the
//     grid before it (programmatic launch), which hides its launch.
//   * Where the block table can only name a few tiles per CTA, the CTAs of a
//     unit form a cluster and join over its shared memory instead: one launch
//     and no workspace.
//   * Each warp has its own ring of K/V chunks in shared memory, filled by TMA
//     (or 16-byte asynchronous copies) through page ids looked up chunks
//     ahead; warps meet only where a unit ends.  The chunk freed last is the
//     scratch space of that meeting, so the ring stays full meanwhile.
//
// Two kernels share that frame: attn_decode_mma_kernel (fp16/bf16, D a
// multiple of 8, 16-byte rows) on warp-level tensor cores, and
// attn_decode_simt_kernel (fp32, any D <= 256, any strides).
//
// Measured on B200 (calls in a row): 64 sequences of up to 16384 tokens, 64/8
// heads of 128, fp16, 2.75 GB of K and V: 402 to 433 us on different GPUs, 6.4
// to 6.8 TB/s, where a copy does 6.54; 24 of up to 4096, 32/8 heads, bf16, with
// weights: 55 us (floor 41); one of 517 tokens: 7.9 us.  A call in two launches
// has about 8 us that are not reading: lengths and first look-ups 3, first fill
// of the rings 2.5, the ends of the runs and the join the rest.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

#include "paged_cache.h"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace ra {

namespace {

// What went wrong since the word was last read (kFault* bits).
__device__ int g_page_fault = 0;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;
constexpr int kSimtRows = 8;  // query heads per unit of the SIMT kernel, at most

struct DecodeArgs {
  PagedView c;
  const void* q;
  long long q_b, q_h;  // element strides of q over (batch, head)
  void* out;           // [B, Hq, D] contiguous
  int Hq, group, rows, row_tiles;  // group = Hq / heads, in row_tiles tiles of `rows` heads
  float scale_log2;
  const int* pages;  // [B, heads, n_pages] contiguous, or null
  int n_pages;
  int cluster;      // CTAs per unit (a cluster), or 0: runs of tiles over the whole grid
  float* x;         // [B, Hq, x_stride] scores in the exp2 domain, or null
  long long x_stride;
  float* lse2;      // [B, Hq] M + log2 L, or null
  int4* meta;       // [gridDim.x]: first output row, rows, CTAs that continue the unit begun last
  float2* part_ml;  // [2 gridDim.x][rows]
  float* part_o;    // [2 gridDim.x][rows][D4]
  int D4;           // D rounded up to 4
  // pos / page_size for pos < 2^31 as (umulhi(pos, ps_mul) + pos) >> ps_shift:
  // Granlund and Montgomery, Division by Invariant Integers using
  // Multiplication (1994), figure 4.1.
  unsigned ps_mul;
  int ps_shift;
};

__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// 2^(x - m) for a running maximum that may still be -inf (no token yet).
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// The running maximum of tokens starts here, below which only -inf lies, so
// that M = -inf says that there is no token (the result is 0), and a sum of 0
// beside another M that all scores are -inf (the result is 0 / 0).
constexpr float kLowest = -3.402823466e38f;
__device__ __forceinline__ float quotient(float sum, float M, float L) {
  return L == 0.f && M == -INFINITY ? 0.f : sum / L;
}
__device__ __forceinline__ float inverse(float M, float L) {
  return L != 0.f ? 1.f / L : M == -INFINITY ? 0.f : __int_as_float(0x7fffffff);
}
// log2 of the sum, for the weights: 2^(x - this) is 0, or NaN.
__device__ __forceinline__ float log2_sum(float M, float L) {
  return L != 0.f ? M + log2f(L) : M == -INFINITY ? INFINITY : __int_as_float(0x7fffffff);
}

// ---------------------------------------------------------------------------
// The run of tiles of one CTA
// ---------------------------------------------------------------------------

// A place in the row of tiles: tile t of the T tiles of the unit (sequence b,
// kv head h, tile rt of its query heads).
struct Cursor {
  int b, h, rt, t, T, len;
};

template <int kTile>
__device__ __forceinline__ int tiles_of(const DecodeArgs& a, int len) {
  const int n = a.pages ? (len > 0 ? a.n_pages * a.c.page_size : 0) : len;
  return (n + kTile - 1) / kTile;
}

template <int kTile>
__device__ __forceinline__ void advance(const DecodeArgs& a, Cursor& c, int* fault) {
  c.t += max(a.cluster, 1);
  if (c.t < c.T) return;
  c.t = 0;
  if (++c.rt < a.row_tiles) return;
  c.rt = 0;
  if (++c.h < a.c.heads) return;
  c.h = 0;
  c.T = 0;
  while (c.T == 0 && ++c.b < a.c.B) {
    c.len = paged_len(a.c, c.b, fault);
    c.T = tiles_of<kTile>(a, c.len);
  }
}

// This CTA's run of the grid's tiles: `n` of them from tile `first`, and how
// to tell the CTA of a later tile.  The runs differ by one tile at most, the
// longer ones first.
struct Run {
  int first, n;
  int each, longer;  // tiles per CTA, and CTAs with one more
  __device__ __forceinline__ int owner(int tile) const {
    const int cut = longer * (each + 1);
    return tile < cut ? tile / (each + 1) : longer + (tile - cut) / each;
  }
};

struct ScheduleSmem {
  int warp_sum[kWarps];
  Cursor first;
};

// Works out this CTA's run and its first tile.  The host keeps the number of
// tiles the block table can name below 2^31.  kWhole: the threads of the CTA
// share the batch; otherwise each warp looks at all of it by itself, without
// barriers, which is quicker for batches that a few loads per lane cover.
template <int kTile, bool kWhole>
__device__ __forceinline__ Cursor schedule_by(const DecodeArgs& a, ScheduleSmem& s, Run* run, int* fault) {
  constexpr int kShare = kWhole ? kThreads : 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, id = kWhole ? threadIdx.x : lane;
  const int seg = (a.c.B + kShare - 1) / kShare;
  const int b0 = min(a.c.B, id * seg), b1 = min(a.c.B, b0 + seg);
  int mine = 0, len = 0, T = 0;
  for (int b = b0; b < b1; ++b) {
    len = paged_len(a.c, b, fault);
    T = tiles_of<kTile>(a, len);
    mine += T;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  int before = upto - mine, total = __shfl_sync(0xffffffffu, upto, 31);
  if constexpr (kWhole) {
    if (lane == 31) s.warp_sum[warp] = upto;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s.warp_sum[w];
      total += s.warp_sum[w];
    }
  }
  const int units = a.c.heads * a.row_tiles, grid = gridDim.x, c = blockIdx.x;
  total *= units;
  run->each = static_cast<unsigned>(total) / static_cast<unsigned>(grid);
  run->longer = total - run->each * grid;
  run->first = c * run->each + min(c, run->longer);
  run->n = run->each + (c < run->longer ? 1 : 0);
  Cursor at = {};
  const bool here = run->n > 0 && run->first >= before * units && run->first - before * units < mine * units;
  if (here) {
    int in = run->first - before * units, b = b0;
    if (seg > 1) {
      for (;; ++b) {
        len = paged_len(a.c, b, fault);
        T = tiles_of<kTile>(a, len);
        if (in < T * units || b + 1 >= b1) break;
        in -= T * units;
      }
    }
    const int hu = static_cast<unsigned>(in) / static_cast<unsigned>(T), h = a.row_tiles == 1 ? hu : hu / a.row_tiles;
    at = Cursor{b, h, hu - h * a.row_tiles, in - hu * T, T, len};
  }
  if constexpr (kWhole) {
    if (here) s.first = at;
    __syncthreads();
    return s.first;
  } else {
    const unsigned who = __ballot_sync(0xffffffffu, here);
    const int from = who ? __ffs(who) - 1 : 0;
    return Cursor{__shfl_sync(0xffffffffu, at.b, from), __shfl_sync(0xffffffffu, at.h, from),
                  __shfl_sync(0xffffffffu, at.rt, from), __shfl_sync(0xffffffffu, at.t, from),
                  __shfl_sync(0xffffffffu, at.T, from), __shfl_sync(0xffffffffu, at.len, from)};
  }
}

template <int kTile>
__device__ __forceinline__ Cursor schedule(const DecodeArgs& a, ScheduleSmem& s, Run* run, int* fault) {
  return a.c.B <= 128 ? schedule_by<kTile, false>(a, s, run, fault) : schedule_by<kTile, true>(a, s, run, fault);
}

// The first query row of the unit at c.
template <typename T>
__device__ __forceinline__ const T* query_rows(const DecodeArgs& a, const Cursor& c) {
  return static_cast<const T*>(a.q) + c.b * a.q_b + (static_cast<long long>(c.h) * a.group + c.rt * a.rows) * a.q_h;
}

// Output rows of empty sequences are zeros.
template <typename T>
__device__ __forceinline__ void zero_empty_rows(const DecodeArgs& a, int* fault) {
  const long long per_seq = static_cast<long long>(a.Hq) * a.c.D;
  for (int b = blockIdx.x; b < a.c.B; b += gridDim.x) {
    if (paged_len(a.c, b, fault) > 0 && !(a.pages && a.n_pages == 0)) continue;
    T* o = static_cast<T*>(a.out) + b * per_seq;
    for (long long i = threadIdx.x; i < per_seq; i += kThreads) o[i] = from_f32<T>(0.f);
  }
}

// Where token `pos` of (sequence b, kv head h) lies, pos counting the tokens
// of the listed pages when there is a list.  In two steps, each a load whose
// value only the next needs, so that the loads of several tokens overlap: its
// logical page (row < 0: no such token), then its physical page.
__device__ __forceinline__ void locate_logical(const DecodeArgs& a, int b, int h, int pos, int len, int* lp, int* row) {
  const unsigned p = static_cast<unsigned>(pos);
  const int j = static_cast<int>((__umulhi(p, a.ps_mul) + p) >> a.ps_shift);
  *row = pos - j * a.c.page_size;
  *lp = j;
  if (a.pages) {
    if (j < a.n_pages)
      *lp = *(a.pages + (static_cast<long long>(b) * a.c.heads + h) * a.n_pages + j);
    else
      *row = -1;
  } else if (pos >= len) {
    *row = -1;
  }
}
__device__ __forceinline__ void locate_physical(const DecodeArgs& a, int b, int len, int* page, int* row) {
  const int lp = *page;
  // A list's entry that names no page of the sequence adds nothing.
  if (a.pages && (lp < 0 || lp >= a.c.table_width || lp * a.c.page_size + *row >= len)) *row = -1;
  if (*row >= 0) *page = *(a.c.table + static_cast<long long>(b) * a.c.table_stride + lp);
}
// After both: whether there is such a token, in a page of the cache.
__device__ __forceinline__ bool located(const DecodeArgs& a, int page, int row, int* fault) {
  const bool in = static_cast<unsigned>(page) < static_cast<unsigned>(a.c.num_pages);
  if (row >= 0 && !in) *fault |= kFaultPage;
  return row >= 0 && in;
}

// Where a unit's result goes: the output when the whole unit was in this
// CTA's run, otherwise a part of the workspace (the first of the CTA's two
// for a unit begun earlier, the second for one begun here).
struct Place {
  bool whole;
  long long row0;  // first output row
  int rows, slot;
};

__device__ __forceinline__ Place place_of(const DecodeArgs& a, const Cursor& c, bool begun, const Run& run, int tile) {
  Place p;
  p.rows = min(a.rows, a.group - c.rt * a.rows);
  p.row0 = static_cast<long long>(c.b) * a.Hq + c.h * a.group + c.rt * a.rows;
  const bool ends = a.cluster ? true : c.t + 1 == c.T;
  p.whole = begun && ends && a.cluster <= 1;
  p.slot = 2 * blockIdx.x + (begun ? 1 : 0);
  if (begun && !ends && threadIdx.x == 0) {
    const int later = run.owner(tile + c.T - 1 - c.t) - static_cast<int>(blockIdx.x);  // `tile` is tile c.t of the unit
    // row0 < B * Hq, which the host keeps below 2^31
    a.meta[blockIdx.x] = make_int4(static_cast<int>(p.row0), p.rows, later, 0);
  }
  return p;
}

// ---------------------------------------------------------------------------
// Tensor-core kernel
// ---------------------------------------------------------------------------

// Products are taken with the tokens (then the head dim) as the rows of the
// m16n8k16 product and eight query heads as its columns: S^T = K Q^T and O^T =
// V^T P^T.  A group of up to eight heads then fills a product that the other
// way round it would half waste, with half the registers for O and Q; groups
// of up to 32 heads take two or four column tiles over the same K and V
// fragments.  P^T comes out of S^T's accumulators transposed against what the
// second product reads, which one 8x8 transpose (movmatrix) per 8 tokens mends.
//
// A warp's chunk is kKeys tokens: K rows, then V rows, of kD 16-bit elements,
// 16-byte columns XOR-swizzled by the row so that ldmatrix reads every bank
// once.  Its size, 4 kKeys kD bytes, is that of 16 rows of O in fp32 or more,
// which is what the freed chunk holds where a unit ends.  Rings of two chunks:
// with three, 64 long sequences read 6.39 TB/s instead of 6.73.  Two CTAs of
// four warps per SM (one at D = 256, whose accumulators and query heads take
// the registers): while one ends a unit the other reads.
template <int kD>
struct MmaCfg {
  static constexpr int kKeys = kD <= 64 ? 32 : 16;
  static constexpr int kTile = kWarps * kKeys;
  static constexpr int kCtas = kD <= 128 ? 2 : 1;
  static constexpr int kStageBytes = kKeys * kD * 4;
  static constexpr int kStages = 2;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMaxHeads = kD <= 128 ? 32 : 16;  // query heads per unit
};

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A value at the same place in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ float cluster_load(const float* p, int rank) {
  uint32_t at;
  float x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ float4 cluster_load4(const float* p, int rank) {
  uint32_t at;
  float4 x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(at)
               : "memory");
  return x;
}

// The two caches as [num_pages, heads, page_size, D] tensors read in boxes of
// 16 rows by 64 columns.
struct TmaMaps {
  CUtensorMap k, v;
  unsigned long long wait_ns;
  int lose;  // watchdog test build only: CTA 0's first wait is for bytes that never come
};

template <bool kBf16, int kD, int kNT, bool kWeights, bool kTma>
__global__ void __launch_bounds__(kThreads, MmaCfg<kD>::kCtas)
    attn_decode_mma_kernel(const __grid_constant__ DecodeArgs a, const __grid_constant__ TmaMaps maps) {
  using C = MmaCfg<kD>;
  using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  constexpr int kKeys = C::kKeys, kTile = C::kTile, kStages = C::kStages;
  constexpr int kCols = kD / 8;                // 16-byte columns of a row
  constexpr int kSteps = kD / 16;              // 16-wide steps of the head dim
  constexpr int kRowsPerCopy = 32 / kCols;     // rows of one 16-byte copy of the warp
  // A warp's weights, and so its L and O, are kept times this power of two:
  // fp16 has its full precision down to 2^-14 and nothing below 2^-25, where
  // the tokens beside one that takes nearly everything lie.  With it weights
  // down to 2^-29 of the largest keep their bits, and those down to 2^-40 count.
  constexpr float kUp = kBf16 ? 1.f : 32768.f;

  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ ScheduleSmem s_sched;
  __shared__ float s_m[kWarps][8 * kNT], s_l[kWarps][8 * kNT];
  __shared__ uint32_t s_mask[kWarps][kStages];
  __shared__ uint64_t s_full[kWarps][kStages];
  __shared__ int s_abort, s_code, s_late;
  __shared__ float s_cm[8 * kNT], s_cl[8 * kNT];  // of this CTA's part of a cluster's unit

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int fault = 0;
  if constexpr (kTma) {
    if (lane == 0) {
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
#pragma unroll
      for (int s = 0; s < kStages; ++s) mbar_init(&s_full[warp][s], 1);
      fence_mbar_init();
    }
    if (threadIdx.x == 0) s_abort = s_code = s_late = 0;
  }
  launch_dependents();
  grid_dependency_wait();
  int n;
  Run run = {};
  Cursor cur;
  if (a.cluster) {
    // Tiles rank, rank + cluster, ... of one unit.  Which they are does not
    // depend on the length, so the first look-ups need not wait for it.
    const int unit = blockIdx.x / a.cluster, hu = unit % (a.c.heads * a.row_tiles);
    cur.b = unit / (a.c.heads * a.row_tiles);
    cur.h = hu / a.row_tiles;
    cur.rt = hu - cur.h * a.row_tiles;
    cur.t = blockIdx.x % a.cluster;
    cur.len = a.pages ? paged_len(a.c, cur.b, &fault) : a.c.capacity();
    cur.T = tiles_of<kTile>(a, cur.len);
    n = (cur.T - cur.t + a.cluster - 1) / a.cluster;
    if (threadIdx.x < 8 * kNT) s_cm[threadIdx.x] = -INFINITY, s_cl[threadIdx.x] = 0.f;
  } else {
    if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    cur = schedule<kTile>(a, s_sched, &run, &fault);
    n = run.n;
    zero_empty_rows<T>(a, &fault);
    __syncthreads();  // the set-up above
  }

  unsigned char* ring = smem + warp * (kStages * C::kStageBytes);
  const uint32_t ring_addr = smem_addr(ring);
  // Without TMA a lane copies one 16-byte column (zeros behind D) of every
  // kRowsPerCopy-th row; the swizzle of later rows is an XOR with a constant.
  const int my_row = lane / kCols;
  const bool my_col_ok = (lane % kCols) * 8 < a.c.D;
  const int my_col = my_col_ok ? (lane % kCols) * 8 : 0;
  const uint32_t my_dst = (lane % kCols) / 8 * (kKeys * 128) + my_row * 128 + (((lane % 8) ^ my_row) << 4);
  const T* kbase = static_cast<const T*>(a.c.k) + my_col;
  const T* vbase = static_cast<const T*>(a.c.v) + my_col;

  auto prefetch_q = [&](const Cursor& c) {
    constexpr int kLines = kD / 64;  // of 128 bytes in a row
    const int rows = min(a.rows, a.group - c.rt * a.rows);
    const T* q = query_rows<T>(a, c);
    for (int e = lane; e < rows * kLines; e += 32)
      if (e % kLines * 64 < a.c.D) prefetch_l1(q + (e / kLines) * a.q_h + e % kLines * 64);
  };

  // The chunks whose copies go out next, with the page and row of each token
  // (lane = token): logical pages are looked up kStages + 1 chunks ahead of
  // the copies and physical pages kStages ahead, so that no copy waits for a
  // look-up and the first ones wait for one together.
  int page[kStages + 1], row[kStages + 1], head[kStages + 1];
  Cursor ahead = cur;
  int looked = 0, last_b = 0, last_len = 0;
  auto logical = [&](int s) {
    row[s] = -1;
    if (looked < n) {
      last_b = ahead.b;
      last_len = ahead.len;
      head[s] = ahead.h;
      // The query heads of a unit to come, so that its first product does not
      // wait for them.
      if (warp == 0 && ahead.t == 0) prefetch_q(ahead);
      if (kKeys == 32 || lane < kKeys)
        locate_logical(a, last_b, ahead.h, ahead.t * kTile + warp * kKeys + lane, last_len, &page[s], &row[s]);
      advance<kTile>(a, ahead, &fault);
      ++looked;
    }
  };
  auto physical = [&](int s) { locate_physical(a, last_b, last_len, &page[s], &row[s]); };
  const uint64_t policy = l2_policy_evict_first();
  uint32_t phase = 0, in_flight = 0;  // of each stage's barrier; chunks asked for and not yet seen
  bool gave_up = false;
  auto issue = [&](int stage) {
    uint32_t mask = __ballot_sync(0xffffffffu, located(a, page[0], row[0], &fault));
    if (gave_up) mask = 0;
    if (lane == 0) s_mask[warp][stage] = mask;
    if constexpr (kTma) {
      // One lane asks for the boxes, of 16 rows, that hold tokens.  All rows of
      // a box lie in one page; its first row holds a token if any does.
      if (mask != 0) {
        int boxes = 0;
#pragma unroll
        for (int g = 0; g < kKeys / 16; ++g) boxes += mask >> (g * 16) & 1u;
        int bytes = boxes * 16 * (kD * 4);
#ifdef RA_WATCHDOG_TEST
        if (maps.lose && blockIdx.x == 0 && threadIdx.x == 0 && in_flight == 0 && phase == 0) bytes += 16;
#endif
        if (lane == 0) mbar_arrive_expect_tx(&s_full[warp][stage], bytes);
        in_flight |= 1u << stage;
#pragma unroll
        for (int g = 0; g < kKeys / 16; ++g) {
          const int pg = __shfl_sync(0xffffffffu, page[0], g * 16), in = __shfl_sync(0xffffffffu, row[0], g * 16);
          if (lane == 0 && (mask >> (g * 16) & 1u)) {
            const uint32_t dst = ring_addr + stage * C::kStageBytes + g * 16 * 128;
#pragma unroll
            for (int c = 0; c < kD / 64; ++c) {
              tma_load_4d(dst + c * (kKeys * 128), &maps.k, &s_full[warp][stage], c * 64, in, head[0], pg, policy);
              tma_load_4d(dst + c * (kKeys * 128) + kKeys * kD * 2, &maps.v, &s_full[warp][stage], c * 64, in, head[0],
                          pg, policy);
            }
          }
        }
      }
    } else {
      if (mask != 0) {
        const uint32_t dst = ring_addr + stage * C::kStageBytes + my_dst;
        const T* kh = kbase + head[0] * a.c.ks[1];
        const T* vh = vbase + head[0] * a.c.vs[1];
#pragma unroll
        for (int i = 0; i < kKeys / kRowsPerCopy; ++i) {
          const int tok = i * kRowsPerCopy + my_row;
          const int pg = __shfl_sync(0xffffffffu, page[0], tok), in = __shfl_sync(0xffffffffu, row[0], tok);
          const bool ok = (mask >> tok & 1u) && my_col_ok;
          const uint32_t at = (dst ^ ((i * kRowsPerCopy & 7) << 4)) + i * kRowsPerCopy * 128;
          cp_async16(at, kh + (ok ? pg * a.c.ks[0] + in * a.c.ks[2] : 0), ok);
          cp_async16(at + kKeys * kD * 2, vh + (ok ? pg * a.c.vs[0] + in * a.c.vs[2] : 0), ok);
        }
      }
      cp_async_commit();
    }
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      page[s] = page[s + 1];
      row[s] = row[s + 1];
      head[s] = head[s + 1];
    }
    physical(kStages - 1);
    logical(kStages);
  };

  // The first kStages physical look-ups overlap: each needs its own sequence,
  // and only the first look-ups of a run can span several.
  {
    int bs[kStages], ls[kStages];
#pragma unroll
    for (int s = 0; s <= kStages; ++s) {
      page[s] = head[s] = 0;
      logical(s);
      if (s < kStages) bs[s] = last_b, ls[s] = last_len;
    }
#pragma unroll
    for (int s = 0; s < kStages; ++s) locate_physical(a, bs[s], ls[s], &page[s], &row[s]);
  }
  if (a.cluster) {
    if (!a.pages) {
      // The length: what was looked up behind it does not count.
      cur.len = ahead.len = last_len = paged_len(a.c, cur.b, &fault);
      cur.T = ahead.T = tiles_of<kTile>(a, cur.len);
      n = max(0, (cur.T - cur.t + a.cluster - 1) / a.cluster);
#pragma unroll
      for (int s = 0; s <= kStages; ++s)
        if ((cur.t + s * a.cluster) * kTile + warp * kKeys + lane >= cur.len) row[s] = -1;
    }
    __syncthreads();  // the set-up above
  }

  const int cur_rt = cur.rt, unit_T = cur.T;
  const long long unit_row0 = static_cast<long long>(cur.b) * a.Hq + cur.h * a.group + cur.rt * a.rows;
  uint32_t qf[kNT][kSteps][2];
  float o[kNT][kSteps][4];
  float m[kNT][2], l[kNT][2];  // of query heads 8 t + 2 (lane % 4) + {0, 1}
  bool begun = a.cluster ? true : cur.t == 0, fresh = true;
  int stage = 0;

  // Scores of tokens lane / 4 + {0, 8} of the chunk's g-th 16 and of two heads
  // of column tile t, for the weights: -inf where there is no token, and a
  // token's own -inf as the lowest finite value, which weighs nothing either.
  auto keep_scores = [&](int t, int g, float x0, float x1, float y0, float y1) {
    const int rows = min(a.rows, a.group - cur.rt * a.rows), r = t * 8 + (lane & 3) * 2;
    const long long row0 = static_cast<long long>(cur.b) * a.Hq + cur.h * a.group + cur.rt * a.rows;
    float* x = a.x + (row0 + r) * a.x_stride + cur.t * kTile + warp * kKeys + g * 16 + (lane >> 2);
    if (r < rows) x[0] = x0, x[8] = y0;
    if (r + 1 < rows) x[a.x_stride] = x1, x[a.x_stride + 8] = y1;
  };

  // Row r of this CTA's part of its cluster's unit: in the chunk of warp r / 16
  // that the unit's end leaves free.
  static_assert(kStages >= 2, "one chunk is scratch space, another holds the part");
  auto cluster_part = [&](int r) {
    const int other = n % kStages;  // the last chunk was n - 1
    return reinterpret_cast<float*>(smem + ((r >> 4) * kStages + other) * C::kStageBytes) + (r & 15) * kD;
  };

  // The first kStages turns only fill the ring (one copy of the code: a CTA's
  // first pass over it comes from a cold instruction cache).
  for (int i = -kStages; i < n; ++i) {
    if (i >= 0) {
      if (fresh) {
        // A new unit: its query heads as B fragments (heads behind the last are zero).
        const int rows = min(a.rows, a.group - cur.rt * a.rows);
        const T* q = query_rows<T>(a, cur);
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
          const int r = t * 8 + (lane >> 2);
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int d = ks * 16 + j * 8 + (lane & 3) * 2;
              qf[t][ks][j] = (r < rows && d < a.c.D) ? *reinterpret_cast<const uint32_t*>(q + r * a.q_h + d) : 0u;
            }
            o[t][ks][0] = o[t][ks][1] = o[t][ks][2] = o[t][ks][3] = 0.f;
          }
          m[t][0] = m[t][1] = -INFINITY;
          l[t][0] = l[t][1] = 0.f;
        }
        fresh = false;
      }
      if constexpr (!kTma) cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t mask = s_mask[warp][stage];
      if (mask != 0 || kWeights) {
        const uint32_t chunk = ring_addr + stage * C::kStageBytes;
        const uint32_t kaddr = chunk + (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
        const uint32_t vaddr =
            chunk + kKeys * kD * 2 + ((lane >> 4) * 8 + (lane & 7)) * 128 + (((lane >> 3 & 1) ^ (lane & 7)) << 4);
        if constexpr (kTma) {
          if (mask != 0) {
            // A wait that runs out marks the launch; the warp asks for nothing
            // more, whose barrier could not tell it from what is missing, and
            // goes on without, so that the CTA's warps still meet.
            if (!gave_up) {
              const bool there = mbar_wait(&s_full[warp][stage], phase >> stage & 1u, &s_abort, &s_code, 1, maps.wait_ns);
              if (__all_sync(0xffffffffu, there)) {
                phase ^= 1u << stage;
                in_flight &= ~(1u << stage);
              } else {
                gave_up = true;
                fault |= kFaultWait;
              }
            }
            if (mask != 0xffffffffu >> (32 - kKeys)) {
              // Rows of a box that hold no token have come along; V's are
              // cleared, as no weight, not even zero, may meet them.
#pragma unroll 1
              for (int e = lane; e < kKeys * kCols; e += 32) {
                const int r = e % kKeys, c = e / kKeys;
                unsigned char* v_at = ring + stage * C::kStageBytes + kKeys * kD * 2 + (c / 8) * (kKeys * 128);
                if (!(mask >> r & 1u))
                  *reinterpret_cast<uint4*>(v_at + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
        }
#pragma unroll
        for (int g = 0; g < kKeys / 16; ++g) {
          const uint32_t live = mask >> (g * 16) & 0xffffu;
          if (live == 0) {
            if constexpr (kWeights) {
#pragma unroll
              for (int t = 0; t < kNT; ++t) keep_scores(t, g, -INFINITY, -INFINITY, -INFINITY, -INFINITY);
            }
            continue;
          }
          // Scores of 16 tokens: thread has tokens lane / 4 + {0, 8} of its two
          // heads.  Even and odd steps of the head dim in two accumulators.
          float s[kNT][4], s2[kNT][4];
#pragma unroll
          for (int t = 0; t < kNT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = s2[t][e] = 0.f;
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks) {
            uint32_t kf[4];
            ldsm_x4((kaddr ^ (ks % 4 * 32)) + (ks / 4 * kKeys + g * 16) * 128, kf);
#pragma unroll
            for (int t = 0; t < kNT; ++t)
              mma16816<kBf16>(ks % 2 ? s2[t] : s[t], kf, qf[t][ks][0], qf[t][ks][1]);
          }
          uint32_t pf[kNT][2];
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = (s[t][e] + s2[t][e]) * a.scale_log2;
            if (live != 0xffffu) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(live >> ((e >> 1) * 8 + (lane >> 2)) & 1u)) s[t][e] = -INFINITY;
            }
            if constexpr (kWeights) {
              float x[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                x[e] = live >> ((e >> 1) * 8 + (lane >> 2)) & 1u ? fmaxf(s[t][e], kLowest) : -INFINITY;
              keep_scores(t, g, x[0], x[1], x[2], x[3]);
            }
            float f[2], top[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(s[t][e], s[t][e + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              top[e] = fmaxf(fmaxf(m[t][e], mx), kLowest);  // there is a token among the 16
              f[e] = ex2_approx(m[t][e] - top[e]);
              m[t][e] = top[e];
            }
            if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
              l[t][0] *= f[0];
              l[t][1] *= f[1];
#pragma unroll
              for (int j = 0; j < kSteps; ++j) {
                o[t][j][0] *= f[0];
                o[t][j][1] *= f[1];
                o[t][j][2] *= f[0];
                o[t][j][3] *= f[1];
              }
            }
            // P is rounded to the input type for P V, by half a step (2^-8 or
            // 2^-11 of each weight) at most; its sum is taken before that.
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = ex2_approx(s[t][e] - top[e & 1]) * kUp;
            l[t][0] += s[t][0] + s[t][2];
            l[t][1] += s[t][1] + s[t][3];
            pf[t][0] = transpose_8x8(pack2<kBf16>(s[t][0], s[t][1]));
            pf[t][1] = transpose_8x8(pack2<kBf16>(s[t][2], s[t][3]));
          }
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            uint32_t vf[4];
            ldsm_x4_trans((vaddr ^ (j % 4 * 32)) + (j / 4 * kKeys + g * 16) * 128, vf);
#pragma unroll
            for (int t = 0; t < kNT; ++t) mma16816<kBf16>(o[t][j], vf, pf[t][0], pf[t][1]);
          }
        }
      }

      if ((!a.cluster && cur.t + 1 == cur.T) || i + 1 == n) {
        // The unit, or this CTA's part of it, ends: the warps leave their parts
        // in the chunks just freed, 16 heads at a time, and their sum is taken
        // with each scaled to the common maximum.
        const Place p = place_of(a, cur, begun, run, run.first + i);
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
            l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
            l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
            if (lane < 4) {
              s_m[warp][t * 8 + lane * 2 + e] = m[t][e];
              s_l[warp][t * 8 + lane * 2 + e] = l[t][e];
            }
          }
        float* ot = reinterpret_cast<float*>(ring + stage * C::kStageBytes);
#pragma unroll
        for (int t0 = 0; t0 < kNT; t0 += 2) {
#pragma unroll
          for (int t = t0; t < (t0 + 2 < kNT ? t0 + 2 : kNT); ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = t * 8 + (lane & 3) * 2 + e, at = r - t0 * 8;
              if (r < p.rows) {
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
#pragma unroll
                  for (int up = 0; up < 2; ++up) {
                    const int d = j * 16 + up * 8 + (lane >> 2);
                    ot[at * kD + (((d >> 2) ^ ((lane & 3) << 1)) << 2) + (d & 3)] = o[t][j][2 * up + e];
                  }
              }
            }
          __syncthreads();
          const int here = min(p.rows - t0 * 8, 16);
          for (int e = threadIdx.x; e < here * (kD / 4); e += kThreads) {
            const int at = e / (kD / 4), c4 = e % (kD / 4), r = t0 * 8 + at;
            if (c4 * 4 >= a.c.D) continue;
            float M = s_m[0][r], L = 0.f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][r]);
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float f = ex2_approx(s_m[w][r] - finite_max(M)) * (1.f / kUp);
              const float4 y = *reinterpret_cast<const float4*>(
                  reinterpret_cast<const float*>(smem + (w * kStages + stage) * C::kStageBytes) + at * kD +
                  ((c4 ^ ((at >> 1 & 3) << 1)) << 2));
              L += s_l[w][r] * f;
              sum.x += y.x * f;
              sum.y += y.y * f;
              sum.z += y.z * f;
              sum.w += y.w * f;
            }
            if (p.whole) {
              const float inv = inverse(M, L);
              T* out = static_cast<T*>(a.out) + (p.row0 + r) * a.c.D + c4 * 4;
              *reinterpret_cast<uint2*>(out) =
                  make_uint2(pack2<kBf16>(sum.x * inv, sum.y * inv), pack2<kBf16>(sum.z * inv, sum.w * inv));
              if (kWeights && c4 == 0) a.lse2[p.row0 + r] = log2_sum(M, L);
            } else if (a.cluster) {
              // kept for the cluster in the other chunk of warp 0 (or 1), which is free: there are no more tiles
              *reinterpret_cast<float4*>(cluster_part(r) + c4 * 4) = sum;
              if (c4 == 0) s_cm[r] = M, s_cl[r] = L;
            } else {
              const long long slot = static_cast<long long>(p.slot) * a.rows + r;
              *reinterpret_cast<float4*>(a.part_o + slot * a.D4 + c4 * 4) = sum;
              if (c4 == 0) a.part_ml[slot] = make_float2(M, L);
            }
          }
          if constexpr (kTma) fence_proxy_async_smem();
          __syncthreads();  // all this is read before it is written again
        }
        begun = true;
        fresh = true;
      }
    }
    __syncwarp();
    issue(stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (i >= 0) advance<kTile>(a, cur, &fault);
  }
  if (a.cluster > 1) {
    // The parts of the cluster's CTAs are joined in their order, each CTA
    // taking its share of the columns; none leaves before all have read.
    cluster_sync();
    const int rank = blockIdx.x % a.cluster, rows = min(a.rows, a.group - cur_rt * a.rows);
    for (int e = rank * kThreads + threadIdx.x; e < rows * (kD / 4); e += a.cluster * kThreads) {
      const int r = e / (kD / 4), c4 = e % (kD / 4);
      if (c4 * 4 >= a.c.D) continue;
      // All loads first: each takes a good part of a microsecond.
      float ms[kMaxCluster], ls[kMaxCluster];
      float4 ys[kMaxCluster];
#pragma unroll
      for (int w = 0; w < kMaxCluster; ++w) {
        if (w < a.cluster) {
          const int n_w = (unit_T - w + a.cluster - 1) / a.cluster;
          ms[w] = cluster_load(&s_cm[r], w);
          ls[w] = cluster_load(&s_cl[r], w);
          const unsigned char* part = smem + ((r >> 4) * kStages + n_w % kStages) * C::kStageBytes;
          ys[w] = cluster_load4(reinterpret_cast<const float*>(part) + (r & 15) * kD + c4 * 4, w);
        }
      }
      float M = -INFINITY, L = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kMaxCluster; ++w)
        if (w < a.cluster) M = fmaxf(M, ms[w]);
#pragma unroll
      for (int w = 0; w < kMaxCluster; ++w) {
        if (w < a.cluster && ls[w] != 0.f) {  // 0: no token, and no part
          const float f = ex2_approx(ms[w] - finite_max(M));
          L += ls[w] * f;
          sum.x += ys[w].x * f;
          sum.y += ys[w].y * f;
          sum.z += ys[w].z * f;
          sum.w += ys[w].w * f;
        }
      }
      const float inv = inverse(M, L);
      T* out = static_cast<T*>(a.out) + (unit_row0 + r) * a.c.D + c4 * 4;
      *reinterpret_cast<uint2*>(out) =
          make_uint2(pack2<kBf16>(sum.x * inv, sum.y * inv), pack2<kBf16>(sum.z * inv, sum.w * inv));
      if (kWeights && c4 == 0) a.lse2[unit_row0 + r] = log2_sum(M, L);
    }
    cluster_sync();
  } else if (a.cluster == 1 && n == 0) {
    const int rows = min(a.rows, a.group - cur_rt * a.rows);
    T* out = static_cast<T*>(a.out) + unit_row0 * a.c.D;
    for (int e = threadIdx.x; e < rows * a.c.D; e += kThreads) out[e] = from_f32<T>(0.f);
  }
  if constexpr (kTma) {
    // Copies still in flight must not outlive the CTA's shared memory.
    if (gave_up) {
      for (int s = 0; s < kStages; ++s)
        if (in_flight >> s & 1u) mbar_wait(&s_full[warp][s], phase >> s & 1u, &s_late, &s_code, 1);
    }
  } else {
    cp_async_wait<0>();
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// SIMT kernel: fp32, any head dim, any strides
// ---------------------------------------------------------------------------

// A warp takes 32 tokens, kKeys at a time, the next ones on their way while
// these are used, and the tokens of its next tile looked up meanwhile (17
// sequences of up to 8192 tokens, 64/8 heads of 128 in fp32: 374 us without,
// 199 us with).  Lane holds dims lane + 32 i of q, K, V and O.  The kRows *
// kKeys dot products of a step are summed over the lanes by a butterfly that
// halves the number of values at each step, which leaves each lane one product
// (31 shuffles for 32 products).
constexpr int kSimtChunk = 32, kSimtTile = kWarps * kSimtChunk;
template <int kPer, int kRows>
struct SimtCfg {
  static constexpr int kKeys = kPer == 8 ? 2 : kPer == 4 || kRows == 8 ? 4 : 8;
  static constexpr int kCtas = kPer <= 2 ? 4 : kPer == 4 ? 3 : 2;  // per SM
};

template <typename T, int kPer, int kRows, bool kWeights>
__global__ void __launch_bounds__(kThreads, SimtCfg<kPer, kRows>::kCtas)
    attn_decode_simt_kernel(const __grid_constant__ DecodeArgs a) {
  using C = SimtCfg<kPer, kRows>;
  constexpr int kKeys = C::kKeys, kTile = kSimtTile, kChunk = kSimtChunk;
  constexpr int kVals = kRows * kKeys;
  constexpr int kSame = 32 / kVals;    // lanes that hold the same product
  constexpr int kRowLanes = 32 / kRows;  // lanes of one row
  __shared__ ScheduleSmem s_sched;
  __shared__ float s_m[2][kWarps][kRows], s_l[2][kWarps][kRows];
  __shared__ float s_o[kWarps][kRows][kPer * 32];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int fault = 0;
  launch_dependents();
  grid_dependency_wait();
  if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  Run run;
  Cursor cur = schedule<kTile>(a, s_sched, &run, &fault);
  const int n = run.n;
  zero_empty_rows<T>(a, &fault);
  const T* kbase = static_cast<const T*>(a.c.k);
  const T* vbase = static_cast<const T*>(a.c.v);

  float q[kRows][kPer], o[kRows][kPer];
  float m = -INFINITY, l = 0.f;  // of the row this lane's product belongs to
  bool begun = cur.t == 0, fresh = true;
  int parity = 0;
  const int my_row = lane / kRowLanes, my_key = (lane / kSame) % kKeys;
  int page = -1, row = -1;  // of token `lane` of the warp's part of a tile
  auto look_up = [&](const Cursor& c) {
    locate_logical(a, c.b, c.h, c.t * kTile + warp * kChunk + lane, c.len, &page, &row);
    locate_physical(a, c.b, c.len, &page, &row);
  };
  if (n > 0) look_up(cur);

  for (int i = 0; i < n; ++i) {
    const int h = cur.h, rt = cur.rt;
    const int rows = min(a.rows, a.group - rt * a.rows);
    const long long row0 = static_cast<long long>(cur.b) * a.Hq + h * a.group + rt * a.rows;
    if (fresh) {
      const T* qp = query_rows<T>(a, cur);
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int d = lane + 32 * e;
          q[r][e] = (r < rows && d < a.c.D) ? to_f32(qp[r * a.q_h + d]) : 0.f;
          o[r][e] = 0.f;
        }
      m = -INFINITY;
      l = 0.f;
      fresh = false;
    }
    const int pos0 = cur.t * kTile + warp * kChunk;
    const uint32_t mask = __ballot_sync(0xffffffffu, located(a, page, row, &fault));
    const int this_page = page, this_row = row;
    Cursor next = cur;
    advance<kTile>(a, next, &fault);
    if (i + 1 < n) look_up(next);
    if (mask != 0 || kWeights) {
      const T* kh = kbase + h * a.c.ks[1];
      const T* vh = vbase + h * a.c.vs[1];
      T kn[kKeys][kPer], vn[kKeys][kPer];
      auto fetch = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const int pg = __shfl_sync(0xffffffffu, this_page, k0 + k), in = __shfl_sync(0xffffffffu, this_row, k0 + k);
          const bool live = mask >> (k0 + k) & 1u;
          const T* kp = kh + (live ? pg * a.c.ks[0] + in * a.c.ks[2] : 0);
          const T* vp = vh + (live ? pg * a.c.vs[0] + in * a.c.vs[2] : 0);
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const int d = lane + 32 * e;
            const bool ok = live && d < a.c.D;
            kn[k][e] = ok ? kp[d] : from_f32<T>(0.f);
            vn[k][e] = ok ? vp[d] : from_f32<T>(0.f);
          }
        }
      };
      fetch(0);
#pragma unroll 1
      for (int k0 = 0; k0 < kChunk; k0 += kKeys) {
        float kv[kKeys][kPer], vv[kKeys][kPer];
#pragma unroll
        for (int k = 0; k < kKeys; ++k)
#pragma unroll
          for (int e = 0; e < kPer; ++e) kv[k][e] = to_f32(kn[k][e]), vv[k][e] = to_f32(vn[k][e]);
        if (k0 + kKeys < kChunk) fetch(k0 + kKeys);
        float s[kVals];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int k = 0; k < kKeys; ++k) {
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < kPer; ++e) x = fmaf(q[r][e], kv[k][e], x);
            s[r * kKeys + k] = x;
          }
        int off = 16;
#pragma unroll
        for (int left = kVals; left > 1; left >>= 1) {
          const bool up = lane & off;
#pragma unroll
          for (int j = 0; j < left / 2; ++j) {
            const float keep = up ? s[j + left / 2] : s[j], give = up ? s[j] : s[j + left / 2];
            s[j] = keep + __shfl_xor_sync(0xffffffffu, give, off);
          }
          off >>= 1;
        }
#pragma unroll
        for (int rest = kSame / 2; rest > 0; rest >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], rest);
        const bool is = mask >> (k0 + my_key) & 1u;
        const float x = is ? s[0] * a.scale_log2 : -INFINITY;
        float mx = is ? fmaxf(x, kLowest) : -INFINITY;  // what the weights keep: -inf is an absent token alone
        if (kWeights && my_row < rows && lane % kSame == 0)
          a.x[(row0 + my_row) * a.x_stride + pos0 + k0 + my_key] = mx;
#pragma unroll
        for (int w = kSame; w < kRowLanes; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float mn = fmaxf(m, mx);
        const float f = ex2_approx(m - finite_max(mn));
        m = mn;
        const float pr = ex2_approx(x - finite_max(mn));
        float sum = pr;
#pragma unroll
        for (int w = kSame; w < kRowLanes; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l = l * f + sum;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float fr = __shfl_sync(0xffffffffu, f, r * kRowLanes);
#pragma unroll
          for (int e = 0; e < kPer; ++e) o[r][e] *= fr;
#pragma unroll
          for (int k = 0; k < kKeys; ++k) {
            const float w = __shfl_sync(0xffffffffu, pr, (r * kKeys + k) * kSame);
#pragma unroll
            for (int e = 0; e < kPer; ++e) o[r][e] = fmaf(w, vv[k][e], o[r][e]);
          }
        }
      }
    }
    if (cur.t + 1 == cur.T || i + 1 == n) {
      const Place p = place_of(a, cur, begun, run, run.first + i);
      if (lane % kRowLanes == 0) {
        s_m[parity][warp][my_row] = m;
        s_l[parity][warp][my_row] = l;
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int e = 0; e < kPer; ++e) s_o[warp][r][lane + 32 * e] = o[r][e];
      __syncthreads();
      for (int e = threadIdx.x; e < p.rows * (kPer * 32); e += kThreads) {
        const int r = e / (kPer * 32), d = e % (kPer * 32);
        if (d >= a.c.D) continue;
        float M = s_m[parity][0][r], L = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[parity][w][r]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ex2_approx(s_m[parity][w][r] - finite_max(M));
          L += s_l[parity][w][r] * f;
          sum += s_o[w][r][d] * f;
        }
        if (p.whole) {
          static_cast<T*>(a.out)[(p.row0 + r) * a.c.D + d] = from_f32<T>(quotient(sum, M, L));
          if (kWeights && d == 0) a.lse2[p.row0 + r] = log2_sum(M, L);
        } else {
          const long long at = static_cast<long long>(p.slot) * a.rows + r;
          a.part_o[at * a.D4 + d] = sum;
          if (d == 0) a.part_ml[at] = make_float2(M, L);
        }
      }
      __syncthreads();  // s_o is read before it is written again
      parity ^= 1;
      begun = true;
      fresh = true;
    }
    cur = next;
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Join of units cut between CTAs, and the weights
// ---------------------------------------------------------------------------

// CTA (c, r): row r of the unit that CTA c of the grid before began and did
// not finish.  First every part's maximum and sum at once, then the parts
// themselves, warp w parts w, w + 8, ..., lane four columns of each 128, whose
// loads depend on nothing; the warps' sums meet in shared memory in their order.
constexpr int kJoinWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_decode_join_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr int kAtOnce = kJoinWarps * 32;  // parts
  __shared__ float4 s_o[kJoinWarps][2][32];
  __shared__ float s_f[kAtOnce], s_m[kJoinWarps], s_l[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  launch_dependents();
  grid_dependency_wait();
  const int c = blockIdx.x, r = blockIdx.y;
  auto slot = [&](int i) { return static_cast<long long>(i == 0 ? 2 * c + 1 : 2 * (c + i)) * a.rows + r; };
  // Most units have few parts: the first eight are asked for before it is
  // known that they are parts of it.
  const bool ask = c + warp < gridDim.x;
  float2 early_ml = make_float2(-INFINITY, 0.f);
  float4 early[2] = {};
  if (lane < kJoinWarps && c + lane < gridDim.x) early_ml = a.part_ml[slot(lane)];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (ask && k * 128 + lane * 4 < a.D4)
      early[k] = *reinterpret_cast<const float4*>(a.part_o + slot(warp) * a.D4 + k * 128 + lane * 4);
  const int4 meta = a.meta[c];
  if (meta.z == 0 || r >= meta.y) return;
  float M = -INFINITY, L = 0.f;
  float4 o[2] = {};
  if (meta.z < kJoinWarps) {
    const bool part = lane <= meta.z;
    float m = part ? early_ml.x : -INFINITY;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    m = __shfl_sync(0xffffffffu, m, 0);
    const float f = part ? ex2_approx(early_ml.x - finite_max(m)) : 0.f;
    M = m;
    L = part ? early_ml.y * f : 0.f;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    L = __shfl_sync(0xffffffffu, L, 0);
    const float g = __shfl_sync(0xffffffffu, f, warp);
    if (warp <= meta.z) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        o[k] = make_float4(early[k].x * g, early[k].y * g, early[k].z * g, early[k].w * g);
    }
  } else
  for (int i0 = 0; i0 <= meta.z; i0 += kAtOnce) {
    const int here = min(kAtOnce, meta.z + 1 - i0);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (threadIdx.x < here) ml = a.part_ml[slot(i0 + threadIdx.x)];
    float m = ml.x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if (i0 > 0) __syncthreads();  // the turn before has read s_f
    if (lane == 0) s_m[warp] = m;
    __syncthreads();
    float mn = M;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) mn = fmaxf(mn, s_m[w]);
    const float back = ex2_approx(M - finite_max(mn)), f = ex2_approx(ml.x - finite_max(mn));
    M = mn;
    s_f[threadIdx.x] = f;
    float l = ml.y * f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    L *= back;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) L += s_l[w];
#pragma unroll
    for (int k = 0; k < 2; ++k) o[k].x *= back, o[k].y *= back, o[k].z *= back, o[k].w *= back;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int d = k * 128 + lane * 4;
      if (d >= a.D4) break;
#pragma unroll 8
      for (int i = warp; i < here; i += kJoinWarps) {
        const float4 y = *reinterpret_cast<const float4*>(a.part_o + slot(i0 + i) * a.D4 + d);
        const float g = s_f[i];
        o[k].x = fmaf(y.x, g, o[k].x);
        o[k].y = fmaf(y.y, g, o[k].y);
        o[k].z = fmaf(y.z, g, o[k].z);
        o[k].w = fmaf(y.w, g, o[k].w);
      }
    }
  }
  s_o[warp][0][lane] = o[0];
  s_o[warp][1][lane] = o[1];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.c.D) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) sum += reinterpret_cast<const float*>(s_o[w])[d];
  const long long row = meta.x + r;
  static_cast<T*>(a.out)[row * a.c.D + d] = from_f32<T>(quotient(sum, M, L));
  if (a.lse2 && d == 0) a.lse2[row] = log2_sum(M, L);
}

// weights[b, h, t] += sum over the group of 2^(x_t - lse2), one thread per
// token: reads the scores the kernel before kept.
__global__ void __launch_bounds__(256) attn_decode_weights_kernel(const __grid_constant__ DecodeArgs a, float* weights,
                                                                  long long w_b, long long w_h) {
  launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.z, h = blockIdx.y;
  int fault = 0;  // recorded by the first kernel
  const int len = paged_len(a.c, b, &fault);
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= len) return;
  const long long r0 = static_cast<long long>(b) * a.Hq + static_cast<long long>(h) * a.group;
  float sum = 0.f;
#pragma unroll 4
  for (int g = 0; g < a.group; ++g) {
    const float x = a.x[(r0 + g) * a.x_stride + t], p = ex2_approx(x - a.lse2[r0 + g]);
    sum += x == -INFINITY ? 0.f : p;  // an absent token gets nothing, not even of a sum that is NaN
  }
  float* w = weights + b * w_b + h * w_h + t;
  *w += sum;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct Plan {
  bool mma;
  int kd;  // head dim the kernel is compiled for (mma), or dims per lane (simt)
  int rows, row_tiles, tile;
  int grid, cluster;  // see DecodeArgs
  long long tiles;      // the block table can name
  long long x_stride;
  size_t meta_at, ml_at, o_at, lse_at, x_at, bytes;
};

bool mma_takes(const AttnPagedCache* c) {
  if (c->dtype == ATTN_F32 || c->D % 8 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] % 8 != 0 || c->v_strides[i] % 8 != 0) return false;
  return aligned_to(c->k, 16) && aligned_to(c->v, 16);
}

// `fast`: q and out allow the tensor-core kernel too.
Plan make_plan(const AttnPagedCache* c, bool fast, int Hq, int n_pages, bool listed, bool weights, int sms) {
  Plan p;
  const int group = Hq / c->heads;
  const int D = c->D;
  int per_sm;
  p.mma = fast && mma_takes(c);
  if (p.mma) {
    p.kd = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    const int most = p.kd == 256 ? MmaCfg<256>::kMaxHeads : MmaCfg<128>::kMaxHeads;
    p.rows = group < most ? group : most;
    p.tile = p.kd == 64 ? MmaCfg<64>::kTile : p.kd == 128 ? MmaCfg<128>::kTile : MmaCfg<256>::kTile;
    per_sm = p.kd == 64 ? MmaCfg<64>::kCtas : p.kd == 128 ? MmaCfg<128>::kCtas : MmaCfg<256>::kCtas;
  } else {
    p.kd = D <= 32 ? 1 : D <= 64 ? 2 : D <= 128 ? 4 : 8;
    p.rows = group == 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : kSimtRows;
    if (p.rows > group) p.rows = group;
    p.tile = kSimtTile;
    per_sm = p.kd <= 2 ? SimtCfg<2, 1>::kCtas : p.kd == 4 ? SimtCfg<4, 1>::kCtas : SimtCfg<8, 1>::kCtas;
  }
  p.row_tiles = (group + p.rows - 1) / p.rows;
  const long long capacity = static_cast<long long>(listed ? n_pages : c->table_width) * c->page_size;
  const long long tiles = (capacity + p.tile - 1) / p.tile * c->B * c->heads * p.row_tiles;
  long long grid = static_cast<long long>(sms) * per_sm;
  if (grid > tiles) grid = tiles;
  if (grid < 1) grid = 1;
  p.cluster = 0;
  if (p.mma) {
    const long long unit_tiles = (capacity + p.tile - 1) / p.tile;
    const long long units = static_cast<long long>(c->B) * c->heads * p.row_tiles;
    const long long slots = static_cast<long long>(sms) * per_sm;
    // One launch of clusters where a CTA gets at most two tiles, or four if
    // the clusters leave no more than three quarters of the GPU idle; not where
    // units far outnumber the CTAs that fit, whose set-up would then repeat.
    // Clusters grow beyond half of the GPU only for more than four tiles per
    // CTA, as up to there a call starts beside the one before it.  Measured at
    // D = 128 and full lengths, calls in a row, us, as this rule has it in
    // clusters / in runs: 8 units of 1 tile 4.5 / 6.5, of 8 tiles 6.7 / 7.2, of 16
    // 8.0 / 8.5; 32 units of 1 tile 4.9 / 7.1, of 4 tiles 7.1 / 7.6, of 8 8.4 / 8.2,
    // of 16 11.0 / 10.7, of 32 14.4 / 13.9; 128 of 4 tiles 9.0 / 10.0; 512 of 2 tiles
    // 13.2 / 14.1.  Left to runs: 8 of 32 tiles 10.4 / 9.5, 512 of 4 tiles 18.7 /
    // 19.7, of 8 28.7 / 29.5, 2048 of 2 tiles 42.7 / 32.2.  32 units of 8 tiles in
    // clusters of eight, 256 CTAs, take 9.9.
    int cl = 1;
    while (cl < kMaxCluster && cl < unit_tiles && units * cl * 2 <= slots &&
           (units * cl * 4 <= slots || unit_tiles > 4 * cl))
      cl *= 2;
    const int most = units * cl * 4 >= slots && units * cl <= slots ? 4 : 2;
    if (unit_tiles <= cl * most && units * cl <= 2 * slots) {
      p.cluster = cl;
      grid = units * cl;
    }
  }
  p.grid = static_cast<int>(grid);
  p.tiles = tiles;
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  const size_t D4 = (D + 3) / 4 * 4, parts = p.cluster ? 0 : grid;
  p.meta_at = 0;
  p.ml_at = up(sizeof(int4) * parts);
  p.o_at = p.ml_at + up(sizeof(float2) * 2 * parts * p.rows);
  p.lse_at = p.o_at + up(sizeof(float) * 2 * parts * p.rows * D4);
  p.x_at = p.lse_at;
  p.bytes = p.x_at;
  p.x_stride = (capacity + p.tile - 1) / p.tile * p.tile;
  if (weights) {
    p.x_at += up(sizeof(float) * static_cast<size_t>(c->B) * Hq);
    p.bytes = p.x_at + up(sizeof(float) * static_cast<size_t>(c->B) * Hq * p.x_stride);
  }
  return p;
}

// The checks of a call that need no device.  Returns ATTN_OK or a status.
int check_decode(const AttnPagedCache* c, int Hq, const void* pages, int n_pages, bool weights, PagedView* view) {
  const int st = check_paged_cache(c, kCacheK | kCacheV, view);
  if (st != ATTN_OK) return st;
  if (Hq < 0 || n_pages < 0) return ATTN_ERR_INVALID_ARGUMENT;
  if (Hq % c->heads != 0) return ATTN_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(c->B) * Hq > 0x7fffffffLL) return ATTN_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(n_pages) * c->page_size > kMaxCapacity) return ATTN_ERR_INVALID_ARGUMENT;
  if (pages && weights) return ATTN_ERR_UNSUPPORTED;
  if (weights && (c->B > 65535 || c->heads > 65535)) return ATTN_ERR_UNSUPPORTED;
  return ATTN_OK;
}

// The first launch on a device opts the kernel in to its shared memory and to
// the largest shared-memory share of the SM, so that two CTAs fit.
template <bool kBf16, int kD, int kNT, bool kWeights, bool kTma>
bool launch_mma(const DecodeArgs& a, const TmaMaps& maps, int grid, cudaStream_t stream) {
  auto kern = attn_decode_mma_kernel<kBf16, kD, kNT, kWeights, kTma>;
  static bool done[64] = {};
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  {
    std::lock_guard<std::mutex> g(mu);
    if (!done[dev]) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MmaCfg<kD>::kRingBytes) !=
              cudaSuccess ||
          cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                               static_cast<int>(cudaSharedmemCarveoutMaxShared)) != cudaSuccess)
        return false;
      done[dev] = true;
    }
  }
  const bool ahead = a.cluster <= 1 || 2 * grid <= MmaCfg<kD>::kCtas * sm_count();
  return launch_after(kern, dim3(grid), dim3(kThreads), MmaCfg<kD>::kRingBytes, stream, a.cluster, ahead, a, maps);
}

// Column tiles of eight query heads: 1, 2 or 4.
template <bool kBf16, int kD, bool kWeights, bool kTma>
bool launch_mma_tiles(const DecodeArgs& a, const TmaMaps& maps, int grid, cudaStream_t stream) {
  if (a.rows <= 8) return launch_mma<kBf16, kD, 1, kWeights, kTma>(a, maps, grid, stream);
  if (a.rows <= 16) return launch_mma<kBf16, kD, 2, kWeights, kTma>(a, maps, grid, stream);
  if constexpr (MmaCfg<kD>::kMaxHeads > 16) return launch_mma<kBf16, kD, 4, kWeights, kTma>(a, maps, grid, stream);
  return false;
}

template <bool kBf16, bool kWeights, bool kTma>
bool launch_mma_d(const DecodeArgs& a, const TmaMaps& maps, int kd, int grid, cudaStream_t stream) {
  switch (kd) {
    case 64: return launch_mma_tiles<kBf16, 64, kWeights, kTma>(a, maps, grid, stream);
    case 128: return launch_mma_tiles<kBf16, 128, kWeights, kTma>(a, maps, grid, stream);
    default: return launch_mma_tiles<kBf16, 256, kWeights, kTma>(a, maps, grid, stream);
  }
}

// TMA where 16 divides the page size (a box is rows of one page) and the
// strides suit it, else 16-byte copies (pages of 24 rows of 128 bytes: boxes
// of 8 rows 143 us, copies 135 us).
template <bool kBf16, bool kWeights>
bool launch_mma_any(const DecodeArgs& a, const Plan& p, cudaStream_t stream) {
  TmaMaps maps;
  const unsigned long long limit = wait_limit_ns();
  maps.wait_ns = limit != 0 ? limit : kWaitTimeoutNs;
  maps.lose = drop_arrival_requested();
  auto encode = [&](CUtensorMap* map, const void* base, const long long* st) {
    return make_tensor_map_4d(map, base, kBf16, a.c.D, a.c.page_size, a.c.heads, a.c.num_pages, st[2], st[1], st[0], 64,
                              16) == 0;
  };
  if (a.c.page_size % 16 == 0 && a.c.num_pages > 0 && encode(&maps.k, a.c.k, a.c.ks) && encode(&maps.v, a.c.v, a.c.vs))
    return launch_mma_d<kBf16, kWeights, true>(a, maps, p.kd, p.grid, stream);
  return launch_mma_d<kBf16, kWeights, false>(a, maps, p.kd, p.grid, stream);
}

template <typename T, int kPer, bool kWeights>
bool launch_simt_rows(const DecodeArgs& a, int grid, cudaStream_t stream) {
  const auto kern = a.rows <= 1   ? attn_decode_simt_kernel<T, kPer, 1, kWeights>
                    : a.rows <= 2 ? attn_decode_simt_kernel<T, kPer, 2, kWeights>
                    : a.rows <= 4 ? attn_decode_simt_kernel<T, kPer, 4, kWeights>
                                  : attn_decode_simt_kernel<T, kPer, 8, kWeights>;
  return launch_after(kern, dim3(grid), dim3(kThreads), 0, stream, 1, true, a);
}

template <typename T, bool kWeights>
bool launch_simt(const DecodeArgs& a, int per, int grid, cudaStream_t stream) {
  switch (per) {
    case 1: return launch_simt_rows<T, 1, kWeights>(a, grid, stream);
    case 2: return launch_simt_rows<T, 2, kWeights>(a, grid, stream);
    case 4: return launch_simt_rows<T, 4, kWeights>(a, grid, stream);
    default: return launch_simt_rows<T, 8, kWeights>(a, grid, stream);
  }
}

template <bool kWeights>
bool launch_first(const DecodeArgs& a, const Plan& p, AttnDType dtype, cudaStream_t stream) {
  if (p.mma)
    return dtype == ATTN_BF16 ? launch_mma_any<true, kWeights>(a, p, stream)
                              : launch_mma_any<false, kWeights>(a, p, stream);
  switch (dtype) {
    case ATTN_F16: return launch_simt<__half, kWeights>(a, p.kd, p.grid, stream);
    case ATTN_BF16: return launch_simt<__nv_bfloat16, kWeights>(a, p.kd, p.grid, stream);
    default: return launch_simt<float, kWeights>(a, p.kd, p.grid, stream);
  }
}

}  // namespace

int page_word_read_clear_decode(cudaStream_t stream, int* host) {
  static const int zero = 0;
  return cudaMemcpyFromSymbolAsync(host, g_page_fault, sizeof(int), 0, cudaMemcpyDeviceToHost, stream) ==
                     cudaSuccess &&
                 cudaMemcpyToSymbolAsync(g_page_fault, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream) ==
                     cudaSuccess
             ? 0
             : -1;
}

}  // namespace ra

extern "C" int attn_decode_workspace_bytes(const AttnPagedCache* cache, int Hq, bool listed, int n_pages, bool weights,
                                           size_t* bytes) {
  using namespace ra;
  if (!bytes) return ATTN_ERR_INVALID_ARGUMENT;
  PagedView view;
  int st = check_decode(cache, Hq, nullptr, n_pages, weights, &view);
  if (st != ATTN_OK) return st;
  *bytes = 0;
  if (cache->B == 0 || Hq == 0) return ATTN_OK;
  st = check_device();
  if (st != ATTN_OK) return st;
  const int sms = sm_count();
  // q or out may turn out to need the other kernel: room for either
  const Plan fast = make_plan(cache, true, Hq, n_pages, listed, weights, sms);
  const Plan other = make_plan(cache, false, Hq, n_pages, listed, weights, sms);
  *bytes = fast.bytes > other.bytes ? fast.bytes : other.bytes;
  return ATTN_OK;
}

extern "C" int launch_attn_decode(const AttnPagedCache* cache, const void* q, const long long* q_strides, void* out,
                                  int Hq, float softmax_scale, const int* pages, int n_pages, float* weights,
                                  const long long* weights_strides, void* workspace, size_t workspace_bytes,
                                  cudaStream_t stream) {
  using namespace ra;
  PagedView view;
  int st = check_decode(cache, Hq, pages, n_pages, weights != nullptr, &view);
  if (st != ATTN_OK) return st;
  if (cache->B == 0 || Hq == 0) return ATTN_OK;
  if (!q || !out || !workspace || (weights && !weights_strides)) return ATTN_ERR_INVALID_ARGUMENT;
  const int D = cache->D;
  const long long contiguous[2] = {static_cast<long long>(Hq) * D, D};
  const long long* qs = q_strides ? q_strides : contiguous;
  if (qs[0] < 0 || qs[1] < 0) return ATTN_ERR_INVALID_ARGUMENT;
  if (weights && (weights_strides[0] < 0 || weights_strides[1] < 0)) return ATTN_ERR_INVALID_ARGUMENT;
  const size_t elem = cache->dtype == ATTN_F32 ? 4 : 2;
  if (!aligned_to(q, elem) || !aligned_to(out, elem) || !aligned_to(pages, 4) || !aligned_to(weights, 4) ||
      !aligned_to(workspace, 16))
    return ATTN_ERR_MISALIGNED;
  st = check_device();
  if (st != ATTN_OK) return st;
  const bool fast = aligned_to(q, 16) && aligned_to(out, 16) && qs[0] % 8 == 0 && qs[1] % 8 == 0;
  const Plan p = make_plan(cache, fast, Hq, n_pages, pages != nullptr, weights != nullptr, sm_count());
  if (workspace_bytes < p.bytes || p.tiles > 0x7fffffffLL - 65536) return ATTN_ERR_INVALID_ARGUMENT;

  float scale = softmax_scale;
  if (!(scale > 0.f) || !isfinite(scale)) scale = 1.0f / sqrtf(static_cast<float>(D));
  char* ws = static_cast<char*>(workspace);
  DecodeArgs a;
  a.c = view;
  a.q = q;
  a.q_b = qs[0];
  a.q_h = qs[1];
  a.out = out;
  a.Hq = Hq;
  a.group = Hq / cache->heads;
  a.rows = p.rows;
  a.row_tiles = p.row_tiles;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.pages = pages;
  a.n_pages = n_pages;
  a.cluster = p.cluster;
  a.x = weights ? reinterpret_cast<float*>(ws + p.x_at) : nullptr;
  a.x_stride = p.x_stride;
  a.lse2 = weights ? reinterpret_cast<float*>(ws + p.lse_at) : nullptr;
  a.meta = reinterpret_cast<int4*>(ws + p.meta_at);
  a.part_ml = reinterpret_cast<float2*>(ws + p.ml_at);
  a.part_o = reinterpret_cast<float*>(ws + p.o_at);
  a.D4 = (D + 3) / 4 * 4;
  const unsigned long long ps = static_cast<unsigned long long>(cache->page_size);
  a.ps_shift = 0;
  while ((1ull << a.ps_shift) < ps) ++a.ps_shift;
  a.ps_mul = static_cast<unsigned>((((1ull << a.ps_shift) - ps) << 32) / ps + 1);

  if (!(weights ? launch_first<true>(a, p, cache->dtype, stream) : launch_first<false>(a, p, cache->dtype, stream)))
    return ATTN_ERR_LAUNCH;
  const dim3 grid(p.grid, p.rows), block(kJoinWarps * 32);
  bool ok = true;
  if (!p.cluster) switch (cache->dtype) {
    case ATTN_F16: ok = launch_after(attn_decode_join_kernel<__half>, grid, block, 0, stream, 1, true, a); break;
    case ATTN_BF16: ok = launch_after(attn_decode_join_kernel<__nv_bfloat16>, grid, block, 0, stream, 1, true, a); break;
    default: ok = launch_after(attn_decode_join_kernel<float>, grid, block, 0, stream, 1, true, a); break;
  }
  if (ok && weights) {
    const dim3 wgrid((view.capacity() + 255) / 256, cache->heads, cache->B);
    ok = wgrid.x == 0 || launch_after(attn_decode_weights_kernel, wgrid, dim3(256), 0, stream, 1, true, a, weights,
                                      weights_strides[0], weights_strides[1]);
  }
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}
