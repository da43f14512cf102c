// Attention of drafted tokens over a paged key-value cache (launch_attn_tree).
//
// Sequence b has n drafted tokens at its end, token s at position base + s,
// base = seq_lens[b] - n.  For query head i of the g heads that read kv head h,
// drafted token s, and the tokens t of the sequence that s may see (t < base,
// or t = base + a for a = s, parent(s), parent(parent(s)), ...):
//   x_t = scale * log2(e) * (q_{i,s} . k_t),  M = max x_t,  L = sum 2^(x_t - M),
//   o_{i,s} = sum 2^(x_t - M) v_t / L,  and 0 where there is no token
//   (where there are tokens and every x_t is -inf, 0 / 0: NaN, as the formula).
//
// The g S rows (i, s) of a kv head read the same K and V, i outermost, so that
// rows r = i S + s are contiguous in the output.  The work is dealt out by
// tokens: a unit is one (sequence, kv head, tile of rows), its tokens are cut in
// tiles, and the tiles of all units in a row are dealt out in equal runs to a
// grid that fills the GPU once; each CTA works out its own run from seq_lens,
// so the host needs no lengths and a ragged batch loads every SM alike.  A
// unit cut by the ends of runs leaves its parts (M, L and the unscaled O, fp32)
// in the workspace and a second kernel joins them in the order of the tokens.
//
// What carries the products depends on the rows:
//   up to 8, 16-bit   attn_decode's kernel, the rows as columns of mma.sync: 17
//                     sequences of up to 2047 tokens, 16 kv heads of 64, five
//                     rows 32.4 us, 35.5 here
//   up to 128         tcgen05, tiles of 64 tokens, two CTAs per SM: 273 MB in 61
//                     to 65 us on different GPUs, of which the join takes 3
//   above             tcgen05, 256 rows in two streams over the same tiles of
//                     128 tokens: K and V cross the copy engine once for both
//   fp32, odd strides dot products on the plain cores
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

__device__ int g_page_fault = 0;

constexpr int kMaxDrafted = 1024;  // tokens of a tree, at most: parents lie in shared memory

struct TreeArgs {
  PagedView c;
  const void* q;
  long long q_b, q_h, q_s;  // element strides of q over (batch, head, token)
  void* out;                // [B, Hq, S, D] contiguous
  int Hq, group, S;
  int rows;                  // group * S rows per kv head, in row_tiles tiles of unit_rows
  int unit_rows, row_tiles;
  int tile;                  // tokens per tile
  float scale_log2;
  const int* parents;        // or null: a chain
  long long parents_stride;
  const int* new_lens;       // or null: S
  int4* meta;                // [gridDim.x]: kv head's first output row, tile of rows, CTAs that continue the unit begun last
  float2* part_ml;           // [2 gridDim.x][unit_rows]
  float4* part_o;            // [2 gridDim.x][D4][unit_rows]: a row of threads writes and reads it in a row
  int D4;                    // D / 4, rounded up
  // x / page_size, x / S and x / tile for x < 2^31 as (umulhi(x, mul) + x) >> shift:
  // Granlund and Montgomery, Division by Invariant Integers using
  // Multiplication (1994), figure 4.1.
  unsigned ps_mul, s_mul, t_mul;
  int ps_shift, s_shift, t_shift;
  __device__ __forceinline__ int page_at(int pos) const {
    const unsigned p = static_cast<unsigned>(pos);
    return static_cast<int>((__umulhi(p, ps_mul) + p) >> ps_shift);
  }
  __device__ __forceinline__ int head_at(int row) const {
    const unsigned r = static_cast<unsigned>(row);
    return static_cast<int>((__umulhi(r, s_mul) + r) >> s_shift);
  }
};

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
__device__ __forceinline__ float inverse(float M, float L) {
  return L != 0.f ? 1.f / L : M == -INFINITY ? 0.f : __int_as_float(0x7fffffff);
}

// ---------------------------------------------------------------------------
// Sequences and runs of tiles
// ---------------------------------------------------------------------------

// The tokens of a sequence: `len` in the cache, the last `n` from position
// `base` on drafted (base < 0: the first of them are not there).  base is len
// at most, so that a tile up to base is whole: drafted tokens that lie behind
// the table's end are not there, wherever they lie.
struct Seq {
  int len, n, base;
};

// What memory holds of a sequence, asked for well before it is used.
struct RawSeq {
  int len, n;
};
__device__ __forceinline__ RawSeq raw_seq(const TreeArgs& a, int b) {
  RawSeq r{0, 0};
  if (b < a.c.B) {
    r.len = *(a.c.lens + b);
    r.n = a.new_lens ? *(a.new_lens + b) : a.S;
  }
  return r;
}
__device__ __forceinline__ Seq seq_from(const TreeArgs& a, const RawSeq& r, int* fault) {
  Seq s;
  s.n = max(min(r.n, a.S), 0);
  s.len = max(min(r.len, a.c.capacity()), 0);
  s.base = min(max(r.len, 0) - s.n, s.len);
  if (r.n > a.S || r.len > a.c.capacity()) *fault |= kFaultPage;
  return s;
}
__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int b, int* fault) { return seq_from(a, raw_seq(a, b), fault); }

// A place in the row of tiles: tile t of the T tiles of the unit (sequence b,
// kv head h, tile rt of its rows).
struct Cursor {
  int b, h, rt, t, T;
  Seq s;
};

__device__ __forceinline__ int tiles_of(const TreeArgs& a, const Seq& s) {
  const unsigned x = static_cast<unsigned>(s.len + a.tile - 1);
  return s.n > 0 ? static_cast<int>((__umulhi(x, a.t_mul) + x) >> a.t_shift) : 0;
}

// To the next unit; `ahead` is the sequence behind c.b, on its way.
__device__ __forceinline__ void next_unit(const TreeArgs& a, Cursor& c, RawSeq& ahead, int* fault) {
  c.t = 0;
  if (++c.rt < a.row_tiles) return;
  c.rt = 0;
  if (++c.h < a.c.heads) return;
  c.h = 0;
  c.T = 0;
#pragma unroll 1
  while (c.T == 0 && ++c.b < a.c.B) {
    c.s = seq_from(a, ahead, fault);
    ahead = raw_seq(a, c.b + 1);
    c.T = tiles_of(a, c.s);
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

template <int kThreads>
struct ScheduleSmem {
  int warp_sum[kThreads / 32];
  Cursor first;
};

// Works out this CTA's run and its first tile; all its threads share the
// batch.  The host keeps the number of tiles the block table can name below
// 2^31.
template <int kThreads>
__device__ __forceinline__ Cursor schedule(const TreeArgs& a, ScheduleSmem<kThreads>& s, Run* run, int* fault) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = (a.c.B + kThreads - 1) / kThreads;
  const long long from = static_cast<long long>(threadIdx.x) * seg;
  const int b0 = from < a.c.B ? static_cast<int>(from) : a.c.B, b1 = min(a.c.B - b0, seg) + b0;
  int mine = 0, T = 0;
  Seq q = {};
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    q = seq_of(a, b, fault);
    T = tiles_of(a, q);
    mine += T;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  if (lane == 31) s.warp_sum[warp] = upto;
  __syncthreads();
  int before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s.warp_sum[w];
    total += s.warp_sum[w];
  }
  const int units = a.c.heads * a.row_tiles, grid = gridDim.x, c = blockIdx.x;
  total *= units;
  run->each = static_cast<unsigned>(total) / static_cast<unsigned>(grid);
  run->longer = total - run->each * grid;
  run->first = c * run->each + min(c, run->longer);
  run->n = run->each + (c < run->longer ? 1 : 0);
  if (run->n > 0 && run->first >= before * units && run->first - before * units < mine * units) {
    int in = run->first - before * units, b = b0;
    if (seg > 1) {
#pragma unroll 1
      for (;; ++b) {
        q = seq_of(a, b, fault);
        T = tiles_of(a, q);
        if (in < T * units || b + 1 >= b1) break;
        in -= T * units;
      }
    }
    const int hu = in / T, h = hu / a.row_tiles;
    s.first = Cursor{b, h, hu - h * a.row_tiles, in - hu * T, T, q};
  }
  __syncthreads();
  return run->n > 0 ? s.first : Cursor{};  // nobody has written a first tile of an empty run
}

// Output rows of sequences without tokens, or without drafted ones, are zeros.
template <typename T, int kThreads>
__device__ __forceinline__ void zero_empty_rows(const TreeArgs& a, int* fault) {
  const long long bytes = static_cast<long long>(a.Hq) * a.S * a.c.D * sizeof(T);
  const bool wide = bytes % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
#pragma unroll 1
  for (int b = blockIdx.x; b < a.c.B; b += gridDim.x) {
    const Seq s = seq_of(a, b, fault);
    if (s.len > 0 && s.n > 0) continue;
    unsigned char* o = static_cast<unsigned char*>(a.out) + b * bytes;
    if (wide) {
#pragma unroll 1
      for (long long i = threadIdx.x; i < bytes / 16; i += kThreads) reinterpret_cast<uint4*>(o)[i] = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll 1
      for (long long i = threadIdx.x; i < bytes / static_cast<long long>(sizeof(T)); i += kThreads)
        reinterpret_cast<T*>(o)[i] = from_f32<T>(0.f);
    }
  }
}

// The drafted tokens that each one follows: the first kParShared of them in
// shared memory, the others where they are.
constexpr int kParShared = 256;
struct Tree {
  const int* shared;
  const int* global;  // null: a chain
  __device__ __forceinline__ int parent(int s, int* fault) const {
    if (!global) return s - 1;
    const int p = s < kParShared ? shared[s] : global[s];
    if (p >= -1 && p < s) return p;
    *fault |= kFaultPage;
    return -1;
  }
};
__device__ __forceinline__ const int* tree_of(const TreeArgs& a, int b) {
  return a.parents ? a.parents + b * a.parents_stride : nullptr;
}

// Bits of the kWords * 32 positions from `pos0` on that drafted token s of the
// sequence may see (s < n), beside those the sequence has there.
template <int kWords>
__device__ __forceinline__ void visible(const Seq& q, int s, int pos0, const Tree& tree, uint32_t (&bits)[kWords],
                                        int* fault) {
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    // positions below base: all of them
    const int in = q.base - (pos0 + 32 * w);
    bits[w] = in >= 32 ? 0xffffffffu : in > 0 ? (1u << in) - 1u : 0u;
  }
  if (!tree.global) {
    // a chain: also those up to s
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const int in = q.base + s + 1 - (pos0 + 32 * w);
      const uint32_t upto = in >= 32 ? 0xffffffffu : in > 0 ? (1u << in) - 1u : 0u;
      bits[w] |= upto;
    }
    if (q.base < 0) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) bits[w] = q.base + s >= 0 ? bits[w] : 0u;
    }
    return;
  }
#pragma unroll 1
  for (int p = s; p >= 0; p = tree.parent(p, fault)) {
    const int at = q.base + p - pos0;
    if (at < 0) break;  // ancestors only lie further ahead
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      if (at >> 5 == w) bits[w] |= 1u << (at & 31);
  }
}

// Where token `pos` lies: its physical page and row, or page -1.
__device__ __forceinline__ int page_of(const TreeArgs& a, const Cursor& c, int pos, int* row, int* fault) {
  if (pos >= c.s.len) return -1;
  const int lp = a.page_at(pos);
  *row = pos - lp * a.c.page_size;
  return paged_page(a.c, c.b, lp, fault);
}

// Where a unit's result goes: the output when the whole unit was in this
// CTA's run, otherwise a part of the workspace (the first of the CTA's two
// for a unit begun earlier, the second for one begun here).
struct Place {
  bool whole;
  long long row0;  // first output row of the kv head
  int slot;
};

__device__ __forceinline__ Place place_of(const TreeArgs& a, const Cursor& c, bool begun, const Run& run, int tile,
                                          bool record) {
  Place p;
  p.row0 = (static_cast<long long>(c.b) * a.Hq + static_cast<long long>(c.h) * a.group) * a.S;
  const bool ends = c.t + 1 == c.T;
  p.whole = begun && ends;
  p.slot = 2 * blockIdx.x + (begun ? 1 : 0);
  if (begun && !ends && record) {
    const int later = run.owner(tile + c.T - 1 - c.t) - static_cast<int>(blockIdx.x);  // `tile` is tile c.t of the unit
    // b * Hq + head < 2^31, which the host checks
    a.meta[blockIdx.x] = make_int4(c.b * a.Hq + c.h * a.group, c.rt, later, 0);
  }
  return p;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---------------------------------------------------------------------------
// SIMT kernel: fp32, any head dim, any strides
// ---------------------------------------------------------------------------

// 32 rows by 64 tokens per tile.  Thread (ty, tx) of 8 x 16 has rows 4 ty + {0
// .. 3}: scores of tokens tx + 16 {0 .. 3}, and of O the columns 4 tx + {0 .. 3}
// + 64 j.  K and V lie in 32 bits, in a buffer each where copies of 16 bytes can
// fill them (kWide: fp32, 16-byte rows), so that the next tile's come while this
// one is worked on; else one after the other in one buffer.  fp32, n sequences of
// 1/n, 2/n ... of the given length, us (in brackets one buffer and an element per
// load): 3 of 1500 tokens, 16/4 heads of 64, 7 drafted 16.0 (30.5); 16 of 8192 97
// (446); 16 of 4096, 32/8 heads of 128, 8 drafted 227 (808); 8 of 4096, 16/4 of
// 256, 8 drafted 152 (596).  16 bits, element by element: 16 of 4096, 32/8 heads of
// 100, 8 drafted 374.  Two buffers cost CTAs per SM (4, 2 and 1 at D = 64, 128 and 256 instead of 5, 3 and 2).
constexpr int kSimtThreads = 128, kSimtRows = 32, kSimtTile = 64;

template <int kDP, bool kWide>
struct SimtCfg {
  static constexpr int kPitch = kDP + 4;  // floats; rows 4 banks apart
  static constexpr int kPPitch = kSimtTile + 4;
  static constexpr size_t kBytes = sizeof(float) * ((kSimtRows + (kWide ? 2 : 1) * kSimtTile) * kPitch + kSimtRows * kPPitch) +
                                   sizeof(long long) * 4 * kSimtTile + sizeof(int) * kParShared;
};

template <typename T, int kDP, bool kWide>
__global__ void __launch_bounds__(kSimtThreads) attn_tree_simt_kernel(const __grid_constant__ TreeArgs a) {
  using C = SimtCfg<kDP, kWide>;
  constexpr int kCols = kDP / 16;
  extern __shared__ __align__(16) float sm[];
  float* s_q = sm;
  float* s_k = s_q + kSimtRows * C::kPitch;
  float* s_v = kWide ? s_k + kSimtTile * C::kPitch : s_k;
  float* s_p = s_v + kSimtTile * C::kPitch;
  long long* s_at = reinterpret_cast<long long*>(s_p + kSimtRows * C::kPPitch);  // K, then V offsets; -1: no token
  long long* s_next = s_at + 2 * kSimtTile;                                      // those of the next tile (kWide)
  int* s_par = reinterpret_cast<int*>(s_next + 2 * kSimtTile);
  Tree tree{s_par, nullptr};
  __shared__ ScheduleSmem<kSimtThreads> s_sched;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, D = a.c.D;
  int fault = 0;
  launch_dependents();
  grid_dependency_wait();
  if (tid == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  Run run;
  Cursor cur = schedule(a, s_sched, &run, &fault);
  zero_empty_rows<T, kSimtThreads>(a, &fault);
  RawSeq ahead = raw_seq(a, cur.b + 1);
  float o[4][kCols], m[4], l[4];
  bool begun = cur.t == 0, fresh = true;
  const T* kbase = static_cast<const T*>(a.c.k);
  const T* vbase = static_cast<const T*>(a.c.v);

  // Rows of the cache to `to`, zeros behind D and where there is no token.
  auto load = [&](float* to, const T* base, const long long* at) {
    if constexpr (kWide) {
#pragma unroll
      for (int e = tid; e < kSimtTile * kDP / 4; e += kSimtThreads) {
        const int r = e / (kDP / 4), d = e % (kDP / 4) * 4;
        const bool is = at[r] >= 0 && d < D;
        cp_async16(smem_addr(to + r * C::kPitch + d), base + (is ? at[r] + d : 0), is);
      }
      cp_async_commit();
    } else {
#pragma unroll 1
      for (int e0 = tid; e0 < kSimtTile * kDP; e0 += 8 * kSimtThreads) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = e0 + k * kSimtThreads, r = e / kDP, d = e % kDP;
          x[k] = at[r] >= 0 && d < D ? to_f32(base[at[r] + d]) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = e0 + k * kSimtThreads;
          to[e / kDP * C::kPitch + e % kDP] = x[k];
        }
      }
    }
  };
  // Token `pos`, this thread's of a tile, to its place in `at`.
  auto locate = [&](int page, int row, long long* at) {
    at[tid] = page < 0 ? -1 : page * a.c.ks[0] + cur.h * a.c.ks[1] + row * a.c.ks[2];
    at[kSimtTile + tid] = page < 0 ? -1 : page * a.c.vs[0] + cur.h * a.c.vs[1] + row * a.c.vs[2];
  };

  for (int i = 0; i < run.n; ++i) {
    const int pos0 = cur.t * kSimtTile;
    int page = -1, row = 0;
    if (fresh || !kWide) {
      if (tid < kSimtTile) {
        page = page_of(a, cur, pos0 + tid, &row, &fault);
        locate(page, row, s_at);
      }
      __syncthreads();
      load(s_k, kbase, s_at);
      if constexpr (kWide) load(s_v, vbase, s_at + kSimtTile);
    }
    if (fresh) {
      const T* q = static_cast<const T*>(a.q) + cur.b * a.q_b + static_cast<long long>(cur.h) * a.group * a.q_h;
#pragma unroll 16
      for (int e = tid; e < kSimtRows * kDP; e += kSimtThreads) {
        const int r = e / kDP, d = e % kDP, gr = cur.rt * kSimtRows + r;
        const int head = a.head_at(gr), s = gr - head * a.S;
        s_q[r * C::kPitch + d] = gr < a.rows && d < D ? to_f32(q[head * a.q_h + s * a.q_s + d]) : 0.f;
      }
      tree.global = tree_of(a, cur.b);
      for (int e = tid; tree.global && e < min(cur.s.n, kParShared); e += kSimtThreads) s_par[e] = tree.global[e];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[r][c] = 0.f;
      }
      fresh = false;
    }
    const bool more = kWide && cur.t + 1 < cur.T && i + 1 < run.n;  // another tile of this unit
    if (more && tid < kSimtTile) page = page_of(a, cur, pos0 + kSimtTile + tid, &row, &fault);
    if constexpr (kWide) cp_async_wait<1>();  // V may be on its way
    __syncthreads();
    float x[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < kDP; d += 4) {
      float4 q[4], k[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) q[r] = *reinterpret_cast<const float4*>(s_q + (ty * 4 + r) * C::kPitch + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) k[c] = *reinterpret_cast<const float4*>(s_k + (tx + 16 * c) * C::kPitch + d);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[r][c] = fmaf(q[r].x, k[c].x, x[r][c]);
          x[r][c] = fmaf(q[r].y, k[c].y, x[r][c]);
          x[r][c] = fmaf(q[r].z, k[c].z, x[r][c]);
          x[r][c] = fmaf(q[r].w, k[c].w, x[r][c]);
        }
    }
    // Which tokens each row may see: lane r of the 16 that share four rows finds it for row r.
    uint32_t see[2] = {0, 0};
    if (tx < 4) {
      const int gr = cur.rt * kSimtRows + ty * 4 + tx, s = gr % a.S;
      if (gr < a.rows && s < cur.s.n) visible<2>(cur.s, s, pos0, tree, see, &fault);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int from = (tid & 16) + r;
      const uint32_t lo = __shfl_sync(0xffffffffu, see[0], from), hi = __shfl_sync(0xffffffffu, see[1], from);
      float top = -INFINITY;
      bool is[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int t = tx + 16 * c;
        is[c] = ((t < 32 ? lo >> t : hi >> (t - 32)) & 1u) && s_at[t] >= 0;
        x[r][c] = is[c] ? x[r][c] * a.scale_log2 : -INFINITY;
        if (is[c]) top = fmaxf(top, fmaxf(x[r][c], kLowest));
      }
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = fmaxf(m[r], top), f = ex2_approx(m[r] - finite_max(mn));
      m[r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = is[c] ? ex2_approx(x[r][c] - finite_max(mn)) : -0.f;  // -0: not a token of this row
        s_p[(ty * 4 + r) * C::kPPitch + tx + 16 * c] = p;
        sum += p;
      }
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * f + sum;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[r][c] *= f;
    }
    if (more && tid < kSimtTile) locate(page, row, s_next);
    __syncthreads();  // K is used up
    if constexpr (kWide) {
      if (more) load(s_k, kbase, s_next);
      else cp_async_commit();  // a group either way
      cp_async_wait<1>();
    } else {
      load(s_v, vbase, s_at + kSimtTile);
    }
    __syncthreads();
    const bool drafts = pos0 + kSimtTile > cur.s.base;
    for (int t = 0; t < kSimtTile; t += 4) {
      float4 p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = *reinterpret_cast<const float4*>(s_p + (ty * 4 + r) * C::kPPitch + t);
#pragma unroll
      for (int j = 0; j < kDP / 64; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 v = *reinterpret_cast<const float4*>(s_v + (t + k) * C::kPitch + j * 64 + tx * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = k == 0 ? p[r].x : k == 1 ? p[r].y : k == 2 ? p[r].z : p[r].w;
            // A drafted token the row does not follow adds nothing, be it infinite or NaN.
            if (drafts && __float_as_uint(w) == 0x80000000u) continue;
            o[r][j * 4 + 0] = fmaf(w, v.x, o[r][j * 4 + 0]);
            o[r][j * 4 + 1] = fmaf(w, v.y, o[r][j * 4 + 1]);
            o[r][j * 4 + 2] = fmaf(w, v.z, o[r][j * 4 + 2]);
            o[r][j * 4 + 3] = fmaf(w, v.w, o[r][j * 4 + 3]);
          }
        }
    }
    if (cur.t + 1 == cur.T || i + 1 == run.n) {
      const Place p = place_of(a, cur, begun, run, run.first + i, tid == 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int in = ty * 4 + r, gr = cur.rt * kSimtRows + in;
        if (gr >= a.rows) continue;
        const float inv = inverse(m[r], l[r]);
#pragma unroll
        for (int j = 0; j < kCols / 4; ++j) {
          const int d = j * 64 + tx * 4;
          if (d >= D) continue;
          if (p.whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + e < D)
                static_cast<T*>(a.out)[(p.row0 + gr) * D + d + e] =
                    from_f32<T>(m[r] == -INFINITY ? 0.f : o[r][j * 4 + e] * inv);
          } else {
            a.part_o[(static_cast<long long>(p.slot) * a.D4 + d / 4) * kSimtRows + in] =
                make_float4(o[r][j * 4], o[r][j * 4 + 1], o[r][j * 4 + 2], o[r][j * 4 + 3]);
          }
        }
        if (!p.whole && tx == 0) a.part_ml[static_cast<long long>(p.slot) * kSimtRows + in] = make_float2(m[r], l[r]);
      }
      begun = true;
      fresh = true;
    }
    __syncthreads();  // the tile's buffers are free
    if (more) {
      load(s_v, vbase, s_next + kSimtTile);
      long long* at = s_at;
      s_at = s_next;
      s_next = at;
    }
    if (++cur.t == cur.T) next_unit(a, cur, ahead, &fault);
  }
  if constexpr (kWide) cp_async_wait_all();
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Tensor-core kernel: fp16 and bf16, D a multiple of 8, 16-byte rows
// ---------------------------------------------------------------------------

// The rows of a kv head are the rows of the tcgen05 products: S = Q K^T into
// tensor memory, a thread per row takes the softmax of it and writes P over it,
// O += P V.  Up to 128 rows the floor is the time to read the cache, 2800 clocks
// for 64 KB as an SM's share, the K and V of 128 tokens at D = 128.
//   up to 128 rows   tiles of 64 tokens, two score buffers, so that S(j + 1) is
//                    there when the softmax of tile j ends; two CTAs per SM (one
//                    at D = 256).  With 64 rows each takes 3390 clocks for a tile,
//                    the two of an SM 1690, where reading takes 1400 and the
//                    chain of product, softmax and product alone 1600; no unit
//                    is busy, and which wait it is has not been found.  One CTA with
//                    two tiles in turn is slower (66 to 76 us for 62).
//                    Q of the next unit is copied during this one where there
//                    is room (up to 64 rows; at D = 64 up to 128): a load takes
//                    some 5000 clocks beside so many copies.
//   more rows        256 at a time over the same tiles of 128 tokens: two
//                    streams, each with its S and O in tensor memory and a
//                    warpgroup for the softmax, one CTA per SM.  A tile's chain
//                    is 3900 clocks; Q of the next unit is asked for when this
//                    one has ended.
// Warp roles: softmax warpgroups, then one warp of which a thread issues the
// products, and one that copies K and V (one for each with two streams), page ids
// looked up ahead: boxes of rows by TMA where 8 divides the page size, else by
// 16-byte asynchronous copies.  It also mends V of tiles that end early.
template <int kD_, bool kTwo_>
struct TcCfg {
  static constexpr int kD = kD_;
  static constexpr bool kTwo = kTwo_;
  static constexpr int kStreams = kTwo ? 2 : 1;
  static constexpr int kCtas = kTwo || kD == 256 ? 1 : 2;  // per SM
  static constexpr int kBN = kTwo ? 128 : 64;              // tokens per tile
  static constexpr int kRows = 128 * kStreams;
  static constexpr uint32_t kQBytes = 128u * kD * 2;       // a Q tile
  // Q tiles there is room for: two row tiles; at D = 64 this unit's and the
  // next one's; otherwise one, or two of up to 64 rows.
  static constexpr int kQTiles = kTwo || kD == 64 ? 2 : 1;
  static constexpr uint32_t kSlotBytes = kBN * kD * 2u;  // a K or V tile
  static constexpr uint32_t kSlotBlock = kBN * 128u;     // 64 columns of it
  static constexpr int kKSlots = kTwo ? (kD == 64 ? 5 : 2) : kD == 64 ? 4 : 2;
  static constexpr int kVSlots = kTwo ? (kD == 64 ? 5 : 3) : kD == 64 ? 4 : kD == 128 ? 2 : 3;
  static constexpr uint32_t kColO = 2 * kBN;               // after the scores: two buffers, or one of each stream
  static constexpr uint32_t kTmemCols = kColO + kStreams * kD <= 256 ? 256 : 512;
  static constexpr int kSoftThreads = 128 * kStreams;
  static constexpr int kMmaWarp = 4 * kStreams, kCopyWarp = kMmaWarp + 1;
  static constexpr int kThreads = kSoftThreads + 32 + 32 * kStreams;
  static constexpr uint32_t kTileBytes = kQTiles * kQBytes + (kKSlots + kVSlots) * kSlotBytes;
  static constexpr size_t kCtlBytes = 3 * 1024;
  static constexpr size_t kSmemBytes = kTileBytes + kCtlBytes;
  static_assert(kSmemBytes <= (kCtas == 1 ? 232448 : 115712), "shared memory of a CTA");
};
// A wait that did not end at once: mbar_wait's polling, once in the program.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* code,
                                       unsigned long long limit_ns) {
  return mbar_wait(bar, parity, abort_flag, code, 1, limit_ns);
}

constexpr int kHoles = 8;  // tiles, and units, that are remembered: more than the copies may be ahead

template <typename C>
struct __align__(16) TcCtl {
  uint64_t q_full;                          // a unit's Q (kSoftThreads arrivals)
  uint64_t k_full[C::kKSlots], k_empty[C::kKSlots], v_full[C::kVSlots], v_empty[C::kVSlots];
  uint64_t v_raw[C::kVSlots];               // V has come, and is to be mended before it is full
  uint64_t s_full[2], p_full[2];            // of a score buffer
  uint64_t o_done;                          // the last product of a unit
  uint64_t met;                             // the softmax threads meet
  uint64_t mma_done;
  unsigned long long hole[kHoles][2];       // tokens of a tile that lie in no page of the cache
  int4 mend[kHoles];                        // of tiles to mend: first drafted row, rows, draft of row 0, unit
  uint32_t odd[kHoles][kMaxDrafted / 256];  // of a unit: eights of drafted tokens with infinite or NaN values
  ScheduleSmem<C::kThreads> sched;
  uint32_t tmem_base;
  int abort_flag, code;
  int par[2][kParShared];
};

// The two caches as [num_pages, heads, page_size, D] tensors read in boxes of
// `rows` rows by 64 columns.
struct TcMaps {
  CUtensorMap k, v;
  int rows, boxes;  // rows of a box, boxes of a tile; 0: no boxes, 16-byte copies
  unsigned long long wait_ns;
  int lose;  // watchdog test build only: CTA 0's first K copy is for bytes that never come, or is never told
};

// Whether the phase has completed, without waiting for it.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

template <bool kBf16, int kD, bool kTwo>
__global__ void __launch_bounds__(TcCfg<kD, kTwo>::kThreads, TcCfg<kD, kTwo>::kCtas)
    attn_tree_tc_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ TcMaps maps) {
  using C = TcCfg<kD, kTwo>;
  using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  constexpr int kBN = C::kBN, kWords = kBN / 32;
  static_assert(sizeof(TcCtl<C>) <= C::kCtlBytes, "control block");
  // fp16 has its full precision down to 2^-14: P is kept times 2^7 (at most
  // 2^15, as the maximum it refers to may be 2^8 below the largest score).
  constexpr float kUp = kBf16 ? 0.f : 7.f;

  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::kQTiles * C::kQBytes;
  uint8_t* sV = sK + C::kKSlots * C::kSlotBytes;
  TcCtl<C>& ctl = *reinterpret_cast<TcCtl<C>*>(smem + C::kTileBytes);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0), lane = threadIdx.x & 31;
  int fault = 0;

  if (threadIdx.x == 0) {
    ctl.abort_flag = ctl.code = 0;
    mbar_init(&ctl.q_full, C::kSoftThreads);
    for (int s = 0; s < C::kKSlots; ++s) {
      mbar_init(&ctl.k_full[s], 1);
      mbar_init(&ctl.k_empty[s], 1);
    }
    for (int s = 0; s < C::kVSlots; ++s) {
      mbar_init(&ctl.v_full[s], 1);
      mbar_init(&ctl.v_empty[s], 1);
      mbar_init(&ctl.v_raw[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl.s_full[s], 1);
      mbar_init(&ctl.p_full[s], 128);
    }
    mbar_init(&ctl.o_done, 1);
    mbar_init(&ctl.met, C::kSoftThreads);
    mbar_init(&ctl.mma_done, 1);
    fence_mbar_init();
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(smem_addr(&ctl.tmem_base), C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == C::kCopyWarp && lane == 0) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base;
  // The next kernel's CTAs may come once every CTA of this one has its tensor
  // memory, so that none of them can take what this one waits for.
  launch_dependents();
  grid_dependency_wait();
  if (threadIdx.x == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  Run run;
  Cursor cur = schedule(a, ctl.sched, &run, &fault);
  const int n = run.n;
  RawSeq ahead = raw_seq(a, cur.b + 1);

  const unsigned long long wait_ns = maps.wait_ns;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool there = __all_sync(0xffffffffu, mbar_try_wait(smem_addr(bar), parity) ||
                                                   wait_long(bar, parity, &ctl.abort_flag, &ctl.code, wait_ns));
    if (!there) fault |= kFaultWait;
    return there;
  };
  int last_copy[2] = {-1, -1};  // the last tile whose copies of K and V went out (copying warps)
  // The tile of V to mend, when the copies of the next one are out, and the
  // parities of v_raw.
  int late = -1, late_slot = 0;
  uint32_t raw = 0;
  // Q of the next unit is copied during this one where there is room for two.
  const bool early_q = !kTwo && (C::kQTiles == 2 || a.rows <= 64);
  const int q_rows = early_q && C::kQTiles == 1 ? 64 : 128;  // of a Q tile
  const uint32_t q_block = q_rows * 128, q_tile = q_block * (kD / 64);

  if (warp >= C::kCopyWarp) {
    // ---------------------------------------------------------------- copies
    const bool does[2] = {!kTwo || warp == C::kCopyWarp, !kTwo || warp != C::kCopyWarp};  // K, V
    int left = n, slot[2] = {0, 0};
    uint32_t parity[2] = {1, 1};  // of the slots' `empty`: the first round finds it so
    bool ok = true;
    auto full = [&](int kv, int s) { return kv ? &ctl.v_full[s] : &ctl.k_full[s]; };
    auto empty = [&](int kv, int s) { return kv ? &ctl.v_empty[s] : &ctl.k_empty[s]; };
    auto to_next = [&](int kv) {
      if (++slot[kv] == (kv ? C::kVSlots : C::kKSlots)) slot[kv] = 0, parity[kv] ^= 1;
    };

    // V of a tile as the product may see it: rows that are no tokens are zeros
    // (no weight, not even zero, may meet what lies there), and so are infinite and
    // NaN values of drafted tokens, which some rows do not follow; the rows
    // that do add them at the end.
    constexpr int kCols = kD / 8, kPer = kCols >= 32 ? 1 : 32 / kCols;  // 16-byte columns of a row, rows at once
    const int col = lane % kCols, my_row = lane / kCols;
    int unit = -1;
    bool unit_begins = true;
    // Notes what there is to mend of tile j, cur's or the look-up's; whether there is anything.
    auto note_mend = [&](int j, const Seq& q, int t, bool begins, bool holes) {
      if (begins) {
        ++unit;
        if (lane < kMaxDrafted / 256) ctl.odd[unit % kHoles][lane] = 0;
      }
      const int pos0 = t * a.tile;
      if (pos0 + a.tile <= q.base && !holes) return false;
      if (lane == 0)
        ctl.mend[j % kHoles] = make_int4(max(0, q.base - pos0), min(q.len - pos0, a.tile), pos0 - q.base, unit % kHoles);
      __syncwarp();
      return true;
    };
    auto mend = [&](int j, int in_slot, unsigned long long hole0, unsigned long long hole1) {
      const int4 what = ctl.mend[j % kHoles];
      uint8_t* v = sV + in_slot * C::kSlotBytes + (col / 8) * C::kSlotBlock;
      auto place = [&](int r) { return reinterpret_cast<uint4*>(v + r * 128 + (((col % 8) ^ (r & 7)) << 4)); };
#pragma unroll 1
      for (int r = what.y + my_row; r < kBN; r += kPer) *place(r) = make_uint4(0, 0, 0, 0);
      if (hole0 | hole1) {
#pragma unroll 1
        for (int r = my_row; r < kBN; r += kPer)
          if ((r < 64 ? hole0 >> r : hole1 >> (r & 63)) & 1u) *place(r) = make_uint4(0, 0, 0, 0);
      }
#pragma unroll 1
      for (int r = what.x + my_row; r < what.y; r += kPer) {
        uint4* at = place(r);
        uint32_t x[4] = {at->x, at->y, at->z, at->w};
        bool odd = false;
        constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((x[i] & kExp) == kExp) x[i] &= 0xffff0000u, odd = true;
          if ((x[i] >> 16 & kExp) == kExp) x[i] &= 0xffffu, odd = true;
        }
        if (odd) {
          *at = make_uint4(x[0], x[1], x[2], x[3]);
          const int eight = (what.z + r) >> 3;
          atomicOr(&ctl.odd[what.w][eight >> 5], 1u << (eight & 31));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    if (maps.boxes > 0) {
      const int R = maps.rows, boxes = maps.boxes, group = 32 / boxes;  // tiles per look-up
      const uint64_t policy = a.row_tiles > 1 ? l2_policy_evict_last() : l2_policy_evict_first();
      const int my_tile = lane / boxes, my_box = lane - my_tile * boxes;
      struct Group {
        int page, row, live;  // of this lane's box: table entry, first row, whether it has tokens
        int count, h, t;
        bool begins;  // the unit, or this run's part of it
        Seq s;
      };
      auto look_up = [&](Group& g) {
        g = Group{-1, 0, 0, 0, cur.h, cur.t, unit_begins, cur.s};
        if (left <= 0) return;
        g.count = min(min(group, cur.T - cur.t), left);
        const int pos = (cur.t + my_tile) * a.tile + my_box * R;
        if (my_tile < g.count && pos < cur.s.len) {
          const int lp = a.page_at(pos);
          g.row = pos - lp * a.c.page_size;
          g.live = 1;
          g.page = *(a.c.table + static_cast<long long>(cur.b) * a.c.table_stride + lp);
        }
        left -= g.count;
        cur.t += g.count;
        unit_begins = cur.t == cur.T;
        if (left > 0 && unit_begins) next_unit(a, cur, ahead, &fault);
      };
      if (does[1] && a.tile < kBN) {
        // Rows behind a tile's tokens: no copy reaches them.
#pragma unroll 1
        for (int v = 0; v < C::kVSlots; ++v)
#pragma unroll 1
          for (int r = a.tile + my_row; r < kBN; r += kPer)
            *reinterpret_cast<uint4*>(sV + v * C::kSlotBytes + (col / 8) * C::kSlotBlock + r * 128 +
                                      (((col % 8) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      Group now, next;
      look_up(now);
      look_up(next);
      int in = 0;
      unsigned long long late_hole[2] = {0, 0};
      auto mend_late = [&] {
        const bool there = wait(&ctl.v_raw[late_slot], raw >> late_slot & 1u);
        raw ^= 1u << late_slot;
        if (there) {
          mend(late, late_slot, late_hole[0], late_hole[1]);
          if (lane == 0) mbar_arrive(&ctl.v_full[late_slot]);
        }
        late = -1;
        return there;
      };
      for (int j = 0; j < n && ok; ++j) {
        const bool mine = my_tile == in && now.live;
        const bool good = mine && static_cast<unsigned>(now.page) < static_cast<unsigned>(a.c.num_pages);
        const uint32_t have = __ballot_sync(0xffffffffu, good);
        const uint32_t gone = __ballot_sync(0xffffffffu, mine && !good) >> (in * boxes);
        unsigned long long hole[2] = {0, 0};
#pragma unroll 1
        for (int b = 0; gone && b < boxes; ++b)
          if (gone >> b & 1u)
#pragma unroll 1
            for (int r = b * R; r < (b + 1) * R; r += 8) hole[r >> 6] |= 0xffull << (r & 63);
        if (gone) fault |= kFaultPage;
        bool to_mend = false;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!does[kv] || !ok) continue;
          if (late >= 0 && !__all_sync(0xffffffffu, mbar_test(empty(kv, slot[kv]), parity[kv]))) ok = mend_late();
          ok = ok && wait(empty(kv, slot[kv]), parity[kv]);
          if (!ok) continue;
          uint64_t* arrives = full(kv, slot[kv]);
          if (kv == 1) {
            to_mend = note_mend(j, now.s, now.t + in, now.begins && in == 0, gone != 0);
            if (to_mend) arrives = &ctl.v_raw[slot[1]];
          }
          if (lane == 0) {
            if (kv == 0) ctl.hole[j % kHoles][0] = hole[0], ctl.hole[j % kHoles][1] = hole[1];
            uint32_t bytes = __popc(have) * R * (kD * 2);
#ifdef RA_WATCHDOG_TEST
            if (maps.lose && blockIdx.x == 0 && j == 0 && kv == 0) bytes += 16;
#endif
            mbar_arrive_expect_tx(arrives, bytes);
          }
          __syncwarp();
          if (good) {
            const uint32_t dst = smem_addr((kv ? sV : sK) + slot[kv] * C::kSlotBytes) + my_box * R * 128;
#pragma unroll
            for (int c = 0; c < kD / 64; ++c)
              tma_load_4d(dst + c * C::kSlotBlock, kv ? &maps.v : &maps.k, arrives, c * 64, now.row, now.h, now.page,
                          policy);
          }
          last_copy[kv] = j;
          if (kv == 1) {
            if (late >= 0) ok = mend_late();
            if (to_mend) late = j, late_slot = slot[1], late_hole[0] = hole[0], late_hole[1] = hole[1];
          }
          to_next(kv);
        }
        if (++in == now.count) {
          in = 0;
          now = next;
          look_up(next);
        }
      }
      if (ok && late >= 0) ok = mend_late();
    } else {
      // Lane looks up tokens lane + 32 w of a tile, and copies one 16-byte
      // column (zeros behind D and where there is no token) of every kPer-th row.
      constexpr int kLag = 2;  // tiles in flight before the first is waited for
      const bool col_ok = col * 8 < a.c.D;
      struct Look {
        int page[kWords], row[kWords];  // row -1: no such token
        int h, t;
        bool begins;
        Seq s;
      };
      auto look_up = [&](Look& k) {
        k.h = cur.h;
        k.t = cur.t;
        k.s = cur.s;
        k.begins = unit_begins;
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const int in = w * 32 + lane, pos = cur.t * a.tile + in;
          k.page[w] = -1;
          k.row[w] = -1;
          if (left > 0 && in < a.tile && pos < cur.s.len) {
            const int lp = a.page_at(pos);
            k.row[w] = pos - lp * a.c.page_size;
            k.page[w] = *(a.c.table + static_cast<long long>(cur.b) * a.c.table_stride + lp);
          }
        }
        unit_begins = ++cur.t == cur.T;
        if (--left > 0 && unit_begins) next_unit(a, cur, ahead, &fault);
      };
      int told = 0, told_slot[2] = {0, 0};  // tiles whose arrival has been told
      uint32_t to_mend = 0;         // of the tiles from `told` on
      auto tell = [&](int upto) {
        fence_proxy_async_smem();
        __syncwarp();
#pragma unroll 1
        for (; told < upto; ++told) {
          if (to_mend & 1u) mend(told, told_slot[1], 0, 0);
          to_mend >>= 1;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (!does[kv]) continue;
#ifdef RA_WATCHDOG_TEST
            const bool lost = maps.lose && blockIdx.x == 0 && told == 0 && kv == 0;
#else
            constexpr bool lost = false;
#endif
            if (lane == 0 && !lost) mbar_arrive(full(kv, told_slot[kv]));
            if (++told_slot[kv] == (kv ? C::kVSlots : C::kKSlots)) told_slot[kv] = 0;
          }
        }
      };
      Look now, next;
      look_up(now);
      look_up(next);
      for (int j = 0; j < n && ok; ++j) {
        unsigned long long hole[2] = {0, 0};
        bool good[kWords];
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          good[w] = static_cast<unsigned>(now.page[w]) < static_cast<unsigned>(a.c.num_pages);
          const uint32_t gone = __ballot_sync(0xffffffffu, now.row[w] >= 0 && !good[w]);
          if (gone) fault |= kFaultPage;
          hole[w / 2] |= static_cast<unsigned long long>(gone) << (w % 2 * 32);
          good[w] = good[w] && now.row[w] >= 0;
        }
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (!does[kv] || !ok) continue;
          if (!__all_sync(0xffffffffu, mbar_test(empty(kv, slot[kv]), parity[kv]))) {
            // Nothing may wait for what has arrived meanwhile.
            cp_async_wait_all();
            tell(j);
            ok = wait(empty(kv, slot[kv]), parity[kv]);
            if (!ok) continue;
          }
          if (kv == 0 && lane == 0) ctl.hole[j % kHoles][0] = hole[0], ctl.hole[j % kHoles][1] = hole[1];
          if (kv == 1 && note_mend(j, now.s, now.t, now.begins, false)) to_mend |= 1u << (j - told);
          const long long* st = kv ? a.c.vs : a.c.ks;
          const T* from = static_cast<const T*>(kv ? a.c.v : a.c.k) + (col_ok ? col * 8 : 0) + now.h * st[1];
          const uint32_t dst = smem_addr((kv ? sV : sK) + slot[kv] * C::kSlotBytes) + (col / 8) * C::kSlotBlock;
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            // element offset of this lane's token, or -1
            const long long at = good[w] ? now.page[w] * st[0] + now.row[w] * st[2] : -1;
#pragma unroll 4
            for (int i = 0; i < 32; i += kPer) {
              const int r = i + (kPer > 1 ? my_row : 0);
              const long long off = __shfl_sync(0xffffffffu, at, r);
              const bool there = off >= 0 && col_ok;
              cp_async16(dst + (w * 32 + r) * 128 + (((col % 8) ^ (r & 7)) << 4), from + (there ? off : 0), there);
            }
          }
          last_copy[kv] = j;
          to_next(kv);
        }
        if (!ok) break;
        cp_async_commit();
        now = next;
        look_up(next);
        if (j >= kLag) {
          cp_async_wait<kLag>();
          tell(j - kLag + 1);
        }
      }
      cp_async_wait_all();
      if (ok) tell(n);
    }
  } else if (warp == C::kMmaWarp) {
    // -------------------------------------------------------------- products
    // One thread, and as few instructions as can be: it shares its scheduler
    // with softmax warps, and every wait and product it issues is in the
    // streams' way.
    constexpr uint32_t idesc_s = umma_idesc_f16(kBf16, 128, kBN, false);
    constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, 128, kD, true);
    if (elect_one()) {
      auto wait_one = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_try_wait(smem_addr(bar), parity) ||
            wait_long(bar, parity, &ctl.abort_flag, &ctl.code, wait_ns))
          return true;
        fault |= kFaultWait;
        return false;
      };
      const uint64_t qd0 = sw128_desc(smem_addr(sQ), 16, 1024), kd0 = sw128_desc(smem_addr(sK), 16, 1024);
      const uint64_t vd0 = sw128_desc(smem_addr(sV), C::kSlotBlock, 1024);
      int k_slot = 0, v_slot = 0;
      uint32_t k_parity = 0, v_parity = 0, p_parity = 0;
      const uint32_t q_step = q_block >> 4;
      // S into buffer st for the K at hand, of the run's u-th unit, whose Q is
      // waited for at its first tile.  `begins`: the first product with this K,
      // `frees`: the last.
      auto issue_s = [&](int st, bool begins, bool frees, bool first, int u) {
        if (begins && !wait_one(&ctl.k_full[k_slot], k_parity)) return false;
        if (first && !wait_one(&ctl.q_full, u & 1)) return false;
        tc_fence_after();
        const uint64_t kd = sw128_desc_step(kd0, k_slot * C::kSlotBytes);
        const uint64_t qd = sw128_desc_step(qd0, (kTwo ? st : early_q ? u & 1 : 0) * q_tile);
#pragma unroll
        for (int k = 0; k < kD / 16; ++k)
          umma_ss(tmem + st * kBN, qd + (k / 4) * q_step + (k % 4) * 2,
                  sw128_desc_step(kd, (k / 4) * C::kSlotBlock + (k % 4) * 32), idesc_s, k > 0 ? 1u : 0u);
        umma_commit(&ctl.s_full[st]);
        if (frees) {
          umma_commit(&ctl.k_empty[k_slot]);
          if (++k_slot == C::kKSlots) k_slot = 0, k_parity ^= 1;
        }
        return true;
      };
      // O += P V from buffer st with the V at hand; `anew`: O begins, `ends`: the
      // unit's last product.
      auto issue_pv = [&](int st, bool begins, bool frees, bool anew, bool ends) {
        if (begins && !wait_one(&ctl.v_full[v_slot], v_parity)) return false;
        if (!wait_one(&ctl.p_full[st], p_parity >> st & 1u)) return false;
        p_parity ^= 1u << st;
        tc_fence_after();
        const uint64_t vd = sw128_desc_step(vd0, v_slot * C::kSlotBytes);
#pragma unroll
        for (int k = 0; k < kBN / 16; ++k)
          umma_ts(tmem + C::kColO + (kTwo ? st * kD : 0), tmem + st * kBN + k * 8, sw128_desc_step(vd, k * 2048), idesc_o,
                  (!anew || k > 0) ? 1u : 0u);
        if (frees) {
          umma_commit(&ctl.v_empty[v_slot]);
          if (++v_slot == C::kVSlots) v_slot = 0, v_parity ^= 1;
        }
        if (ends) umma_commit(&ctl.o_done);
        return true;
      };
      bool ok = n > 0;
      int unit = 0, j = 0;
      if constexpr (!kTwo) ok = ok && issue_s(0, true, true, true, 0);
      while (ok && j < n) {
        const int count = min(cur.T - cur.t, n - j);  // tiles of the unit in this run
        for (int i = 0; i < count && ok; ++i, ++j) {
          const bool closes = i + 1 == count;
          if constexpr (!kTwo) {
            // S(j + 1), then P(j) V(j); the other way round before a new unit,
            // whose Q may still be on its way.
            if (!closes) ok = issue_s((j + 1) & 1, true, true, false, unit);
            ok = ok && issue_pv(j & 1, true, true, i == 0, closes);
            if (closes && j + 1 < n) ok = ok && issue_s((j + 1) & 1, true, true, true, unit + 1);
          } else {
            // S0(j), P1(j - 1) V(j - 1), S1(j), P0(j) V(j): each stream's softmax
            // runs beside the other's products.  (V(j - 1) is at hand until P1.)
            ok = issue_s(0, true, false, i == 0, unit);
            if (i > 0) ok = ok && issue_pv(1, false, true, i == 1, false);
            ok = ok && issue_s(1, false, true, false, unit);
            ok = ok && issue_pv(0, true, false, i == 0, false);
            if (closes) ok = ok && issue_pv(1, false, true, i == 0, true);
          }
        }
        ++unit;
        if (ok && j < n) next_unit(a, cur, ahead, &fault);
      }
      // Every product has retired before tensor memory is given back.
      umma_commit(&ctl.mma_done);
      volatile int no_abort = 0;
      mbar_wait(&ctl.mma_done, 0, &no_abort, &ctl.code, 1);
    }
    __syncwarp();
  } else {
    // --------------------------------------------------------------- softmax
    const int st = warp >> 2, in_tile = (warp & 3) * 32 + lane;
    const int row_off = st * 128 + in_tile;  // row within the unit
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_off + C::kColO + st * kD;
    const float c = a.scale_log2;
    const uint64_t c2 = f2(c, c);
    uint32_t met = 0;
    // The softmax threads meet (by a wait that ends, as all here).
    auto meet = [&] {
      mbar_arrive(&ctl.met);
      const bool there = wait(&ctl.met, met);
      met ^= 1;
      return there;
    };
    // Starts the copy of a unit's Q rows, those of warps that have any (zeros
    // behind the last and behind D), and of its sequence's tree.
    auto copy_unit = [&](const Cursor& u, int tile, int par_buf, bool tree) {
      constexpr int kCols = kD / 8, kAtOnce = C::kSoftThreads / kCols;  // columns of a row, rows at once
      static_assert(kAtOnce % 4 == 0, "rows at once");
      const int col = threadIdx.x % kCols, r0 = threadIdx.x / kCols;
      const int used = (min(a.rows - u.rt * C::kRows, C::kRows) + 31) & ~31;
      const T* q = static_cast<const T*>(a.q) + u.b * a.q_b + static_cast<long long>(u.h) * a.group * a.q_h + col * 8;
      const uint32_t to = smem_addr(sQ) + tile * q_tile + (col / 8) * q_block;
#pragma unroll 2
      for (int r = r0; r < used; r += kAtOnce) {
        const int gr = u.rt * C::kRows + r, head = a.head_at(gr), s = gr - head * a.S;
        const bool there = gr < a.rows && col * 8 < a.c.D;
        cp_async16(to + (r >> 7) * q_tile + (r & 127) * 128 + (((col % 8) ^ (r & 7)) << 4),
                   there ? q + head * a.q_h + s * a.q_s : a.q, there);
      }
      if (tree && a.parents) {
        const int* par = tree_of(a, u.b);
#pragma unroll 1
        for (int e = threadIdx.x; e < min(u.s.n, kParShared); e += C::kSoftThreads)
          cp_async4(smem_addr(&ctl.par[par_buf][e]), par + e);
      }
    };
    auto q_arrived = [&] {
      cp_async_wait_all();
      fence_proxy_async_smem();
      mbar_arrive(&ctl.q_full);
    };

    bool ok = n > 0;
    if (ok) copy_unit(cur, 0, 0, true);  // before the flood of K and V
    zero_empty_rows<T, C::kSoftThreads>(a, &fault);
    int par_buf = 0, unit = 0, j = 0;
    if (ok) {
      q_arrived();
      ok = meet();
    }
    bool begun = cur.t == 0;
    while (ok && j < n) {
      // The unit at cur, or the part of it in this run: tiles j .. j + count - 1.
      const int count = min(cur.T - cur.t, n - j), j1 = j + count;
      const bool last = j1 == n;
      Cursor nxt = cur;
      if (!last) next_unit(a, nxt, ahead, &fault);
      const bool new_tree = nxt.b != cur.b;
      if (early_q && !last) copy_unit(nxt, (unit + 1) & 1, par_buf ^ 1, new_tree);
      const Tree tree{ctl.par[par_buf], tree_of(a, cur.b)};
      const int gr = cur.rt * C::kRows + row_off, s_row = gr - a.head_at(gr) * a.S;
      const bool dead = gr >= a.rows || s_row >= cur.s.n;  // no row of the result, or a drafted token that is not there
      const bool warp_dead = __all_sync(0xffffffffu, dead);
      float m = -INFINITY, l = 0.f;  // running maximum of the scaled scores that P refers to, sum of P
      bool first = true;
      for (int jj = j; jj < j1; ++jj) {
        const int buf = kTwo ? st : jj & 1;
        const uint32_t tS = tmem + lane_off + buf * kBN;
        ok = wait(&ctl.s_full[buf], (kTwo ? jj : jj >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (!warp_dead) {
          const int pos0 = (cur.t + jj - j) * a.tile;
          const unsigned long long hole0 = ctl.hole[jj % kHoles][0], hole1 = ctl.hole[jj % kHoles][1];
          const bool masked = pos0 + a.tile > cur.s.base || (hole0 | hole1) != 0;
          bool any = true;
          uint32_t see[kWords];
          if (masked) {
            if (dead) {
#pragma unroll
              for (int w = 0; w < kWords; ++w) see[w] = 0;
            } else {
              visible<kWords>(cur.s, s_row, pos0, tree, see, &fault);
            }
            any = false;
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              // behind the table's end or the tile's, or in no page
              const int in = min(cur.s.len - pos0, a.tile) - 32 * w;
              see[w] &= in >= 32 ? 0xffffffffu : in > 0 ? (1u << in) - 1u : 0u;
              see[w] &= ~static_cast<uint32_t>((w < 2 ? hole0 : hole1) >> (w % 2 * 32));
              any = any || see[w] != 0;
            }
          }
          // Tiles of 128 tokens are read from tensor memory twice, 64 scores at a
          // time, for their maximum and for P: all at once would not fit the
          // registers.  Those that do not count are -inf there after the first
          // time.  (The loops are kept short: a CTA's first pass over them comes
          // from a cold instruction cache.)
          float s[64];
          auto load_scores = [&](int hf) {
            uint32_t u[2][32];
            tmem_ld32(tS + hf * 64, u[0]);
            tmem_ld32(tS + hf * 64 + 32, u[1]);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = __uint_as_float(u[i / 32][i % 32]);
          };
          float top = -INFINITY;
#pragma unroll 1
          for (int hf = 0; hf < kBN / 64; ++hf) {
            load_scores(hf);
            uint32_t lo = see[0], hi = see[1];
            if (kWords == 4 && hf) lo = see[kWords - 2], hi = see[kWords - 1];
            const int tail = a.tile - hf * 64;
            if (masked || tail < 64) {
              if (!masked) lo = 0xffffffffu, hi = tail >= 64 ? 0xffffffffu : (1u << (tail - 32)) - 1u;
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (!((i < 32 ? lo : hi) >> (i % 32) & 1u)) s[i] = -INFINITY;
              if constexpr (kBN > 64) {
                uint32_t u[2][32];
#pragma unroll
                for (int i = 0; i < 64; ++i) u[i / 32][i % 32] = __float_as_uint(s[i]);
                tmem_st32(tS + hf * 64, u[0]);
                tmem_st32(tS + hf * 64 + 32, u[1]);
                tmem_wait_st();
              }
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 60; i += 8) {
              mx[0] = fmax3(mx[0], s[i + 0], s[i + 4]);
              mx[1] = fmax3(mx[1], s[i + 1], s[i + 5]);
              mx[2] = fmax3(mx[2], s[i + 2], s[i + 6]);
              mx[3] = fmax3(mx[3], s[i + 3], s[i + 7]);
            }
            top = fmax3(top, fmax3(mx[0], mx[1], s[60]), fmax3(fmax3(mx[2], mx[3], s[61]), s[62], s[63]));
          }
          const float mb = any ? fmaxf(top * c, kLowest) : -INFINITY;
          // The maximum that P refers to moves, and O is rescaled, only when it
          // has grown by more than 2^8; O / L is the same in exact arithmetic.
          const bool grow = mb > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) {
            float alpha = 1.f;
            if (grow) {
              alpha = ex2_approx(m - mb);  // 0 where m is -inf
              l *= alpha;
              m = mb;
            }
            if (!first) {
              if constexpr (!kTwo) {
                // The product before may not have retired, which frees its V.
                // (With two streams it has, as S has been written over its P.)
                ok = wait(&ctl.v_empty[(jj - 1) % C::kVSlots], ((jj - 1) / C::kVSlots) & 1);
                if (!ok) break;
                tc_fence_after();
              }
#pragma unroll 1
              for (int cc = 0; cc < kD; cc += 32) {
                uint32_t o[32];
                tmem_ld32(tO + cc, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st32(tO + cc, o);
              }
            }
          }
          const float sub = kUp - finite_max(m);
          const uint64_t sub2 = f2(sub, sub);
          uint64_t sum0 = f2(0.f, 0.f), sum1 = f2(0.f, 0.f);
          // P is rounded to the input type for P V, by half a step of each weight
          // at most; its sum is taken before that.
#pragma unroll 1
          for (int hf = 0; hf < kBN / 64; ++hf) {
            uint32_t pk[32];
            if constexpr (kBN > 64) load_scores(hf);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float x0, x1;
              f2_split(f2_fma(f2(s[2 * i], s[2 * i + 1]), c2, sub2), x0, x1);
              x0 = ex2_approx(x0);
              x1 = ex2_approx(x1);
              if (i % 2) sum1 = f2_add(sum1, f2(x0, x1));
              else sum0 = f2_add(sum0, f2(x0, x1));
              pk[i] = pack2<kBf16>(x0, x1);
            }
            tmem_st32(tS + hf * 32, pk);
          }
          float a0, a1, b0, b1;
          f2_split(sum0, a0, a1);
          f2_split(sum1, b0, b1);
          l += (a0 + a1) + (b0 + b1);
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&ctl.p_full[buf]);
        first = false;
      }
      if (!ok) break;

      // The unit, or this run's part of it, ends.
      if (early_q && !last) q_arrived();
      ok = wait(&ctl.o_done, unit & 1);
      if (!ok) break;
      tc_fence_after();
      // (no product reads this unit's Q any more)
      if (!early_q && !last) copy_unit(nxt, 0, par_buf ^ 1, new_tree);
      Cursor at_end = cur;
      at_end.t += count - 1;
      const Place p = place_of(a, at_end, begun, run, run.first + j1 - 1, threadIdx.x == 0);
      // Whether drafted tokens have values that the products left out.
      bool mend = false;
#pragma unroll
      for (int w = 0; w < kMaxDrafted / 256; ++w) mend = mend || ctl.odd[unit % kHoles][w] != 0;
      float M = m;
      if (dead) M = -INFINITY;
      const float inv = inverse(M, l);
      if (!__all_sync(0xffffffffu, gr >= a.rows)) {
#pragma unroll 1
        for (int cc = 0; cc < kD; cc += 32) {
          float o[32];
          {
            uint32_t u[32];
            tmem_ld32(tO + cc, u);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(u[i]);
          }
          if (mend && !dead) {
            // the infinite and NaN values of drafted tokens this row follows, which the products left out
#pragma unroll 1
            for (int f = s_row; f >= 0; f = tree.parent(f, &fault)) {
              if (!(ctl.odd[unit % kHoles][f >> 8] >> (f >> 3 & 31) & 1u)) continue;
              int row = 0;
              const int page = page_of(a, cur, cur.s.base + f, &row, &fault);
              if (page < 0) continue;
              const T* v = static_cast<const T*>(a.c.v) + page * a.c.vs[0] + cur.h * a.c.vs[1] + row * a.c.vs[2];
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float x = cc + i < a.c.D ? to_f32(v[cc + i]) : 0.f;
                if (!isfinite(x)) o[i] += x;
              }
            }
          }
          if (gr >= a.rows) {
          } else if (p.whole) {
            T* out = static_cast<T*>(a.out) + (p.row0 + gr) * a.c.D + cc;
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = M == -INFINITY ? 0.f : o[i] * inv;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              if (cc + i < a.c.D)
                *reinterpret_cast<uint4*>(out + i) =
                    make_uint4(pack2<kBf16>(o[i], o[i + 1]), pack2<kBf16>(o[i + 2], o[i + 3]),
                               pack2<kBf16>(o[i + 4], o[i + 5]), pack2<kBf16>(o[i + 6], o[i + 7]));
          } else {
            float4* part = a.part_o + (static_cast<long long>(p.slot) * a.D4 + cc / 4) * C::kRows + row_off;
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (cc + i < a.c.D) part[i / 4 * C::kRows] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (gr < a.rows && !p.whole)
          a.part_ml[static_cast<long long>(p.slot) * C::kRows + row_off] = make_float2(M, l);
      }
      tc_fence_before();  // O has been read before the next unit's first product overwrites it (p_full orders the two)
      if (!last) {
        if (!early_q) q_arrived();
        ok = meet();  // the tree is there
        if (!ok) break;
      }
      begun = true;
      ++unit;
      if (new_tree) par_buf ^= 1;
      cur = nxt;
      j = j1;
    }
    cp_async_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (warp >= C::kCopyWarp && maps.boxes > 0 && ctl.abort_flag) {
    // Some role gave up on a wait: copies already asked for land before the
    // CTA's shared memory goes.
    for (int kv = 0; kv < 2; ++kv) {
      const int slots = kv ? C::kVSlots : C::kKSlots, last = kv ? last_copy[1] : last_copy[0];
      for (int s = 0; s < slots; ++s) {
        volatile int no_abort = 0;
        const int j = last - (last - s + slots) % slots;  // the last tile in slot s
        if (last < 0 || j < 0) continue;
        if (kv && late >= 0 && s == late_slot)
          wait_long(&ctl.v_raw[s], raw >> s & 1u, &no_abort, &ctl.code, kWaitTimeoutNs);
        else
          wait_long(kv ? &ctl.v_full[s] : &ctl.k_full[s], (j / slots) & 1, &no_abort, &ctl.code, kWaitTimeoutNs);
      }
    }
  }
  if (warp == C::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Join of units cut between CTAs
// ---------------------------------------------------------------------------

// The unit that CTA blockIdx.x of the grid before began and did not finish:
// lane a row and eight columns of it, its parts in the order of the tokens, or
// by `split` warps that take every split-th of them where there are many (one
// sequence of 4096 tokens, 8 kv heads: 37 parts each).
constexpr int kJoinWarps = 8, kJoinCols = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_tree_join_kernel(const __grid_constant__ TreeArgs a, int split) {
  __shared__ float2 s_ml[kJoinWarps][32];
  __shared__ float4 s_o[kJoinWarps][2][32];
  launch_dependents();
  grid_dependency_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col_tiles = (a.c.D + kJoinCols - 1) / kJoinCols, first = warp & (split - 1);
  const int w = (blockIdx.y * kJoinWarps + warp) / split, rows32 = w / col_tiles, d = (w - rows32 * col_tiles) * kJoinCols;
  const int4 meta = a.meta[c];
  if (meta.z == 0) return;
  const int r = rows32 * 32 + lane, gr = meta.y * a.unit_rows + r;
  const bool live = r < a.unit_rows && gr < a.rows, two = d / 4 + 1 < a.D4;
  float M = -INFINITY, L = 0.f;
  float4 o[2] = {};
#pragma unroll 1
  for (int i0 = first; live && i0 <= meta.z; i0 += 4 * split) {
    float2 ml[4];
    float4 y[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int part = i0 + i * split;
      ml[i] = make_float2(-INFINITY, 0.f);
      y[i][0] = y[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (part <= meta.z) {
        const long long slot = part == 0 ? 2 * c + 1 : 2 * (c + part);
        ml[i] = a.part_ml[slot * a.unit_rows + r];
        const float4* at = a.part_o + (slot * a.D4 + d / 4) * a.unit_rows + r;
        y[i][0] = *at;
        if (two) y[i][1] = at[a.unit_rows];
      }
    }
    const float mn = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M);
    const float back = ex2_approx(M - finite_max(mn));
    M = mn;
    L *= back;
#pragma unroll
    for (int k = 0; k < 2; ++k) o[k].x *= back, o[k].y *= back, o[k].z *= back, o[k].w *= back;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ex2_approx(ml[i].x - finite_max(mn));
      L = fmaf(ml[i].y, f, L);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        o[k].x = fmaf(y[i][k].x, f, o[k].x);
        o[k].y = fmaf(y[i][k].y, f, o[k].y);
        o[k].z = fmaf(y[i][k].z, f, o[k].z);
        o[k].w = fmaf(y[i][k].w, f, o[k].w);
      }
    }
  }
  if (split > 1) {
    s_ml[warp][lane] = make_float2(M, L);
    s_o[warp][0][lane] = o[0];
    s_o[warp][1][lane] = o[1];
    __syncthreads();
    if (first != 0) return;
    float top = M;
    for (int k = 1; k < split; ++k) top = fmaxf(top, s_ml[warp + k][lane].x);
    float f = ex2_approx(M - finite_max(top));
    L *= f;
#pragma unroll
    for (int k = 0; k < 2; ++k) o[k].x *= f, o[k].y *= f, o[k].z *= f, o[k].w *= f;
    for (int i = 1; i < split; ++i) {
      const float2 ml = s_ml[warp + i][lane];
      f = ex2_approx(ml.x - finite_max(top));
      L = fmaf(ml.y, f, L);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 y = s_o[warp + i][k][lane];
        o[k].x = fmaf(y.x, f, o[k].x);
        o[k].y = fmaf(y.y, f, o[k].y);
        o[k].z = fmaf(y.z, f, o[k].z);
        o[k].w = fmaf(y.w, f, o[k].w);
      }
    }
    M = top;
  }
  if (!live) return;
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(meta.x) * a.S + gr) * a.c.D + d;
  const float inv = inverse(M, L);
  const float x[8] = {o[0].x, o[0].y, o[0].z, o[0].w, o[1].x, o[1].y, o[1].z, o[1].w};
  struct alignas(16) Eight {
    T v[8];
  };
  Eight z;
#pragma unroll
  for (int e = 0; e < 8; ++e) z.v[e] = from_f32<T>(M == -INFINITY ? 0.f : x[e] * inv);
  if (a.c.D % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0) {
    *reinterpret_cast<Eight*>(out) = z;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (d + e < a.c.D) out[e] = z.v[e];
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct Plan {
  bool tc;  // the tensor-core kernel
  int kd;   // head dim the kernel is compiled for
  bool wide;  // the other, fed by 16-byte copies
  bool two_tiles;  // a CTA takes two tiles of 128 rows at once (tensor cores)
  int unit_rows, row_tiles, tile;
  int box_rows, boxes;  // of a tile of K or V, by TMA; 0: 16-byte copies
  int grid;
  long long tiles;  // the block table can name
  size_t meta_at, ml_at, o_at, bytes;
};

// Whether the cache's rows are read 16 bytes at a time.
bool wide_rows(const AttnPagedCache* c) {
  const int vec = c->dtype == ATTN_F32 ? 4 : 8;
  if (c->D % vec != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] % vec != 0 || c->v_strides[i] % vec != 0) return false;
  return aligned_to(c->k, 16) && aligned_to(c->v, 16);
}

// `fast`: q and out allow 16-byte accesses, where the kernel needs them.
Plan make_plan(const AttnPagedCache* c, bool fast, int Hq, int S, int sms) {
  Plan p;
  const int D = c->D;
  const long long rows = static_cast<long long>(Hq / c->heads) * S;
  int per_sm;
  const bool wide = fast && wide_rows(c);
  p.tc = wide && c->dtype != ATTN_F32 && c->num_pages > 0;
  p.kd = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  p.two_tiles = p.wide = false;
  if (p.tc) {
    p.two_tiles = p.kd <= 128 && rows > 128;
    p.unit_rows = p.two_tiles ? 256 : 128;
    const int most = p.two_tiles ? TcCfg<128, true>::kBN : TcCfg<128, false>::kBN;
    // A box is rows of one page, a multiple of 8 that divides its size, and a
    // tile is whole boxes.  A warp takes some 600 clocks for a tile and 80 for
    // each box of 64 columns; a tile takes 1600 (3900 with two streams) all
    // the same, so a shorter tile of fewer boxes can be the quicker one, but need
    // not: pages of 24 rows at D = 64, tiles of 64 tokens in eight boxes 32.0
    // us, of 48 in two 38.4.
    p.tile = most;
    p.box_rows = p.boxes = 0;
    double best = 0;
    for (int r = 8; r <= most && c->page_size % 8 == 0; r += 8) {
      const int boxes = most / r, tokens = boxes * r;
      if (c->page_size % r != 0 || tokens <= most - 32) continue;  // (the kernel masks the last 31 at most)
      const int copy = 600 + 80 * (p.kd / 64) * boxes * (p.two_tiles ? 1 : 2), least = p.two_tiles ? 3900 : 1600;
      const double cost = static_cast<double>(copy > least ? copy : least) / tokens;
      if (p.boxes > 0 && cost > best) continue;
      best = cost;
      p.box_rows = r;
      p.boxes = boxes;
      p.tile = tokens;
    }
    per_sm = p.two_tiles || p.kd == 256 ? 1 : 2;
  } else {
    p.unit_rows = kSimtRows;
    p.tile = kSimtTile;
    p.wide = wide && c->dtype == ATTN_F32;
    per_sm = p.wide ? (p.kd == 64 ? 4 : p.kd == 128 ? 2 : 1) : p.kd == 64 ? 5 : p.kd == 128 ? 3 : 2;
  }
  p.row_tiles = static_cast<int>((rows + p.unit_rows - 1) / p.unit_rows);
  const long long capacity = static_cast<long long>(c->table_width) * c->page_size;
  p.tiles = (capacity + p.tile - 1) / p.tile * c->B * c->heads * p.row_tiles;
  long long grid = static_cast<long long>(sms) * per_sm;
  if (grid > p.tiles) grid = p.tiles;
  if (grid < 1) grid = 1;
  p.grid = static_cast<int>(grid);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  const size_t D4 = (D + 3) / 4, parts = grid;
  p.meta_at = 0;
  p.ml_at = up(sizeof(int4) * parts);
  p.o_at = p.ml_at + up(sizeof(float2) * 2 * parts * p.unit_rows);
  p.bytes = p.o_at + up(sizeof(float4) * 2 * parts * p.unit_rows * D4);
  return p;
}

// Multiplier and shift of a division by d (see TreeArgs).
void divisor(int d, unsigned* mul, int* shift) {
  const unsigned long long x = static_cast<unsigned long long>(d);
  *shift = 0;
  while ((1ull << *shift) < x) ++*shift;
  *mul = static_cast<unsigned>((((1ull << *shift) - x) << 32) / x + 1);
}

// The checks of a call that need no device.  Returns ATTN_OK or a status.
int check_tree(const AttnPagedCache* c, int Hq, int S, PagedView* view) {
  const int st = check_paged_cache(c, kCacheK | kCacheV, view);
  if (st != ATTN_OK) return st;
  if (Hq < 0 || S < 0 || Hq % c->heads != 0) return ATTN_ERR_INVALID_ARGUMENT;
  if (S > kMaxDrafted) return ATTN_ERR_INVALID_ARGUMENT;
  if (static_cast<long long>(c->B) * Hq > 0x7fffffffLL || static_cast<long long>(Hq) * S > 0x7fffffffLL)
    return ATTN_ERR_INVALID_ARGUMENT;
  return ATTN_OK;
}

// The first launch on a device opts the kernel in to its shared memory and to
// the largest shared-memory share of the SM, so that its CTAs fit.
template <typename... Params, typename... Args>
bool launch_big(void (*kern)(Params...), std::mutex& mu, bool (&done)[64], int grid, int threads, size_t smem,
                cudaStream_t stream, const Args&... args) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  {
    std::lock_guard<std::mutex> g(mu);
    if (!done[dev]) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) !=
              cudaSuccess ||
          cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                               static_cast<int>(cudaSharedmemCarveoutMaxShared)) != cudaSuccess)
        return false;
      done[dev] = true;
    }
  }
  return launch_after(kern, dim3(grid), dim3(threads), smem, stream, 1, true, args...);
}

template <bool kBf16, int kD, bool kTwo>
bool launch_tc(const TreeArgs& a, const TcMaps& maps, int grid, cudaStream_t stream) {
  using C = TcCfg<kD, kTwo>;
  static bool done[64] = {};
  static std::mutex mu;
  return launch_big(attn_tree_tc_kernel<kBf16, kD, kTwo>, mu, done, grid, C::kThreads, C::kSmemBytes, stream, a, maps);
}

template <bool kBf16>
bool launch_tc_d(const TreeArgs& a, const TcMaps& maps, const Plan& p, cudaStream_t stream) {
  switch (p.kd) {
    case 64: return p.two_tiles ? launch_tc<kBf16, 64, true>(a, maps, p.grid, stream)
                                : launch_tc<kBf16, 64, false>(a, maps, p.grid, stream);
    case 128: return p.two_tiles ? launch_tc<kBf16, 128, true>(a, maps, p.grid, stream)
                                 : launch_tc<kBf16, 128, false>(a, maps, p.grid, stream);
    default: return launch_tc<kBf16, 256, false>(a, maps, p.grid, stream);
  }
}

// The caches' tensor maps; boxes = 0 where TMA does not suit them.
TcMaps make_maps(const AttnPagedCache* c, const Plan& p) {
  TcMaps m;
  const unsigned long long limit = wait_limit_ns();
  m.wait_ns = limit != 0 ? limit : kWaitTimeoutNs;
  m.lose = drop_arrival_requested();
  m.rows = p.box_rows;
  m.boxes = p.boxes;
  auto encode = [&](CUtensorMap* map, const void* base, const long long* st) {
    return make_tensor_map_4d(map, base, c->dtype == ATTN_BF16, c->D, c->page_size, c->heads, c->num_pages, st[2], st[1],
                              st[0], 64, m.rows) == 0;
  };
  if (m.boxes > 0 && (c->num_pages == 0 || !encode(&m.k, c->k, c->k_strides) || !encode(&m.v, c->v, c->v_strides)))
    m.boxes = 0;
  return m;
}

template <typename T, int kDP, bool kWide>
bool launch_simt(const TreeArgs& a, int grid, cudaStream_t stream) {
  static bool done[64] = {};
  static std::mutex mu;
  return launch_big(attn_tree_simt_kernel<T, kDP, kWide>, mu, done, grid, kSimtThreads, SimtCfg<kDP, kWide>::kBytes, stream, a);
}

template <typename T, bool kWide = false>
bool launch_simt_d(const TreeArgs& a, const Plan& p, cudaStream_t stream) {
  switch (p.kd) {
    case 64: return launch_simt<T, 64, kWide>(a, p.grid, stream);
    case 128: return launch_simt<T, 128, kWide>(a, p.grid, stream);
    default: return launch_simt<T, 256, kWide>(a, p.grid, stream);
  }
}

}  // namespace

int page_word_read_clear_tree(cudaStream_t stream, int* host) {
  static const int zero = 0;
  return cudaMemcpyFromSymbolAsync(host, g_page_fault, sizeof(int), 0, cudaMemcpyDeviceToHost, stream) ==
                     cudaSuccess &&
                 cudaMemcpyToSymbolAsync(g_page_fault, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream) ==
                     cudaSuccess
             ? 0
             : -1;
}

}  // namespace ra

extern "C" int attn_tree_workspace_bytes(const AttnPagedCache* cache, int Hq, int S, size_t* bytes) {
  using namespace ra;
  if (!bytes) return ATTN_ERR_INVALID_ARGUMENT;
  PagedView view;
  int st = check_tree(cache, Hq, S, &view);
  if (st != ATTN_OK) return st;
  *bytes = 0;
  if (cache->B == 0 || Hq == 0 || S == 0) return ATTN_OK;
  st = check_device();
  if (st != ATTN_OK) return st;
  const int sms = sm_count();
  // q or out may turn out to need the other kernel: room for either
  const Plan fast = make_plan(cache, true, Hq, S, sms), other = make_plan(cache, false, Hq, S, sms);
  *bytes = fast.bytes > other.bytes ? fast.bytes : other.bytes;
  size_t few = 0;
  if (decode_rows_plan(cache, Hq, S, sms, &few) && few > *bytes) *bytes = few;
  return ATTN_OK;
}

extern "C" int launch_attn_tree(const AttnPagedCache* cache, const void* q, const long long* q_strides, void* out,
                                int Hq, int S, float softmax_scale, const int* parents, long long parents_stride,
                                const int* new_lens, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using namespace ra;
  PagedView view;
  int st = check_tree(cache, Hq, S, &view);
  if (st != ATTN_OK) return st;
  if (cache->B == 0 || Hq == 0 || S == 0) return ATTN_OK;
  if (!q || !out || !workspace || (parents && parents_stride < 0)) return ATTN_ERR_INVALID_ARGUMENT;
  const int D = cache->D;
  const long long contiguous[3] = {static_cast<long long>(Hq) * S * D, static_cast<long long>(S) * D, D};
  const long long* qs = q_strides ? q_strides : contiguous;
  if (qs[0] < 0 || qs[1] < 0 || qs[2] < 0) return ATTN_ERR_INVALID_ARGUMENT;
  const size_t elem = cache->dtype == ATTN_F32 ? 4 : 2;
  if (!aligned_to(q, elem) || !aligned_to(out, elem) || !aligned_to(parents, 4) || !aligned_to(new_lens, 4) ||
      !aligned_to(workspace, 16))
    return ATTN_ERR_MISALIGNED;
  st = check_device();
  if (st != ATTN_OK) return st;
  const bool fast = cache->dtype == ATTN_F32 ||
                    (aligned_to(q, 16) && aligned_to(out, 16) && qs[0] % 8 == 0 && qs[1] % 8 == 0 && qs[2] % 8 == 0);
  const int sms = sm_count();
  float scale = softmax_scale;
  if (!(scale > 0.f) || !isfinite(scale)) scale = 1.0f / sqrtf(static_cast<float>(D));
  // Up to eight rows (which must lie evenly in memory) fill one column tile of
  // attn_decode's products, where a tile's softmax is not one warp's work of some
  // 1100 clocks: 8 rows, D = 128, that kernel / this one, us: one sequence of 4096
  // tokens 14.6 / 17.3, of 517 10.4 / 9.8, 24 of up to 4096 55 to 60 / 54, 16 of up
  // to 16384 124 to 133 / 133 to 139; five rows, D = 64, pages of 24 (no box of 16)
  // 32.4 / 35.5.  16 rows: one of 4096 19.9 / 19.7, 24 77.4 / 63.2, 16 172 / 155.
  const bool even = S == 1 || Hq == 1 || qs[1] == S * qs[2];
  size_t few = 0;
  if (fast && even && decode_rows_plan(cache, Hq, S, sms, &few)) {
    if (workspace_bytes < few) return ATTN_ERR_INVALID_ARGUMENT;
    return launch_decode_rows(cache, view, q, qs[0], S == 1 ? qs[1] : qs[2], out, Hq, S, scale, parents, parents_stride,
                              new_lens, workspace, stream)
               ? ATTN_OK
               : ATTN_ERR_LAUNCH;
  }
  const Plan p = make_plan(cache, fast, Hq, S, sms);
  if (workspace_bytes < p.bytes || p.tiles > 0x7fffffffLL - 65536) return ATTN_ERR_INVALID_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  TreeArgs a;
  a.c = view;
  a.q = q;
  a.q_b = qs[0];
  a.q_h = qs[1];
  a.q_s = qs[2];
  a.out = out;
  a.Hq = Hq;
  a.group = Hq / cache->heads;
  a.S = S;
  a.rows = a.group * S;
  a.unit_rows = p.unit_rows;
  a.row_tiles = p.row_tiles;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.parents = parents;
  a.parents_stride = parents_stride;
  a.new_lens = new_lens;
  a.meta = reinterpret_cast<int4*>(ws + p.meta_at);
  a.part_ml = reinterpret_cast<float2*>(ws + p.ml_at);
  a.part_o = reinterpret_cast<float4*>(ws + p.o_at);
  a.D4 = (D + 3) / 4;
  divisor(cache->page_size, &a.ps_mul, &a.ps_shift);
  divisor(S, &a.s_mul, &a.s_shift);
  divisor(p.tile, &a.t_mul, &a.t_shift);
  a.tile = p.tile;

  bool ok;
  if (p.tc) {
    const TcMaps maps = make_maps(cache, p);
    ok = cache->dtype == ATTN_BF16 ? launch_tc_d<true>(a, maps, p, stream) : launch_tc_d<false>(a, maps, p, stream);
  } else switch (cache->dtype) {
    case ATTN_F16: ok = launch_simt_d<__half>(a, p, stream); break;
    case ATTN_BF16: ok = launch_simt_d<__nv_bfloat16>(a, p, stream); break;
    default: ok = p.wide ? launch_simt_d<float, true>(a, p, stream) : launch_simt_d<float>(a, p, stream); break;
  }
  if (!ok) return ATTN_ERR_LAUNCH;
  const int used = a.rows < p.unit_rows ? a.rows : p.unit_rows;
  const long long items = static_cast<long long>((used + 31) / 32) * ((D + kJoinCols - 1) / kJoinCols);
  // About how many CTAs share a unit, at full lengths.
  const long long parts = p.grid / (static_cast<long long>(cache->B) * cache->heads * p.row_tiles);
  int split = 1;
  while (split < kJoinWarps && split * 4 <= parts) split *= 2;
  const dim3 grid(p.grid, static_cast<unsigned>((items * split + kJoinWarps - 1) / kJoinWarps)), block(kJoinWarps * 32);
  switch (cache->dtype) {
    case ATTN_F16: ok = launch_after(attn_tree_join_kernel<__half>, grid, block, 0, stream, 1, true, a, split); break;
    case ATTN_BF16: ok = launch_after(attn_tree_join_kernel<__nv_bfloat16>, grid, block, 0, stream, 1, true, a, split); break;
    default: ok = launch_after(attn_tree_join_kernel<float>, grid, block, 0, stream, 1, true, a, split); break;
  }
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}
