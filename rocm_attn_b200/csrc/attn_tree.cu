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
  float scale_log2;
  const int* parents;        // or null: a chain
  long long parents_stride;
  const int* new_lens;       // or null: S
  int4* meta;                // [gridDim.x]: kv head's first output row, tile of rows, CTAs that continue the unit begun last
  float2* part_ml;           // [2 gridDim.x][unit_rows]
  float* part_o;             // [2 gridDim.x][unit_rows][D4]
  int D4;                    // D rounded up to 4
  // pos / page_size for pos < 2^31 as (umulhi(pos, ps_mul) + pos) >> ps_shift:
  // Granlund and Montgomery, Division by Invariant Integers using
  // Multiplication (1994), figure 4.1.
  unsigned ps_mul;
  int ps_shift;
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
// `base` on drafted (base < 0: the first of them are not there).
struct Seq {
  int len, n, base;
};

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int b, int* fault) {
  Seq s;
  int n = a.S;
  if (a.new_lens) {
    n = *(a.new_lens + b);
    if (n > a.S) {
      *fault |= kFaultPage;
      n = a.S;
    }
    if (n < 0) n = 0;
  }
  s.n = n;
  s.base = max(*(a.c.lens + b), 0) - n;
  s.len = paged_len(a.c, b, fault);
  return s;
}

// A place in the row of tiles: tile t of the T tiles of the unit (sequence b,
// kv head h, tile rt of its rows).
struct Cursor {
  int b, h, rt, t, T;
  Seq s;
};

template <int kTile>
__device__ __forceinline__ int tiles_of(const Seq& s) {
  return s.n > 0 ? (s.len + kTile - 1) / kTile : 0;
}

template <int kTile>
__device__ __forceinline__ void advance(const TreeArgs& a, Cursor& c, int* fault) {
  if (++c.t < c.T) return;
  c.t = 0;
  if (++c.rt < a.row_tiles) return;
  c.rt = 0;
  if (++c.h < a.c.heads) return;
  c.h = 0;
  c.T = 0;
  while (c.T == 0 && ++c.b < a.c.B) {
    c.s = seq_of(a, c.b, fault);
    c.T = tiles_of<kTile>(c.s);
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
template <int kTile, int kThreads>
__device__ __forceinline__ Cursor schedule(const TreeArgs& a, ScheduleSmem<kThreads>& s, Run* run, int* fault) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = (a.c.B + kThreads - 1) / kThreads;
  const long long from = static_cast<long long>(threadIdx.x) * seg;
  const int b0 = from < a.c.B ? static_cast<int>(from) : a.c.B, b1 = min(a.c.B - b0, seg) + b0;
  int mine = 0, T = 0;
  Seq q = {};
  for (int b = b0; b < b1; ++b) {
    q = seq_of(a, b, fault);
    T = tiles_of<kTile>(q);
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
      for (;; ++b) {
        q = seq_of(a, b, fault);
        T = tiles_of<kTile>(q);
        if (in < T * units || b + 1 >= b1) break;
        in -= T * units;
      }
    }
    const int hu = in / T, h = hu / a.row_tiles;
    s.first = Cursor{b, h, hu - h * a.row_tiles, in - hu * T, T, q};
  }
  __syncthreads();
  return s.first;
}

// Output rows of sequences without tokens, or without drafted ones, are zeros.
template <typename T, int kThreads>
__device__ __forceinline__ void zero_empty_rows(const TreeArgs& a, int* fault) {
  const long long bytes = static_cast<long long>(a.Hq) * a.S * a.c.D * sizeof(T);
  const bool wide = bytes % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  for (int b = blockIdx.x; b < a.c.B; b += gridDim.x) {
    const Seq s = seq_of(a, b, fault);
    if (s.len > 0 && s.n > 0) continue;
    unsigned char* o = static_cast<unsigned char*>(a.out) + b * bytes;
    if (wide) {
      for (long long i = threadIdx.x; i < bytes / 16; i += kThreads) reinterpret_cast<uint4*>(o)[i] = make_uint4(0, 0, 0, 0);
    } else {
      for (long long i = threadIdx.x; i < bytes / static_cast<long long>(sizeof(T)); i += kThreads)
        reinterpret_cast<T*>(o)[i] = from_f32<T>(0.f);
    }
  }
}

// The drafted tokens that each one follows, checked: par[s] < s.
template <int kThreads>
__device__ __forceinline__ void load_parents(const TreeArgs& a, int b, int n, int* par, int thread, int* fault) {
  for (int s = thread; s < n; s += kThreads) {
    int p = s - 1;
    if (a.parents) {
      p = *(a.parents + b * a.parents_stride + s);
      if (p < -1 || p >= s) {
        *fault |= kFaultPage;
        p = -1;
      }
    }
    par[s] = p;
  }
}

// Bits of the kWords * 32 positions from `pos0` on that drafted token s of the
// sequence may see (s < n), beside those the sequence has there.
template <int kWords>
__device__ __forceinline__ void visible(const Seq& q, int s, int pos0, const int* par, uint32_t (&bits)[kWords]) {
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    // positions below base: all of them
    const int in = q.base - (pos0 + 32 * w);
    bits[w] = in >= 32 ? 0xffffffffu : in > 0 ? (1u << in) - 1u : 0u;
  }
  for (int p = s; p >= 0; p = par[p]) {
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
  const unsigned p = static_cast<unsigned>(pos);
  const int lp = static_cast<int>((__umulhi(p, a.ps_mul) + p) >> a.ps_shift);
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

// ---------------------------------------------------------------------------
// SIMT kernel: fp32, any head dim, any strides
// ---------------------------------------------------------------------------

// 32 rows by 64 tokens per tile.  Thread (ty, tx) of 8 x 16 has rows 4 ty + {0
// .. 3}: scores of tokens tx + 16 {0 .. 3}, and of O the columns 4 tx + {0 .. 3}
// + 64 j.  K and then V lie in one buffer, in 32 bits.
constexpr int kSimtThreads = 128, kSimtRows = 32, kSimtTile = 64;

template <int kDP>
struct SimtCfg {
  static constexpr int kPitch = kDP + 4;  // floats; rows 4 banks apart
  static constexpr int kPPitch = kSimtTile + 4;
  static constexpr size_t kBytes = sizeof(float) * ((kSimtRows + kSimtTile) * kPitch + kSimtRows * kPPitch) +
                                   sizeof(long long) * 2 * kSimtTile + sizeof(int) * kMaxDrafted;
};

template <typename T, int kDP>
__global__ void __launch_bounds__(kSimtThreads) attn_tree_simt_kernel(const __grid_constant__ TreeArgs a) {
  using C = SimtCfg<kDP>;
  constexpr int kCols = kDP / 16;
  extern __shared__ __align__(16) float sm[];
  float* s_q = sm;
  float* s_kv = s_q + kSimtRows * C::kPitch;
  float* s_p = s_kv + kSimtTile * C::kPitch;
  long long* s_at = reinterpret_cast<long long*>(s_p + kSimtRows * C::kPPitch);  // K, then V offsets; -1: no token
  int* s_par = reinterpret_cast<int*>(s_at + 2 * kSimtTile);
  __shared__ ScheduleSmem<kSimtThreads> s_sched;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, D = a.c.D;
  int fault = 0;
  launch_dependents();
  grid_dependency_wait();
  if (tid == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  Run run;
  Cursor cur = schedule<kSimtTile>(a, s_sched, &run, &fault);
  zero_empty_rows<T, kSimtThreads>(a, &fault);
  float o[4][kCols], m[4], l[4];
  bool begun = cur.t == 0, fresh = true;
  const T* kbase = static_cast<const T*>(a.c.k);
  const T* vbase = static_cast<const T*>(a.c.v);

  // Rows of the cache at s_at to s_kv, zeros behind D and where there is no token.
  auto load = [&](const T* base, const long long* at) {
    for (int e = tid; e < kSimtTile * kDP; e += kSimtThreads) {
      const int r = e / kDP, d = e % kDP;
      s_kv[r * C::kPitch + d] = at[r] >= 0 && d < D ? to_f32(base[at[r] + d]) : 0.f;
    }
  };

  for (int i = 0; i < run.n; ++i) {
    if (fresh) {
      const T* q = static_cast<const T*>(a.q) + cur.b * a.q_b + static_cast<long long>(cur.h) * a.group * a.q_h;
      for (int e = tid; e < kSimtRows * kDP; e += kSimtThreads) {
        const int r = e / kDP, d = e % kDP, gr = cur.rt * kSimtRows + r;
        const int head = gr / a.S, s = gr - head * a.S;
        s_q[r * C::kPitch + d] = gr < a.rows && d < D ? to_f32(q[head * a.q_h + s * a.q_s + d]) : 0.f;
      }
      load_parents<kSimtThreads>(a, cur.b, cur.s.n, s_par, tid, &fault);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[r][c] = 0.f;
      }
      fresh = false;
    }
    const int pos0 = cur.t * kSimtTile;
    if (tid < kSimtTile) {
      int row = 0;
      const int page = page_of(a, cur, pos0 + tid, &row, &fault);
      s_at[tid] = page < 0 ? -1 : page * a.c.ks[0] + cur.h * a.c.ks[1] + row * a.c.ks[2];
      s_at[kSimtTile + tid] = page < 0 ? -1 : page * a.c.vs[0] + cur.h * a.c.vs[1] + row * a.c.vs[2];
    }
    __syncthreads();
    load(kbase, s_at);
    __syncthreads();
    float x[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < kDP; d += 4) {
      float4 q[4], k[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) q[r] = *reinterpret_cast<const float4*>(s_q + (ty * 4 + r) * C::kPitch + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) k[c] = *reinterpret_cast<const float4*>(s_kv + (tx + 16 * c) * C::kPitch + d);
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
      if (gr < a.rows && s < cur.s.n) visible<2>(cur.s, s, pos0, s_par, see);
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
    __syncthreads();  // K is used up
    load(vbase, s_at + kSimtTile);
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
          const float4 v = *reinterpret_cast<const float4*>(s_kv + (t + k) * C::kPitch + j * 64 + tx * 4);
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
        const long long slot = static_cast<long long>(p.slot) * kSimtRows + in;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int d = (c / 4) * 64 + tx * 4 + c % 4;
          if (d >= D) continue;
          if (p.whole)
            static_cast<T*>(a.out)[(p.row0 + gr) * D + d] = from_f32<T>(m[r] == -INFINITY ? 0.f : o[r][c] * inv);
          else
            a.part_o[slot * a.D4 + d] = o[r][c];
        }
        if (!p.whole && tx == 0) a.part_ml[slot] = make_float2(m[r], l[r]);
      }
      begun = true;
      fresh = true;
    }
    __syncthreads();  // the tile's buffers are free
    advance<kSimtTile>(a, cur, &fault);
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Join of units cut between CTAs
// ---------------------------------------------------------------------------

// Warp per row of the unit that CTA blockIdx.x of the grid before began and did
// not finish: its parts in the order of the tokens, 32 maxima and sums at a
// time, lane four columns of each 128.
constexpr int kJoinWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_tree_join_kernel(const __grid_constant__ TreeArgs a) {
  launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, c = blockIdx.x, r = blockIdx.y * kJoinWarps + (threadIdx.x >> 5);
  const int4 meta = a.meta[c];
  const int gr = meta.y * a.unit_rows + r;
  if (meta.z == 0 || r >= a.unit_rows || gr >= a.rows) return;
  auto slot = [&](int i) { return static_cast<long long>(i == 0 ? 2 * c + 1 : 2 * (c + i)) * a.unit_rows + r; };
  float M = -INFINITY, L = 0.f;
  float4 o[2] = {};
  for (int i0 = 0; i0 <= meta.z; i0 += 32) {
    const int here = min(32, meta.z + 1 - i0);
    const float2 ml = lane < here ? a.part_ml[slot(i0 + lane)] : make_float2(-INFINITY, 0.f);
    float mn = ml.x;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
    mn = fmaxf(mn, M);
    const float back = ex2_approx(M - finite_max(mn)), f = ex2_approx(ml.x - finite_max(mn));
    M = mn;
    float sum = lane < here ? ml.y * f : 0.f;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    L = L * back + sum;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int d = k * 128 + lane * 4;
      o[k].x *= back, o[k].y *= back, o[k].z *= back, o[k].w *= back;
#pragma unroll 8
      for (int i = 0; i < here; ++i) {
        const float g = __shfl_sync(0xffffffffu, f, i);
        if (d < a.D4) {
          const float4 y = *reinterpret_cast<const float4*>(a.part_o + slot(i0 + i) * a.D4 + d);
          o[k].x = fmaf(y.x, g, o[k].x);
          o[k].y = fmaf(y.y, g, o[k].y);
          o[k].z = fmaf(y.z, g, o[k].z);
          o[k].w = fmaf(y.w, g, o[k].w);
        }
      }
    }
  }
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(meta.x) * a.S + gr) * a.c.D;
  const float inv = inverse(M, L);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float x[4] = {o[k].x, o[k].y, o[k].z, o[k].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = k * 128 + lane * 4 + e;
      if (d < a.c.D) out[d] = from_f32<T>(M == -INFINITY ? 0.f : x[e] * inv);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct Plan {
  int kd;  // head dim the kernel is compiled for
  int unit_rows, row_tiles, tile;
  int grid;
  long long tiles;  // the block table can name
  size_t meta_at, ml_at, o_at, bytes;
};

Plan make_plan(const AttnPagedCache* c, int Hq, int S, int sms) {
  Plan p;
  const int D = c->D;
  p.kd = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  p.unit_rows = kSimtRows;
  p.tile = kSimtTile;
  const int per_sm = p.kd == 64 ? 5 : p.kd == 128 ? 3 : 2;
  const long long rows = static_cast<long long>(Hq / c->heads) * S;
  p.row_tiles = static_cast<int>((rows + p.unit_rows - 1) / p.unit_rows);
  const long long capacity = static_cast<long long>(c->table_width) * c->page_size;
  p.tiles = (capacity + p.tile - 1) / p.tile * c->B * c->heads * p.row_tiles;
  long long grid = static_cast<long long>(sms) * per_sm;
  if (grid > p.tiles) grid = p.tiles;
  if (grid < 1) grid = 1;
  p.grid = static_cast<int>(grid);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  const size_t D4 = (D + 3) / 4 * 4, parts = grid;
  p.meta_at = 0;
  p.ml_at = up(sizeof(int4) * parts);
  p.o_at = p.ml_at + up(sizeof(float2) * 2 * parts * p.unit_rows);
  p.bytes = p.o_at + up(sizeof(float) * 2 * parts * p.unit_rows * D4);
  return p;
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

template <typename T, int kDP>
bool launch_simt(const TreeArgs& a, int grid, cudaStream_t stream) {
  auto kern = attn_tree_simt_kernel<T, kDP>;
  static bool done[64] = {};
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  {
    std::lock_guard<std::mutex> g(mu);
    if (!done[dev]) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(SimtCfg<kDP>::kBytes)) != cudaSuccess ||
          cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                               static_cast<int>(cudaSharedmemCarveoutMaxShared)) != cudaSuccess)
        return false;
      done[dev] = true;
    }
  }
  return launch_after(kern, dim3(grid), dim3(kSimtThreads), SimtCfg<kDP>::kBytes, stream, 1, true, a);
}

template <typename T>
bool launch_simt_d(const TreeArgs& a, const Plan& p, cudaStream_t stream) {
  switch (p.kd) {
    case 64: return launch_simt<T, 64>(a, p.grid, stream);
    case 128: return launch_simt<T, 128>(a, p.grid, stream);
    default: return launch_simt<T, 256>(a, p.grid, stream);
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
  *bytes = make_plan(cache, Hq, S, sm_count()).bytes;
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
  const Plan p = make_plan(cache, Hq, S, sm_count());
  if (workspace_bytes < p.bytes || p.tiles > 0x7fffffffLL - 65536) return ATTN_ERR_INVALID_ARGUMENT;

  float scale = softmax_scale;
  if (!(scale > 0.f) || !isfinite(scale)) scale = 1.0f / sqrtf(static_cast<float>(D));
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
  a.part_o = reinterpret_cast<float*>(ws + p.o_at);
  a.D4 = (D + 3) / 4 * 4;
  const unsigned long long ps = static_cast<unsigned long long>(cache->page_size);
  a.ps_shift = 0;
  while ((1ull << a.ps_shift) < ps) ++a.ps_shift;
  a.ps_mul = static_cast<unsigned>((((1ull << a.ps_shift) - ps) << 32) / ps + 1);

  bool ok;
  switch (cache->dtype) {
    case ATTN_F16: ok = launch_simt_d<__half>(a, p, stream); break;
    case ATTN_BF16: ok = launch_simt_d<__nv_bfloat16>(a, p, stream); break;
    default: ok = launch_simt_d<float>(a, p, stream); break;
  }
  if (!ok) return ATTN_ERR_LAUNCH;
  const dim3 grid(p.grid, (p.unit_rows + kJoinWarps - 1) / kJoinWarps), block(kJoinWarps * 32);
  switch (cache->dtype) {
    case ATTN_F16: ok = launch_after(attn_tree_join_kernel<__half>, grid, block, 0, stream, 1, true, a); break;
    case ATTN_BF16: ok = launch_after(attn_tree_join_kernel<__nv_bfloat16>, grid, block, 0, stream, 1, true, a); break;
    default: ok = launch_after(attn_tree_join_kernel<float>, grid, block, 0, stream, 1, true, a); break;
  }
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}
