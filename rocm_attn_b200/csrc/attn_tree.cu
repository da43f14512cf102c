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
  float4* part_o;            // [2 gridDim.x][D4][unit_rows]: a row of threads writes and reads it in a row
  int D4;                    // D / 4, rounded up
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

// One of them, where they are not at hand.
__device__ __noinline__ int parent_of(const TreeArgs& a, int b, int s) {
  const int p = a.parents ? *(a.parents + b * a.parents_stride + s) : s - 1;
  return p < -1 || p >= s ? -1 : p;
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
    advance<kSimtTile>(a, cur, &fault);
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// Tensor-core kernel: fp16 and bf16, D a multiple of 8, 16-byte rows
// ---------------------------------------------------------------------------

// 128 rows (or two tiles of 128) of a kv head are the rows of the tcgen05
// products, 64 tokens a tile: S = Q K^T into tensor memory, a thread per row
// takes the softmax of it and writes P over it, O += P V.  Up to 128 rows the
// floor is the time to read the cache: 64 tokens of D = 128 are 32 KB, 1400
// clocks of an SM's share of the bandwidth, beside 384 + 256 of the two products and about 800
// of the softmax.  Warp roles:
//   warps 0-3 (4-7)  softmax of row tile 0 (1), and its Q and O
//   next warp        the products, one elected lane; V of tiles that end early
//   last warp        copies: boxes of K and V rows by TMA, page ids looked up a
//                    group of tiles ahead
// S has two buffers, so S(j + 1) is computed while the softmax takes S(j); the
// products are issued S(j + 1), P(j) V(j), and at the end of a unit P(j) V(j)
// first, as the next unit's Q takes the place of this one's.  Two CTAs per SM
// where they fit hide each other's ends of units and waits.
template <int kD_, int kTiles_>
struct TcCfg {
  static constexpr int kD = kD_, kTiles = kTiles_;
  static constexpr int kBN = 64;
  static constexpr int kRows = 128 * kTiles;
  static constexpr int kCtas = kTiles == 1 && kD <= 128 ? 2 : 1;  // per SM
  static constexpr int kStages = kD == 64 ? 5 : kTiles == 2 ? 4 : 2;  // of K and of V
  static constexpr uint32_t kQBytes = 128u * kD * 2;      // a Q tile
  static constexpr uint32_t kQBlock = 128u * 128;         // 64 columns of it
  static constexpr uint32_t kKVBytes = kBN * kD * 2u;     // a K or V tile
  static constexpr uint32_t kKVBlock = kBN * 128u;        // 64 columns of it
  static constexpr size_t kSmemBytes = 1024 + kTiles * kQBytes + 2 * kStages * kKVBytes;
  static constexpr uint32_t kColO = 2 * kTiles * kBN;     // after the S buffers
  static constexpr uint32_t kTmemCols = kColO + kTiles * kD <= 256 ? 256 : 512;
  static constexpr int kMmaWarp = 4 * kTiles, kTmaWarp = kMmaWarp + 1;
  static constexpr int kThreads = 128 * kTiles + 64;
};
constexpr int kHoles = 8;  // tiles whose holes are remembered: a ring deeper than the stages by two

template <typename C>
struct __align__(8) TcCtl {
  uint64_t q_full[C::kTiles];
  uint64_t k_full[C::kStages], k_empty[C::kStages], v_full[C::kStages], v_empty[C::kStages];
  uint64_t s_full[C::kTiles][2], p_full[C::kTiles][2], pv_done[C::kTiles], o_done[C::kTiles];
  uint64_t mma_done, group_met[C::kTiles];
  unsigned long long hole[kHoles];  // tokens of a tile that lie in no page of the cache
  uint32_t odd[2][kMaxDrafted / 32];  // drafted tokens of this unit (the last) with infinite or NaN values
  uint32_t tmem_base;
  int abort_flag, code;
};

// The two caches as [num_pages, heads, page_size, D] tensors read in boxes of
// `rows` rows by 64 columns.
struct TcMaps {
  CUtensorMap k, v;
  int rows;
  unsigned long long wait_ns;
  int lose;  // watchdog test build only: CTA 0's first K copy is for bytes that never come
};

template <bool kBf16, int kD, int kTiles>
__global__ void __launch_bounds__(TcCfg<kD, kTiles>::kThreads, TcCfg<kD, kTiles>::kCtas)
    attn_tree_tc_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ TcMaps maps) {
  using C = TcCfg<kD, kTiles>;
  using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  constexpr int kBN = C::kBN, kStages = C::kStages, kThreads = C::kThreads;
  static_assert(kHoles >= kStages + 2, "the softmax may be two tiles behind the copies' ring");
  // fp16 has its full precision down to 2^-14: P is kept times 2^7 (at most
  // 2^15, as the maximum it refers to may be 2^8 below the largest score).
  constexpr float kUp = kBf16 ? 0.f : 7.f;

  extern __shared__ uint8_t smem_raw[];
  __shared__ TcCtl<C> ctl;
  __shared__ ScheduleSmem<kThreads> s_sched;
  __shared__ int s_par[kTiles][kMaxDrafted];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + kTiles * C::kQBytes;
  uint8_t* sV = sK + kStages * C::kKVBytes;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0), lane = threadIdx.x & 31;
  int fault = 0;

  if (threadIdx.x == 0) {
    ctl.abort_flag = ctl.code = 0;
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&ctl.q_full[t], 128);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&ctl.s_full[t][i], 1);
        mbar_init(&ctl.p_full[t][i], 128);
      }
      mbar_init(&ctl.pv_done[t], 1);
      mbar_init(&ctl.o_done[t], 1);
      mbar_init(&ctl.group_met[t], 128);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ctl.k_full[s], 1);
      mbar_init(&ctl.k_empty[s], 1);
      mbar_init(&ctl.v_full[s], 1);
      mbar_init(&ctl.v_empty[s], 1);
    }
    mbar_init(&ctl.mma_done, 1);
    fence_mbar_init();
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(smem_addr(&ctl.tmem_base), C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == C::kTmaWarp && lane == 0) {
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
  Cursor cur = schedule<kBN>(a, s_sched, &run, &fault);
  const int n = run.n;
  zero_empty_rows<T, kThreads>(a, &fault);

  const unsigned long long wait_ns = maps.wait_ns;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool there =
        __all_sync(0xffffffffu, mbar_wait(bar, parity, &ctl.abort_flag, &ctl.code, 1, wait_ns));
    if (!there) fault |= kFaultWait;
    return there;
  };
  int last_k = -1, last_v = -1;  // last tiles whose copies went out (copying warp)

  if (warp == C::kTmaWarp) {
    // ---------------------------------------------------------------- copies
    const int R = maps.rows, boxes = kBN / R, group = 32 / boxes;  // tiles per look-up
    const uint64_t policy = a.row_tiles > 1 ? l2_policy_evict_last() : l2_policy_evict_first();
    const int my_tile = lane / boxes, my_box = lane % boxes;
    struct Group {
      int page, row, live;  // of this lane's box: table entry, first row, rows that are tokens
      int count, h;
    };
    Cursor look = cur;
    int left = n;
    auto look_up = [&](Group& g) {
      g.count = min(min(group, look.T - look.t), left);
      g.h = look.h;
      g.page = -1;
      g.row = g.live = 0;
      if (left <= 0) return;
      const int pos = (look.t + my_tile) * kBN + my_box * R;
      if (my_tile < g.count && pos < look.s.len) {
        const unsigned p = static_cast<unsigned>(pos);
        const int lp = static_cast<int>((__umulhi(p, a.ps_mul) + p) >> a.ps_shift);
        g.row = pos - lp * a.c.page_size;
        g.live = min(R, look.s.len - pos);
        g.page = *(a.c.table + static_cast<long long>(look.b) * a.c.table_stride + lp);
      }
      left -= g.count;
      look.t += g.count - 1;
      if (left > 0) advance<kBN>(a, look, &fault);
    };
    Group now, next;
    look_up(now);
    look_up(next);
    int in = 0;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      const int slot = j % kStages;
      const uint32_t parity = ((j / kStages) & 1) ^ 1;
      const bool mine = my_tile == in && now.live > 0;
      const bool there = mine && static_cast<unsigned>(now.page) < static_cast<unsigned>(a.c.num_pages);
      uint32_t bytes = __popc(__ballot_sync(0xffffffffu, there)) * R * (kD * 2);
      unsigned long long hole = 0;
      if (__any_sync(0xffffffffu, mine && !there)) {
        unsigned long long bits = 0;
        if (mine && !there) {
          fault |= kFaultPage;
          bits = (R == 64 ? ~0ull : (1ull << R) - 1) << (my_box * R);
        }
        const uint32_t lo = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(bits));
        const uint32_t hi = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(bits >> 32));
        hole = static_cast<unsigned long long>(hi) << 32 | lo;
      }
      ok = wait(&ctl.k_empty[slot], parity);
      if (!ok) break;
      if (lane == 0) {
        ctl.hole[j % kHoles] = hole;
        uint32_t expected = bytes;
#ifdef RA_WATCHDOG_TEST
        if (maps.lose && blockIdx.x == 0 && j == 0) expected += 16;
#endif
        mbar_arrive_expect_tx(&ctl.k_full[slot], expected);
      }
      __syncwarp();
      if (there) {
#pragma unroll
        for (int c = 0; c < kD / 64; ++c)
          tma_load_4d(smem_addr(sK + slot * C::kKVBytes + c * C::kKVBlock + my_box * R * 128), &maps.k,
                      &ctl.k_full[slot], c * 64, now.row, now.h, now.page, policy);
      }
      last_k = j;
      ok = wait(&ctl.v_empty[slot], parity);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&ctl.v_full[slot], bytes);
      __syncwarp();
      if (there) {
#pragma unroll
        for (int c = 0; c < kD / 64; ++c)
          tma_load_4d(smem_addr(sV + slot * C::kKVBytes + c * C::kKVBlock + my_box * R * 128), &maps.v,
                      &ctl.v_full[slot], c * 64, now.row, now.h, now.page, policy);
      }
      last_v = j;
      if (++in == now.count) {
        in = 0;
        now = next;
        look_up(next);
      }
    }
  } else if (warp == C::kMmaWarp) {
    // -------------------------------------------------------------- products
    constexpr uint32_t idesc_s = umma_idesc_f16(kBf16, 128, kBN, false);
    constexpr uint32_t idesc_o = umma_idesc_f16(kBf16, 128, kD, true);
    const bool leader = elect_one();
    int unit = 0;  // of the run, at tile j (+ 1 while the next unit's S is issued)
    auto issue_s = [&](int j, bool first, int u) {
      const int slot = j % kStages;
      if (!wait(&ctl.k_full[slot], (j / kStages) & 1)) return false;
      if (first) {
        for (int t = 0; t < kTiles; ++t)
          if (!wait(&ctl.q_full[t], u & 1)) return false;
      }
      tc_fence_after();
      if (leader) {
        const uint64_t kd = sw128_desc(smem_addr(sK + slot * C::kKVBytes), 16, 1024);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const uint64_t qd = sw128_desc(smem_addr(sQ + t * C::kQBytes), 16, 1024);
#pragma unroll
          for (int k = 0; k < kD / 16; ++k)
            umma_ss(tmem + (2 * t + (j & 1)) * kBN, sw128_desc_step(qd, (k / 4) * C::kQBlock + (k % 4) * 32),
                    sw128_desc_step(kd, (k / 4) * C::kKVBlock + (k % 4) * 32), idesc_s, k > 0 ? 1u : 0u);
          umma_commit(&ctl.s_full[t][j & 1]);
        }
        umma_commit(&ctl.k_empty[slot]);
      }
      __syncwarp();
      return true;
    };
    // V of a tile as the product may see it: rows that are no tokens are zeros
    // (no weight, not even zero, may meet what lies there), and so are infinite and
    // NaN values of drafted tokens, which some rows do not follow; the rows
    // that do add them at the end.
    auto mend_v = [&](uint8_t* v, const Cursor& c, unsigned long long hole, int u) {
      const int pos0 = c.t * kBN, live = c.s.len - pos0;
      unsigned long long absent = hole;
      if (live < kBN) absent |= ~0ull << live;
      if (absent) {
        for (int e = lane; e < kBN * (kD / 8); e += 32) {
          const int r = e / (kD / 8), col = e % (kD / 8);
          if (absent >> r & 1u)
            *reinterpret_cast<uint4*>(v + (col / 8) * C::kKVBlock + r * 128 + (((col % 8) ^ (r & 7)) << 4)) =
                make_uint4(0, 0, 0, 0);
        }
      }
      const int from = max(0, c.s.base - pos0), rows = min(live, kBN) - from;
      for (int e = lane; e < rows * (kD / 8); e += 32) {
        const int r = from + e / (kD / 8), col = e % (kD / 8);
        uint4* at = reinterpret_cast<uint4*>(v + (col / 8) * C::kKVBlock + r * 128 + (((col % 8) ^ (r & 7)) << 4));
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
          const int s = pos0 + r - c.s.base;
          atomicOr(&ctl.odd[u & 1][s >> 5], 1u << (s & 31));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    bool ok = n > 0 && issue_s(0, true, 0);
    bool first = true;
    for (int j = 0; j < n && ok; ++j) {
      const bool more = j + 1 < n, ends = cur.t + 1 == cur.T;
      if (more && !ends) ok = issue_s(j + 1, false, unit);
      if (!ok) break;
      const int slot = j % kStages;
      if (first) {
        // (the softmax is past the unit before the last: this buffer is free)
        for (int i = lane; i < kMaxDrafted / 32; i += 32) ctl.odd[unit & 1][i] = 0;
        __syncwarp();
      }
      ok = wait(&ctl.v_full[slot], (j / kStages) & 1);
      if (!ok) break;
      const unsigned long long hole = ctl.hole[j % kHoles];
      if ((cur.t + 1) * kBN > cur.s.base || hole) mend_v(sV + slot * C::kKVBytes, cur, hole, unit);
      const uint64_t vd = sw128_desc(smem_addr(sV + slot * C::kKVBytes), C::kKVBlock, 1024);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        ok = ok && wait(&ctl.p_full[t][j & 1], (j >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = 0; k < kBN / 16; ++k)
            umma_ts(tmem + C::kColO + t * kD, tmem + (2 * t + (j & 1)) * kBN + k * 8, sw128_desc_step(vd, k * 2048),
                    idesc_o, (!first || k > 0) ? 1u : 0u);
          umma_commit(&ctl.pv_done[t]);
          // A barrier of its own: by then the softmax may be two phases of pv_done behind or none.
          if (ends || !more) umma_commit(&ctl.o_done[t]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (leader) umma_commit(&ctl.v_empty[slot]);
      __syncwarp();
      first = false;
      advance<kBN>(a, cur, &fault);
      if (ends) {
        first = true;
        ++unit;
        if (more) ok = issue_s(j + 1, true, unit);
      }
    }
    // Every product this warp issued has retired before tensor memory is given back.
    if (leader) umma_commit(&ctl.mma_done);
    __syncwarp();
    volatile int no_abort = 0;
    mbar_wait(&ctl.mma_done, 0, &no_abort, &ctl.code, 1);
  } else {
    // --------------------------------------------------------------- softmax
    const int t = warp >> 2, in_tile = (warp & 3) * 32 + lane, tid = threadIdx.x & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_off + C::kColO + t * kD;
    const float c = a.scale_log2;
    const uint64_t c2 = f2(c, c);
    int* par = s_par[t];
    int par_b = -1;
    uint32_t met = 0;
    // The 128 threads of the row tile meet (by a wait that ends, as all here).
    auto meet = [&] {
      mbar_arrive(&ctl.group_met[t]);
      const bool there = wait(&ctl.group_met[t], met);
      met ^= 1;
      return there;
    };

    // Q of a unit's rows to shared memory (rows behind the last are zeros) and
    // its sequence's tree.  The S products of the unit before have retired.
    auto load_unit = [&](const Cursor& u) {
      if (!meet()) return false;  // nobody looks at the tree before any more
      if (u.b != par_b) {
        load_parents<128>(a, u.b, u.s.n, par, tid, &fault);
        par_b = u.b;
      }
      const T* q = static_cast<const T*>(a.q) + u.b * a.q_b + static_cast<long long>(u.h) * a.group * a.q_h;
      uint8_t* to = sQ + t * C::kQBytes;
      constexpr int kChunks = kD / 8;
#pragma unroll 8
      for (int e = tid; e < 128 * kChunks; e += 128) {
        const int r = e / kChunks, col = e % kChunks, gr = u.rt * C::kRows + t * 128 + r;
        const int head = gr / a.S, s = gr - head * a.S;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (gr < a.rows && col * 8 < a.c.D)
          x = *reinterpret_cast<const uint4*>(q + head * a.q_h + s * a.q_s + col * 8);
        *reinterpret_cast<uint4*>(to + (col / 8) * C::kQBlock + r * 128 + (((col % 8) ^ (r & 7)) << 4)) = x;
      }
      fence_proxy_async_smem();
      mbar_arrive(&ctl.q_full[t]);
      return meet();  // the tree is there
    };

    float m = -INFINITY, l = 0.f;  // running maximum of the scaled scores that P refers to, sum of P
    bool begun = cur.t == 0, first = true;
    int unit = 0, gr = 0, s_row = 0;  // this thread's row of the kv head, and the drafted token it is
    bool dead = true;                 // no row of the result, or a drafted token that is not there
    auto row_of = [&](const Cursor& u) {
      gr = u.rt * C::kRows + t * 128 + in_tile;
      s_row = gr % a.S;
      dead = gr >= a.rows || s_row >= u.s.n;
    };
    bool ok = n > 0 && load_unit(cur);
    if (ok) row_of(cur);
    for (int j = 0; j < n && ok; ++j) {
      const uint32_t tS = tmem + lane_off + (2 * t + (j & 1)) * kBN;
      ok = wait(&ctl.s_full[t][j & 1], (j >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (!__all_sync(0xffffffffu, dead)) {
        uint32_t u[2][32];
        tmem_ld32(tS, u[0]);
        tmem_ld32(tS + 32, u[1]);
        const int pos0 = cur.t * kBN;
        const unsigned long long hole = ctl.hole[j % kHoles];
        bool any = true;
        uint32_t see[2] = {0xffffffffu, 0xffffffffu};
        const bool masked = pos0 + kBN > cur.s.base || hole;
        if (masked) {
          if (dead) see[0] = see[1] = 0;
          else visible<2>(cur.s, s_row, pos0, par, see);
          // behind the table's end, or in no page
          unsigned long long there = ~hole;
          if (cur.s.len - pos0 < kBN) there &= ~(~0ull << (cur.s.len - pos0));
          see[0] &= static_cast<uint32_t>(there);
          see[1] &= static_cast<uint32_t>(there >> 32);
          any = (see[0] | see[1]) != 0;
        }
        tmem_wait_ld();
        float s[kBN];
#pragma unroll
        for (int i = 0; i < kBN; ++i) s[i] = __uint_as_float(u[i / 32][i % 32]);
        if (masked) {
#pragma unroll
          for (int i = 0; i < kBN; ++i)
            if (!(see[i / 32] >> (i % 32) & 1u)) s[i] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < kBN - 4; i += 8) {
          mx[0] = fmax3(mx[0], s[i + 0], s[i + 4]);
          mx[1] = fmax3(mx[1], s[i + 1], s[i + 5]);
          mx[2] = fmax3(mx[2], s[i + 2], s[i + 6]);
          mx[3] = fmax3(mx[3], s[i + 3], s[i + 7]);
        }
        const float top = fmax3(fmax3(mx[0], mx[1], s[kBN - 4]), fmax3(mx[2], mx[3], s[kBN - 3]),
                                fmaxf(s[kBN - 2], s[kBN - 1]));
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
            ok = wait(&ctl.pv_done[t], (j - 1) & 1);
            if (!ok) break;
            tc_fence_after();
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
        uint32_t pk[32];
        // P is rounded to the input type for P V, by half a step of each weight
        // at most; its sum is taken before that.
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
        tmem_st32(tS, pk);
        float a0, a1, b0, b1;
        f2_split(sum0, a0, a1);
        f2_split(sum1, b0, b1);
        l += (a0 + a1) + (b0 + b1);
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive(&ctl.p_full[t][j & 1]);

      const bool ends = cur.t + 1 == cur.T, last = j + 1 == n;
      Cursor nxt = cur;
      if (!last) advance<kBN>(a, nxt, &fault);
      if (ends || last) {
        // The unit, or this CTA's part of it, ends.
        if (!last && !load_unit(nxt)) break;
        ok = wait(&ctl.o_done[t], unit & 1);
        if (!ok) break;
        tc_fence_after();
        const Place p = place_of(a, cur, begun, run, run.first + j, threadIdx.x == 0);
        const float M = dead ? -INFINITY : m, inv = inverse(M, l);
        uint32_t odd = 0;
        if (lane * 32 < cur.s.n) odd = ctl.odd[unit & 1][lane];
        const bool mend = __any_sync(0xffffffffu, odd != 0);
        if (!__all_sync(0xffffffffu, gr >= a.rows)) {
#pragma unroll 1
          for (int cc = 0; cc < kD; cc += 32) {
            uint32_t u[32];
            tmem_ld32(tO + cc, u);
            tmem_wait_ld();
            float o[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(u[i]);
            if (mend && !dead) {
              // the infinite and NaN values of drafted tokens this row follows, which the product left out
              for (int f = s_row; f >= 0; f = nxt.b == cur.b || last ? par[f] : parent_of(a, cur.b, f)) {
                if (!(ctl.odd[unit & 1][f >> 5] >> (f & 31) & 1u)) continue;
                int row = 0, ignore = 0;
                const int page = page_of(a, cur, cur.s.base + f, &row, &ignore);
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
              float4* part = a.part_o + (static_cast<long long>(p.slot) * a.D4 + cc / 4) * C::kRows + t * 128 + in_tile;
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                if (cc + i < a.c.D) part[i / 4 * C::kRows] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
          if (gr < a.rows && !p.whole)
            a.part_ml[static_cast<long long>(p.slot) * C::kRows + t * 128 + in_tile] = make_float2(M, l);
        }
        tc_fence_before();  // O has been read before the next unit's first product overwrites it (p_full orders the two)
        m = -INFINITY;
        l = 0.f;
        begun = true;
        ++unit;
        if (!last) row_of(nxt);
      }
      first = ends;
      cur = nxt;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kTmaWarp && ctl.abort_flag) {
    // Some role gave up on a wait: copies already asked for land before the
    // CTA's shared memory goes.
    for (int s = 0; s < kStages; ++s) {
      volatile int no_abort = 0;
      const int k = last_k - (last_k - s + kStages * 2) % kStages;  // last tile in slot s
      if (k >= 0) mbar_wait(&ctl.k_full[s], (k / kStages) & 1, &no_abort, &ctl.code, 1);
      const int v = last_v - (last_v - s + kStages * 2) % kStages;
      if (v >= 0) mbar_wait(&ctl.v_full[s], (v / kStages) & 1, &no_abort, &ctl.code, 1);
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
// warp (row tile, columns), lane a row and eight columns of it, its parts in the
// order of the tokens.
constexpr int kJoinWarps = 4, kJoinCols = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_tree_join_kernel(const __grid_constant__ TreeArgs a) {
  launch_dependents();
  grid_dependency_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const int col_tiles = (a.c.D + kJoinCols - 1) / kJoinCols;
  const int w = blockIdx.y * kJoinWarps + (threadIdx.x >> 5), rows32 = w / col_tiles, d = (w - rows32 * col_tiles) * kJoinCols;
  const int4 meta = a.meta[c];
  const int r = rows32 * 32 + lane, gr = meta.y * a.unit_rows + r;
  if (meta.z == 0 || r >= a.unit_rows || gr >= a.rows) return;
  const bool two = d / 4 + 1 < a.D4;
  float M = -INFINITY, L = 0.f;
  float4 o[2] = {};
  for (int i0 = 0; i0 <= meta.z; i0 += 4) {
    float2 ml[4];
    float4 y[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      y[i][0] = y[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + i <= meta.z) {
        const long long slot = i0 + i == 0 ? 2 * c + 1 : 2 * (c + i0 + i);
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
  int row_tiles_each;  // tiles of 128 rows a CTA takes at once (tensor cores)
  int unit_rows, row_tiles, tile;
  int grid;
  long long tiles;  // the block table can name
  size_t meta_at, ml_at, o_at, bytes;
};

// What the tensor-core kernel asks of the cache: 16-byte rows, read in boxes
// of 8 rows at least, which lie in one page.
bool tc_takes(const AttnPagedCache* c) {
  if (c->dtype == ATTN_F32 || c->D % 8 != 0 || c->page_size % 8 != 0 || c->num_pages == 0) return false;
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] % 8 != 0 || c->v_strides[i] % 8 != 0) return false;
  return aligned_to(c->k, 16) && aligned_to(c->v, 16);
}

// `fast`: q, out and the tensor maps allow the tensor-core kernel too.
Plan make_plan(const AttnPagedCache* c, bool fast, int Hq, int S, int sms) {
  Plan p;
  const int D = c->D;
  const long long rows = static_cast<long long>(Hq / c->heads) * S;
  int per_sm;
  p.tc = fast && tc_takes(c);
  p.kd = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  p.row_tiles_each = 1;
  if (p.tc) {
    if (p.kd == 128 && rows > 128) p.row_tiles_each = 2;
    p.unit_rows = 128 * p.row_tiles_each;
    p.tile = TcCfg<128, 1>::kBN;
    per_sm = p.kd <= 128 && p.row_tiles_each == 1 ? 2 : 1;
  } else {
    p.unit_rows = kSimtRows;
    p.tile = kSimtTile;
    per_sm = p.kd == 64 ? 5 : p.kd == 128 ? 3 : 2;
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

template <bool kBf16, int kD, int kTiles>
bool launch_tc(const TreeArgs& a, const TcMaps& maps, int grid, cudaStream_t stream) {
  using C = TcCfg<kD, kTiles>;
  static bool done[64] = {};
  static std::mutex mu;
  return launch_big(attn_tree_tc_kernel<kBf16, kD, kTiles>, mu, done, grid, C::kThreads, C::kSmemBytes, stream, a, maps);
}

template <bool kBf16>
bool launch_tc_d(const TreeArgs& a, const TcMaps& maps, const Plan& p, cudaStream_t stream) {
  if (p.kd == 64) return launch_tc<kBf16, 64, 1>(a, maps, p.grid, stream);
  if (p.kd == 256) return launch_tc<kBf16, 256, 1>(a, maps, p.grid, stream);
  return p.row_tiles_each == 2 ? launch_tc<kBf16, 128, 2>(a, maps, p.grid, stream)
                               : launch_tc<kBf16, 128, 1>(a, maps, p.grid, stream);
}

// The caches' tensor maps; false where TMA cannot describe them.
bool make_maps(const AttnPagedCache* c, TcMaps* m) {
  m->rows = c->page_size % 64 == 0 ? 64 : c->page_size % 32 == 0 ? 32 : c->page_size % 16 == 0 ? 16 : 8;
  const unsigned long long limit = wait_limit_ns();
  m->wait_ns = limit != 0 ? limit : kWaitTimeoutNs;
  m->lose = drop_arrival_requested();
  auto encode = [&](CUtensorMap* map, const void* base, const long long* st) {
    return make_tensor_map_4d(map, base, c->dtype == ATTN_BF16, c->D, c->page_size, c->heads, c->num_pages, st[2], st[1],
                              st[0], 64, m->rows) == 0;
  };
  return encode(&m->k, c->k, c->k_strides) && encode(&m->v, c->v, c->v_strides);
}

template <typename T, int kDP>
bool launch_simt(const TreeArgs& a, int grid, cudaStream_t stream) {
  static bool done[64] = {};
  static std::mutex mu;
  return launch_big(attn_tree_simt_kernel<T, kDP>, mu, done, grid, kSimtThreads, SimtCfg<kDP>::kBytes, stream, a);
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
  const int sms = sm_count();
  // q or out may turn out to need the other kernel: room for either
  const Plan fast = make_plan(cache, true, Hq, S, sms), other = make_plan(cache, false, Hq, S, sms);
  *bytes = fast.bytes > other.bytes ? fast.bytes : other.bytes;
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
  TcMaps maps;
  const bool fast = tc_takes(cache) && aligned_to(q, 16) && aligned_to(out, 16) && qs[0] % 8 == 0 && qs[1] % 8 == 0 &&
                    qs[2] % 8 == 0 && make_maps(cache, &maps);
  const Plan p = make_plan(cache, fast, Hq, S, sm_count());
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
  a.part_o = reinterpret_cast<float4*>(ws + p.o_at);
  a.D4 = (D + 3) / 4;
  const unsigned long long ps = static_cast<unsigned long long>(cache->page_size);
  a.ps_shift = 0;
  while ((1ull << a.ps_shift) < ps) ++a.ps_shift;
  a.ps_mul = static_cast<unsigned>((((1ull << a.ps_shift) - ps) << 32) / ps + 1);

  bool ok;
  if (p.tc) ok = cache->dtype == ATTN_BF16 ? launch_tc_d<true>(a, maps, p, stream) : launch_tc_d<false>(a, maps, p, stream);
  else switch (cache->dtype) {
    case ATTN_F16: ok = launch_simt_d<__half>(a, p, stream); break;
    case ATTN_BF16: ok = launch_simt_d<__nv_bfloat16>(a, p, stream); break;
    default: ok = launch_simt_d<float>(a, p, stream); break;
  }
  if (!ok) return ATTN_ERR_LAUNCH;
  const int used = a.rows < p.unit_rows ? a.rows : p.unit_rows;
  const int join_warps = (used + 31) / 32 * ((D + kJoinCols - 1) / kJoinCols);
  const dim3 grid(p.grid, (join_warps + kJoinWarps - 1) / kJoinWarps), block(kJoinWarps * 32);
  switch (cache->dtype) {
    case ATTN_F16: ok = launch_after(attn_tree_join_kernel<__half>, grid, block, 0, stream, 1, true, a); break;
    case ATTN_BF16: ok = launch_after(attn_tree_join_kernel<__nv_bfloat16>, grid, block, 0, stream, 1, true, a); break;
    default: ok = launch_after(attn_tree_join_kernel<float>, grid, block, 0, stream, 1, true, a); break;
  }
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}
