// What keeps a paged key-value cache: its writer (launch_kv_append), the page
// bounds (launch_kv_page_bounds), the choice of pages a new token should read
// (launch_kv_select_pages) and eviction by accumulated attention weight
// (launch_kv_evict).  The attention that reads the cache is in attn_decode.cu.
//
// All of these move bytes: each row or bound is read once and written once,
// by 16-byte accesses where D and the strides allow (element by element
// otherwise), and the time is that of the bytes once there are enough of them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "paged_cache.h"

namespace ra {

namespace {

__device__ int g_page_fault = 0;

// ---------------------------------------------------------------------------
// Vectors of kVec elements and their elementwise minimum and maximum, NaN
// where either is NaN
// ---------------------------------------------------------------------------

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
  T v[kVec];
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ __half min_nan(__half a, __half b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __half max_nan(__half a, __half b) { return __hmax_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 min_nan(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 max_nan(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmax_nan(a, b); }

template <typename T, int kVec>
__device__ __forceinline__ void fold(Vec<T, kVec>& lo, Vec<T, kVec>& hi, const Vec<T, kVec>& a, const Vec<T, kVec>& b) {
  if constexpr (kVec % 2 == 0 && sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      T2 l, h, x, y;
      memcpy(&l, &lo.v[2 * i], 4);
      memcpy(&h, &hi.v[2 * i], 4);
      memcpy(&x, &a.v[2 * i], 4);
      memcpy(&y, &b.v[2 * i], 4);
      l = __hmin2_nan(l, x);
      h = __hmax2_nan(h, y);
      memcpy(&lo.v[2 * i], &l, 4);
      memcpy(&hi.v[2 * i], &h, 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      lo.v[i] = min_nan(lo.v[i], a.v[i]);
      hi.v[i] = max_nan(hi.v[i], b.v[i]);
    }
  }
}

// The vector of the lane `by` lanes up.
template <typename T, int kVec>
__device__ __forceinline__ Vec<T, kVec> shuffle_down(const Vec<T, kVec>& x, int by) {
  Vec<T, kVec> y;
  if constexpr (sizeof(y) >= 4) {
    uint32_t w[sizeof(y) / 4];
    memcpy(w, &x, sizeof(y));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(y) / 4); ++i) w[i] = __shfl_down_sync(0xffffffffu, w[i], by);
    memcpy(&y, w, sizeof(y));
  } else {
    uint16_t h;
    memcpy(&h, &x, 2);
    h = static_cast<uint16_t>(__shfl_down_sync(0xffffffffu, static_cast<unsigned>(h), by));
    memcpy(&y, &h, 2);
  }
  return y;
}

// ---------------------------------------------------------------------------
// Append and page bounds
// ---------------------------------------------------------------------------

struct RowsArgs {
  PagedView c;
  const void *k, *v;           // new rows (append)
  long long k_b, k_h, k_s, v_b, v_h, v_s;
  int S;
  const int* new_lens;
  void* bounds;
  long long b_p, b_h, b_m;     // bounds strides over (page, head, min/max)
  int runs;                    // pages a sequence may touch
  int cols, row_lanes;         // a warp's lanes: row_lanes rows of up to 32 columns
};

constexpr int kRowsWarps = 8;

// Warp (b, run, head): the rows of one page and head that are new (kAppend),
// or that the sequence has there.  Lane (row lane, column): every
// row_lanes-th row of one 16-byte column, kAhead rows in flight, so that a
// page's rows are mostly on their way at once and nothing waits for other
// warps; the row lanes' minima and maxima meet by shuffles.  Bounds of 16
// sequences of up to 16384 tokens, 8 heads of 128, pages of 32, bf16: 65 us,
// 5.7 TB/s (with CTAs that meet in shared memory 104 us; eight rows in flight
// 69, two 76).  Eight prompts of up to 8192 tokens appended: 40 us, 5.4 TB/s of reads and writes.
template <typename T, int kVec, bool kAppend, bool kBounds>
__global__ void __launch_bounds__(kRowsWarps * 32) kv_rows_kernel(const __grid_constant__ RowsArgs a) {
  using V = Vec<T, kVec>;
  constexpr int kAhead = 4;
  launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long task = static_cast<long long>(blockIdx.x) * kRowsWarps + (threadIdx.x >> 5);
  const int heads = a.c.heads, h = static_cast<int>(task % heads);
  const int page_task = static_cast<int>(task / heads), b = page_task / a.runs, run = page_task - b * a.runs;
  if (b >= a.c.B) return;
  const int ps = a.c.page_size, cap = a.c.capacity();
  int fault = 0;
  long long len = *(a.c.lens + b), first = 0;  // positions [first, len) are taken
  long long start = 0;                             // position of token 0 of the new ones
  if (kAppend) {
    int n = a.S;
    if (a.new_lens) {
      n = *(a.new_lens + b);
      if (n > a.S) {
        fault |= kFaultPage;
        n = a.S;
      }
      if (n < 0) n = 0;
    }
    start = len - n;
    first = start > 0 ? start : 0;
  }
  if (len > cap) {
    fault |= kFaultPage;
    len = cap;
  }
  int page = -1;
  long long base = 0;
  if (first < len) {
    // 64 bits: fewer tokens may be new than there is room for in `runs` pages,
    // and the pages behind the last new one may lie past 2^31.
    const long long lp = static_cast<long long>(static_cast<int>(first) / ps) + run;
    base = lp * ps;
    if (base < len) page = paged_page(a.c, b, static_cast<int>(lp), &fault);
  }
  if (fault && lane == 0) atomicOr(&g_page_fault, fault);
  if (page < 0) return;
  const int r0 = first > base ? static_cast<int>(first - base) : 0;
  const int r1 = len - base < ps ? static_cast<int>(len - base) : ps;

  const int width = min(a.cols, 32);  // columns per turn
  const int row_lane = lane / width, in_row = lane - row_lane * width;
  for (int c0 = 0; c0 < a.cols; c0 += 32) {
    const int col = c0 + in_row;
    const bool live = row_lane < a.row_lanes && col < a.cols;
    V lo = {}, hi = {};
    bool any = false;
    const long long d = static_cast<long long>(col) * kVec;
    if (live) {
      T* ck = static_cast<T*>(a.c.k) + page * a.c.ks[0] + h * a.c.ks[1] + d;
      T* cv = kAppend ? static_cast<T*>(a.c.v) + page * a.c.vs[0] + h * a.c.vs[1] + d : nullptr;
      // row r of the page is new token base + r - start
      const T* nk = kAppend ? static_cast<const T*>(a.k) + b * a.k_b + h * a.k_h + (base - start) * a.k_s + d : ck;
      const T* nv = kAppend ? static_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + (base - start) * a.v_s + d : nullptr;
      const long long k_s = kAppend ? a.k_s : a.c.ks[2];
      for (int r = r0 + row_lane; r < r1; r += kAhead * a.row_lanes) {
        V x[kAhead], y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int at = r + i * a.row_lanes;
          if (at < r1) {
            x[i] = *reinterpret_cast<const V*>(nk + at * k_s);
            if (kAppend) y[i] = *reinterpret_cast<const V*>(nv + at * a.v_s);
          }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int at = r + i * a.row_lanes;
          if (at < r1) {
            if (kAppend) {
              *reinterpret_cast<V*>(ck + at * a.c.ks[2]) = x[i];
              *reinterpret_cast<V*>(cv + at * a.c.vs[2]) = y[i];
            }
            if (kBounds) {
              if (!any) {
                lo = hi = x[i];
                any = true;
              } else {
                fold(lo, hi, x[i], x[i]);
              }
            }
          }
        }
      }
    }
    if constexpr (kBounds) {
      // Row lane i has rows if r0 + i < r1; lane 0 always does.
      const int lanes = min(a.row_lanes, r1 - r0);
      for (int i = 1; i < lanes; ++i) {
        const V l = shuffle_down(lo, i * width), x = shuffle_down(hi, i * width);
        if (row_lane == 0) fold(lo, hi, l, x);
      }
      if (live && row_lane == 0) {
        T* out = static_cast<T*>(a.bounds) + page * a.b_p + h * a.b_h + d;
        V* out_lo = reinterpret_cast<V*>(out);
        V* out_hi = reinterpret_cast<V*>(out + a.b_m);
        if (kAppend && r0 > 0) fold(lo, hi, *out_lo, *out_hi);
        *out_lo = lo;
        *out_hi = hi;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Page scores
// ---------------------------------------------------------------------------

// Keys that order as unsigned integers as the values do, NaN above all, the
// two zeros alike.
__device__ __forceinline__ unsigned long long order_key(double x) {
  if (x != x) return ~0ull;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ unsigned order_key(float x) {
  if (x != x) return ~0u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u >> 31) ? ~u : u | (1u << 31);
}

__device__ __forceinline__ float key_value(unsigned key) {  // (a zero comes back as +0)
  return __uint_as_float((key >> 31) ? key & 0x7fffffffu : ~key);
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

struct ScoreArgs {
  PagedView c;
  const void* q;
  long long q_b, q_h;
  int group;
  const void* bounds;
  long long b_p, b_h, b_m;
  unsigned long long* keys;  // [B, heads, table_width]
  int chunks, pages;         // CTAs per (sequence, head), and pages of each
};

constexpr int kScoreLanes = 16;                 // lanes per page
constexpr int kScoreSlots = 256 / kScoreLanes;  // pages a CTA takes at a time

// 16-bit values as doubles without a conversion, of which the hardware does 16
// a clock and SM against 64 multiply-adds: a value's bits at the top of a
// double are the value times 2^-kShift (the difference of the two exponent
// biases), zeros and subnormals included, as a double's own subnormals carry
// on.  Infinities and NaN come out as finite values, so the caller looks for
// them.
template <typename T> struct Bits16 { static constexpr int kShift = 0; };
template <> struct Bits16<__nv_bfloat16> {
  static constexpr int kShift = 1023 - 127, kMove = 3;
  static constexpr unsigned kMask = 0x8fffe000u;
};
template <> struct Bits16<__half> {
  static constexpr int kShift = 1023 - 15, kMove = 6;
  static constexpr unsigned kMask = 0x81fffc00u;
};
template <typename T>
__device__ __forceinline__ double scaled_double(unsigned top) {  // the value in the upper half of `top`
  // an arithmetic shift keeps the sign; its copies in the exponent go
  const unsigned moved = static_cast<unsigned>(static_cast<int>(top) >> Bits16<T>::kMove) & Bits16<T>::kMask;
  return __hiloint2double(static_cast<int>(moved), 0);
}
__device__ __forceinline__ double power_of_two(int e) { return __hiloint2double((1023 + e) << 20, 0); }

// A lane's part of the sum of a page whose bounds hold infinities or NaN, or
// whose sum came out NaN, by the definition: a part of q that is zero adds
// nothing to it, unless the bound is NaN.  Rare, so out of the way.
template <typename T>
__device__ __noinline__ double odd_page_sum(const T* lo, const T* hi, const double* up, const double* down, int D,
                                            int sub) {
  double sum = 0.0;
#pragma unroll 1
  for (int d = sub; d < D; d += kScoreLanes) {
    const double h = to_f32(hi[d]), l = to_f32(lo[d]);
    if (up[d] != 0.0 || h != h) sum = fma(up[d], h, sum);
    if (down[d] != 0.0 || l != l) sum = fma(down[d], l, sum);
  }
  return sum;
}

// max(q min, q max) is q max where q >= 0 and q min where q < 0, so the sum
// over the query heads needs only their summed positive and negative parts:
// one fused multiply-add per bound whatever the group.  Products of 16-bit
// values are exact in 64 bits and their sums as good as exact, so the choice
// of pages does not depend on the order of the sum.  Half the bounds are
// converted, half moved (Bits16): the two take different pipes (32 contexts of
// up to 1024 pages, 85 MB of bounds: 32 us, all converted 41, all moved 47 with
// what looking for infinities costs).  Neither these pipes nor memory bound it:
// 64 full contexts, 268 MB, take 94 us at 2.9 TB/s, with the 64-bit pipe 14 %
// and the converting one 21 % busy, half of the issue slots used and a third
// of the warps' time spent waiting for bounds, which a warp asks for only when
// those before are summed; and 512 CTAs are 1.15 times what fits at once.
template <typename T, int kVec, int kPer>
__global__ void __launch_bounds__(256, kPer == 1 ? 3 : 1) kv_page_score_kernel(const __grid_constant__ ScoreArgs a) {
  using V = Vec<T, kVec>;
  constexpr bool kMoved = sizeof(T) == 2 && kVec == 8;
  constexpr int kBatch = kPer == 1 ? 2 : 1;  // pages on their way together
  __shared__ double s_up[256], s_down[256];
  launch_dependents();
  grid_dependency_wait();
  const int b = static_cast<int>(blockIdx.x / a.chunks);
  const int chunk = static_cast<int>(blockIdx.x - static_cast<unsigned>(b) * a.chunks);
  const int h = blockIdx.y, lane = threadIdx.x & 31;
  const int sub = threadIdx.x % kScoreLanes, slot = threadIdx.x / kScoreLanes;
  int fault = 0;
  const int len = paged_len(a.c, b, &fault);
  const int pages = static_cast<int>((static_cast<long long>(len) + a.c.page_size - 1) / a.c.page_size);
  const int first = chunk * a.pages, last = first + min(pages - first, a.pages);  // first < table_width
  if (first < last) {
    // Page ids of the next 16 turns, one per lane of the page's lanes.
    auto look_up = [&](int p0) {
      const int p = p0 + sub * kScoreSlots + slot;
      return p < last ? paged_page(a.c, b, p, &fault) : -1;
    };
    int ids = look_up(first);
    {
      const int d = threadIdx.x;
      double up = 0.0, down = 0.0;
      if (d < a.c.D) {
        const T* q = static_cast<const T*>(a.q) + b * a.q_b + static_cast<long long>(h) * a.group * a.q_h + d;
#pragma unroll 8
        for (int g = 0; g < a.group; ++g) {
          const double x = to_f32(q[g * a.q_h]);
          // a NaN goes to both
          if (!(x < 0.0)) up += x;
          if (!(x >= 0.0)) down += x;
        }
      }
      s_up[d] = up;
      s_down[d] = down;
    }
    __syncthreads();
    // Half the shift of the moved bounds goes to q, which keeps products of
    // the largest and of the smallest values in range, half to their sum.
    double up[kPer][kVec], down[kPer][kVec];
#pragma unroll
    for (int j = 0; j < kPer; ++j)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int d = (j * kScoreLanes + sub) * kVec + e;
        up[j][e] = s_up[d & 255];
        down[j][e] = kMoved ? s_down[d & 255] * power_of_two(Bits16<T>::kShift / 2) : s_down[d & 255];
      }
    const T* base = static_cast<const T*>(a.bounds) + h * a.b_h;
    unsigned long long* keys = a.keys + (static_cast<long long>(b) * a.c.heads + h) * a.c.table_width;
    int turn = 0;
    for (int p0 = first; p0 < last; p0 += kBatch * kScoreSlots) {
      V lo[kBatch][kPer], hi[kBatch][kPer];
      int page[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        page[i] = __shfl_sync(0xffffffffu, ids, (lane & 16) + turn + i);
        const T* at = base + page[i] * a.b_p;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int d = (j * kScoreLanes + sub) * kVec;
          lo[i][j] = hi[i][j] = V{};
          if (page[i] >= 0 && d < a.c.D) {
            lo[i][j] = *reinterpret_cast<const V*>(at + d);
            hi[i][j] = *reinterpret_cast<const V*>(at + a.b_m + d);
          }
        }
      }
      turn += kBatch;
      if (turn == kScoreLanes) {
        turn = 0;
        ids = look_up(p0 + kBatch * kScoreSlots);
      }
      double sum[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        double s_hi = 0.0, s_lo = 0.0;
        bool odd = false;
        if constexpr (kMoved) {
          using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
          T2 seen(T(0.f), T(0.f));  // 0 * inf and 0 * NaN are NaN
#pragma unroll
          for (int j = 0; j < kPer; ++j)
#pragma unroll
            for (int e = 0; e < kVec / 2; ++e) {
              unsigned w;
              T2 x;
              memcpy(&w, &lo[i][j].v[2 * e], 4);
              memcpy(&x, &lo[i][j].v[2 * e], 4);
              seen = __hfma2(x, T2(T(0.f), T(0.f)), seen);
              s_lo = fma(down[j][2 * e], scaled_double<T>(w << 16), s_lo);
              s_lo = fma(down[j][2 * e + 1], scaled_double<T>(w), s_lo);
              s_hi = fma(up[j][2 * e], static_cast<double>(to_f32(hi[i][j].v[2 * e])), s_hi);
              s_hi = fma(up[j][2 * e + 1], static_cast<double>(to_f32(hi[i][j].v[2 * e + 1])), s_hi);
            }
          odd = __hisnan(seen.x) || __hisnan(seen.y);
          sum[i] = fma(s_lo, power_of_two(Bits16<T>::kShift / 2), s_hi);
        } else {
#pragma unroll
          for (int j = 0; j < kPer; ++j)
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              s_hi = fma(up[j][e], static_cast<double>(to_f32(hi[i][j].v[e])), s_hi);
              s_lo = fma(down[j][e], static_cast<double>(to_f32(lo[i][j].v[e])), s_lo);
            }
          sum[i] = s_hi + s_lo;
        }
        odd = odd || sum[i] != sum[i];
        const unsigned odd_lanes = __ballot_sync(0xffffffffu, odd && page[i] >= 0);
        if (odd_lanes >> (lane & 16) & 0xffffu)
          sum[i] = odd_page_sum(base + page[i] * a.b_p, base + page[i] * a.b_p + a.b_m, s_up, s_down, a.c.D, sub);
      }
      // The sums over the page's lanes; of two pages the halves of the lanes
      // take one each.
      int mine = 0;
      if constexpr (kBatch == 2) {
        constexpr int off = kScoreLanes / 2;
        mine = sub >= off;
        const double keep = mine ? sum[1] : sum[0], give = mine ? sum[0] : sum[1];
        sum[0] = keep + __shfl_xor_sync(0xffffffffu, give, off);
      }
#pragma unroll
      for (int o = kScoreLanes / 2 / kBatch; o > 0; o >>= 1) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
      const int p = p0 + mine * kScoreSlots + slot;
      // a page the table does not name ranks last
      const bool named = (mine ? page[kBatch - 1] : page[0]) >= 0;
      if (p < last && sub % (kScoreLanes / kBatch) == 0) keys[p] = named ? order_key(sum[0]) : 0ull;
    }
  }
  if (fault) atomicOr(&g_page_fault, fault);
}

// ---------------------------------------------------------------------------
// The largest `pick` of n values, in the order of their places
// ---------------------------------------------------------------------------

// CTAs of 32 warps, or of 8 where there are few places (kPickFew): their
// barriers are shorter.
constexpr int kPickFew = 4096;
constexpr int kPickBits = 11;
constexpr int kPickList = 1024;

struct PickSmem {
  unsigned count[1 << kPickBits];
  unsigned scan[32][2], rank[32][2];
  unsigned long long low[32], high[32], list[kPickList];
  unsigned digit, above, in, listed;
};

// Calls emit(rank, place, key) for the places of the `pick` largest of
// key(0..n-1), 0 < pick < n, in the order of their places; of equal keys at the
// border the lower places.  Each warp has a run of n / 32 places, its lanes 32
// in a row at a time.  Memory is read once if the keys fit `room` in shared
// memory (`kept`), else once a pass.
//
// The border is found from the top, eleven bits a pass, beginning at the
// highest bit in which any two keys differ; a pass whose bucket is taken whole
// is the last.  Once the border's bucket holds few keys they are listed, and
// the later passes look at the list alone.  A place is then taken if key &
// mask > prefix, and the first `need` of those that are equal.
template <int kWarps, typename Key, typename Get, typename Emit>
__device__ void pick_largest(PickSmem& s, Key* kept, int room, Get get, int n, int pick, Emit emit) {
  constexpr int kPickThreads = kWarps * 32, kMine = (1 << kPickBits) / kPickThreads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (n + kPickThreads - 1) / kPickThreads * 32;  // places per warp
  const int begin = warp * run, have = min(max(n - begin, 0), run);
  const bool near = n <= room;
  // f(key, place, is) for 32 places in a row at a time, `is` false behind the
  // end; a warp stays together.
  auto each = [&](auto f) {
    const int full = have & ~31;
    if (near) {
      const Key* at = kept + begin + lane;
#pragma unroll 4
      for (int j = 0; j < full; j += 32) f(at[j], begin + j + lane, true);
    } else {
#pragma unroll 4
      for (int j = 0; j < full; j += 32) f(get(begin + j + lane), begin + j + lane, true);
    }
    if (full < have) {
      const int i = begin + full + lane;
      const bool is = i < begin + have;
      f(is ? get(i) : Key(0), i, is);
    }
  };
  Key low = ~Key(0), high = 0;
  for (int j0 = 0; j0 < have; j0 += 8 * 32) {
    Key x[8];  // eight loads on their way at a time
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = get(min(begin + j0 + j * 32 + lane, n - 1));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = j0 + j * 32 + lane;
      if (i < have) {
        if (near) kept[begin + i] = x[j];  // read by this warp only
        low = x[j] < low ? x[j] : low;
        high = x[j] > high ? x[j] : high;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Key l = __shfl_xor_sync(0xffffffffu, low, o), x = __shfl_xor_sync(0xffffffffu, high, o);
    low = l < low ? l : low;
    high = x > high ? x : high;
  }
  if (lane == 0) {
    s.low[warp] = low;
    s.high[warp] = high;
  }
  if (tid == 0) s.listed = 0;
  for (int i = tid; i < (1 << kPickBits); i += kPickThreads) s.count[i] = 0;
  __syncthreads();
  low = static_cast<Key>(s.low[lane % kWarps]);
  high = static_cast<Key>(s.high[lane % kWarps]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Key l = __shfl_xor_sync(0xffffffffu, low, o), x = __shfl_xor_sync(0xffffffffu, high, o);
    low = l < low ? l : low;
    high = x > high ? x : high;
  }
  const unsigned long long differ = static_cast<unsigned long long>(low ^ high);
  int bit = differ == 0 ? 0 : 64 - __clzll(static_cast<long long>(differ));  // keys agree from this bit up
  Key mask = bit >= static_cast<int>(sizeof(Key) * 8) ? Key(0) : static_cast<Key>(~Key(0) << bit);
  Key prefix = low & mask;
  unsigned need = pick;
  bool listed = false;
  while (bit > 0) {
    const int shift = bit > kPickBits ? bit - kPickBits : 0;
    const unsigned top = (1u << (bit - shift)) - 1;
    if (listed) {
      const unsigned m = s.listed;
      for (unsigned i = tid; i < m; i += kPickThreads) {
        const Key x = static_cast<Key>(s.list[i]);
        if ((x & mask) == prefix) atomicAdd(&s.count[static_cast<unsigned>(x >> shift) & top], 1u);
      }
    } else {
      each([&](Key x, int, bool is) {
        if (is && (x & mask) == prefix) atomicAdd(&s.count[static_cast<unsigned>(x >> shift) & top], 1u);
      });
    }
    __syncthreads();
    // Thread t has kMine buckets, those of thread 0 the highest.
    unsigned c[kMine], upto = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) upto += c[j] = s.count[(1 << kPickBits) - 1 - (kMine * tid + j)];
    const unsigned mine = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) s.scan[warp][0] = upto;
    __syncthreads();
    unsigned before = lane < warp ? s.scan[lane][0] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    unsigned above = before + upto - mine;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int at = (1 << kPickBits) - 1 - (kMine * tid + j);
      if (above < need && above + c[j] >= need) {
        s.digit = at;
        s.above = above;
        s.in = c[j];
      }
      above += c[j];
      s.count[at] = 0;  // for the next pass
    }
    __syncthreads();
    need -= s.above;
    prefix |= static_cast<Key>(s.digit) << shift;
    mask |= static_cast<Key>(top) << shift;
    bit = shift;
    const unsigned in = s.in;
    if (in == need) break;
    if (!listed && in <= kPickList && bit > 0) {
      listed = true;
      each([&](Key x, int, bool is) {
        const bool hit = is && (x & mask) == prefix;
        if (hit) s.list[atomicAdd(&s.listed, 1u)] = x;
      });
      __syncthreads();
    }
  }
  unsigned gt = 0, eq = 0;
  each([&](Key x, int, bool is) {
    gt += is && (x & mask) > prefix;
    eq += is && (x & mask) == prefix;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  if (lane == 0) {
    s.rank[warp][0] = gt;
    s.rank[warp][1] = eq;
  }
  __syncthreads();
  gt = lane < warp ? s.rank[lane][0] : 0;
  eq = lane < warp ? s.rank[lane][1] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  const unsigned under = (1u << lane) - 1;
  each([&](Key x, int i, bool is) {
    const bool is_gt = is && (x & mask) > prefix, is_eq = is && (x & mask) == prefix;
    const unsigned g = __ballot_sync(0xffffffffu, is_gt), e = __ballot_sync(0xffffffffu, is_eq);
    if ((g | e) == 0) return;
    const unsigned eq_here = eq + __popc(e & under);
    if (is_gt || (is_eq && eq_here < need)) emit(static_cast<int>(gt + __popc(g & under) + min(eq_here, need)), i, x);
    gt += __popc(g);
    eq += __popc(e);
  });
}

// Shared memory for the keys of up to `most` places.
constexpr int kPickRoomBytes = 160 * 1024;
int pick_room(long long most, int key_bytes) {
  const long long room = kPickRoomBytes / key_bytes;
  return static_cast<int>(most < room ? most : room);
}

template <typename... Params, typename... Args>
bool launch_pick(void (*kern)(Params...), int warps, unsigned units, size_t smem, cudaStream_t stream,
                 const Args&... args) {
  // 48 KiB without asking, PickSmem among them
  if (smem + sizeof(PickSmem) > 48 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickRoomBytes) != cudaSuccess)
    return false;
  return launch_after(kern, dim3(units), dim3(warps * 32), smem, stream, 1, true, args...);
}

// CTA (head, b): the last place, and the pick - 1 largest of the others.
template <int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
    kv_pick_pages_kernel(PagedView c, const unsigned long long* keys, int top, int* pages, int room) {
  __shared__ PickSmem s;
  extern __shared__ __align__(16) unsigned char kept[];
  launch_dependents();
  grid_dependency_wait();
  const int h = blockIdx.x % c.heads, b = blockIdx.x / c.heads;
  int fault = 0;  // recorded by the kernel before
  const int len = paged_len(c, b, &fault);
  const int n = static_cast<int>((static_cast<long long>(len) + c.page_size - 1) / c.page_size);
  const unsigned long long* k = keys + (static_cast<long long>(b) * c.heads + h) * c.table_width;
  int* out = pages + (static_cast<long long>(b) * c.heads + h) * top;
  if (n <= top) {
    // unsigned: `top` may be the largest int, and a step past it must not wrap
    for (unsigned i = threadIdx.x; i < static_cast<unsigned>(top); i += kWarps * 32)
      out[i] = i < static_cast<unsigned>(n) ? static_cast<int>(i) : -1;
    return;
  }
  if (threadIdx.x == 0) out[top - 1] = n - 1;
  if (top == 1) return;
  pick_largest<kWarps>(
      s, reinterpret_cast<unsigned long long*>(kept), room, [&](int i) { return k[i]; }, n - 1, top - 1,
      [&](int rank, int i, unsigned long long) { out[rank] = i; });
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------

struct EvictArgs {
  PagedView c;
  const float* w;
  long long w_b, w_h;
  const int* new_table;
  long long new_stride;
  int new_width, budget, recent;
  float* new_w;
  int* kept;
  int* new_lens;
  int cols, rows_per_cta, chunks;
  int room;  // keys in shared memory
};

// CTA (head, b): the kept positions and their weights.
template <int kWarps>
__global__ void __launch_bounds__(kWarps * 32) kv_evict_pick_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ PickSmem s;
  extern __shared__ __align__(16) unsigned char keys[];
  grid_dependency_wait();
  const int h = blockIdx.x % a.c.heads, b = blockIdx.x / a.c.heads;
  int fault = 0;
  const int n = paged_len(a.c, b, &fault);
  if (fault && threadIdx.x == 0) atomicOr(&g_page_fault, 1);
  const float* w = a.w + b * a.w_b + h * a.w_h;
  const long long unit = static_cast<long long>(b) * a.c.heads + h;
  int* kept = a.kept + unit * a.budget;
  const int new_cap = a.new_width * a.c.page_size;
  float* new_w = a.new_w + unit * new_cap;
  const int m = min(n, a.budget);
  if (h == 0 && threadIdx.x == 0) a.new_lens[b] = m;
  for (int i = m + threadIdx.x; i < new_cap; i += kWarps * 32) new_w[i] = 0.f;
  for (int i = m + threadIdx.x; i < a.budget; i += kWarps * 32) kept[i] = -1;
  // positions [0, sure) compete for `pick` places, those behind are kept
  const int pick = n <= a.budget ? 0 : a.budget - a.recent;
  const int sure = n <= a.budget ? 0 : n - a.recent;
  for (int i = sure + threadIdx.x; i < n; i += kWarps * 32) {
    kept[pick + i - sure] = i;
    new_w[pick + i - sure] = w[i];
  }
  if (pick == 0) return;
  pick_largest<kWarps>(
      s, reinterpret_cast<unsigned*>(keys), a.room, [&](int i) { return order_key(w[i]); }, sure, pick,
      [&](int rank, int i, unsigned key) {
        kept[rank] = i;
        new_w[rank] = key_value(key);
      });
}

constexpr int kCopyRows = 2;  // 4 and 8 measured 3 % and 23 % slower: CTAs on the SM do more than loads per thread

// Keeping 4096 of up to 32768 tokens of 16 sequences, 8 heads of 128, fp16: the
// choice 24 us, the copy 90 us, 5.9 TB/s of scattered 256-byte rows.
//
// CTA (b, chunk of rows; head): copies kept rows to the new pages, a column
// of kVec elements of kCopyRows rows per thread, K and V.
template <typename T, int kVec>
__global__ void __launch_bounds__(256) kv_evict_copy_kernel(const __grid_constant__ EvictArgs a) {
  using V = Vec<T, kVec>;
  constexpr int kAhead = kCopyRows;
  grid_dependency_wait();
  const int b = static_cast<int>(blockIdx.x / a.chunks);
  const int chunk = static_cast<int>(blockIdx.x - static_cast<unsigned>(b) * a.chunks);
  const int h = blockIdx.y, ps = a.c.page_size;
  int fault = 0;
  const int m = min(paged_len(a.c, b, &fault), a.budget);
  fault = 0;  // recorded by the kernel before
  const int col = threadIdx.x % a.cols, lane = threadIdx.x / a.cols;
  if (lane >= a.rows_per_cta) return;
  const int* kept = a.kept + (static_cast<long long>(b) * a.c.heads + h) * a.budget;
  const long long d = static_cast<long long>(col) * kVec;
  T* ck = static_cast<T*>(a.c.k) + h * a.c.ks[1] + d;
  T* cv = static_cast<T*>(a.c.v) + h * a.c.vs[1] + d;
  V x[kAhead], y[kAhead];
  int to[kAhead], row[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const long long place = static_cast<long long>(chunk) * (kAhead * a.rows_per_cta) + i * a.rows_per_cta + lane;
    to[i] = -1;
    if (place < m) {
      const int src = kept[place];
      const int lp = src / ps, page = paged_page(a.c, b, lp, &fault);
      const int np = static_cast<int>(place) / ps;
      row[i] = static_cast<int>(place) - np * ps;
      const int t = *(a.new_table + b * a.new_stride + np);
      const bool good = static_cast<unsigned>(t) < static_cast<unsigned>(a.c.num_pages);
      if (!good) fault |= kFaultPage;
      if (good && page >= 0) {
        to[i] = t;
        x[i] = *reinterpret_cast<const V*>(ck + page * a.c.ks[0] + (src - lp * ps) * a.c.ks[2]);
        y[i] = *reinterpret_cast<const V*>(cv + page * a.c.vs[0] + (src - lp * ps) * a.c.vs[2]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (to[i] >= 0) {
      *reinterpret_cast<V*>(ck + to[i] * a.c.ks[0] + row[i] * a.c.ks[2]) = x[i];
      *reinterpret_cast<V*>(cv + to[i] * a.c.vs[0] + row[i] * a.c.vs[2]) = y[i];
    }
  if (fault) atomicOr(&g_page_fault, 1);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

bool all_multiples(const long long* s, int n, int of) {
  for (int i = 0; i < n; ++i)
    if (s[i] % of != 0) return false;
  return true;
}

// Elements per 16-byte access when D, the given strides and pointers allow
// them, else 1.
struct Width {
  int vec;
  explicit Width(const AttnPagedCache* c) : vec(c->dtype == ATTN_F32 ? 4 : 8) {
    if (c->D % vec != 0) vec = 1;
  }
  void need(const void* p, const long long* strides, int n) {
    if (!aligned_to(p, 16) || !all_multiples(strides, n, vec)) vec = 1;
  }
};

size_t elem_size(AttnDType t) { return t == ATTN_F32 ? 4 : 2; }

template <typename T, int kVec>
bool launch_rows_typed(const RowsArgs& a, bool append, dim3 grid, cudaStream_t stream) {
  const auto kern = !append    ? kv_rows_kernel<T, kVec, false, true>
                    : a.bounds ? kv_rows_kernel<T, kVec, true, true>
                               : kv_rows_kernel<T, kVec, true, false>;
  return launch_after(kern, grid, dim3(kRowsWarps * 32), 0, stream, 1, true, a);
}

int launch_rows(RowsArgs& a, AttnDType dtype, int vec, bool append, cudaStream_t stream) {
  a.cols = a.c.D / vec;
  a.row_lanes = a.cols >= 32 ? 1 : 32 / a.cols;
  const long long pages = static_cast<long long>(a.c.B) * a.runs;
  if (pages == 0) return ATTN_OK;
  if (pages > 0x7fffffffLL || (pages * a.c.heads + kRowsWarps - 1) / kRowsWarps > 0x7fffffffLL)
    return ATTN_ERR_INVALID_ARGUMENT;
  const dim3 grid(static_cast<unsigned>((pages * a.c.heads + kRowsWarps - 1) / kRowsWarps));
  bool ok;
  switch (dtype) {
    case ATTN_F16:
      ok = vec == 8 ? launch_rows_typed<__half, 8>(a, append, grid, stream)
                    : launch_rows_typed<__half, 1>(a, append, grid, stream);
      break;
    case ATTN_BF16:
      ok = vec == 8 ? launch_rows_typed<__nv_bfloat16, 8>(a, append, grid, stream)
                    : launch_rows_typed<__nv_bfloat16, 1>(a, append, grid, stream);
      break;
    default:
      ok = vec == 4 ? launch_rows_typed<float, 4>(a, append, grid, stream)
                    : launch_rows_typed<float, 1>(a, append, grid, stream);
      break;
  }
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}

bool negative(const long long* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0) return true;
  return false;
}

template <typename T, int kVec, int kPer>
bool launch_score(const ScoreArgs& a, dim3 grid, cudaStream_t stream) {
  return launch_after(kv_page_score_kernel<T, kVec, kPer>, grid, dim3(256), 0, stream, 1, true, a);
}

template <typename T>
bool launch_score_typed(const ScoreArgs& a, int vec, dim3 grid, cudaStream_t stream) {
  if (vec == 1) return launch_score<T, 1, 16>(a, grid, stream);
  constexpr int kVec = sizeof(T) == 2 ? 8 : 4;
  const int per = (a.c.D + kScoreLanes * kVec - 1) / (kScoreLanes * kVec);
  if (per == 1) return launch_score<T, kVec, 1>(a, grid, stream);
  if (per == 2) return launch_score<T, kVec, 2>(a, grid, stream);
  return launch_score<T, kVec, 256 / (kScoreLanes * kVec)>(a, grid, stream);
}

}  // namespace

int check_paged_cache(const AttnPagedCache* c, int tensors, PagedView* view) {
  if (!c) return ATTN_ERR_INVALID_ARGUMENT;
  if (c->dtype != ATTN_F16 && c->dtype != ATTN_BF16 && c->dtype != ATTN_F32) return ATTN_ERR_UNSUPPORTED;
  if (c->B < 0 || c->heads < 1 || c->page_size < 1 || c->num_pages < 0 || c->table_width < 0 || c->table_stride < 0 ||
      c->D < 1)
    return ATTN_ERR_INVALID_ARGUMENT;
  if (c->D > 256) return ATTN_ERR_UNSUPPORTED;
  if (static_cast<long long>(c->table_width) * c->page_size > kMaxCapacity) return ATTN_ERR_INVALID_ARGUMENT;
  if (c->B > 0 && (!c->seq_lens || (c->table_width > 0 && !c->block_table))) return ATTN_ERR_INVALID_ARGUMENT;
  if (!aligned_to(c->seq_lens, 4) || !aligned_to(c->block_table, 4)) return ATTN_ERR_MISALIGNED;
  const void* ptr[2] = {c->k, c->v};
  const long long* st[2] = {c->k_strides, c->v_strides};
  for (int i = 0; i < 2; ++i) {
    if (!(tensors >> i & 1)) continue;
    if ((c->num_pages > 0 && !ptr[i]) || negative(st[i], 3)) return ATTN_ERR_INVALID_ARGUMENT;
    if (!aligned_to(ptr[i], elem_size(c->dtype))) return ATTN_ERR_MISALIGNED;
  }
  *view = PagedView{c->k,
                    c->v,
                    {c->k_strides[0], c->k_strides[1], c->k_strides[2]},
                    {c->v_strides[0], c->v_strides[1], c->v_strides[2]},
                    c->block_table,
                    c->table_stride,
                    c->seq_lens,
                    c->table_width,
                    c->num_pages,
                    c->heads,
                    c->page_size,
                    c->D,
                    c->B};
  return ATTN_OK;
}

int page_word_read_clear_cache(cudaStream_t stream, int* host) {
  static const int zero = 0;
  return cudaMemcpyFromSymbolAsync(host, g_page_fault, sizeof(int), 0, cudaMemcpyDeviceToHost, stream) ==
                     cudaSuccess &&
                 cudaMemcpyToSymbolAsync(g_page_fault, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream) ==
                     cudaSuccess
             ? 0
             : -1;
}

}  // namespace ra

extern "C" int launch_kv_append(const AttnPagedCache* cache, const void* k, const long long* k_strides, const void* v,
                                const long long* v_strides, int S, const int* new_lens, void* bounds,
                                const long long* bounds_strides, cudaStream_t stream) {
  using namespace ra;
  PagedView view;
  int st = check_paged_cache(cache, kCacheK | kCacheV, &view);
  if (st != ATTN_OK) return st;
  if (S < 0) return ATTN_ERR_INVALID_ARGUMENT;
  if (cache->B == 0 || S == 0) return ATTN_OK;
  if (!k || !v || !k_strides || !v_strides || negative(k_strides, 3) || negative(v_strides, 3) ||
      (bounds && (!bounds_strides || negative(bounds_strides, 3))))
    return ATTN_ERR_INVALID_ARGUMENT;
  const size_t elem = elem_size(cache->dtype);
  if (!aligned_to(k, elem) || !aligned_to(v, elem) || !aligned_to(bounds, elem) || !aligned_to(new_lens, 4))
    return ATTN_ERR_MISALIGNED;
  st = check_device();
  if (st != ATTN_OK) return st;
  Width w(cache);
  w.need(cache->k, cache->k_strides, 3);
  w.need(cache->v, cache->v_strides, 3);
  w.need(k, k_strides, 3);
  w.need(v, v_strides, 3);
  if (bounds) w.need(bounds, bounds_strides, 3);
  RowsArgs a = {};
  a.c = view;
  a.k = k;
  a.v = v;
  a.k_b = k_strides[0], a.k_h = k_strides[1], a.k_s = k_strides[2];
  a.v_b = v_strides[0], a.v_h = v_strides[1], a.v_s = v_strides[2];
  a.S = S;
  a.new_lens = new_lens;
  a.bounds = bounds;
  if (bounds) a.b_p = bounds_strides[0], a.b_h = bounds_strides[1], a.b_m = bounds_strides[2];
  // S tokens touch at most this many pages of the table
  const long long runs = (static_cast<long long>(S) - 1 + cache->page_size - 1) / cache->page_size + 1;
  a.runs = static_cast<int>(runs < cache->table_width ? runs : cache->table_width > 0 ? cache->table_width : 1);
  return launch_rows(a, cache->dtype, w.vec, true, stream);
}

extern "C" int launch_kv_page_bounds(const AttnPagedCache* cache, void* bounds, const long long* bounds_strides,
                                     cudaStream_t stream) {
  using namespace ra;
  PagedView view;
  int st = check_paged_cache(cache, kCacheK, &view);
  if (st != ATTN_OK) return st;
  if (cache->B == 0) return ATTN_OK;
  if ((cache->num_pages > 0 && !bounds) || !bounds_strides || negative(bounds_strides, 3))
    return ATTN_ERR_INVALID_ARGUMENT;
  if (!aligned_to(bounds, elem_size(cache->dtype))) return ATTN_ERR_MISALIGNED;
  st = check_device();
  if (st != ATTN_OK) return st;
  Width w(cache);
  w.need(cache->k, cache->k_strides, 3);
  w.need(bounds, bounds_strides, 3);
  RowsArgs a = {};
  a.c = view;
  a.bounds = bounds;
  a.b_p = bounds_strides[0], a.b_h = bounds_strides[1], a.b_m = bounds_strides[2];
  a.runs = cache->table_width > 0 ? cache->table_width : 1;
  return launch_rows(a, cache->dtype, w.vec, false, stream);
}

extern "C" int kv_select_pages_workspace_bytes(const AttnPagedCache* cache, size_t* bytes) {
  using namespace ra;
  if (!bytes) return ATTN_ERR_INVALID_ARGUMENT;
  PagedView view;
  const int st = check_paged_cache(cache, 0, &view);
  if (st != ATTN_OK) return st;
  *bytes = sizeof(unsigned long long) * static_cast<size_t>(cache->B) * cache->heads * cache->table_width;
  return ATTN_OK;
}

extern "C" int launch_kv_select_pages(const AttnPagedCache* cache, const void* q, const long long* q_strides, int Hq,
                                      const void* bounds, const long long* bounds_strides, int top, int* pages,
                                      void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  using namespace ra;
  PagedView view;
  int st = check_paged_cache(cache, 0, &view);
  if (st != ATTN_OK) return st;
  if (top < 1 || Hq < 0 || Hq % cache->heads != 0 || cache->heads > 65535) return ATTN_ERR_INVALID_ARGUMENT;
  if (cache->B == 0) return ATTN_OK;
  const long long units = static_cast<long long>(cache->B) * cache->heads;
  // Pages per CTA: as many as leave four CTAs per SM, three of which run at
  // once (32 contexts of 1024 pages: 34.8 us with eight, 32.9 us with four).
  // In 64 bits: the width rounded up can pass 2^31.
  const long long target = 4LL * sm_count(), wanted = units < target ? target / units : 1;
  constexpr int kTurns = 4 * kScoreSlots;
  const long long per = ((cache->table_width + wanted - 1) / wanted + kTurns - 1) / kTurns * kTurns;
  const long long chunks = per > 0 ? (cache->table_width + per - 1) / per : 0;
  if (units > 0x7fffffffLL || cache->B * chunks > 0x7fffffffLL) return ATTN_ERR_INVALID_ARGUMENT;
  const long long contiguous[2] = {static_cast<long long>(Hq) * cache->D, cache->D};
  const long long* qs = q_strides ? q_strides : contiguous;
  if ((Hq > 0 && !q) || !pages || (cache->num_pages > 0 && !bounds) || !bounds_strides || negative(bounds_strides, 3) ||
      negative(qs, 2) || (cache->table_width > 0 && !workspace))
    return ATTN_ERR_INVALID_ARGUMENT;
  const size_t elem = elem_size(cache->dtype);
  if (!aligned_to(q, elem) || !aligned_to(bounds, elem) || !aligned_to(pages, 4) || !aligned_to(workspace, 16))
    return ATTN_ERR_MISALIGNED;
  if (workspace_bytes < sizeof(unsigned long long) * static_cast<size_t>(units) * cache->table_width)
    return ATTN_ERR_INVALID_ARGUMENT;
  st = check_device();
  if (st != ATTN_OK) return st;
  Width w(cache);
  w.need(bounds, bounds_strides, 3);
  ScoreArgs a;
  a.c = view;
  a.q = q;
  a.q_b = qs[0];
  a.q_h = qs[1];
  a.group = Hq / cache->heads;
  a.bounds = bounds;
  a.b_p = bounds_strides[0], a.b_h = bounds_strides[1], a.b_m = bounds_strides[2];
  a.keys = static_cast<unsigned long long*>(workspace);
  a.chunks = static_cast<int>(chunks);
  a.pages = static_cast<int>(per);  // kTurns divides 2^31 - 65536, the widest table and one, so this fits too
  if (chunks > 0) {
    const dim3 grid(static_cast<unsigned>(cache->B * chunks), cache->heads);
    bool ok;
    switch (cache->dtype) {
      case ATTN_F16: ok = launch_score_typed<__half>(a, w.vec, grid, stream); break;
      case ATTN_BF16: ok = launch_score_typed<__nv_bfloat16>(a, w.vec, grid, stream); break;
      default: ok = launch_score_typed<float>(a, w.vec, grid, stream); break;
    }
    if (!ok) return ATTN_ERR_LAUNCH;
  }
  const int room = pick_room(cache->table_width, sizeof(unsigned long long));
  const bool few = cache->table_width <= kPickFew;
  return launch_pick(few ? kv_pick_pages_kernel<8> : kv_pick_pages_kernel<32>, few ? 8 : 32,
                     static_cast<unsigned>(units), room * sizeof(unsigned long long), stream, view,
                     static_cast<const unsigned long long*>(a.keys), top, pages, room)
             ? ATTN_OK
             : ATTN_ERR_LAUNCH;
}

extern "C" int launch_kv_evict(const AttnPagedCache* cache, const float* weights, const long long* weights_strides,
                               const int* new_table, long long new_stride, int new_width, int budget, int recent,
                               float* new_weights, int* kept, int* new_lens, cudaStream_t stream) {
  using namespace ra;
  PagedView view;
  int st = check_paged_cache(cache, kCacheK | kCacheV, &view);
  if (st != ATTN_OK) return st;
  if (budget < 1 || recent < 0 || recent > budget || new_width < 0 || new_stride < 0 || cache->heads > 65535 ||
      static_cast<long long>(new_width) * cache->page_size > kMaxCapacity ||
      budget > static_cast<long long>(new_width) * cache->page_size)
    return ATTN_ERR_INVALID_ARGUMENT;
  if (cache->B == 0) return ATTN_OK;
  if ((!weights && view.capacity() > 0) || !weights_strides || negative(weights_strides, 2) || !new_table ||
      !new_weights || !kept || !new_lens)
    return ATTN_ERR_INVALID_ARGUMENT;
  if (!aligned_to(weights, 4) || !aligned_to(new_table, 4) || !aligned_to(new_weights, 4) || !aligned_to(kept, 4) ||
      !aligned_to(new_lens, 4))
    return ATTN_ERR_MISALIGNED;
  Width w(cache);
  w.need(cache->k, cache->k_strides, 3);
  w.need(cache->v, cache->v_strides, 3);
  EvictArgs a;
  a.c = view;
  a.w = weights;
  a.w_b = weights_strides[0];
  a.w_h = weights_strides[1];
  a.new_table = new_table;
  a.new_stride = new_stride;
  a.new_width = new_width;
  a.budget = budget;
  a.recent = recent;
  a.new_w = new_weights;
  a.kept = kept;
  a.new_lens = new_lens;
  a.cols = cache->D / w.vec;
  a.rows_per_cta = 256 / a.cols;
  const long long units = static_cast<long long>(cache->B) * cache->heads;
  a.chunks = (budget + kCopyRows * a.rows_per_cta - 1) / (kCopyRows * a.rows_per_cta);
  const long long x = static_cast<long long>(cache->B) * a.chunks;
  if (units > 0x7fffffffLL || x > 0x7fffffffLL) return ATTN_ERR_INVALID_ARGUMENT;
  st = check_device();
  if (st != ATTN_OK) return st;
  a.room = pick_room(view.capacity(), sizeof(unsigned));
  const bool few = view.capacity() <= kPickFew;
  if (!launch_pick(few ? kv_evict_pick_kernel<8> : kv_evict_pick_kernel<32>, few ? 8 : 32, static_cast<unsigned>(units),
                   a.room * sizeof(unsigned), stream, a))
    return ATTN_ERR_LAUNCH;
  const dim3 grid(static_cast<unsigned>(x), cache->heads), block(256);
  bool ok;
  switch (cache->dtype) {
    case ATTN_F16:
      ok = w.vec == 8 ? launch_after(kv_evict_copy_kernel<__half, 8>, grid, block, 0, stream, 1, true, a)
                      : launch_after(kv_evict_copy_kernel<__half, 1>, grid, block, 0, stream, 1, true, a);
      break;
    case ATTN_BF16:
      ok = w.vec == 8 ? launch_after(kv_evict_copy_kernel<__nv_bfloat16, 8>, grid, block, 0, stream, 1, true, a)
                      : launch_after(kv_evict_copy_kernel<__nv_bfloat16, 1>, grid, block, 0, stream, 1, true, a);
      break;
    default:
      ok = w.vec == 4 ? launch_after(kv_evict_copy_kernel<float, 4>, grid, block, 0, stream, 1, true, a)
                      : launch_after(kv_evict_copy_kernel<float, 1>, grid, block, 0, stream, 1, true, a);
      break;
  }
  return ok ? ATTN_OK : ATTN_ERR_LAUNCH;
}
