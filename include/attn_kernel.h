/*
 * C-ABI launch interface of the sm_100a attention-forward library
 * (librocm_attn.so).  Plain pointers and sizes only; no framework types.
 *
 * Replaces the reference's `launch_attn_forward` declared at
 * src/attn_kernel.h:18-20 of JoursBleu/rocm_attn (enum AttnDType at
 * src/attn_kernel.h:12-16), whose definitions live at
 * src/attn_kernel_torch.cu:625-689 and src/attn_kernel.hip.cpp:304-367.
 *
 * Differences from the reference signature, all deliberate:
 *   - returns an int status (the reference returns void and checks nothing);
 *   - takes an explicit softmax scale (the reference hard-wires rsqrt(D),
 *     src/attn_kernel_torch.cu:111); a value <= 0 or non-finite selects the
 *     reference default 1/sqrt(D);
 *   - the stream is a cudaStream_t (the reference takes a hipStream_t).
 * The argument order otherwise matches the reference.
 */
#ifndef ROCM_ATTN_B200_ATTN_KERNEL_H_
#define ROCM_ATTN_B200_ATTN_KERNEL_H_

#include <cuda_runtime.h>
#include <stdbool.h>
#include <stddef.h>

#if defined(__GNUC__)
#define ATTN_API __attribute__((visibility("default")))
#else
#define ATTN_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of q/k/v/out.  Values match the reference enum
 * (src/attn_kernel.h:12-16) so the ABI stays compatible. */
typedef enum AttnDType {
  ATTN_F16 = 0,
  ATTN_BF16 = 1,
  ATTN_F32 = 2,
} AttnDType;

/* Status codes returned by the entry points below. */
enum AttnStatus {
  ATTN_OK = 0,
  ATTN_ERR_INVALID_ARGUMENT = 1, /* null pointer, negative size, overflow   */
  ATTN_ERR_UNSUPPORTED = 2,      /* unknown dtype or head_dim > 256         */
  ATTN_ERR_MISALIGNED = 3,       /* pointer not aligned to its element size */
  ATTN_ERR_TENSOR_MAP = 4,       /* TMA descriptor could not be encoded     */
  ATTN_ERR_LAUNCH = 5,           /* CUDA runtime error at launch            */
  ATTN_ERR_DEVICE = 6,           /* current device is not an sm_100 GPU     */
  ATTN_ERR_WATCHDOG = 7,         /* a kernel wait timed out (see below)     */
  ATTN_ERR_BAD_PAGE = 8          /* page id or length out of range (below)  */
};

/*
 * Scaled dot-product attention forward, O = softmax(scale * Q K^T [+ mask]) V.
 *   q   [B, H, Sq,  D]  contiguous, row-major
 *   k,v [B, H, Skv, D]  contiguous, row-major
 *   out [B, H, Sq,  D]  contiguous, row-major, fully overwritten
 * causal: key j is masked for query i when j > i (top-left aligned, the
 * reference's rule at src/attn_kernel_torch.cu:54,238,263).  Skv == 0 gives
 * an all-zero output, like the reference's empty-denominator rule
 * (src/attn_kernel_torch.cu:335-336).
 * Supported: dtype ATTN_F16 / ATTN_BF16 / ATTN_F32 and 1 <= D <= 256, every
 * pointer aligned to its element size.  fp16/bf16 with D in {64, 128} and
 * 16-byte aligned buffers run the tcgen05 tensor-core kernel; every other
 * supported call runs the general kernel (fp32 arithmetic), which covers the
 * reference's fp32 and D=16 routes (src/attn_kernel_torch.cu:625-689).
 * Asynchronous on `stream`; allocates nothing; re-entrant.
 * Returns ATTN_OK or an AttnStatus code; on error nothing was launched.
 */
ATTN_API int launch_attn_forward(const void* q, const void* k, const void* v, void* out, int B, int H, int Sq, int Skv,
                        int D, bool causal, float softmax_scale, AttnDType dtype, cudaStream_t stream);

/*
 * launch_attn_forward on strided q, k and v: each *_strides array holds the
 * element strides over (batch, head, row), the head dim being contiguous; a
 * null array means the contiguous layout.  For example the [B, L, H, D]
 * layout of flash-style callers viewed as [B, H, L, D] has strides
 * {L*H*D, D, H*D}.  out stays contiguous [B, H, Sq, D].  The tensor-core
 * kernel reads strided inputs directly through TMA when every stride is a
 * multiple of 16 bytes; otherwise the general kernel runs.  Strides must be
 * >= 0.  No counterpart in the reference, whose binding copies inputs to
 * contiguous tensors first (src/attn_torch.cpp:20-22).
 */
ATTN_API int launch_attn_forward_strided(const void* q, const void* k, const void* v, void* out, int B, int H,
                                         int Sq, int Skv, int D, bool causal, float softmax_scale, AttnDType dtype,
                                         const long long* q_strides, const long long* k_strides,
                                         const long long* v_strides, cudaStream_t stream);

/*
 * One problem of launch_attn_forward_batch: the arguments of
 * launch_attn_forward_strided for one call (null strides: contiguous).
 */
typedef struct AttnProblem {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int B, H, Sq, Skv, D;
  bool causal;
  float softmax_scale;
  const long long* q_strides;
  const long long* k_strides;
  const long long* v_strides;
} AttnProblem;

/*
 * Runs n independent problems of one dtype, as launch_attn_forward_strided
 * would one by one, with the same results bit for bit, in fewer launches:
 * the problems that run the tcgen05 tensor-core kernel with the same head
 * dim, masking and tile shape share one grid (up to 16 problems per grid),
 * whose work units are ordered longest first, so the short units of one
 * problem fill the last wave of another and no launch waits for the tail of
 * the previous one.  Short problems (fp16/bf16, at most 16 queries and 64
 * keys) with the same head dim and 16-key group count share one grid of the
 * warp-level tensor-core kernel the same way.  The others are launched one
 * by one.  Every problem is
 * checked before anything is launched; on an error nothing was launched.
 * The output buffers must not overlap any input or each other.  No
 * counterpart in the reference, whose benchmark launches one shape at a time
 * (benchmark/bench_attention.py:81-100,171-175).
 */
ATTN_API int launch_attn_forward_batch(const AttnProblem* problems, int n, AttnDType dtype, cudaStream_t stream);

/*
 * Reads and clears the device status word of the current device, after
 * synchronising `stream`.  *status receives ATTN_OK, or ATTN_ERR_WATCHDOG when a
 * kernel launched earlier gave up on a wait (its output is then invalid), or
 * ATTN_ERR_BAD_PAGE when a kernel of the paged cache met a block-table entry
 * outside the cache or a length beyond the block table (see below; both words
 * are cleared, the watchdog is reported first).
 * No counterpart in the reference, whose launcher has no error reporting.
 * Returns ATTN_OK, or ATTN_ERR_LAUNCH if the synchronisation itself failed.
 */
ATTN_API int attn_get_status(cudaStream_t stream, int* status);

/*
 * Sets the limit, in nanoseconds, of each pipeline wait inside the
 * tensor-core kernel for launches queued from now on (all devices); 0 restores
 * the default of 2 s.  The clock is checked each time the hardware's own
 * suspension of an mbarrier wait ends without the awaited arrival, so a
 * legitimate wait (microseconds) never expires whatever the limit, and a
 * lost arrival ends the wait after about the limit: the kernel then records
 * ATTN_ERR_WATCHDOG (read with attn_get_status), lets the copies and products
 * it already issued finish under the default limit, frees its tensor memory
 * and returns.  Returns the previous limit (0 = default).  No counterpart in
 * the reference, whose kernels have no bounded waits.
 */
ATTN_API unsigned long long attn_set_wait_limit_ns(unsigned long long ns);

/* Library version, major * 10000 + minor * 100 + patch.  No reference
 * counterpart; lets a binding check which build it loaded. */
ATTN_API int attn_library_version(void);

/*
 * ---------------------------------------------------------------------------
 * Paged key-value cache.  No counterpart in the reference, which has no cache.
 *
 * K and V of all sequences live in num_pages pages of page_size tokens:
 *   k, v  [num_pages, heads, page_size, D], element strides over (page, head,
 *         row) in k_strides / v_strides, the head dim contiguous.  Other
 *         orders (such as [num_pages, page_size, heads, D]) are given by their
 *         strides.
 * Token t of sequence b lies in page block_table[b * table_stride + t /
 * page_size], row t % page_size.  block_table (int32) has table_width entries
 * per sequence; those behind a sequence's last page do not matter.  seq_lens
 * (int32) holds the tokens of each sequence in the cache, the newest
 * included; a length of zero or less is an empty sequence (such as the unused
 * rows of a padded batch).  Both are device memory and read by the kernels
 * only, so captured calls follow lengths and pages that change.
 *
 * The kernels check what they read: an entry of the block table outside
 * [0, num_pages) is never followed (its tokens count as absent and are not
 * written), and tokens behind table_width * page_size are left out.  Either
 * is recorded and reported by attn_get_status as ATTN_ERR_BAD_PAGE.
 *
 * All entry points are asynchronous on `stream`, allocate nothing and return
 * ATTN_OK or an AttnStatus code; on an error of the arguments nothing was
 * launched.  A workspace is 16-byte aligned device memory of the size the
 * matching *_workspace_bytes call gives, needs no initialisation and is in use
 * until the call's work on `stream` is done; calls that may run at the same
 * time need one each.
 * Limits: 1 <= D <= 256, page_size >= 1, heads >= 1,
 * table_width * page_size <= 2^31 - 65537, and for launch_attn_decode as many
 * tiles of 64 tokens in B * heads sequences of that capacity as fit 31 bits.
 */
typedef struct AttnPagedCache {
  void* k;
  void* v;
  int num_pages, heads, page_size, D;
  AttnDType dtype;
  long long k_strides[3], v_strides[3]; /* elements over (page, head, row), >= 0 */
  const int* block_table;
  long long table_stride; /* entries from one sequence to the next */
  int table_width;
  const int* seq_lens;
  int B;
} AttnPagedCache;

/*
 * Attention of one new token per sequence: out = softmax(scale * q K^T) V over
 * the sequence's tokens.
 *   q    [B, Hq, D], element strides over (batch, head) in q_strides, null =
 *        contiguous; Hq a multiple of cache->heads, query heads
 *        [h * Hq / heads, (h + 1) * Hq / heads) read kv head h
 *   out  [B, Hq, D] contiguous, fully overwritten; zeros for a sequence with
 *        no token (one whose every score is -inf gives NaN, as the formula)
 *   pages  null, or int32 [B, heads, n_pages]: only the tokens of these logical
 *        pages (t / page_size) are attended to.  Entries that name no page of
 *        the sequence (such as -1) add nothing, one named twice counts twice.
 *   weights  null, or fp32 with strides weights_strides over (batch, head) and
 *        at least table_width * page_size contiguous values per (batch, head),
 *        no two of which share memory: weights[b, h, t] += the sum of the
 *        softmax weights of token t over the query heads of kv head h.  Not
 *        together with `pages` (ATTN_ERR_UNSUPPORTED).
 * Products are summed and the softmax is held in 32 bits; for fp16 and bf16
 * caches with 16-byte rows each softmax weight is rounded to the cache's type
 * before the product with V (half a step; fp16 weights below 2^-29 of the
 * largest by at most 2^-40 of that).
 * softmax_scale as in launch_attn_forward.  With weights the workspace holds
 * the scores, 4 * B * Hq * table_width * page_size bytes; without, it does not
 * grow with the lengths and may be empty (the pointer is then only checked).
 * `listed` tells the workspace call whether `pages` will be given, `weights`
 * whether weights will be.
 */
ATTN_API int attn_decode_workspace_bytes(const AttnPagedCache* cache, int Hq, bool listed, int n_pages, bool weights,
                                         size_t* bytes);
ATTN_API int launch_attn_decode(const AttnPagedCache* cache, const void* q, const long long* q_strides, void* out,
                                int Hq, float softmax_scale, const int* pages, int n_pages, float* weights,
                                const long long* weights_strides, void* workspace, size_t workspace_bytes,
                                cudaStream_t stream);

/*
 * Writes new tokens to the cache.
 *   k, v  [B, heads, S, D], element strides over (batch, head, token)
 *   new_lens  null (every sequence has S new tokens), or int32 [B] device
 *         memory: the first new_lens[b] of the S are new
 * seq_lens counts the new tokens: token s of the n new ones of sequence b goes
 * to position seq_lens[b] - n + s.  Positions below zero are left out, so a
 * sequence of length zero takes nothing.
 *   bounds  null, or the page bounds [num_pages, heads, 2, D] (see
 *         launch_kv_page_bounds), element strides over (page, head, min/max):
 *         the new keys are folded in; a page whose row 0 is new begins anew.
 * Two sequences of a call must not write to one page.
 */
ATTN_API int launch_kv_append(const AttnPagedCache* cache, const void* k, const long long* k_strides, const void* v,
                              const long long* v_strides, int S, const int* new_lens, void* bounds,
                              const long long* bounds_strides, cudaStream_t stream);

/*
 * Bounds of the pages of every sequence: bounds[page, h, 0, :] and
 * bounds[page, h, 1, :] are the elementwise minimum and maximum of the keys of
 * the sequence's tokens in the page (NaN where one is NaN), in the cache's
 * type.  Pages of no sequence are left as they are; a page that sequences
 * share should hold the same tokens of each (a full page of a common prefix),
 * otherwise it gets the bounds of one of them.  cache->v is not used.
 */
ATTN_API int launch_kv_page_bounds(const AttnPagedCache* cache, void* bounds, const long long* bounds_strides,
                                   cudaStream_t stream);

/*
 * Picks the pages of each (sequence, kv head) that may matter most to a new
 * token: pages int32 [B, heads, top] receives ascending logical pages, -1
 * behind them where the sequence has fewer than `top`.  The newest page is
 * always in; of the others those with the largest
 *   score = sum over the dims d of max[d] * p[d] + min[d] * m[d],
 * p and m being the sums of q's positive and negative parts over the query
 * heads of the kv head: the sum of max(q * min, q * max), an upper bound of the
 * summed scores of any token of the page.  A part of q that is zero adds
 * nothing, even beside an infinite bound; a bound that is NaN makes the score
 * NaN.  Ties go to the lower page, NaN counts as largest.  Sums are taken in 64
 * bits, since a score next to the border decides a page.  top >= 1; cache->k
 * and v are not used.
 */
ATTN_API int kv_select_pages_workspace_bytes(const AttnPagedCache* cache, size_t* bytes);
ATTN_API int launch_kv_select_pages(const AttnPagedCache* cache, const void* q, const long long* q_strides, int Hq,
                                    const void* bounds, const long long* bounds_strides, int top, int* pages,
                                    void* workspace, size_t workspace_bytes, cudaStream_t stream);

/*
 * Evicts tokens by accumulated attention weight: of each (sequence, kv head)
 * the last `recent` tokens are kept and, of the others, those with the largest
 * weights, `budget` in all (ties to the lower position, NaN counts as largest;
 * all of them when there are no more than budget).  The kept tokens are copied in
 * their order to positions 0, 1, ... of the pages that new_table (int32,
 * new_width entries per sequence, new_stride apart) names; heads keep different
 * tokens.  The old pages are left as they are, so pages shared with other
 * sequences stay valid; new pages must be distinct and none an old page of
 * a sequence of the call.
 *   weights      fp32, strides over (batch, head), as for launch_attn_decode
 *   new_weights  [B, heads, new_width * page_size] contiguous: the weights of
 *                the kept tokens, zeros behind them
 *   kept         int32 [B, heads, budget]: the old positions, -1 behind them
 *   new_lens     int32 [B]: min(seq_lens, budget)
 * 1 <= budget <= new_width * page_size, 0 <= recent <= budget.
 */
ATTN_API int launch_kv_evict(const AttnPagedCache* cache, const float* weights, const long long* weights_strides,
                             const int* new_table, long long new_stride, int new_width, int budget, int recent,
                             float* new_weights, int* kept, int* new_lens, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* ROCM_ATTN_B200_ATTN_KERNEL_H_ */
