/* q36_attn.h -- C ABI of the attention side of a layer on B200 (sm_100a): a paged
 * key/value cache held in 4 bits, its tables, its writer and reader, attention
 * over it, and the matrix product that leads back into the residual stream.
 *
 * This half of a layer is: append to the cache, attention, output projection,
 * residual add.  q36_attn_block runs that chain and leaves h where q36_moe_block
 * takes it up.
 *
 * The conventions are those of q36_moe.h: device pointers, launch-only (no host
 * synchronisation, no allocation, capturable in a CUDA graph), a stream per
 * call, a Q36_MOE_* status back.  The library keeps no state between calls;
 * calls that may run at the same time need a workspace each, and so do calls
 * that two host threads make at a time, on one stream too: a call is several
 * launches, which hand partial results over in it.  Pointers, and
 * the rows that strides lead to, must lie on 16 bytes where a 16-byte vector
 * is read or written: q, k, v, x, w, out, the cache and the workspace.
 *
 * Cache: n_blocks blocks of block_size tokens (16, 32, 64 or 128), for each
 * block and kv head one region of block_size * head_dim * 17/16 bytes
 * (head_dim 64, 128 or 256): K codes, V codes, K scales, V scales.  A value is
 * e2m1(code) * 2^(scale-127), one scale byte per 32 consecutive dims.
 *   K codes: token t, word j * (head_dim/32) + b of head_dim/8 words (4 bytes)
 *            holds dims 32b + 8j .. 32b + 8j + 7, low nibble first (j < 4)
 *   V codes: token pair t/2, group g of 8, token t%2: halfword b of head_dim/32
 *            holds dims 32b + 4g .. 32b + 4g + 3, low nibble first
 *   scales:  [token][head_dim/32], 1 .. 252 (what the writer makes)
 * The order inside a row is the one in which the lanes of a warp hold a tensor
 * core operand, so that attention reads a row with full-width loads.
 * A slot is block * block_size + offset; offsets into the cache are 64-bit. */
#ifndef Q36_ATTN_H
#define Q36_ATTN_H

#include "q36_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one block over all kv heads; 0 for a geometry that is not supported. */
uint64_t q36_kv_block_bytes(int block_size, int n_kv_head, int head_dim);

/* Tables of one step from the lengths of its requests.  Request b has kv_old[b]
 * tokens in the cache and brings q_len[b] new ones (0 allowed).  It keeps its
 * ceil(kv_old/block_size) blocks and takes what it lacks, in request order, from
 * free_blocks[*free_head ..n_free).
 *   block_table [n_seq][max_blocks]  new entries are written, others left alone
 *   cu_q [n_seq+1]   first row of each request; row cu_q[b]+i is its i-th new token
 *   kv_len [n_seq]   kv_old + q_len (may be kv_old itself)
 *   slots [T], positions [T]  per row: cache slot and position; -1 in the rows
 *                    behind the last request (so that a padded, replayed step
 *                    writes nothing there)
 *   *free_head_out   entries of the free list used so far (may be free_head itself)
 *   *status          0, or the sum of: 1 the free list is too short, 2 the table is
 *                    too narrow, 4 a negative length, 8 more rows than T
 * With kv_len or free_head_out in place one thread block does the work: as fast for
 * decoding steps, 30 to 40 us for prompts of 32,768 tokens together (4 otherwise).
 * A request that cannot be served takes no block: its kv_len is 0 (attention
 * gives zeros for its rows) and its slots are -1.  When the free list is too
 * short, the requests behind the first unserved one that need blocks are not
 * served either.  Block ids outside [0, n_blocks) give slot -1.
 * 1 <= n_seq <= 16384; T, n_free <= 2^29; n_blocks * block_size < 2^31;
 * max_blocks * block_size <= 2^30.  The outputs may not overlap the inputs but as said. */
int q36_kv_tables(const int *kv_old, const int *q_len, int n_seq, int block_size, int n_blocks, const int *free_blocks,
                  int n_free, const int *free_head, int *block_table, int max_blocks, int *cu_q, int *kv_len, int *slots,
                  int *positions, int T, int *free_head_out, int *status, void *stream);

/* Rows k, v [T][n_kv_head][head_dim] (f32, or bf16 when x_is_bf16; strides between
 * tokens in elements) into the cache at slots[T]; slots outside
 * [0, n_blocks*block_size) are skipped.  Per 32 elements: e = smallest exponent
 * with amax <= 6 * 2^e, kept in [-126, 125], scale byte e + 127, codes rounded to
 * nearest even.  NaN is stored as 0; an infinity is stored as 6 * 2^125.
 * No slot may appear twice in one call. */
int q36_kv_append(const void *k, const void *v, int x_is_bf16, int64_t k_stride, int64_t v_stride, const int *slots,
                  void *cache, int n_blocks, int block_size, int n_kv_head, int head_dim, int T, void *stream);
/* The rows at slots[T] back as values: k, v [T][n_kv_head][head_dim], contiguous;
 * zeros for a slot outside the cache. */
int q36_kv_read(const void *cache, int n_blocks, int block_size, int n_kv_head, int head_dim, const int *slots, void *k,
                void *v, int x_is_bf16, int T, void *stream);

/* Attention of q [T][n_head][head_dim] over the cache.  The rows of request b are
 * cu_q[b] .. cu_q[b+1], cu_q[0] = 0; with n = cu_q[b+1] - cu_q[b] its row i has position
 * p = kv_len[b] - n + i and sees the cached tokens j with p - window < j <= p
 * (window 0: all j <= p).  Query head h reads kv head h / (n_head / n_kv_head).
 * out [T][n_head][head_dim] has the type of q; lse (or NULL) [T][n_head] f32
 * receives the natural logarithm of the sum of exponentials.  A row that sees
 * nothing gets zeros and -infinity.  Rows behind cu_q[n_seq] are left as they
 * were.  kv_len beyond max_blocks * block_size is cut there; tokens in blocks
 * whose id is outside [0, n_blocks) are left out.
 * max_q: the largest number of new tokens of a request, as far as the host
 * knows it; it chooses kernels only, any value >= 1 gives right results.
 * n_head / n_kv_head <= 128, n_head <= 4096, 1 <= n_seq <= 16384, T * n_head <= 2^30.
 * f32 prompts run on the kernel for few rows: right at every length, 6 to 14 times bf16's time. */
uint64_t q36_kv_attention_workspace_bytes(int n_head, int n_kv_head, int head_dim, int max_q);
int q36_kv_attention(const void *q, int x_is_bf16, int64_t q_stride, const void *cache, int n_blocks, int block_size,
                     int n_head, int n_kv_head, int head_dim, const int *block_table, int max_blocks, const int *cu_q,
                     const int *kv_len, int n_seq, float scale, int window, void *out, int64_t out_stride, float *lse,
                     int T, int max_q, void *ws, uint64_t ws_bytes, void *stream);

/* At -infinity every activation but NONE gives its limit, zero; NaN passes.  SILU and GELU_TANH are good to
 * 2^-17 of their value, 2^-14 where that nears f32's smallest; GELU to 2^-20 in all below zero. */
#define Q36_ACT_NONE 0
#define Q36_ACT_RELU 1
#define Q36_ACT_SILU 2
#define Q36_ACT_GELU 3       /* x * Phi(x)                                     */
#define Q36_ACT_GELU_TANH 4  /* 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) */
/* y [T][N] = act(x W^T + bias) + residual: x bf16 [T][K], w bf16 [N][K]
 * contiguous, bias f32 [N] or NULL, residual [T][N] f32 or bf16 or NULL, y f32 or
 * bf16; strides between rows in elements.  Sums in f32, one rounding at the end.
 * residual may be y itself (same type and stride); y overlaps nothing else.  rows_used (or NULL): device
 * count of rows; rows of y from *rows_used on are left as they were.  K and
 * x_stride are multiples of 8; T, N, K <= 2^30. */
int q36_linear(const void *x, int64_t x_stride, const void *w, const float *bias, int act, const void *residual,
               int res_is_bf16, int64_t res_stride, void *y, int y_is_bf16, int64_t y_stride, int T, int N, int K,
               const int *rows_used, void *stream);

/* The attention half of a layer from projected, rotated q, k, v: append,
 * attention, then h [T][D] += attention W_o^T + bias_o, w_o bf16
 * [D][n_head*head_dim].  The attention output is rounded once to bf16 in between.
 * Rows of h behind cu_q[n_seq] are left as they were. */
uint64_t q36_attn_block_workspace_bytes(int T, int n_head, int n_kv_head, int head_dim, int max_q);
int q36_attn_block(const void *q, const void *k, const void *v, int x_is_bf16, int64_t q_stride, int64_t k_stride,
                   int64_t v_stride, const int *slots, void *cache, int n_blocks, int block_size, int n_head,
                   int n_kv_head, int head_dim, const int *block_table, int max_blocks, const int *cu_q,
                   const int *kv_len, int n_seq, float scale, int window, const void *w_o, const float *bias_o, float *h,
                   int D, int T, int max_q, void *ws, uint64_t ws_bytes, void *stream);

/* The long waits of the tensor core kernels (on a copy, on a product) are bounded.
 * Synchronises the stream and returns Q36_MOE_EDEVICE when one gave up on the
 * current device since the last call of this function (results written since then
 * are not to be used; which one: q36_moe_last_cuda_error()), else 0.  One check
 * covers every call before it, as q36_moe_ws_status does: the record is the device's,
 * and the check clears it, so let one thread of the process ask. */
int q36_attn_status(void *stream);
/* A 32-thread kernel that waits for what nobody completes, with a short limit, and
 * records that it gave up: lets a test see q36_attn_status report it. */
int q36_attn_selftest_wait_timeout(void *stream);

#ifdef __cplusplus
}
#endif
#endif
