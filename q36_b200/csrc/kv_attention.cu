// Attention over the paged 4-bit cache.
#include <math.h>

#include "attn_plan.cuh"

namespace q36 {

constexpr int JOIN_THREADS = 128;

// The join.  Row r of the span whose first piece CTA i had, if it had one of a cut span: piece p counts l_p 2^(m_p - m); a piece that
// saw nothing has no row to read.
__device__ __forceinline__ const float *join_slot(const float *part, const AttnPart &d, int cta, int p, int stride) {
    return part + (size_t)(p == 0 ? d.slot : 2 * (cta + p)) * stride;
}

// Which CTAs had the first piece of a cut span (n of them), into list[].  Every block finds out for itself and takes its share of (span,
// rows): a block per CTA and row, most of which leave at once, took 7 us at 296 x 16 and 12 at 148 x 64.
__device__ __forceinline__ int join_list(const AttnPart *desc, int grid, int *list) {
    __shared__ int cnt[JOIN_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int n = 0;
    for (int i0 = 0; i0 < grid; i0 += JOIN_THREADS) {
        const int i = i0 + threadIdx.x;
        const bool cut = i < grid && desc[i].parts > 0;
        const unsigned in = __ballot_sync(0xffffffffu, cut);
        if (lane == 0) cnt[warp] = __popc(in);
        __syncthreads();
        int at = n;
#pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; w++) {
            if (w < warp) at += cnt[w];
            n += cnt[w];
        }
        if (cut) list[at + __popc(in & ((1u << lane) - 1))] = i;      // in order: the blocks have to agree
        __syncthreads();
    }
    return n;
}

// Spans in up to hundreds of pieces (few rows): block (i, r), the pieces over its threads.
template <int DH>
__global__ void __launch_bounds__(JOIN_THREADS)
k_attn_join(AttnArgs a, int tile_rows, int grid, const AttnPart *__restrict__ desc, const float *__restrict__ part) {
    Q36_GDS();
    constexpr int C4 = DH / 4, LANES = JOIN_THREADS / C4;      // threads over the dims, and pieces in parallel
    extern __shared__ float w[];                               // one weight per piece, then the list
    __shared__ float red[2][JOIN_THREADS / 32];
    __shared__ float4 acc[LANES][C4];
    int *list = reinterpret_cast<int *>(w + grid);
    const int n = join_list(desc, grid, list), tid = threadIdx.x;
    for (int item = blockIdx.x; item < n * tile_rows; item += gridDim.x) {
        const int cta = list[item / tile_rows], r = item % tile_rows;
        const AttnPart d = desc[cta];
        if (r >= d.rows) continue;
        const int stride = attn_part_floats(tile_rows, DH);
        float m = -3.0e38f;
        for (int p = tid; p < d.parts; p += JOIN_THREADS) m = fmaxf(m, join_slot(part, d, cta, p, stride)[2 * r]);
        m = warp_max(m);
        if ((tid & 31) == 0) red[0][tid >> 5] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        float l = 0.f;
        for (int p = tid; p < d.parts; p += JOIN_THREADS) {
            const float *s = join_slot(part, d, cta, p, stride);
            l += w[p] = s[2 * r + 1] * exp2f(s[2 * r] - m);
        }
        l = warp_sum(l);
        if ((tid & 31) == 0) red[1][tid >> 5] = l;
        __syncthreads();
        l = red[1][0] + red[1][1] + red[1][2] + red[1][3];
        const int c = tid % C4, lane = tid / C4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int p = lane; p < d.parts; p += LANES) {
            const float f = w[p];
            if (f == 0.f) continue;
            const float4 v = *reinterpret_cast<const float4 *>(join_slot(part, d, cta, p, stride) + 2 * tile_rows + r * DH + 4 * c);
            o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
        }
        acc[lane][c] = o;
        __syncthreads();
        if (lane == 0) {
#pragma unroll
            for (int i = 1; i < LANES; i++) { const float4 v = acc[i][c]; o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w; }
            const float f = l == 0.f ? 0.f : 1.f / l;
            attn_store(a, d.t0, d.n, d.hk, d.row0 + r, 4 * c, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
            if (c == 0) attn_store_lse(a, d.t0, d.n, d.hk, d.row0 + r, m, l);
        }
        __syncthreads();
    }
}

// Many rows, few pieces: a warp per row.
template <int DH>
__global__ void __launch_bounds__(JOIN_THREADS)
k_attn_join_rows(AttnArgs a, int tile_rows, int grid, const AttnPart *__restrict__ desc, const float *__restrict__ part) {
    Q36_GDS();
    constexpr int N4 = (DH + 127) / 128;      // 16-byte pieces of a row per lane
    extern __shared__ int list[];
    constexpr int WARPS = JOIN_THREADS / 32;
    const int n = join_list(desc, grid, list), lane = threadIdx.x & 31, groups = tile_rows / WARPS;
    for (int item = blockIdx.x; item < n * groups; item += gridDim.x) {
        const int cta = list[item / groups], r = item % groups * WARPS + (threadIdx.x >> 5);
        const AttnPart d = desc[cta];
        if (r >= d.rows) continue;
        const int stride = attn_part_floats(tile_rows, DH);
        float m = -3.0e38f;
        for (int p = lane; p < d.parts; p += 32) m = fmaxf(m, join_slot(part, d, cta, p, stride)[2 * r]);
        m = warp_max(m);
        float l = 0.f;
        float4 o[N4];
#pragma unroll
        for (int k = 0; k < N4; k++) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p0 = 0; p0 < d.parts; p0 += 32) {
            float mine = 0.f;
            if (p0 + lane < d.parts) {
                const float *s = join_slot(part, d, cta, p0 + lane, stride);
                mine = s[2 * r + 1] * exp2f(s[2 * r] - m);
            }
            l += warp_sum(mine);
#pragma unroll 4
            for (int p = 0; p < min(32, d.parts - p0); p++) {
                const float f = __shfl_sync(0xffffffffu, mine, p);
                if (f == 0.f) continue;
                const float4 *s = reinterpret_cast<const float4 *>(join_slot(part, d, cta, p0 + p, stride) + 2 * tile_rows + r * DH);
#pragma unroll
                for (int k = 0; k < N4; k++) {
                    if (DH < 128 && lane >= DH / 4) continue;
                    const float4 v = s[32 * k + lane];
                    o[k].x = fmaf(f, v.x, o[k].x); o[k].y = fmaf(f, v.y, o[k].y); o[k].z = fmaf(f, v.z, o[k].z); o[k].w = fmaf(f, v.w, o[k].w);
                }
            }
        }
        const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int k = 0; k < N4; k++) {
            if (DH < 128 && lane >= DH / 4) continue;
            attn_store(a, d.t0, d.n, d.hk, d.row0 + r, 4 * (32 * k + lane), make_float4(o[k].x * f, o[k].y * f, o[k].z * f, o[k].w * f));
        }
        if (lane == 0) attn_store_lse(a, d.t0, d.n, d.hk, d.row0 + r, m, l);
    }
}

int launch_attn_join(const AttnArgs &a, int tile_rows, int grid, const AttnPart *desc, const float *part, cudaStream_t st) {
    const dim3 blocks((tile_rows > 16 ? 14 : 8) * sm_count()), threads(JOIN_THREADS);
    if (tile_rows > 16) {
        if (a.kv.Dh == 64) launch_k(k_attn_join_rows<64>, blocks, threads, grid * 4, st, a, tile_rows, grid, desc, part);
        else if (a.kv.Dh == 128) launch_k(k_attn_join_rows<128>, blocks, threads, grid * 4, st, a, tile_rows, grid, desc, part);
        else launch_k(k_attn_join_rows<256>, blocks, threads, grid * 4, st, a, tile_rows, grid, desc, part);
        return check_launch();
    }
    if (a.kv.Dh == 64) launch_k(k_attn_join<64>, blocks, threads, grid * 8, st, a, tile_rows, grid, desc, part);
    else if (a.kv.Dh == 128) launch_k(k_attn_join<128>, blocks, threads, grid * 8, st, a, tile_rows, grid, desc, part);
    else launch_k(k_attn_join<256>, blocks, threads, grid * 8, st, a, tile_rows, grid, desc, part);
    return check_launch();
}

static int rows_of(int Hq, int Hkv, int max_q) { return (int)min((long)(Hq / Hkv) * max_q, (long)INT32_MAX); }

uint64_t attention_ws_bytes(int Hq, int Hkv, int Dh, int max_q) {
    const int rows = rows_of(Hq, Hkv, max_q);
    const uint64_t few = decode_ws_bytes(Dh, rows);
    return rows < LONG_ROWS ? few : max(few, prefill_ws_bytes(Dh));      // (one after the other on the stream: the same memory)
}

int launch_attention(const AttnArgs &a, int max_q, void *ws, uint64_t ws_bytes, cudaStream_t st) {
    (void)ws_bytes;
    const int rows = rows_of(a.Hq, a.kv.Hkv, max_q);
    if (!a.q_bf16 || rows < LONG_ROWS) return launch_decode(a, rows, 1, ws, st);
    int rc;
    if ((rc = launch_decode(a, rows, 0, ws, st))) return rc;
    return launch_prefill(a, ws, st);
}

}  // namespace q36

using namespace q36;

static bool off16(const void *p) { return ((uintptr_t)p & 15) != 0; }

// Checks what the attention entries have in common and fills in their arguments.
static int attn_args(AttnArgs &a, const void *q, int x_is_bf16, int64_t q_stride, const void *cache, int n_blocks, int block_size, int n_head,
                     int n_kv_head, int head_dim, const int *block_table, int max_blocks, const int *cu_q, const int *kv_len, int n_seq,
                     float scale, int window, int T, int max_q) {
    if ((T && !q) || !cache || !block_table || !cu_q || !kv_len || !kv_geom_ok(block_size, n_kv_head, head_dim)) return Q36_MOE_EINVAL;
    if (n_head <= 0 || n_head % n_kv_head || n_head / n_kv_head > 128 || n_head > 4096 || n_seq <= 0 || n_seq > 16384 || T < 0 || max_q <= 0 || window < 0) return Q36_MOE_EINVAL;
    if (n_blocks <= 0 || (int64_t)n_blocks * block_size > INT32_MAX || max_blocks <= 0 || (int64_t)max_blocks * block_size > (1 << 30)) return Q36_MOE_EINVAL;
    if (!isfinite(scale) || q_stride < (int64_t)n_head * head_dim || q_stride % (x_is_bf16 ? 8 : 4) || off16(q) || off16(cache)) return Q36_MOE_EINVAL;
    if ((int64_t)T * n_head > INT32_MAX) return Q36_MOE_EINVAL;
    a.kv = KvGeom{(const uint8_t *)cache, n_blocks, block_size, log2_of(block_size), n_kv_head, head_dim};
    a.q = q;
    a.q_stride = q_stride;
    a.table = block_table;
    a.cu_q = cu_q;
    a.kv_len = kv_len;
    a.max_blocks = max_blocks;
    a.B = n_seq;
    a.T = T;
    a.Hq = n_head;
    a.G = n_head / n_kv_head;
    a.window = window;
    a.scale2 = scale * 1.4426950408889634f;
    a.q_bf16 = x_is_bf16 != 0;
    return Q36_MOE_OK;
}

extern "C" {

uint64_t q36_kv_attention_workspace_bytes(int n_head, int n_kv_head, int head_dim, int max_q) {
    if (!kv_geom_ok(16, n_kv_head, head_dim) || n_head <= 0 || n_head % n_kv_head || n_head / n_kv_head > 128 || n_head > 4096 || max_q <= 0) return 0;
    return attention_ws_bytes(n_head, n_kv_head, head_dim, max_q);
}

int q36_kv_attention(const void *q, int x_is_bf16, int64_t q_stride, const void *cache, int n_blocks, int block_size, int n_head,
                     int n_kv_head, int head_dim, const int *block_table, int max_blocks, const int *cu_q, const int *kv_len, int n_seq,
                     float scale, int window, void *out, int64_t out_stride, float *lse, int T, int max_q, void *ws, uint64_t ws_bytes,
                     void *stream) {
    AttnArgs a;
    const int rc = attn_args(a, q, x_is_bf16, q_stride, cache, n_blocks, block_size, n_head, n_kv_head, head_dim, block_table, max_blocks, cu_q,
                             kv_len, n_seq, scale, window, T, max_q);
    if (rc) return rc;
    if ((T && !out) || off16(out) || out_stride < (int64_t)n_head * head_dim || out_stride % (x_is_bf16 ? 8 : 4) || !ws || off16(ws)) return Q36_MOE_EINVAL;
    if (ws_bytes < attention_ws_bytes(n_head, n_kv_head, head_dim, max_q)) return Q36_MOE_ENOSPACE;
    if (T == 0) return Q36_MOE_OK;
    a.out = out;
    a.o_stride = out_stride;
    a.o_bf16 = a.q_bf16;
    a.lse = lse;
    return launch_attention(a, max_q, ws, ws_bytes, (cudaStream_t)stream);
}

uint64_t q36_attn_block_workspace_bytes(int T, int n_head, int n_kv_head, int head_dim, int max_q) {
    const uint64_t at = q36_kv_attention_workspace_bytes(n_head, n_kv_head, head_dim, max_q);
    if (!at || T < 0) return 0;
    return ((at + 255) & ~(uint64_t)255) + (uint64_t)T * n_head * head_dim * 2;
}

int q36_attn_block(const void *q, const void *k, const void *v, int x_is_bf16, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                   const int *slots, void *cache, int n_blocks, int block_size, int n_head, int n_kv_head, int head_dim,
                   const int *block_table, int max_blocks, const int *cu_q, const int *kv_len, int n_seq, float scale, int window,
                   const void *w_o, const float *bias_o, float *h, int D, int T, int max_q, void *ws, uint64_t ws_bytes, void *stream) {
    AttnArgs a;
    int rc = attn_args(a, q, x_is_bf16, q_stride, cache, n_blocks, block_size, n_head, n_kv_head, head_dim, block_table, max_blocks, cu_q, kv_len,
                       n_seq, scale, window, T, max_q);
    if (rc) return rc;
    const int64_t row = (int64_t)n_kv_head * head_dim, vec = x_is_bf16 ? 8 : 4;
    if ((T && (!k || !v || !slots || !h)) || !w_o || !ws || D <= 0 || off16(k) || off16(v) || off16(w_o) || off16(ws)) return Q36_MOE_EINVAL;
    if (k_stride < row || v_stride < row || k_stride % vec || v_stride % vec) return Q36_MOE_EINVAL;
    if (ws_bytes < q36_attn_block_workspace_bytes(T, n_head, n_kv_head, head_dim, max_q)) return Q36_MOE_ENOSPACE;
    if (T == 0) return Q36_MOE_OK;
    const cudaStream_t st = (cudaStream_t)stream;
    const uint64_t at = (attention_ws_bytes(n_head, n_kv_head, head_dim, max_q) + 255) & ~(uint64_t)255;
    const int K = n_head * head_dim;
    a.out = (uint8_t *)ws + at;
    a.o_stride = K;
    a.o_bf16 = 1;
    a.lse = nullptr;
    if ((rc = launch_kv_append(k, v, x_is_bf16, k_stride, v_stride, slots, a.kv, T, st))) return rc;
    if ((rc = launch_attention(a, max_q, ws, at, st))) return rc;
    return launch_linear(a.out, K, w_o, bias_o, Q36_ACT_NONE, h, 0, D, h, 0, D, T, D, K, cu_q + n_seq, st);
}

}  // extern "C"
