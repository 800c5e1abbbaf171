// Attention over the paged 4-bit cache.
#include <math.h>

#include "attn_plan.cuh"

namespace q36 {

constexpr int JOIN_THREADS = 128, JOIN_PIECES = 256;
constexpr int JOIN_ID = 0xffff, JOIN_LONG = 0x10000;      // list entries: the CTA, and whether its span is in more than 32 pieces

// Which CTAs had the first piece of a cut span (n of them), into list[].  Every block finds out for itself and takes its share of (span,
// rows): a block per CTA and row, most of which leave at once, took 7 us at 296 x 16 and 12 at 148 x 64.
template <int THREADS>
__device__ __forceinline__ int join_list(const AttnPart *desc, int grid, int *list) {
    constexpr int PER = (DEC_MAX_OCC * 160 + THREADS - 1) / THREADS;      // all of them on their way at once, on up to 160 SMs
    __shared__ int cnt[PER][THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int n = 0;
    for (int base = 0; base < grid; base += PER * THREADS) {
        int parts[PER];
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int i = base + k * THREADS + threadIdx.x;
            parts[k] = i < grid ? desc[i].parts : 0;
        }
        unsigned in[PER];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; k++) {
            in[k] = __ballot_sync(0xffffffffu, parts[k] > 0);
            if (lane == 0) cnt[k][warp] = __popc(in[k]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int at = n;
#pragma unroll
            for (int w = 0; w < THREADS / 32; w++) {
                if (w < warp) at += cnt[k][w];
                n += cnt[k][w];
            }
            if (parts[k] > 0) list[at + __popc(in[k] & ((1u << lane) - 1))] = (base + k * THREADS + threadIdx.x) | (parts[k] > 32 ? JOIN_LONG : 0);      // in order: the blocks have to agree
        }
    }
    __syncthreads();
    return n;
}

// The join.  Row r of the span whose first piece CTA i had: piece p counts l_p 2^(m_p - m) / l, divided by the sum before it meets the row,
// so that rows as large as f32 holds stay finite; a piece that saw nothing has no row to read.
__device__ __forceinline__ const float *join_slot(const float *part, const AttnPart &d, int cta, int p, int stride) {
    return part + (size_t)(p == 0 ? d.slot : 2 * (cta + p)) * stride;
}

// The weights of a row's pieces, lane p has those of pieces p, p + 32, ..; l: what they were divided by, m: the largest one.
template <bool KEEP>
__device__ __forceinline__ void join_weights(const AttnPart &d, const float *part, int cta, int stride, int r, int lane, float *w, float &first, float &m, float &l) {
    m = -3.0e38f;
    l = first = 0.f;
    for (int p = lane; p < d.parts; p += 32) m = fmaxf(m, join_slot(part, d, cta, p, stride)[2 * r]);
    m = warp_max(m);
    for (int p = lane; p < d.parts; p += 32) {
        const float2 ml = *reinterpret_cast<const float2 *>(join_slot(part, d, cta, p, stride) + 2 * r);
        const float f = ml.y * exp2f(ml.x - m);
        if (p == lane) first = f;
        l += f;
        if (KEEP) w[p] = f;
    }
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    first *= inv;
    if (KEEP)
        for (int p = lane; p < d.parts; p += 32) w[p] *= inv;
}
// a lane's share of the weighted rows of pieces p0, p0 + step, ..: several on their way at a time
template <int DH, typename W>
__device__ __forceinline__ void join_rows(const AttnPart &d, const float *part, int cta, int stride, int tile_rows, int r, int lane, int p0, int step, W weight,
                                          float4 (&o)[(DH + 127) / 128]) {
    constexpr int N4 = (DH + 127) / 128, AT_ONCE = 8 / N4;
#pragma unroll
    for (int k = 0; k < N4; k++) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (; p0 < d.parts; p0 += step * AT_ONCE) {
        float4 v[AT_ONCE][N4];
#pragma unroll
        for (int x = 0; x < AT_ONCE; x++) {
            const float4 *s = reinterpret_cast<const float4 *>(join_slot(part, d, cta, min(p0 + x * step, d.parts - 1), stride) + 2 * tile_rows + r * DH);
#pragma unroll
            for (int k = 0; k < N4; k++) v[x][k] = s[32 * k + (DH < 128 ? lane % (DH / 4) : lane)];
        }
#pragma unroll
        for (int x = 0; x < AT_ONCE; x++) {
            const float f = weight(p0 + x * step);      // (0 behind the last piece)
            if (f == 0.f) continue;
#pragma unroll
            for (int k = 0; k < N4; k++) {
                o[k].x = fmaf(f, v[x][k].x, o[k].x); o[k].y = fmaf(f, v[x][k].y, o[k].y); o[k].z = fmaf(f, v[x][k].z, o[k].z); o[k].w = fmaf(f, v[x][k].w, o[k].w);
            }
        }
    }
}
template <int DH>
__device__ __forceinline__ void join_store(const AttnArgs &a, const AttnPart &d, int r, int lane, int k, float4 o) {
    if (DH < 128 && lane >= DH / 4) return;
    attn_store(a, d.t0, d.n, d.hk, d.row0 + r, 4 * (32 * k + lane), o);
}

// Tiles of 8 or 16 rows.  Spans in up to 32 pieces: a block per span, a warp per row.  Longer ones: a block per row, its warps share
// the pieces.  The latency of four reads in a row bounds it (list, piece, weights, rows): 7 to 8 us cold, 4 to 5 behind the kernel before it.
constexpr int JOIN_WIDE = 256;
template <int DH>
__global__ void __launch_bounds__(JOIN_WIDE)
k_attn_join(AttnArgs a, int tile_rows, int grid, const AttnPart *desc, const float *part) {
    Q36_GDS();
    constexpr int N4 = (DH + 127) / 128, WARPS = JOIN_WIDE / 32;      // 16-byte pieces of a row per lane
    extern __shared__ float w[];                                      // one weight per piece, then the list
    __shared__ float4 acc[WARPS][N4][32];
    int *list = reinterpret_cast<int *>(w + grid);
    const int n = join_list<JOIN_WIDE>(desc, grid, list), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int stride = attn_part_floats(tile_rows, DH);
    float m, l, first;
    float4 o[N4];
    for (int item = blockIdx.x; item < n * tile_rows; item += gridDim.x) {
        const int cta = list[item % n] & JOIN_ID, row = item / n;
        if (!(list[item % n] & JOIN_LONG)) {
            if (row) continue;
            const AttnPart d = desc[cta];
            for (int r = warp; r < d.rows; r += WARPS) {
                join_weights<false>(d, part, cta, stride, r, lane, nullptr, first, m, l);
                join_rows<DH>(d, part, cta, stride, tile_rows, r, lane, 0, 1, [&](int p) { return p < 32 ? __shfl_sync(0xffffffffu, first, p) : 0.f; }, o);
#pragma unroll
                for (int k = 0; k < N4; k++) join_store<DH>(a, d, r, lane, k, o[k]);
                if (lane == 0) attn_store_lse(a, d.t0, d.n, d.hk, d.row0 + r, m, l);
            }
            continue;
        }
        const AttnPart d = desc[cta];
        if (row >= d.rows) continue;
        if (warp == 0) join_weights<true>(d, part, cta, stride, row, lane, w, first, m, l);
        else join_weights<false>(d, part, cta, stride, row, lane, nullptr, first, m, l);
        __syncthreads();
        join_rows<DH>(d, part, cta, stride, tile_rows, row, lane, warp, WARPS, [&](int p) { return p < d.parts ? w[p] : 0.f; }, o);
#pragma unroll
        for (int k = 0; k < N4; k++) acc[warp][k][lane] = o[k];
        __syncthreads();
        if (warp < N4) {
            float4 t = acc[0][warp][lane];
#pragma unroll
            for (int i = 1; i < WARPS; i++) { const float4 v = acc[i][warp][lane]; t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w; }
            join_store<DH>(a, d, row, lane, warp, t);
        }
        if (threadIdx.x == 0) attn_store_lse(a, d.t0, d.n, d.hk, d.row0 + row, m, l);
        __syncthreads();
    }
}

// Tiles of 128 or 256 rows, mostly in two or three pieces: a warp per four rows, so that the loads of all four are on their way at once
// (three chunks of up to 777 tokens on up to 6000 beside 37 single tokens: 14.5 us, 25 with a row at a time).
template <int DH>
__global__ void __launch_bounds__(JOIN_THREADS)
k_attn_join_rows(AttnArgs a, int tile_rows, int grid, const AttnPart *desc, const float *part) {
    Q36_GDS();
    constexpr int N4 = (DH + 127) / 128, WARPS = JOIN_THREADS / 32, RB = 4;
    extern __shared__ int list[];
    __shared__ float4 w[WARPS][JOIN_PIECES];      // four rows' weights of each piece (a tile kernel has one CTA per SM)
    const int n = join_list<JOIN_THREADS>(desc, grid, list), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = tile_rows / (WARPS * RB);
    const int stride = attn_part_floats(tile_rows, DH);
    for (int item = blockIdx.x; item < n * groups; item += gridDim.x) {
        const int cta = list[item / groups] & JOIN_ID, r = (item % groups * WARPS + warp) * RB;
        const AttnPart d = desc[cta];
        if (r >= d.rows) continue;
        float m[RB], l[RB] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < RB; i++) m[i] = -3.0e38f;
        // (m, l) of the four rows lie side by side
        for (int p = lane; p < d.parts; p += 32) {
            const float4 *s = reinterpret_cast<const float4 *>(join_slot(part, d, cta, p, stride) + 2 * r);
            const float4 x = s[0], y = s[1];
            m[0] = fmaxf(m[0], x.x); m[1] = fmaxf(m[1], x.z); m[2] = fmaxf(m[2], y.x); m[3] = fmaxf(m[3], y.z);
        }
#pragma unroll
        for (int i = 0; i < RB; i++) m[i] = warp_max(m[i]);
        for (int p = lane; p < d.parts; p += 32) {
            const float4 *s = reinterpret_cast<const float4 *>(join_slot(part, d, cta, p, stride) + 2 * r);
            const float4 x = s[0], y = s[1];
            const float4 f = make_float4(x.y * exp2f(x.x - m[0]), x.w * exp2f(x.z - m[1]), y.y * exp2f(y.x - m[2]), y.w * exp2f(y.z - m[3]));
            w[warp][p] = f;
            l[0] += f.x; l[1] += f.y; l[2] += f.z; l[3] += f.w;
        }
#pragma unroll
        for (int i = 0; i < RB; i++) l[i] = warp_sum(l[i]);
        {
            float inv[RB];
#pragma unroll
            for (int i = 0; i < RB; i++) inv[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
            for (int p = lane; p < d.parts; p += 32) {
                const float4 f = w[warp][p];
                w[warp][p] = make_float4(f.x * inv[0], f.y * inv[1], f.z * inv[2], f.w * inv[3]);
            }
        }
        __syncwarp();
        float4 o[RB][N4];
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int k = 0; k < N4; k++) o[i][k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int p = 0; p < d.parts; p++) {
            const float4 f4 = w[warp][p];
            const float f[RB] = {f4.x, f4.y, f4.z, f4.w};
            float4 v[RB][N4];
#pragma unroll
            for (int i = 0; i < RB; i++) {
                const float4 *s = reinterpret_cast<const float4 *>(join_slot(part, d, cta, p, stride) + 2 * tile_rows + (r + i) * DH);
#pragma unroll
                for (int k = 0; k < N4; k++) v[i][k] = s[32 * k + (DH < 128 ? lane % (DH / 4) : lane)];
            }
#pragma unroll
            for (int i = 0; i < RB; i++) {
                if (f[i] == 0.f) continue;      // (a piece that saw nothing has no row: what was read is not used)
#pragma unroll
                for (int k = 0; k < N4; k++) {
                    o[i][k].x = fmaf(f[i], v[i][k].x, o[i][k].x); o[i][k].y = fmaf(f[i], v[i][k].y, o[i][k].y);
                    o[i][k].z = fmaf(f[i], v[i][k].z, o[i][k].z); o[i][k].w = fmaf(f[i], v[i][k].w, o[i][k].w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RB; i++) {
            if (r + i >= d.rows) break;
#pragma unroll
            for (int k = 0; k < N4; k++) join_store<DH>(a, d, r + i, lane, k, o[i][k]);
            if (lane == 0) attn_store_lse(a, d.t0, d.n, d.hk, d.row0 + r + i, m[i], l[i]);
        }
        __syncwarp();
    }
}

int launch_attn_join(const AttnArgs &a, int tile_rows, int grid, const AttnPart *desc, const float *part, cudaStream_t st) {
    if (tile_rows > 16) {
        const dim3 blocks(8 * sm_count()), threads(JOIN_THREADS);
        if (a.kv.Dh == 64) launch_k(k_attn_join_rows<64>, blocks, threads, grid * 4, st, a, tile_rows, grid, desc, part);
        else if (a.kv.Dh == 128) launch_k(k_attn_join_rows<128>, blocks, threads, grid * 4, st, a, tile_rows, grid, desc, part);
        else launch_k(k_attn_join_rows<256>, blocks, threads, grid * 4, st, a, tile_rows, grid, desc, part);
        return check_launch();
    }
    const dim3 blocks(6 * sm_count()), threads(JOIN_WIDE);
    if (a.kv.Dh == 64) launch_k(k_attn_join<64>, blocks, threads, grid * 8, st, a, tile_rows, grid, desc, part);
    else if (a.kv.Dh == 128) launch_k(k_attn_join<128>, blocks, threads, grid * 8, st, a, tile_rows, grid, desc, part);
    else launch_k(k_attn_join<256>, blocks, threads, grid * 8, st, a, tile_rows, grid, desc, part);
    return check_launch();
}

static int rows_of(int Hq, int Hkv, int max_q) { return (int)min((long)(Hq / Hkv) * max_q, (long)INT32_MAX); }

uint64_t attention_ws_bytes(int Hq, int Hkv, int Dh, int max_q) {
    const int rows = rows_of(Hq, Hkv, max_q);
    const uint64_t few = decode_ws_bytes(Dh);
    return rows < LONG_ROWS ? few : max(few, prefill_ws_bytes(Dh));      // (one after the other on the stream: the same memory)
}

int launch_attention(AttnArgs a, int max_q, void *ws, cudaStream_t st) {
    const long long all = (long long)a.T * a.G;
    const int rows = (int)min((long long)rows_of(a.Hq, a.kv.Hkv, max_q), all);      // of one request, at most
    a.long_work = all <= LONG_FEW_ROWS ? LONG_WORK_FEW : LONG_WORK;
    const bool any = a.q_bf16 && rows >= LONG_ROWS && rows * ((long long)a.max_blocks << a.kv.log_bs) >= a.long_work;
    if (!any) return launch_decode(a, rows, 1, ws, st);
    int rc;
    if ((rc = launch_decode(a, rows, 0, ws, st))) return rc;
    return launch_prefill(a, ws, st);
}

}  // namespace q36

using namespace q36;

static bool off16(const void *p) { return ((uintptr_t)p & 15) != 0; }
static bool off4(const void *p) { return ((uintptr_t)p & 3) != 0; }

// Checks what the attention entries have in common and fills in their arguments.
static int attn_args(AttnArgs &a, const void *q, int x_is_bf16, int64_t q_stride, const void *cache, int n_blocks, int block_size, int n_head,
                     int n_kv_head, int head_dim, const int *block_table, int max_blocks, const int *cu_q, const int *kv_len, int n_seq,
                     float scale, int window, int T, int max_q) {
    if ((T && !q) || !cache || !block_table || !cu_q || !kv_len || !kv_geom_ok(block_size, n_kv_head, head_dim)) return Q36_MOE_EINVAL;
    if (n_head <= 0 || n_head % n_kv_head || n_head / n_kv_head > 128 || n_head > 4096 || n_seq <= 0 || n_seq > 16384 || T < 0 || max_q <= 0 || window < 0 || T > (1 << 30) / n_head) return Q36_MOE_EINVAL;
    if (n_blocks <= 0 || (int64_t)n_blocks * block_size > INT32_MAX || max_blocks <= 0 || (int64_t)max_blocks * block_size > (1 << 30)) return Q36_MOE_EINVAL;
    if (!isfinite(scale * 1.4426950408889634f) || q_stride < (int64_t)n_head * head_dim || q_stride % (x_is_bf16 ? 8 : 4) || off16(q) || off16(cache)) return Q36_MOE_EINVAL;
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
    a.window = window < 1 << 30 ? window : 0;      // (no position is 2^30 or more: such a window hides nothing, and sums with it stay in 32 bits)
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
    if ((T && !out) || off16(out) || off4(lse) || out_stride < (int64_t)n_head * head_dim || out_stride % (x_is_bf16 ? 8 : 4) || !ws || off16(ws)) return Q36_MOE_EINVAL;
    if (ws_bytes < attention_ws_bytes(n_head, n_kv_head, head_dim, max_q)) return Q36_MOE_ENOSPACE;
    if (T == 0) return Q36_MOE_OK;
    a.out = out;
    a.o_stride = out_stride;
    a.o_bf16 = a.q_bf16;
    a.lse = lse;
    return launch_attention(a, max_q, ws, (cudaStream_t)stream);
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
    if ((T && (!k || !v || !slots || !h)) || !w_o || !ws || D <= 0 || D > (1 << 30) || off4(bias_o) || off4(h) || off16(k) || off16(v) || off16(w_o) || off16(ws)) return Q36_MOE_EINVAL;
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
    if ((rc = launch_attention(a, max_q, ws, st))) return rc;
    return launch_linear(a.out, K, w_o, bias_o, Q36_ACT_NONE, h, 0, D, h, 0, D, T, D, K, cu_q + n_seq, st);
}

int q36_attn_status(void *stream) {
    int where[2] = {0, 0}, rc;
    if (cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess) return check_launch();
    if ((rc = prefill_wait_status(&where[0])) || (rc = linear_wait_status(&where[1]))) return rc;
    if (!where[0] && !where[1]) return Q36_MOE_OK;
    last_cuda_error() = where[0] ? 300000 + where[0] : 400000 + where[1];
    return Q36_MOE_EDEVICE;
}
int q36_attn_selftest_wait_timeout(void *stream) { return launch_prefill_wait_timeout((cudaStream_t)stream); }

}  // extern "C"
