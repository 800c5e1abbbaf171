// Attention over the paged 4-bit cache.
#include <math.h>

#include "attn.cuh"

namespace q36 {

constexpr int SA_THREADS = 128;

// One block per (row, query head): each warp takes every fourth token and keeps its own running maximum and sum.
template <int DH>
__global__ void __launch_bounds__(SA_THREADS) k_attn_simple(AttnArgs a) {
    Q36_GDS();
    constexpr int NB = DH / 32;
    __shared__ float qs[DH], sm_o[4][DH], sm_m[4], sm_l[4];
    const int t = blockIdx.x, hq = blockIdx.y, hk = hq / a.G, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int b = -1, t0 = 0, n = 0, len = 0;
    for (int s = 0; s < a.B; s++) {
        seq_span(a, s, t0, n, len);
        if (t >= t0 && t < t0 + n) { b = s; break; }
    }
    if (b < 0) return;
    const int pos = len - n + (t - t0), lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    for (int d = tid; d < DH; d += SA_THREADS) {
        const size_t e = (size_t)t * a.q_stride + (size_t)hq * DH + d;
        qs[d] = (a.q_bf16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(a.q)[e] << 16) : reinterpret_cast<const float *>(a.q)[e]) * a.scale2;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[NB] = {};
    for (int j = lo + warp; j <= pos; j += 4) {
        const int blk = a.table[(size_t)b * a.max_blocks + (j >> a.kv.log_bs)];
        if (blk < 0 || blk >= a.kv.n_blocks) continue;
        const uint8_t *reg = a.kv.at(blk, hk);
        const int tok = j & (a.kv.bs - 1), half = a.kv.bs * DH / 2;
        float s = 0.f, v[NB];
#pragma unroll
        for (int c = 0; c < NB; c++) {     // lane = dim inside block c
            const uint8_t kb = reg[kv_k_off(tok, lane >> 3, c, DH) + ((lane & 7) >> 1)];
            const uint8_t vb = reg[half + kv_v_off(tok, lane >> 2, c, DH) + ((lane & 3) >> 1)];
            const float2 kf = e2m1x2_to_f32x2(kb), vf = e2m1x2_to_f32x2(vb);
            s += qs[32 * c + lane] * ((lane & 1) ? kf.y : kf.x) * ue8m0_to_f32(reg[2 * half + tok * NB + c]);
            v[c] = ((lane & 1) ? vf.y : vf.x) * ue8m0_to_f32(reg[2 * half + a.kv.bs * NB + tok * NB + c]);
        }
        s = warp_sum(s);
        const float mn = fmaxf(m, s), f = exp2f(m - mn), p = exp2f(s - mn);
        m = mn;
        l = l * f + p;
#pragma unroll
        for (int c = 0; c < NB; c++) o[c] = o[c] * f + p * v[c];
    }
#pragma unroll
    for (int c = 0; c < NB; c++) sm_o[warp][32 * c + lane] = o[c];
    if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
    __syncthreads();
    float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3])), L = 0.f, w[4];
    for (int i = 0; i < 4; i++) { w[i] = M == -INFINITY ? 0.f : exp2f(sm_m[i] - M); L += w[i] * sm_l[i]; }
    for (int d = tid; d < DH; d += SA_THREADS) {
        float acc = 0.f;
        for (int i = 0; i < 4; i++) acc += w[i] * sm_o[i][d];
        acc = L > 0.f ? acc / L : 0.f;
        const size_t e = (size_t)t * a.o_stride + (size_t)hq * DH + d;
        if (a.o_bf16) reinterpret_cast<__nv_bfloat16 *>(a.out)[e] = __float2bfloat16_rn(acc);
        else reinterpret_cast<float *>(a.out)[e] = acc;
    }
    if (a.lse && tid == 0) a.lse[(size_t)t * a.Hq + hq] = L > 0.f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

uint64_t attention_ws_bytes(int Hq, int Hkv, int Dh, int max_q) { (void)Hq; (void)Hkv; (void)Dh; (void)max_q; return 256; }

int launch_attention(const AttnArgs &a, int max_q, void *ws, uint64_t ws_bytes, cudaStream_t st) {
    (void)max_q; (void)ws; (void)ws_bytes;
    const dim3 grid(a.T, a.Hq), block(SA_THREADS);
    if (a.kv.Dh == 64) launch_k(k_attn_simple<64>, grid, block, 0, st, a);
    else if (a.kv.Dh == 128) launch_k(k_attn_simple<128>, grid, block, 0, st, a);
    else launch_k(k_attn_simple<256>, grid, block, 0, st, a);
    return check_launch();
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
