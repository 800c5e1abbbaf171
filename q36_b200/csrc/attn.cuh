// Cache geometry and launcher prototypes of the attention side of a layer (include/q36_attn.h).
#pragma once
#include "../../include/q36_attn.h"
#include "common.cuh"
#include "kernels.cuh"

namespace q36 {

// One (block, kv head) region: K codes | V codes | K scales | V scales.
struct KvGeom {
    const uint8_t *base;
    int n_blocks, bs, log_bs, Hkv, Dh;
    __host__ __device__ size_t region() const { return (size_t)bs * Dh * 17 / 16; }
    __host__ __device__ const uint8_t *at(int block, int head) const { return base + ((size_t)block * Hkv + head) * region(); }
};
__host__ __device__ __forceinline__ int kv_k_off(int t, int j, int b, int Dh) { return t * (Dh / 2) + j * (Dh / 8) + b * 4; }
__host__ __device__ __forceinline__ int kv_v_off(int t, int g, int b, int Dh) { return (t >> 1) * Dh + g * (Dh / 8) + (t & 1) * (Dh / 16) + b * 2; }

inline bool kv_geom_ok(int bs, int Hkv, int Dh) {
    return (bs == 16 || bs == 32 || bs == 64 || bs == 128) && (Dh == 64 || Dh == 128 || Dh == 256) && Hkv > 0 && Hkv <= 1024;
}
inline int log2_of(int v) { int n = 0; while ((1 << n) < v) n++; return n; }

// What an attention kernel is given.
struct AttnArgs {
    KvGeom kv;
    const void *q;
    long long q_stride, o_stride;    // elements between tokens
    const int *table, *cu_q, *kv_len;
    int max_blocks, B, T, Hq, G, window;
    float scale2;                    // scale * log2(e)
    void *out;
    float *lse;
    int q_bf16, o_bf16;
    int long_work;                   // rows times cached tokens from which on a request goes to the tile kernel
};
// First row, number of rows and cached length of request b, each kept inside what the host stated.
__device__ __forceinline__ void seq_span(const AttnArgs &a, int b, int &t0, int &n, int &len) {
    t0 = min(max(a.cu_q[b], 0), a.T);
    n = max(min(a.cu_q[b + 1], a.T) - t0, 0);
    len = min(max(a.kv_len[b], 0), a.max_blocks << a.kv.log_bs);
}

// One lane of a warp that runs as a whole, for the threads that issue to the tensor core.  Against `lane == 0` around the same loops: tiles
// of 64 x 128 over K = 2048 10.9 instead of 13.7 us, prompt of 8192 tokens 337 instead of 344.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// eight elements from element e on
__device__ __forceinline__ void load8(const void *p, size_t e, int bf16, float (&v)[8]) {
    if (bf16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + e);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
        const float4 *f = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + e);
        const float4 a = f[0], b = f[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}

int launch_attention(AttnArgs a, int max_q, void *ws, cudaStream_t st);
uint64_t attention_ws_bytes(int Hq, int Hkv, int Dh, int max_q);
int launch_kv_append(const void *k, const void *v, int bf16, long long ks, long long vs, const int *slots, KvGeom g, int T, cudaStream_t st);
int launch_linear(const void *x, long long xs, const void *w, const float *bias, int act, const void *res, int res_bf16, long long rs,
                  void *y, int y_bf16, long long ys, int T, int N, int K, const int *rows_used, cudaStream_t st);

}  // namespace q36
