// y = act(x W^T + bias) + residual, bf16 operands, f32 sums.
#include "attn.cuh"

namespace q36 {

// What happens to a sum between the matrix product and the store.
struct Epilogue {
    const float *bias;
    const void *res;
    void *y;
    long long rs, ys;
    int act, res_bf16, y_bf16;
};
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case Q36_ACT_RELU: return v < 0.f ? 0.f : v;
        case Q36_ACT_SILU: return v / (1.f + expf(-v));
        case Q36_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
        case Q36_ACT_GELU_TANH: return 0.5f * v * (1.f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}
__device__ __forceinline__ void finish(const Epilogue &e, int t, int n, float v) {
    if (e.bias) v += e.bias[n];
    v = activate(v, e.act);
    if (e.res) {
        const size_t i = (size_t)t * e.rs + n;
        v += e.res_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(e.res)[i]) : reinterpret_cast<const float *>(e.res)[i];
    }
    const size_t i = (size_t)t * e.ys + n;
    if (e.y_bf16) reinterpret_cast<__nv_bfloat16 *>(e.y)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float *>(e.y)[i] = v;
}

// 16 x 16 outputs per block, K in steps of 16.
__global__ void __launch_bounds__(256)
k_linear_simple(const uint16_t *__restrict__ x, long long xs, const uint16_t *__restrict__ w, Epilogue e, int T, int N, int K, const int *rows_used) {
    Q36_GDS();
    __shared__ float sx[16][17], sw[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
    const int rows = rows_used ? min(T, *rows_used) : T;
    float acc = 0.f;
    for (int k0 = 0; k0 < K; k0 += 16) {
        sx[ty][tx] = (t0 + ty < rows && k0 + tx < K) ? __uint_as_float((uint32_t)x[(size_t)(t0 + ty) * xs + k0 + tx] << 16) : 0.f;
        sw[ty][tx] = (n0 + ty < N && k0 + tx < K) ? __uint_as_float((uint32_t)w[(size_t)(n0 + ty) * K + k0 + tx] << 16) : 0.f;
        __syncthreads();
        for (int k = 0; k < 16; k++) acc = fmaf(sx[ty][k], sw[tx][k], acc);
        __syncthreads();
    }
    if (t0 + ty < rows && n0 + tx < N) finish(e, t0 + ty, n0 + tx, acc);
}

int launch_linear(const void *x, long long xs, const void *w, const float *bias, int act, const void *res, int res_bf16, long long rs,
                  void *y, int y_bf16, long long ys, int T, int N, int K, const int *rows_used, cudaStream_t st) {
    const Epilogue e{bias, res, y, rs, ys, act, res_bf16, y_bf16};
    launch_k(k_linear_simple, dim3((N + 15) / 16, (T + 15) / 16), dim3(256), 0, st, (const uint16_t *)x, xs, (const uint16_t *)w, e, T, N, K, rows_used);
    return check_launch();
}

}  // namespace q36

using namespace q36;

extern "C" int q36_linear(const void *x, int64_t x_stride, const void *w, const float *bias, int act, const void *residual, int res_is_bf16,
                          int64_t res_stride, void *y, int y_is_bf16, int64_t y_stride, int T, int N, int K, const int *rows_used,
                          void *stream) {
    if ((T && (!x || !y)) || !w || T < 0 || N <= 0 || K <= 0 || K % 8 || x_stride < K || x_stride % 8 || y_stride < N) return Q36_MOE_EINVAL;
    if (act < Q36_ACT_NONE || act > Q36_ACT_GELU_TANH || (residual && res_stride < N)) return Q36_MOE_EINVAL;
    if ((((uintptr_t)x | (uintptr_t)w) & 15) || ((uintptr_t)y & (y_is_bf16 ? 1 : 3))) return Q36_MOE_EINVAL;
    if (residual && ((uintptr_t)residual & (res_is_bf16 ? 1 : 3))) return Q36_MOE_EINVAL;
    if (residual && residual == y && (!res_is_bf16 != !y_is_bf16 || res_stride != y_stride)) return Q36_MOE_EINVAL;
    if (T == 0) return Q36_MOE_OK;
    return launch_linear(x, x_stride, w, bias, act, residual, res_is_bf16 != 0, res_stride, y, y_is_bf16 != 0, y_stride, T, N, K, rows_used,
                         (cudaStream_t)stream);
}
