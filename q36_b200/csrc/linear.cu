// y = act(x W^T + bias) + residual, bf16 operands, f32 sums.
#include "attn.cuh"
#include "tc_ptx.cuh"

namespace q36 {

// What happens to a sum between the matrix product and the store.
struct Epilogue {
    const float *bias;
    const void *res;
    void *y;
    long long rs, ys;
    int act, res_bf16, y_bf16;
};
// An activation over N sums (the choice outside the loop).  x times the logistic function of u, which has x's sign: with h = e^(-|u|/2) it is
// x / (1 + h^2), and below 0 that times h^2, one h after the other: nothing leaves f32's range on the way, and the result goes to zero where
// the function does, in relative precision.  -infinity counts as the lowest finite number, so that zero is its limit too.
// 0.5 (1 + tanh u/2) is the logistic function of u.
__device__ __forceinline__ float floor_finite(float x) {
    float r;
    asm("max.NaN.f32 %0, %1, 0fFF7FFFFF;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float times_logistic(float x, float u) {
    const float h = __expf(-0.5f * fabsf(u)), q = __fdividef(x, fmaf(h, h, 1.f));
    return u < 0.f ? q * h * h : q;
}
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
    switch (act) {
        case Q36_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = v[i] < 0.f ? 0.f : v[i];
            break;
        case Q36_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[i] = floor_finite(v[i]);
                v[i] = times_logistic(v[i], v[i]);
            }
            break;
        case Q36_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[i] = floor_finite(v[i]);
                v[i] = 0.5f * v[i] * (1.f + erff(v[i] * 0.70710678118654752f));
            }
            break;
        case Q36_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[i] = floor_finite(v[i]);
                v[i] = times_logistic(v[i], 1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]));
            }
            break;
        default: break;
    }
}
__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// Residual of column n, rows t .. t + N - 1 (those below `rows`), as it lies in memory: turned into f32 where it is added, so that
// nothing waits for the loads before.
template <int N>
__device__ __forceinline__ void load_res(const Epilogue &e, int n, int t, int rows, uint32_t (&r)[N]) {
    if (!e.res) return;
    if (e.res_bf16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(e.res) + (size_t)t * e.rs + n;
        if (t + N <= rows) {
#pragma unroll
            for (int i = 0; i < N; i++, p += e.rs) r[i] = *p;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++, p += e.rs) r[i] = t + i < rows ? *p : 0;
        }
    } else {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(e.res) + (size_t)t * e.rs + n;
#pragma unroll
        for (int i = 0; i < N; i++, p += e.rs) r[i] = t + i < rows ? *p : 0;
    }
}
// the residual of a tile on its way to L2, by one group of threads (a hint)
template <int BN, int THREADS>
__device__ __forceinline__ void prefetch_res(const Epilogue &e, int n0, int cols, int t0, int rows, int N, int tid) {
    if (!e.res) return;
    const int size = e.res_bf16 ? 2 : 4, bytes = min(cols, N - n0) * size;
    for (int t = t0 + tid; t < min(t0 + BN, rows); t += THREADS) {
        const uint8_t *p = reinterpret_cast<const uint8_t *>(e.res) + ((size_t)t * e.rs + n0) * size;
        for (int o = 0; o < bytes; o += 128) prefetch_l2(p + o);
        prefetch_l2(p + bytes - 1);
    }
}
// Sums of column n, rows t .. t + N - 1 (those below `rows`), to their place; r: their residual.
template <int N>
__device__ __forceinline__ void finish(const Epilogue &e, int n, float bias, int t, int rows, float (&v)[N], const uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += bias;
    activate(v, e.act);
    if (e.res) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __uint_as_float(e.res_bf16 ? r[i] << 16 : r[i]);
    }
    if (e.y_bf16) {
        __nv_bfloat16 *p = reinterpret_cast<__nv_bfloat16 *>(e.y) + (size_t)t * e.ys + n;
#pragma unroll
        for (int i = 0; i < N; i++, p += e.ys)
            if (t + i < rows) *p = __float2bfloat16_rn(v[i]);
    } else {
        float *p = reinterpret_cast<float *>(e.y) + (size_t)t * e.ys + n;
#pragma unroll
        for (int i = 0; i < N; i++, p += e.ys)
            if (t + i < rows) *p = v[i];
    }
}

// ---------------------------------------------------------------- few rows: the weights' stream
// Up to 8 rows: the stream of W bounds it, and below 10 MB the latency of one round trip (1 x 2048 x 2048, 8.4 MB: 5.2 us behind one
// another with W in L2, 7.8 cold).  A block has
// 16 columns of y (rows of W) and splits K over its warps; a lane reads 16 bytes of two rows of W
// and of one row of x, which is a fragment of m16n8k16 with k permuted alike on both sides.
constexpr int LS_WARPS = 8, LS_THREADS = 32 * LS_WARPS, LS_COLS = 16;
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__global__ void __launch_bounds__(LS_THREADS)
k_linear_few(const uint16_t *x, long long xs, const uint16_t *__restrict__ w, Epilogue e, int T, int N, int K, const int *rows_used) {
    constexpr int U = 8;      // steps of 32 k in flight
    cudaTriggerProgrammaticLaunchCompletion();
    __shared__ float red[LS_WARPS][8][LS_COLS + 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
    const int n0 = blockIdx.x * LS_COLS;
    const int steps = (K + 31) / 32;
    const uint16_t *wp[2] = {w + (size_t)min(n0 + g, N - 1) * K + 8 * j, w + (size_t)min(n0 + g + 8, N - 1) * K + 8 * j};
    // the first round of W on its way to L2 while the launch before this one runs (a hint: nothing is read yet)
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int k = (warp + u * LS_WARPS) * 32;
        if (k + 8 * j < K) { prefetch_l2(wp[0] + k); prefetch_l2(wp[1] + k); }
    }
    cudaGridDependencySynchronize();
    const int rows = rows_used ? min(T, *rows_used) : T;
    const uint16_t *xp = x + (size_t)min(g, T - 1) * xs + 8 * j;
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int s0 = warp; s0 < steps; s0 += LS_WARPS * U) {
        uint4 a[U][2], b[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = (s0 + u * LS_WARPS) * 32;
            const bool in = k + 8 * j < K;     // K is a multiple of 8
#pragma unroll
            for (int h = 0; h < 2; h++) a[u][h] = in ? __ldcs(reinterpret_cast<const uint4 *>(wp[h] + k)) : zero;
            b[u] = in ? *reinterpret_cast<const uint4 *>(xp + k) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            mma_bf16(c, a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u].x, b[u].y);
            mma_bf16(c, a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u].z, b[u].w);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) red[warp][2 * j + (i & 1)][g + 8 * (i >> 1)] = c[i];
    __syncthreads();
    if (tid < 8 * LS_COLS) {
        const int t = tid / LS_COLS, n = tid % LS_COLS;
        float v[1] = {0.f};
#pragma unroll
        for (int k = 0; k < LS_WARPS; k++) v[0] += red[k][t][n];
        uint32_t r[1];
        if (t < rows && n0 + n < N) {
            load_res(e, n0 + n, t, rows, r);
            finish(e, n0 + n, e.bias ? e.bias[n0 + n] : 0.f, t, rows, v, r);
        }
    }
}

// ---------------------------------------------------------------- tiles on tcgen05
// A tile is 128 columns of y (rows of W, the 128 lanes of the accumulator) by BN rows (its columns): in the epilogue a thread is
// one column of y, so that bias is a register and a warp's accesses to residual and y are 32 neighbours.
// The tensor pipe bounds large products, the loads from L2 those of few rows.  At 1965 MHz, short bursts: 4096 x 4096 x 4096 102 us, 1347
// TFLOP/s; 8000 x 4100 x 2048 108 plain, 115 with silu, 116 with gelu or gelu_tanh, 122 with a bf16 residual, 128 with gelu_tanh, bias and
// residual (16 epilogue warps; 8 took 8 us more).  A second of the last is under the power cap: 153 at 1470 MHz, 130 of the plain one.
// SPLIT > 1: a cluster shares a tile, each CTA a part of K; the parts are added in rank order over distributed shared memory.
constexpr int LT_M = 128, LT_K = 64;
template <int BN, int SPLIT>
struct LtCfg {
    static constexpr int STAGE = LT_M * LT_K * 2 + BN * LT_K * 2;
    static constexpr int STAGES = SPLIT > 1 ? (BN == 64 ? 3 : 4) : BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int PARTS = SPLIT > 1 ? BN * LT_M * 4 : 0;      // what the cluster's CTAs send: [rank][row of mine][column]
    static constexpr int SMEM = STAGE * STAGES + PARTS + 1024;
    static constexpr int EPI = BN == 256 ? 16 : 8, GROUPS = EPI / 4;      // warps of the epilogue, in groups of a warp per 32 lanes of TMEM
    static constexpr int THREADS = 32 * (2 + EPI);
};
struct LtMaps { CUtensorMap w, x; };
__device__ int g_linear_status;      // where a wait gave up (0: nowhere)

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_cluster(uint32_t addr, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }

template <int BN, int SPLIT>
__global__ void __launch_bounds__(LtCfg<BN, SPLIT>::THREADS, 1)
k_linear_tc(const __grid_constant__ LtMaps maps, Epilogue e, int T, int N, int K, const int *rows_used, int t_tiles, int n_tiles) {
    using C = LtCfg<BN, SPLIT>;
    constexpr int TM_COLS = SPLIT == 1 ? 2 * BN : BN;
    constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(LT_M >> 4) << 24);
    cudaTriggerProgrammaticLaunchCompletion();
    extern __shared__ uint8_t raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full_b[C::STAGES], empty_b[C::STAGES], acc_full_b[2], acc_empty_b[2];
    __shared__ uint32_t tmem_s;
    __shared__ volatile int abort_flag;
    constexpr int PER = BN / SPLIT;       // rows of a tile that one CTA of a cluster finishes
    const uint32_t parts = smem_u32(smem + C::STAGE * C::STAGES);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t full0 = smem_u32(full_b), empty0 = smem_u32(empty_b), accf0 = smem_u32(acc_full_b), acce0 = smem_u32(acc_empty_b);
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < C::STAGES; i++) { mbar_init(full0 + 8 * i, 1); mbar_init(empty0 + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(accf0 + 8 * i, 1); mbar_init(acce0 + 8 * i, C::EPI); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(TM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (SPLIT > 1) cluster_arrive();       // "I run": awaited before anything is sent to another CTA
    cudaGridDependencySynchronize();
    const uint32_t tmem = tmem_s;
    const int rows = rows_used ? min(T, *rows_used) : T;
    const int tiles = t_tiles * n_tiles, all_steps = (K + LT_K - 1) / LT_K;
    const int rank = SPLIT == 1 ? 0 : (int)(blockIdx.x % SPLIT);
    const int k0 = all_steps * rank / SPLIT, k_steps = all_steps * (rank + 1) / SPLIT - k0;
    const int first = SPLIT == 1 ? blockIdx.x : blockIdx.x / SPLIT, step = SPLIT == 1 ? gridDim.x : tiles;
    // Order of tiles: eight row tiles by all column tiles at a time, rows fastest, so that what runs at one time shares W and x in L2.
    auto place = [&](int i, int &n0, int &t0) {
        constexpr int GT = 8;
        const int grp = i / (GT * n_tiles), in = i - grp * GT * n_tiles, gt = min(GT, t_tiles - grp * GT);
        n0 = in / gt * LT_M;
        t0 = (grp * GT + in % gt) * BN;
    };
    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int i = first; i < tiles && ok; i += step) {
                int n0, t0;
                place(i, n0, t0);
                if (t0 >= rows) continue;
                for (int k = 0; k < k_steps; k++, it++) {
                    const uint32_t s = it % C::STAGES, ph = (it / C::STAGES) & 1;
                    if (!(ok = mbar_wait(empty0 + 8 * s, ph ^ 1, &abort_flag, &g_linear_status, 0x100 + s, TC_SPIN_LIMIT, TC_BACKOFF_NS))) break;
                    const uint32_t sa = smem_u32(smem + s * C::STAGE);
                    mbar_expect_tx(full0 + 8 * s, C::STAGE);
                    tma_load_2d(sa, &maps.w, (k0 + k) * LT_K, n0, full0 + 8 * s);
                    tma_load_2d(sa + LT_M * LT_K * 2, &maps.x, (k0 + k) * LT_K, t0, full0 + 8 * s);
                }
            }
            // gave up: let the copies in flight land before the block ends
            if (!ok)
                for (uint32_t i = it > C::STAGES ? it - C::STAGES : 0; i < it; i++)
                    for (uint32_t n = 0; n < TC_SPIN_LIMIT && !mbar_try(full0 + 8 * (i % C::STAGES), (i / C::STAGES) & 1); n++) {}
        }
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t it = 0, tc = 0;
            bool ok = true;
            for (int i = first; i < tiles && ok; i += step) {
                int n0, t0;
                place(i, n0, t0);
                if (t0 >= rows) continue;
                const uint32_t buf = SPLIT == 1 ? tc & 1 : 0;
                if (!(ok = mbar_wait(acce0 + 8 * buf, ((tc >> 1) & 1) ^ 1, &abort_flag, &g_linear_status, 0x200 + buf))) break;
                tc_fence_after();
                for (int k = 0; k < k_steps; k++, it++) {
                    const uint32_t s = it % C::STAGES, ph = (it / C::STAGES) & 1;
                    if (!(ok = mbar_wait(full0 + 8 * s, ph, &abort_flag, &g_linear_status, 0x300 + s))) break;
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + s * C::STAGE);
#pragma unroll
                    for (int kk = 0; kk < LT_K / 16; kk++)
                        mma_f16_ss(tmem + buf * BN, desc_sw128(sa + kk * 32), desc_sw128(sa + LT_M * LT_K * 2 + kk * 32), IDESC, (k | kk) ? 1u : 0u);
                    tc_commit(empty0 + 8 * s);
                }
                if (ok) tc_commit(accf0 + 8 * buf);
                tc++;
            }
        }
    } else {
        const int q = warp & 3, group = (warp - 2) >> 2;
        uint32_t tc = 0;
        if (SPLIT > 1) cluster_wait();
        for (int i = first; i < tiles; i += step) {
            int n0, t0;
            place(i, n0, t0);
            if (t0 >= rows) continue;
            const uint32_t buf = SPLIT == 1 ? tc & 1 : 0;
            const int n = n0 + 32 * q + lane, c0 = group * (BN / C::GROUPS), c1 = c0 + BN / C::GROUPS;
            const float bias = e.bias && n < N ? e.bias[n] : 0.f;
            // The next tile's residual starts for L2 now, so that the loads below, 16 rows at a time, wait for L2 and not for HBM
            // (8000 x 4100 x 2048 with a bf16 residual: 122 us, 188 with plain loads).
            if (SPLIT == 1) {
                if (tc == 0) prefetch_res<BN, 32 * C::EPI>(e, n0, LT_M, t0, rows, N, tid - 64);
                if (i + step < tiles) {
                    int n2, t2;
                    place(i + step, n2, t2);
                    prefetch_res<BN, 32 * C::EPI>(e, n2, LT_M, t2, rows, N, tid - 64);
                }
            }
            uint32_t res[2][16];       // one chunk ahead
            if (SPLIT == 1 && n < N) load_res(e, n, t0 + c0, rows, res[0]);
            if (!mbar_wait(accf0 + 8 * buf, SPLIT == 1 ? (tc >> 1) & 1 : 0, &abort_flag, &g_linear_status, 0x400 + buf, TC_SPIN_LIMIT, TC_BACKOFF_NS)) break;
            __syncwarp();
            tc_fence_after();
#pragma unroll 2
            for (int c = c0; c < c1; c += 16) {
                if (SPLIT == 1 && t0 + c >= rows) break;
                uint32_t r[16];
                tc_ld16(tmem + buf * BN + ((uint32_t)(32 * q) << 16) + c, r);
                if (SPLIT == 1 && n < N && c + 16 < c1) load_res(e, n, t0 + c + 16, rows, res[((c - c0) / 16 + 1) & 1]);
                tc_ld_wait();
                float v[16];
#pragma unroll
                for (int x = 0; x < 16; x++) v[x] = __uint_as_float(r[x]);
                if constexpr (SPLIT == 1) {
                    if (n < N) finish(e, n, bias, t0 + c, rows, v, res[((c - c0) / 16) & 1]);
                } else {
                    // to the CTA of the cluster that finishes these rows, [my rank][row][column]
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const int to = (c + x) / PER, row = (c + x) % PER;
                        st_cluster(map_cluster(parts + ((rank * PER + row) * LT_M + 32 * q + lane) * 4, to), v[x]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acce0 + 8 * buf);
            tc++;
        }
    }
    if constexpr (SPLIT > 1) {
        __syncwarp();
        if (warp < 2) cluster_wait();
        cluster_arrive();
        cluster_wait();
        int n0, t0;
        place(first, n0, t0);
        if (warp >= 2 && t0 < rows && !abort_flag) {
            const int f = (tid - 64) % LT_M, half = (tid - 64) / LT_M, n = n0 + f;
            constexpr int CH = PER >= 16 ? 8 : PER / 2;      // two groups of threads
            const float bias = e.bias && n < N ? e.bias[n] : 0.f;
            const float *p = reinterpret_cast<const float *>(smem + C::STAGE * C::STAGES) + f;
            for (int c = half * (PER / 2); c < (half + 1) * (PER / 2); c += CH) {
                const int t = t0 + rank * PER + c;
                if (t >= rows) break;
                float v[CH];
                uint32_t res[CH];
                if (n < N) load_res(e, n, t, rows, res);
#pragma unroll
                for (int x = 0; x < CH; x++) {
                    v[x] = p[(c + x) * LT_M];
#pragma unroll
                    for (int r = 1; r < SPLIT; r++) v[x] += p[(r * PER + c + x) * LT_M];
                }
                if (n < N) finish(e, n, bias, t, rows, v, res);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (abort_flag)
#pragma unroll 1
            for (int i = 0; i < 200; i++) __nanosleep(1000);      // products and copies in flight land before the block gives its memory back
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TM_COLS) : "memory");
    }
}

static int make_map_bf16(CUtensorMap *m, const void *base, long rows, long cols, long long stride, int box_rows) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return Q36_MOE_ECUDA;
        fn = (Encode)p;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {LT_K, (cuuint32_t)box_rows}, el[2] = {1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { last_cuda_error() = 100000 + (int)r; return Q36_MOE_ECUDA; }
    return Q36_MOE_OK;
}

template <int BN, int SPLIT>
static int run_tc(const LtMaps &maps, const Epilogue &e, int T, int N, int K, const int *rows_used, cudaStream_t st) {
    using C = LtCfg<BN, SPLIT>;
    static bool attr_done[MAX_DEVICES] = {false};
    int rc;
    if ((rc = ensure_smem_attr((const void *)k_linear_tc<BN, SPLIT>, C::SMEM, attr_done))) return rc;
    const int t_tiles = (T + BN - 1) / BN, n_tiles = (N + LT_M - 1) / LT_M;
    const long tiles = (long)t_tiles * n_tiles;
    if (SPLIT == 1) {
        launch_k(k_linear_tc<BN, SPLIT>, dim3((unsigned)min(tiles, (long)sm_count())), dim3(C::THREADS), C::SMEM, st, maps, e, T, N, K, rows_used, t_tiles, n_tiles);
        return check_launch();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * SPLIT));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SPLIT;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, k_linear_tc<BN, SPLIT>, maps, e, T, N, K, rows_used, t_tiles, n_tiles);
    return check_launch();
}
template <int BN>
static int run_split(int split, const LtMaps &maps, const Epilogue &e, int T, int N, int K, const int *rows_used, cudaStream_t st) {
    if (split == 8) return run_tc<BN, 8>(maps, e, T, N, K, rows_used, st);
    if (split == 4) return run_tc<BN, 4>(maps, e, T, N, K, rows_used, st);
    if (split == 2) return run_tc<BN, 2>(maps, e, T, N, K, rows_used, st);
    return run_tc<BN, 1>(maps, e, T, N, K, rows_used, st);
}

int launch_linear(const void *x, long long xs, const void *w, const float *bias, int act, const void *res, int res_bf16, long long rs,
                  void *y, int y_bf16, long long ys, int T, int N, int K, const int *rows_used, cudaStream_t st) {
    const Epilogue e{bias, res, y, rs, ys, act, res_bf16, y_bf16};
    // The stream up to 8 rows while its warps have all of W in flight at once; us at 2048 columns against the split tiles: K 2048 5.8 /
    // 6.0, K 4096 11.4 / 7.5.
    if (T <= 8 && K <= 2048) {
        launch_k(k_linear_few, dim3((N + LS_COLS - 1) / LS_COLS), dim3(LS_THREADS), 0, st, (const uint16_t *)x, xs, (const uint16_t *)w, e, T, N, K, rows_used);
        return check_launch();
    }
    // Tile height and split of K by what an SM has to load (166 KB per us, at least 0.22 us per 64 of K; two CTAs of 32 or 64 rows at a
    // time), what the exchange of a cluster costs and what a second round of CTAs costs.  Measured us at 2048 columns, K 2048, for
    // (rows, split): 64 tokens (32, 4) 6.6, (64, 8) 7.6, (64, 1) 10.9; 200 tokens (32, 2) 8.6, (64, 4) 9.4, (32, 4) 13.4; 300
    // tokens (64, 1) 11.2, (128, 4) 17.0; 1000 tokens (128, 1) 12.5, (256, 1) 15.6, (128, 4) 35.
    int bn = 0, split = 1;
    float best = 0.f;
    const int steps = (K + LT_K - 1) / LT_K, sms = sm_count();
    for (int cb = 32; cb <= 256; cb *= 2)
        for (int cs = 1; cs <= (cb == 256 ? 1 : 8) && (cs == 1 || steps >= 2 * cs); cs *= 2) {
            const long ctas = (long)((T + cb - 1) / cb) * ((N + LT_M - 1) / LT_M) * cs, per_sm = (ctas + sms - 1) / sms;
            const long rounds = cs == 1 ? 1 : (per_sm + (cb <= 64 ? 1 : 0)) / (cb <= 64 ? 2 : 1);
            const float kb = (LT_M + cb) * (LT_K * 2 / 1024.f);
            const float us = cs == 1 ? per_sm * steps * fmaxf(0.22f, kb / 166.f)
                                     : (steps + cs - 1) / cs * fmaxf(0.22f * rounds, per_sm * kb / 166.f) + 0.05f * cb + 4.9f * (rounds - 1);
            if (!bn || us < best) { best = us; bn = cb; split = cs; }
        }
    LtMaps maps;
    int rc;
    if ((rc = make_map_bf16(&maps.w, w, N, K, K, LT_M)) || (rc = make_map_bf16(&maps.x, x, T, K, xs, bn))) return rc;
    if (bn == 32) return run_split<32>(split, maps, e, T, N, K, rows_used, st);
    if (bn == 64) return run_split<64>(split, maps, e, T, N, K, rows_used, st);
    if (bn == 128) return run_split<128>(split, maps, e, T, N, K, rows_used, st);
    return run_tc<256, 1>(maps, e, T, N, K, rows_used, st);
}

// Where a bounded wait gave up (0: nowhere) since this was last asked, on the current device; the stream has been synchronised.
int linear_wait_status(int *out) {
    const int zero = 0;
    if (cudaMemcpyFromSymbol(out, g_linear_status, sizeof(int)) != cudaSuccess) return check_launch();
    if (*out && cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int)) != cudaSuccess) return check_launch();
    return Q36_MOE_OK;
}

}  // namespace q36

using namespace q36;

extern "C" int q36_linear(const void *x, int64_t x_stride, const void *w, const float *bias, int act, const void *residual, int res_is_bf16,
                          int64_t res_stride, void *y, int y_is_bf16, int64_t y_stride, int T, int N, int K, const int *rows_used,
                          void *stream) {
    if ((T && (!x || !y)) || !w || T < 0 || T > (1 << 30) || N <= 0 || N > (1 << 30) || K <= 0 || K > (1 << 30) || K % 8 || x_stride < K || x_stride % 8 || y_stride < N) return Q36_MOE_EINVAL;
    if (act < Q36_ACT_NONE || act > Q36_ACT_GELU_TANH || (residual && res_stride < N)) return Q36_MOE_EINVAL;
    if ((((uintptr_t)x | (uintptr_t)w) & 15) || ((uintptr_t)bias & 3) || ((uintptr_t)y & (y_is_bf16 ? 1 : 3))) return Q36_MOE_EINVAL;
    if (residual && ((uintptr_t)residual & (res_is_bf16 ? 1 : 3))) return Q36_MOE_EINVAL;
    if (residual && residual == y && (!res_is_bf16 != !y_is_bf16 || res_stride != y_stride)) return Q36_MOE_EINVAL;
    if (T == 0) return Q36_MOE_OK;
    return launch_linear(x, x_stride, w, bias, act, residual, res_is_bf16 != 0, res_stride, y, y_is_bf16 != 0, y_stride, T, N, K, rows_used,
                         (cudaStream_t)stream);
}
