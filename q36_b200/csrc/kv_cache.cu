// The paged 4-bit cache: tables of a step from its request lengths, the writer and the reader of cache rows.
#include "attn.cuh"

namespace q36 {

constexpr int TB_THREADS = 512;
constexpr int TB_MAX_SEQ = 16384;

// ---------------------------------------------------------------- tables
// Two prefix sums over the requests (rows, new blocks), then one pass over all rows and all new blocks, each of which finds
// its request by bisection.  Sums saturate just above what is available (min(a + b, cap) is associative for a, b >= 0), so
// that no lengths overflow them.  Every CTA makes the sums for itself: 16 KB of lengths at 2000 requests come out of L2 in
// less time than a second launch takes.  Latency bounds it: 8 requests 5 us, 2000 requests 8 (46 CTAs); behind one another 2.8 and 6.5.
// In place (lengths or list head written where they were read) one CTA does it all, since another could read what it has written: behind
// one another 3.0 and 10.5, 1024 rows 4.4 (3.7 separate), 8192 rows 9.3 (3.4), 32,768 rows 29 of one request, 42 of 16 (3.6, 3.9).
struct TbReq { int rows, need, ok; };
__device__ __forceinline__ TbReq tb_request(int old, int q, int log_bs, int max_blocks, int row_cap, int blk_cap, int &flags) {
    TbReq r;
    r.ok = 1;
    r.rows = min(max(q, 0), row_cap);
    r.need = 0;
    if (old < 0 || q < 0) { flags |= 4; r.ok = 0; return r; }
    const long long last = (1 << log_bs) - 1, held = (old + last) >> log_bs, all = ((long long)old + q + last) >> log_bs;
    if (all > max_blocks) { flags |= 2; r.ok = 0; return r; }
    r.need = (int)min(all - held, (long long)blk_cap);
    return r;
}
__device__ __forceinline__ int sat_add(int a, int b, int cap) { return min(a + b, cap); }

// largest b in [0, n) with pre[b] <= v (pre[0] <= v)
__device__ __forceinline__ int bisect(const int *pre, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (pre[m] <= v) lo = m; else hi = m;
    }
    return lo;
}

__global__ void __launch_bounds__(TB_THREADS)
k_kv_tables(const int *kv_old, const int *q_len, int B, int log_bs, int n_blocks, const int *free_blocks,
            int n_free, const int *free_head, int *block_table, int max_blocks, int *__restrict__ cu_q, int *kv_len,
            int *__restrict__ slots, int *__restrict__ positions, int T, int *free_head_out, int *status) {
    Q36_GDS();
    extern __shared__ int sm[];
    int *pre_r = sm, *pre_b = sm + B + 1;     // exclusive prefix sums; entry B: the total
    __shared__ int wr[TB_THREADS / 32], wb[TB_THREADS / 32], fl;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bs = 1 << log_bs;
    const int head = min(max(*free_head, 0), n_free), avail = n_free - head;
    const int row_cap = T + 1, blk_cap = avail + 1;
    if (tid == 0) fl = 0;
    const int per = (B + TB_THREADS - 1) / TB_THREADS, b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int flags = 0, sr = 0, sb = 0;
    for (int b = b0; b < b1; b++) {
        const TbReq r = tb_request(kv_old[b], q_len[b], log_bs, max_blocks, row_cap, blk_cap, flags);
        pre_r[b] = sr;
        pre_b[b] = sb;
        sr = sat_add(sr, r.rows, row_cap);
        sb = sat_add(sb, r.need, blk_cap);
    }
    int ir = sr, ib = sb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int r = __shfl_up_sync(0xffffffffu, ir, o), n = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) { ir = sat_add(ir, r, row_cap); ib = sat_add(ib, n, blk_cap); }
    }
    if (lane == 31) { wr[warp] = ir; wb[warp] = ib; }
    int er = __shfl_up_sync(0xffffffffu, ir, 1), eb = __shfl_up_sync(0xffffffffu, ib, 1);
    if (lane == 0) er = eb = 0;
    __syncthreads();
    for (int w = 0; w < warp; w++) { er = sat_add(er, wr[w], row_cap); eb = sat_add(eb, wb[w], blk_cap); }
    for (int b = b0; b < b1; b++) { pre_r[b] = sat_add(pre_r[b], er, row_cap); pre_b[b] = sat_add(pre_b[b], eb, blk_cap); }
    if (tid == TB_THREADS - 1) { pre_r[B] = sat_add(er, sr, row_cap); pre_b[B] = sat_add(eb, sb, blk_cap); }
    __syncthreads();
    const int total_rows = min(pre_r[B], T), total_new = pre_b[B];
    auto served = [&](int b, const TbReq &r) { return r.ok && (r.need == 0 || pre_b[b] + r.need <= avail) && (r.rows == 0 || pre_r[b + 1] <= T); };

    const int stride = gridDim.x * TB_THREADS, first = blockIdx.x * TB_THREADS + tid;
    int dummy = 0;
    // new table entries
    for (int i = first; i < min(total_new, avail); i += stride) {
        const int b = bisect(pre_b, B, i);
        const int old = kv_old[b];
        const TbReq r = tb_request(old, q_len[b], log_bs, max_blocks, row_cap, blk_cap, dummy);
        if (!served(b, r)) continue;
        const int held = (old + bs - 1) >> log_bs;
        block_table[(size_t)b * max_blocks + held + (i - pre_b[b])] = free_blocks[head + i];
    }
    // rows; a row's block is an old table entry or a free-list entry (the table's new entries may not be written yet)
    for (int t = first; t < T; t += stride) {
        int slot = -1, pos = -1;
        if (t < total_rows) {
            const int b = bisect(pre_r, B, t);
            const int old = kv_old[b];
            const TbReq r = tb_request(old, q_len[b], log_bs, max_blocks, row_cap, blk_cap, dummy);
            if (served(b, r)) {
                pos = old + (t - pre_r[b]);
                const int held = (old + bs - 1) >> log_bs, col = pos >> log_bs;
                const int blk = col < held ? block_table[(size_t)b * max_blocks + col] : free_blocks[head + pre_b[b] + (col - held)];
                if (blk >= 0 && blk < n_blocks) slot = blk * bs + (pos & (bs - 1));
            }
        }
        slots[t] = slot;
        positions[t] = pos;
    }
    // The requests' own outputs: block 0, after everything that reads the lengths and the head (kv_len and free_head_out may be
    // kv_old and free_head, with one block).
    if (blockIdx.x == 0) {
        __syncthreads();
        int used = 0;
        for (int b = tid; b < B; b += TB_THREADS) {
            const int old = kv_old[b], q = q_len[b];
            const TbReq r = tb_request(old, q, log_bs, max_blocks, row_cap, blk_cap, flags);
            const bool s = served(b, r);
            if (r.ok && r.need > 0 && pre_b[b] + r.need > avail) flags |= 1;
            if (r.rows > 0 && pre_r[b + 1] > T) flags |= 8;
            cu_q[b] = min(pre_r[b], T);
            kv_len[b] = s ? old + q : 0;
            // (from the first unserved request on that needs blocks or rows none of that kind is served: no holes)
            if (s && r.need > 0) used = max(used, pre_b[b] + r.need);
        }
        if (tid == 0) cu_q[B] = total_rows;
        used = (int)__reduce_max_sync(0xffffffffu, (unsigned)used);
        flags = (int)__reduce_or_sync(0xffffffffu, (unsigned)flags);
        if (lane == 0) { wr[warp] = used; atomicOr(&fl, flags); }
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < TB_THREADS / 32; w++) used = max(used, wr[w]);
            *free_head_out = head + used;
            *status = fl;
        }
    }
}

// ---------------------------------------------------------------- rows in and out
// Smallest e with amax <= 6 * 2^e in [-126, 125]; 6 = 1.5 * 2^2.
__device__ __forceinline__ int e2_of_amax_fp4(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 129 + ((u & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    return max(-126, min(125, e));
}
// eight f32 -> eight E2M1 nibbles, element 0 in the low one; round to nearest even, saturating at 6
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// Instructions bound both, the ALU first: 32,768 tokens of 2 x 128, bf16, are written in 14.4 us and read in 11.2 (43 MB each, 6.5 at the
// copy rate).
constexpr int KVC_THREADS = 256;
// A thread's eight dims of a row of K and of V: token t, kv head, scale block b, quarter j of it.  Four lanes share a block, so that rows
// are read and K codes written in whole sectors.
struct RowPart { int t, head, b, j, r; };
// Parts per row and how to divide a part's number, below 2^31, by them: n m / 2^(31 + s) with m = ceil(2^(31 + s) / row8), 2^s >= row8, is at
// most n / 2^31 2^-s above n / row8: less than the 1 / row8 that the next whole number is away.
struct RowDiv {
    unsigned row8, m;
    int s, log_head8;
};
static RowDiv row_div(const KvGeom &g) {
    RowDiv d;
    d.row8 = g.Hkv * g.Dh / 8;
    d.s = log2_of((int)d.row8);
    d.m = (unsigned)(((1ull << (31 + d.s)) + d.row8 - 1) / d.row8);
    d.log_head8 = log2_of(g.Dh / 8);
    return d;
}
__device__ __forceinline__ RowPart row_part(const RowDiv &d, unsigned i) {
    const unsigned t = __umulhi(i, d.m) >> (d.s - 1), r = i - t * d.row8, head = r >> d.log_head8, c = r & ((1u << d.log_head8) - 1);
    return RowPart{(int)t, (int)head, (int)(c >> 2), (int)(c & 3), (int)r};
}
// eight values, and the whole block's largest magnitude's exponent -> codes; NaN counts as 0
__device__ __forceinline__ uint32_t quant8(float (&x)[8], int &e2) {
    float am = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = x[e] == x[e] ? x[e] : 0.f;
        am = fmaxf(am, fabsf(x[e]));
    }
    am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
    am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
    e2 = e2_of_amax_fp4(am);
    const float inv = inv_scale_of_e2(e2);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= inv;
    return f32x8_to_e2m1(x);
}
__global__ void __launch_bounds__(KVC_THREADS)
k_kv_append(const void *k, const void *v, int bf16, long long ks, long long vs, const int *slots, KvGeom g,
            RowDiv div, unsigned n8) {
    Q36_GDS();
    const unsigned i = blockIdx.x * KVC_THREADS + threadIdx.x;
    const RowPart p = row_part(div, min(i, n8 - 1));
    const int slot = i < n8 ? slots[p.t] : -1, block = slot >> g.log_bs;
    const bool put = slot >= 0 && block < g.n_blocks;
    float x[8] = {}, y[8] = {};
    if (put) {
        load8(k, (size_t)p.t * ks + (size_t)p.r * 8, bf16, x);
        load8(v, (size_t)p.t * vs + (size_t)p.r * 8, bf16, y);
    }
    int ek, ev;
    const uint32_t kc = quant8(x, ek), vc = quant8(y, ev);
    if (!put) return;
    uint8_t *reg = const_cast<uint8_t *>(g.at(block, p.head));
    const int tok = slot & (g.bs - 1), half = g.bs * g.Dh / 2, nb = g.Dh / 32;
    *reinterpret_cast<uint32_t *>(reg + kv_k_off(tok, p.j, p.b, g.Dh)) = kc;
    *reinterpret_cast<uint16_t *>(reg + half + kv_v_off(tok, 2 * p.j, p.b, g.Dh)) = (uint16_t)vc;
    *reinterpret_cast<uint16_t *>(reg + half + kv_v_off(tok, 2 * p.j + 1, p.b, g.Dh)) = (uint16_t)(vc >> 16);
    if (p.j == 0) reg[2 * half + tok * nb + p.b] = (uint8_t)(127 + ek);
    if (p.j == 1) reg[2 * half + (g.bs + tok) * nb + p.b] = (uint8_t)(127 + ev);
}

__device__ __forceinline__ void store8_exact(void *p, size_t at, int bf16, uint32_t codes, float sc) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float2 f = e2m1x2_to_f32x2((codes >> (8 * e)) & 0xff);
        x[2 * e] = f.x * sc;
        x[2 * e + 1] = f.y * sc;
    }
    if (bf16) {      // exact: a code has two significant bits
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = (__float_as_uint(x[2 * e]) >> 16) | (__float_as_uint(x[2 * e + 1]) & 0xffff0000u);
        *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        float4 *o = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}
__global__ void __launch_bounds__(KVC_THREADS)
k_kv_read(KvGeom g, const int *slots, void *__restrict__ k, void *__restrict__ v, int bf16, RowDiv div, unsigned n8) {
    Q36_GDS();
    const unsigned i = blockIdx.x * KVC_THREADS + threadIdx.x;
    if (i >= n8) return;
    const RowPart p = row_part(div, i);
    const int slot = slots[p.t], block = slot >> g.log_bs;
    uint32_t kc = 0, vc = 0;
    float sk = 0.f, sv = 0.f;
    if (slot >= 0 && block < g.n_blocks) {
        const uint8_t *reg = g.at(block, p.head);
        const int tok = slot & (g.bs - 1), half = g.bs * g.Dh / 2, nb = g.Dh / 32;
        kc = *reinterpret_cast<const uint32_t *>(reg + kv_k_off(tok, p.j, p.b, g.Dh));
        vc = *reinterpret_cast<const uint16_t *>(reg + half + kv_v_off(tok, 2 * p.j, p.b, g.Dh)) |
             (uint32_t)*reinterpret_cast<const uint16_t *>(reg + half + kv_v_off(tok, 2 * p.j + 1, p.b, g.Dh)) << 16;
        sk = ue8m0_to_f32(reg[2 * half + tok * nb + p.b]);
        sv = ue8m0_to_f32(reg[2 * half + (g.bs + tok) * nb + p.b]);
    }
    store8_exact(k, (size_t)i * 8, bf16, kc, sk);
    store8_exact(v, (size_t)i * 8, bf16, vc, sv);
}

// n8 < 2^31: rows are launched in lots of that many parts
template <typename F>
static int by_lots(KvGeom g, int T, F launch) {
    const RowDiv div = row_div(g);
    const long long row8 = div.row8;
    const int lot = (int)min((long long)T, (1ll << 30) / row8);
    for (int t = 0; t < T; t += lot) {
        const int n = min(lot, T - t);
        launch(t, div, (unsigned)(n * row8), dim3((unsigned)((n * row8 + KVC_THREADS - 1) / KVC_THREADS)));
    }
    return check_launch();
}
int launch_kv_append(const void *k, const void *v, int bf16, long long ks, long long vs, const int *slots, KvGeom g, int T, cudaStream_t st) {
    const int size = bf16 ? 2 : 4;
    return by_lots(g, T, [&](int t, RowDiv div, unsigned n8, dim3 grid) {
        launch_k(k_kv_append, grid, dim3(KVC_THREADS), 0, st, (const void *)((const uint8_t *)k + (size_t)t * ks * size),
                 (const void *)((const uint8_t *)v + (size_t)t * vs * size), bf16, ks, vs, slots + t, g, div, n8);
    });
}

}  // namespace q36

using namespace q36;

static bool off16(const void *p) { return ((uintptr_t)p & 15) != 0; }

extern "C" {

uint64_t q36_kv_block_bytes(int block_size, int n_kv_head, int head_dim) {
    if (!kv_geom_ok(block_size, n_kv_head, head_dim)) return 0;
    return (uint64_t)block_size * head_dim * 17 / 16 * n_kv_head;
}

int q36_kv_tables(const int *kv_old, const int *q_len, int n_seq, int block_size, int n_blocks, const int *free_blocks, int n_free,
                  const int *free_head, int *block_table, int max_blocks, int *cu_q, int *kv_len, int *slots, int *positions, int T,
                  int *free_head_out, int *status, void *stream) {
    if (!kv_old || !q_len || !free_head || !block_table || !cu_q || !kv_len || !free_head_out || !status) return Q36_MOE_EINVAL;
    if ((n_free > 0 && !free_blocks) || (T > 0 && (!slots || !positions))) return Q36_MOE_EINVAL;
    if (n_seq <= 0 || n_seq > TB_MAX_SEQ || T < 0 || T > (1 << 29) || n_free < 0 || n_free > (1 << 29) || max_blocks <= 0 || n_blocks <= 0) return Q36_MOE_EINVAL;
    if (!kv_geom_ok(block_size, 1, 64) || (int64_t)n_blocks * block_size > INT32_MAX || (int64_t)max_blocks * block_size > (1 << 30)) return Q36_MOE_EINVAL;
    const int smem = 2 * (n_seq + 1) * 4;
    static bool attr_done[MAX_DEVICES] = {false};
    int rc;
    // (whatever the size: the limit without it, 48 KB, counts the kernel's static arrays too)
    if ((rc = ensure_smem_attr((const void *)k_kv_tables, 2 * (TB_MAX_SEQ + 1) * 4, attr_done))) return rc;
    const long work = (long)T + n_seq;
    // in place: one block, since another could read what it has written
    const bool in_place = kv_len == kv_old || free_head_out == free_head;
    const int grid = in_place ? 1 : (int)min((work + TB_THREADS - 1) / TB_THREADS, (long)sm_count());
    launch_k(k_kv_tables, dim3(grid), dim3(TB_THREADS), smem, (cudaStream_t)stream, kv_old, q_len, n_seq, log2_of(block_size), n_blocks, free_blocks, n_free,
             free_head, block_table, max_blocks, cu_q, kv_len, slots, positions, T, free_head_out, status);
    return check_launch();
}

int q36_kv_append(const void *k, const void *v, int x_is_bf16, int64_t k_stride, int64_t v_stride, const int *slots, void *cache,
                  int n_blocks, int block_size, int n_kv_head, int head_dim, int T, void *stream) {
    if ((T && (!k || !v || !slots)) || !cache || !kv_geom_ok(block_size, n_kv_head, head_dim) || T < 0) return Q36_MOE_EINVAL;
    const int64_t row = (int64_t)n_kv_head * head_dim, vec = x_is_bf16 ? 8 : 4;
    if (n_blocks <= 0 || (int64_t)n_blocks * block_size > INT32_MAX || k_stride < row || v_stride < row || k_stride % vec || v_stride % vec) return Q36_MOE_EINVAL;
    if (off16(k) || off16(v) || off16(cache)) return Q36_MOE_EINVAL;
    if (T == 0) return Q36_MOE_OK;
    const KvGeom g{(const uint8_t *)cache, n_blocks, block_size, log2_of(block_size), n_kv_head, head_dim};
    return launch_kv_append(k, v, x_is_bf16, k_stride, v_stride, slots, g, T, (cudaStream_t)stream);
}

int q36_kv_read(const void *cache, int n_blocks, int block_size, int n_kv_head, int head_dim, const int *slots, void *k, void *v,
                int x_is_bf16, int T, void *stream) {
    if ((T && (!k || !v || !slots)) || !cache || !kv_geom_ok(block_size, n_kv_head, head_dim) || T < 0) return Q36_MOE_EINVAL;
    if (n_blocks <= 0 || (int64_t)n_blocks * block_size > INT32_MAX || off16(k) || off16(v) || off16(cache)) return Q36_MOE_EINVAL;
    if (T == 0) return Q36_MOE_OK;
    const KvGeom g{(const uint8_t *)cache, n_blocks, block_size, log2_of(block_size), n_kv_head, head_dim};
    const size_t row = (size_t)n_kv_head * head_dim * (x_is_bf16 ? 2 : 4);
    return by_lots(g, T, [&](int t, RowDiv div, unsigned n8, dim3 grid) {
        launch_k(k_kv_read, grid, dim3(KVC_THREADS), 0, (cudaStream_t)stream, g, slots + t, (void *)((uint8_t *)k + t * row),
                 (void *)((uint8_t *)v + t * row), x_is_bf16, div, n8);
    });
}

}  // extern "C"
