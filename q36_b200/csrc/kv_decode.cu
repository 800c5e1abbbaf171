// Attention of few rows per request over the paged 4-bit cache: decoding, short continuations, and f32 activations.
//
// Mathematics.  With c the E2M1 codes and s their block exponents, the score of row r and token t is
//   S[t][r] = sum_b 2^ks[t][b] * (sum_{d in b} c[t][d] q[r][d])
// and the output sum_t p[t][r] 2^vs[t][b] c[t][d].  Both products run on f16 tensor core instructions (m16n8k16, f32 sums) with
// the codes, which f16 holds exactly, as the 16-row operand and eight rows as the narrow one, so that a group of eight query
// heads wastes nothing.  K's exponents multiply the partial sums of each 32-dim block; V's cannot leave the sum over tokens, so
// they go to the weights.  While the V exponents of what a warp has read stay in a window of 13 (anchor - 8 .. anchor + 4, the
// anchor being the first group's largest), the weight 2^(S - mm[r]) is rounded to f16 once (half a step 2^-11, against
// bf16's 2^-8 of the output) and block b uses it times 2^(vs[t][b] - anchor), which is exact: mm keeps weights at 2^7 and
// below 2^11, so the strongest token of any block of dims has at least 2^-1 there and f16 is precise down to 2^-14.
// When an exponent leaves the window (a block of V 2^8 times weaker, 2^4 times stronger than the first tokens'), the warp goes over
// to a reference per row and block of dims and rounds the weights of every block by themselves: f16 keeps them to 2^-36 of the block's
// strongest (weight times 2^exponent), whatever the other blocks' exponents.
// It does so too at K exponents of 65 and more, whose sums with q as it is in f16 would not all fit f32: there they are kept 2^23 lower.
// Blocks of scale byte 1 need no place in the window: zeros, or values up to 6 * 2^-126, which count as zeros beside an anchor 2^9 or more above.
// The normaliser is the sum of the unrounded weights in f32.
// q enters as f16 after an exact power of two per row (bf16 and f16 fit); f32 activations enter as two f16 terms, and so do
// their weights, which leaves 2^-22.
//
// Work.  A unit is 16 tokens of one (request, kv head, row tile).  The units of all requests, in order, are cut into equal
// ranges, one per CTA, so that ragged lengths load every SM alike.  A range's first and last pieces may be parts of what a
// neighbour has the rest of: they go to the workspace and k_attn_join adds them up in a fixed order.
// With the join, 16 heads of 128 on 2, from HBM: 64 requests of 266,000 tokens together 36 us, of 533,000 53, of 1,065,000 86 (4.2 to 4.4 TB/s
// between them; the first 20 us are launches, plan, the first reads of a page, of its data, and the join), one of 131,072 32; one of 700
// tokens 10.  Tokens all in the second form: 266,000 43.
#include <math.h>

#include "attn_plan.cuh"

namespace q36 {

constexpr int DEC_WARPS = 4, DEC_THREADS = 32 * DEC_WARPS, DEC_UNIT = 16;
constexpr float DEC_NONE = -3.0e38f;      // "no token yet" of the running references: finite, so that differences stay defined
constexpr float DEC_TOP = 7.f, DEC_MAX = 11.f;        // log2 of the largest weight when the reference moves, and when it has to
constexpr int DEC_WIN_LO = 8, DEC_WIN_HI = 4;         // window of V exponents around the anchor
constexpr uint32_t DEC_NO_BLOCK = 32 - (15 - DEC_WIN_LO);     // the place in the window whose f16 factor is -0
constexpr float DEC_WIDE_TOP = 11.f, DEC_WIDE_MAX = 15.f;   // the same with a reference per block of dims
// What the wide form takes off K's scales until its sums meet the rows' powers of two: eight blocks' sums of 32 products, below 32 * 6 * 2^15
// as q is in f16, stay in f32 at exponents up to 125; 2^-126 remains a number.
constexpr float DEC_K_DOWN = 1.f / (1 << 23);

// the four bytes of w, two E2M1 codes each (low nibble first), as f16x2
__device__ __forceinline__ void e2m1x8_to_f16x2(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 8x8 matrix of 16-bit elements across the warp, transposed
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// largest of the eight lanes that hold a column (lanes with the same j)
__device__ __forceinline__ float column_max(float v) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
    return v;
}
// weights of tokens (g, g + 8) x rows (2j, 2j + 1), as f16 terms, transposed into the narrow operand of the second product
template <int TERMS, int NT>
__device__ __forceinline__ void weights_f16(const float (&p)[4], uint32_t (&w)[TERMS][NT][2], int nt) {
    const uint32_t w0 = pack_f16(p[0], p[1]), w1 = pack_f16(p[2], p[3]);
    w[0][nt][0] = transpose8x8(w0);
    w[0][nt][1] = transpose8x8(w1);
    if constexpr (TERMS == 2) {
        const float2 h0 = unpack_f16(w0), h1 = unpack_f16(w1);
        w[1][nt][0] = transpose8x8(pack_f16(p[0] - h0.x, p[1] - h0.y));
        w[1][nt][1] = transpose8x8(pack_f16(p[2] - h1.x, p[3] - h1.y));
    }
}
// BYTES from global to shared memory behind the thread's back; what a thread has asked for is there for itself after cp_wait
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t to, const uint8_t *from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// What a lane holds of 16 tokens, and where it waits in shared memory until then.  Lane (g, j): g = lane / 4, j = lane % 4.  A lane
// copies exactly what it reads itself (scales of a token come as a word), so that nobody waits for anybody else.
template <int DH>
struct DecFrag {
    static constexpr int NB = DH / 32, W = DH / 32, SW = (NB + 3) / 4, VB = NB >= 4 ? NB / 4 : 1;
    static constexpr int CB = W == 2 ? 8 : 16, NCH = W * 4 / CB, SB = NB == 8 ? 8 : 4;         // a piece of codes, pieces of a token half, a piece of scales
    static constexpr int CODES = 4 * NCH * 32 * CB, STAGE = CODES + 4 * 32 * SB, STAGES = 2;
    uint32_t k[2][W];      // K words of tokens g and g + 8: word b = dims 32b + 8j ..
    uint32_t v[2][W];      // V of token pairs j and j + 4, group g: first half token 2p, second half token 2p + 1
    uint32_t ks[2][SW];    // K scales of tokens g and g + 8
    uint32_t vs[VB];       // V scales of tokens g (low half) and g + 8, blocks VB j ..
    // pk, pv, pks, pvs: this lane's part of the group's codes and scales
    static __device__ __forceinline__ void copy(uint32_t st, const uint8_t *pk, const uint8_t *pv, const uint8_t *pks, const uint8_t *pvs, int lane) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int c = 0; c < NCH; c++) cp_async<CB>(st + ((h * NCH + c) * 32 + lane) * CB, pk + h * 8 * (DH / 2) + c * CB);
            cp_async<SB>(st + CODES + (h * 32 + lane) * SB, pks + h * 8 * NB);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            cp_async<SB>(st + CODES + ((2 + h) * 32 + lane) * SB, pvs + h * 8 * NB);
#pragma unroll
            for (int c = 0; c < NCH; c++) cp_async<CB>(st + (((2 + h) * NCH + c) * 32 + lane) * CB, pv + h * 4 * DH + c * CB);
        }
    }
    static __device__ __forceinline__ void get(const uint8_t *st, int half, int lane, uint32_t (&r)[W]) {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const uint8_t *p = st + ((half * NCH + c) * 32 + lane) * CB;
            if constexpr (CB == 8) {
                const uint2 u = *reinterpret_cast<const uint2 *>(p);
                r[0] = u.x; r[1] = u.y;
            } else {
                const uint4 u = *reinterpret_cast<const uint4 *>(p);
                r[4 * c] = u.x; r[4 * c + 1] = u.y; r[4 * c + 2] = u.z; r[4 * c + 3] = u.w;
            }
        }
    }
    static __device__ __forceinline__ void get_ks(const uint8_t *st, int h, int lane, uint32_t (&r)[SW]) {
        const uint32_t *p = reinterpret_cast<const uint32_t *>(st + CODES + (h * 32 + lane) * SB);
        if constexpr (NB == 2) r[0] = *p >> (lane & 4 ? 16 : 0);      // (the word has two tokens; what is above is not looked at)
        else r[0] = p[0];
        if constexpr (NB == 8) r[1] = p[1];
    }
    __device__ __forceinline__ void get_k(const uint8_t *st, int lane) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            get(st, h, lane, k[h]);
            get_ks(st, h, lane, ks[h]);
        }
    }
    // not zero: token g + 8h has a K exponent of 65 or more (a scale byte with its two top bits set)
    static __device__ __forceinline__ uint32_t high_k(const uint8_t *st, int h, int lane) {
        uint32_t r[SW], any = 0;
        get_ks(st, h, lane, r);
#pragma unroll
        for (int w = 0; w < SW; w++) any |= r[w] & (r[w] << 1);
        return any & (NB == 2 ? 0x8080u : 0x80808080u);
    }
    __device__ __forceinline__ void get_v(const uint8_t *st, int lane) {
        get(st, 2, lane, v[0]);
        get(st, 3, lane, v[1]);
    }
    __device__ __forceinline__ void get_vs(const uint8_t *st, int lane) {
        const int j = lane & 3, word = NB == 8 ? j >> 1 : 0, first = NB == 8 ? 2 * (j & 1) : NB == 4 ? j : (lane & 4) / 2 + (j & 1);
        const uint8_t *p = st + CODES + (2 * 32 + lane) * SB + 4 * word;
        const uint32_t a = *reinterpret_cast<const uint32_t *>(p), b = *reinterpret_cast<const uint32_t *>(p + 32 * SB);
#pragma unroll
        for (int c = 0; c < VB; c++) vs[c] = __byte_perm(a, b, (first + c) * 0x11 | (first + c + 4) * 0x1100) & 0x00ff00ffu;
    }
};

// The wide form's weights of block b: 2^(S - m + vs - M), M per row and block and relative to m, so that exponents of V are not lost beside
// large scores; moves M, and with it the block's sums.  s: S - m.
template <int DH, int NT, int TERMS, int VB>
__device__ __forceinline__ void wide_weights(float (*Ms)[8 * NT], const uint32_t (&vs)[VB], const float (&s)[NT][4], uint32_t (&w)[TERMS][NT][2],
                                             float (&o)[NT][DH / 32][2][4], int b, int lane) {
    const int j = lane & 3;
    const uint32_t vv = __shfl_sync(0xffffffffu, vs[b % VB], (lane & 28) | (b / VB));
    const float v0 = (float)(vv & 0xffff) - 127.f, v1 = (float)(vv >> 16) - 127.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float p[4];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float *Mp = &Ms[b][nt * 8 + 2 * j + c];
            const float x0 = s[nt][c] + v0, x1 = s[nt][c + 2] + v1;
            __syncwarp();
            float M = *Mp;
            const float t = column_max(fmaxf(x0, x1));
            if (t > M + (DEC_WIDE_MAX - DEC_WIDE_TOP)) {
                const float f = ex2(M - t);
                M = t;
                o[nt][b][0][c] *= f; o[nt][b][0][c + 2] *= f;
                o[nt][b][1][c] *= f; o[nt][b][1][c + 2] *= f;
            }
            __syncwarp();
            if (lane < 4) *Mp = M;
            p[c] = ex2((x0 - M) + DEC_WIDE_TOP);
            p[c + 2] = ex2((x1 - M) + DEC_WIDE_TOP);
        }
        weights_f16<TERMS>(p, w, nt);
    }
}

template <int DH, int NT, int TERMS>
struct DecSmem {
    static constexpr int R = 8 * NT, LD = DH + 4;
    // (the stages are empty when a piece's results are added up)
    union {
        alignas(16) float o[DEC_WARPS][R][LD];
        alignas(16) uint8_t st[DEC_WARPS][DecFrag<DH>::STAGES][DecFrag<DH>::STAGE];
    };
    float m[DEC_WARPS][R], l[DEC_WARPS][R], M[DEC_WARPS][DH / 32][R];      // M: the wide form's references
    alignas(16) uint16_t sc[DEC_WARPS][4][DH / 32][4];     // f16 2^(vs - anchor): [j][block][tokens 2j, 2j+1, 2j+8, 2j+9]
    alignas(16) uint4 q[TERMS][NT][DH / 32][32];           // operand fragments of q, by lane
    int hi[R], lo[R];                                      // first and last token that a row sees
    PlanSmem<DEC_THREADS> plan;
};

template <int DH, int NT, bool F32>
// What bounds it: instructions, 350 per warp and 16 tokens of 128 dims.  16 warps per SM at 128 registers are better than 20 at 102
// (64 requests, 266,000 tokens: 35 against 39 us, when these were chosen) and 12 at 168 (43); wider accumulators (256 dims, or 16 rows of 128) keep 8 warps at 255
// (37 us at 112,000 tokens of 256; 38 with 12 warps).  Tokens come by asynchronous copies one group ahead (35 us; 38 with loads into
// registers behind their last use), two ahead gain nothing.  The stages share their place with the results: with a place of their own, 35.3,
// and 33.2 against 32.0 for one request of 131,072, since more shared memory leaves less of L1.
__global__ void __launch_bounds__(DEC_THREADS, NT * DH <= 128 ? 4 : 2)
k_attn_decode(AttnArgs a, int all, AttnPart *__restrict__ desc, float *__restrict__ part) {
    constexpr int NB = DH / 32, R = 8 * NT, TERMS = F32 ? 2 : 1;
    using Frag = DecFrag<DH>;
    Q36_GDS();
    extern __shared__ __align__(16) uint8_t smem_raw[];
    DecSmem<DH, NT, F32 ? 2 : 1> &sm = *reinterpret_cast<DecSmem<DH, NT, F32 ? 2 : 1> *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
    const SpanRule rule{R, DEC_UNIT, all};
    PlanPos pos;
    if (!plan_start<DEC_THREADS>(a, rule, DEC_WARPS, sm.plan, pos)) {
        if (tid == 0) desc[blockIdx.x].parts = 0;
        return;
    }
    if (tid == 0) desc[blockIdx.x].parts = 0;
    bool first = true;
    while (pos.at < pos.end) {
        const PlanSeg sg = plan_segment(pos);
        // ---- q: operand fragments of the row tile, lane = (row g, quarter j): dims 32b + 8j + 4s + 0..3.  They are the same for
        // every warp and stay in shared memory: a read per block and group costs less than the registers.
        float fac[NT][2];       // scale * log2(e) / 2^(power of two of the row), of columns 2j, 2j + 1
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = sg.rt * R + nt * 8 + g, rows = sg.n * a.G;
            const bool in = r < rows;
            const int i = in ? r / a.G : 0, hq = sg.hk * a.G + (in ? r - i * a.G : 0);
            float x[NB][8];
            float am = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                load8(a.q, (size_t)(sg.t0 + i) * a.q_stride + (size_t)hq * DH + 32 * b + 8 * j, !F32, x[b]);
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    x[b][c] = in ? x[b][c] : 0.f;
                    am = fmaxf(am, fabsf(x[b][c]));
                }
            }
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
            const int ea = (int)(__float_as_uint(am) >> 23) - 127;                     // amax in [2^ea, 2^(ea+1))
            const int up = am > 0.f ? min(14 - ea, 126) : 0;
            const float f = __uint_as_float((uint32_t)(up + 127) << 23), inv = a.scale2 * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (b % DEC_WARPS != warp) continue;
                uint32_t h[4], t[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float x0 = x[b][2 * c] * f, x1 = x[b][2 * c + 1] * f;
                    h[c] = pack_f16(x0, x1);
                    const float2 back = unpack_f16(h[c]);
                    t[c] = pack_f16(x0 - back.x, x1 - back.y);
                }
                sm.q[0][nt][b][lane] = make_uint4(h[0], h[1], h[2], h[3]);
                if constexpr (F32) sm.q[1][nt][b][lane] = make_uint4(t[0], t[1], t[2], t[3]);
            }
            const int p = sg.len - sg.n + i;
            if (warp == 0 && j == 0) {
                sm.hi[nt * 8 + g] = in ? p : -1;
                sm.lo[nt * 8 + g] = a.window > 0 ? p - a.window + 1 : 0;
            }
#pragma unroll
            for (int c = 0; c < 2; c++) fac[nt][c] = __shfl_sync(0xffffffffu, inv, 8 * j + 4 * c);
        }
        __syncthreads();
        // tokens that every row of the tile sees (rows beyond the last one see none: their tile is never interior; its last rows'
        // results are not stored)
        const int i_first = sg.rt * R / a.G, i_last = min(sg.rt * R + R - 1, sg.n * a.G - 1) / a.G;
        const int any_hi = sg.len - sg.n + i_last, any_lo = a.window > 0 ? sg.len - sg.n + i_first - a.window + 1 : 0;
        const int all_hi = sg.len - sg.n + i_first, all_lo = a.window > 0 ? sg.len - sg.n + i_last - a.window + 1 : 0;

        float m[NT][2], l[NT][2], o[NT][NB][2][4];
        int anchor = 0;          // 0: no group read yet
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int c = 0; c < 2; c++) { m[nt][c] = DEC_NONE; l[nt][c] = 0.f; }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[nt][b][u][c] = 0.f;
        }

        // ---- this warp's groups: a quarter of the piece.  Block ids come 32 groups at a time, one per lane.
        const int *row = a.table + (size_t)sg.b * a.max_blocks;
        const int n_all = sg.u1 - sg.u0, first_mine = n_all * warp / DEC_WARPS, n_mine = n_all * (warp + 1) / DEC_WARPS - first_mine;
        const int unit0 = sg.u_first + sg.u0 + first_mine;
        const uint8_t *head_base = a.kv.base + (size_t)sg.hk * a.kv.region();
        const uint32_t block_bytes = (uint32_t)(a.kv.region() * a.kv.Hkv);
        // a lane's part of the addresses: codes of K and V, scales of K and V (of 64 dims a token has two bytes of scales: the word with them)
        const uint32_t sc_row = (NB == 2 ? g & ~1 : g) * NB;
        const uint32_t lane_k = g * (DH / 2) + j * (DH / 8), lane_v = a.kv.bs * (DH / 2) + j * DH + g * (DH / 8), lane_ks = a.kv.bs * DH + sc_row,
                       lane_vs = lane_ks + a.kv.bs * NB;
        int ids = -1;
        // group k's page and its first token there; false when the group is not there
        auto page_of = [&](int k, const uint8_t *&reg, int &t) {
            if ((k & 31) == 0) {
                const int col = (unit0 + k + lane) * DEC_UNIT >> a.kv.log_bs;
                ids = k + lane < n_mine && col < a.max_blocks ? row[col] : -1;
            }
            const int id = __shfl_sync(0xffffffffu, ids, k & 31);
            t = (unit0 + k) * DEC_UNIT & (a.kv.bs - 1);
            reg = head_base + (size_t)(uint32_t)id * block_bytes;
            return (unsigned)id < (unsigned)a.kv.n_blocks;
        };
        // Groups are asked for one ahead; `there`: a bit per stage, whether its group exists.
        constexpr int ST = Frag::STAGES;
        Frag f;
        uint32_t there = 0;
        uint8_t *stages = sm.st[warp][0];
        auto ask = [&](int k) {
            const uint8_t *reg;
            int t;
            const uint32_t s = (uint32_t)k % ST;
            const bool is = k < n_mine && page_of(k, reg, t);
            if (is)
                Frag::copy((uint32_t)__cvta_generic_to_shared(stages) + s * Frag::STAGE, reg + t * (DH / 2) + lane_k, reg + t * (DH / 2) + lane_v, reg + t * NB + lane_ks,
                           reg + t * NB + lane_vs, lane);
            cp_commit();
            there = (there & ~(1u << s)) | (uint32_t)is << s;
        };
        const uint8_t *st = stages;
        // group k's stage, and whether there is anything in it
        auto arrive = [&](int k) {
            ask(k + ST - 1);
            cp_wait<ST - 1>();
            const uint32_t s = (uint32_t)k % ST;
            st = stages + s * Frag::STAGE;
            return (there >> s & 1) != 0;
        };
#pragma unroll
        for (int k = 0; k < ST - 1; k++) ask(k);
        int k = 0, tok = 0;
        bool inner = false;
        float s[NT][4];
        uint32_t w[TERMS][NT][2];
        // S of the group (log2 units), -infinity where a row does not see the token; m moved when needed
        auto scores = [&](bool is_wide) {
            f.get_k(st, lane);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[nt][c] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t k0[4], k1[4];
                e2m1x8_to_f16x2(f.k[0][b], k0);
                e2m1x8_to_f16x2(f.k[1][b], k1);
                float sc0 = __uint_as_float(((f.ks[0][b / 4] >> (8 * (b & 3))) & 0xff) << 23);
                float sc1 = __uint_as_float(((f.ks[1][b / 4] >> (8 * (b & 3))) & 0xff) << 23);
                if (is_wide) { sc0 *= DEC_K_DOWN; sc1 *= DEC_K_DOWN; }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < TERMS; t++) {
                        const uint4 q = sm.q[t][nt][b][lane];
                        mma_f16(c, k0[0], k1[0], k0[1], k1[1], q.x, q.y);
                        mma_f16(c, k0[2], k1[2], k0[3], k1[3], q.z, q.w);
                    }
                    s[nt][0] = fmaf(c[0], sc0, s[nt][0]);
                    s[nt][1] = fmaf(c[1], sc0, s[nt][1]);
                    s[nt][2] = fmaf(c[2], sc1, s[nt][2]);
                    s[nt][3] = fmaf(c[3], sc1, s[nt][3]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[nt][c] = is_wide ? s[nt][c] * fac[nt][c & 1] * (1.f / DEC_K_DOWN) : s[nt][c] * fac[nt][c & 1];
            if (!inner) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int tt = tok + g + (c >> 1) * 8, r = nt * 8 + 2 * j + (c & 1);
                        if (tt > sm.hi[r] || tt < sm.lo[r]) s[nt][c] = -INFINITY;
                    }
            }
            bool move = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) move |= fmaxf(s[nt][c], s[nt][c + 2]) > m[nt][c] + DEC_MAX;
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const float mn = fmaxf(m[nt][c], column_max(fmaxf(s[nt][c], s[nt][c + 2])) - DEC_TOP), by = ex2(m[nt][c] - mn);
                        l[nt][c] *= by;
                        if (is_wide && lane < 4) {
                            // (they are relative to m)
#pragma unroll
                            for (int b = 0; b < NB; b++) {
                                float *M = &sm.M[warp][b][nt * 8 + 2 * j + c];
                                *M = fmaxf(*M + (m[nt][c] - mn), DEC_NONE);
                            }
                        }
                        m[nt][c] = mn;
                        if (!is_wide) {
#pragma unroll
                            for (int b = 0; b < NB; b++)
#pragma unroll
                                for (int u = 0; u < 2; u++) { o[nt][b][u][c] *= by; o[nt][b][u][c + 2] *= by; }
                        }
                    }
            }
        };
        // the f16 operand of two blocks of V: rows dims 4g + 2u (+1), columns tokens
        auto v_codes = [&](int b2, uint32_t (&ev)[2][4], uint32_t (&od)[2][4]) {
#pragma unroll
            for (int e = 0; e < 2; e++) {       // [token pair j, j + 4][byte: block 2 b2 codes 0/1, 2/3, block 2 b2 + 1 codes ...]
                const uint32_t A = f.v[e][b2], B = f.v[e][NB / 2 + b2];
                e2m1x8_to_f16x2((A & 0x0f0f0f0fu) | ((B << 4) & 0xf0f0f0f0u), ev[e]);
                e2m1x8_to_f16x2(((A >> 4) & 0x0f0f0f0fu) | (B & 0xf0f0f0f0u), od[e]);
            }
        };
#pragma unroll 1
        for (; k < n_mine; k++) {
            if (!arrive(k)) continue;
            f.get_vs(st, lane);
            tok = (unit0 + k) * DEC_UNIT;
            inner = tok >= all_lo && tok + DEC_UNIT - 1 <= all_hi;
            // V exponents (own: tokens g, g + 8, blocks VB j ..): inside the window?  vs - (anchor - 8) of both tokens at once (a
            // borrow between them comes with a low half that is outside); only when that says no, token by token.
            auto seen = [&](int e) { const int t = tok + g + 8 * e; return t <= any_hi && t >= any_lo; };
            if (anchor == 0) {
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < Frag::VB; c++) top = max(top, max(seen(0) ? f.vs[c] & 0xffff : 0u, seen(1) ? f.vs[c] >> 16 : 0u));
                anchor = (int)__reduce_max_sync(0xffffffffu, top);
            }
            constexpr uint32_t WIDTH2 = (DEC_WIN_LO + DEC_WIN_HI) * 0x10001u;
            uint32_t d[Frag::VB], far = Frag::high_k(st, 0, lane) | Frag::high_k(st, 1, lane);
#pragma unroll
            for (int c = 0; c < Frag::VB; c++) {
                d[c] = f.vs[c] - (uint32_t)(anchor - DEC_WIN_LO) * 0x10001u;
                far |= __vmaxu2(d[c], WIDTH2) ^ WIDTH2;
            }
            if (__any_sync(0xffffffffu, far != 0)) {
                bool out = (seen(0) && Frag::high_k(st, 0, lane)) || (seen(1) && Frag::high_k(st, 1, lane));
#pragma unroll
                for (int c = 0; c < Frag::VB; c++) {
                    const int v0 = f.vs[c] & 0xffff, v1 = f.vs[c] >> 16, e0 = v0 - anchor + DEC_WIN_LO, e1 = v1 - anchor + DEC_WIN_LO;
                    const bool in0 = (unsigned)e0 <= (unsigned)(DEC_WIN_LO + DEC_WIN_HI), in1 = (unsigned)e1 <= (unsigned)(DEC_WIN_LO + DEC_WIN_HI);
                    out |= seen(0) && v0 > 1 && !in0;
                    out |= seen(1) && v1 > 1 && !in1;
                    // (scale byte 1, or a token that no row sees: a factor of -0)
                    d[c] = (in0 ? (uint32_t)e0 : DEC_NO_BLOCK) | (in1 ? (uint32_t)e1 : DEC_NO_BLOCK) << 16;
                }
                if (__any_sync(0xffffffffu, out)) break;
            }
            __syncwarp();
            if (NB >= 4 || j < NB) {
#pragma unroll
                for (int c = 0; c < Frag::VB; c++) {
                    // f16 2^(vs - anchor): exponent field vs - anchor + 15
                    const uint32_t e = (d[c] + (15 - DEC_WIN_LO) * 0x10001u) << 10;
                    uint16_t *to = sm.sc[warp][g >> 1][Frag::VB * j + c];
                    to[g & 1] = (uint16_t)e;
                    to[2 + (g & 1)] = (uint16_t)(e >> 16);
                }
            }
            scores(false);
            // weights, transposed into the narrow operand: (token 2j, 2j+1 | 2j+8, 2j+9) of row g
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float p[4];
#pragma unroll
                for (int c = 0; c < 4; c++) p[c] = ex2(s[nt][c] - m[nt][c & 1]);
                l[nt][0] += p[0] + p[2];
                l[nt][1] += p[1] + p[3];
                weights_f16<TERMS>(p, w, nt);
            }
            f.get_v(st, lane);
            __syncwarp();
#pragma unroll
            for (int b2 = 0; b2 < NB / 2; b2++) {
                uint32_t ev[2][4], od[2][4];
                v_codes(b2, ev, od);
#pragma unroll
                for (int bb = 0; bb < 2; bb++) {
                    const int b = 2 * b2 + bb;
                    const uint2 sc = *reinterpret_cast<const uint2 *>(sm.sc[warp][j][b]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int t = 0; t < TERMS; t++) {
                            const uint32_t x0 = hmul2(w[t][nt][0], sc.x), x1 = hmul2(w[t][nt][1], sc.y);
#pragma unroll
                            for (int u = 0; u < 2; u++)
                                mma_f16(o[nt][b][u], ev[0][2 * bb + u], od[0][2 * bb + u], ev[1][2 * bb + u], od[1][2 * bb + u], x0, x1);
                        }
                }
            }
        }
        const bool wide = k < n_mine;
        if (wide) {
            // The sums so far count 2^(m + anchor - 127).  What they are makes the reference, not the anchor, which may be another block's or a
            // weak token's, far above what comes here; where they are nothing, the next token does.
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        float (&r0)[4] = o[nt][b][0], (&r1)[4] = o[nt][b][1];
                        const float most = column_max(fmaxf(fmaxf(fabsf(r0[c]), fabsf(r0[c + 2])), fmaxf(fabsf(r1[c]), fabsf(r1[c + 2]))));
                        const float e = (float)max((int)(__float_as_uint(most) >> 23) - 127, -100), f = ex2(DEC_WIDE_TOP - e);
                        r0[c] *= f; r0[c + 2] *= f; r1[c] *= f; r1[c + 2] *= f;
                        if (lane < 4) sm.M[warp][b][nt * 8 + 2 * j + c] = most > 0.f ? (float)(anchor - 127) + e : DEC_NONE;
                    }
            __syncwarp();
#pragma unroll 1
            for (bool fresh = true; k < n_mine; k++, fresh = false) {
                if (!fresh && !arrive(k)) continue;      // (the first group is there)
                f.get_vs(st, lane);
                f.get_v(st, lane);
                tok = (unit0 + k) * DEC_UNIT;
                inner = tok >= all_lo && tok + DEC_UNIT - 1 <= all_hi;
                scores(true);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        s[nt][c] -= m[nt][c & 1];
                        l[nt][c & 1] += ex2(s[nt][c]);
                    }
#pragma unroll
                for (int b2 = 0; b2 < NB / 2; b2++) {
                    uint32_t ev[2][4], od[2][4];
                    v_codes(b2, ev, od);
#pragma unroll
                    for (int bb = 0; bb < 2; bb++) {
                        const int b = 2 * b2 + bb;
                        wide_weights<DH, NT, TERMS, Frag::VB>(sm.M[warp], f.vs, s, w, o, b, lane);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int t = 0; t < TERMS; t++)
#pragma unroll
                                for (int u = 0; u < 2; u++)
                                    mma_f16(o[nt][b][u], ev[0][2 * bb + u], od[0][2 * bb + u], ev[1][2 * bb + u], od[1][2 * bb + u], w[t][nt][0], w[t][nt][1]);
                    }
                }
            }
        }

        // ---- the warps' shares into one result
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
                if (g == 0) { sm.m[warp][nt * 8 + 2 * j + c] = m[nt][c]; sm.l[warp][nt * 8 + 2 * j + c] = l[nt][c]; }
            }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float ma2[2], lg[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int r = nt * 8 + 2 * j + c;
                float ma = sm.m[0][r], la = 0.f;
#pragma unroll
                for (int w = 1; w < DEC_WARPS; w++) ma = fmaxf(ma, sm.m[w][r]);
#pragma unroll
                for (int w = 0; w < DEC_WARPS; w++) la += sm.l[w][r] * ex2(sm.m[w][r] - ma);
                ma2[c] = ma;
                lg[c] = la == 0.f ? INFINITY : log2f(la);      // (nothing seen: a factor of 0)
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                // 2^(m + reference) / (2^ma la), the sum in the exponent: V may be as large or small as f32
                float f[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float ref = wide ? sm.M[warp][b][nt * 8 + 2 * j + c] - DEC_WIDE_TOP : (float)(anchor - 127);
                    f[c] = exp2f((m[nt][c] - ma2[c]) + (ref - lg[c]));
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int d = 32 * b + 4 * g + 2 * u;
                    *reinterpret_cast<float2 *>(&sm.o[warp][nt * 8 + 2 * j][d]) = make_float2(o[nt][b][u][0] * f[0], o[nt][b][u][2] * f[0]);
                    *reinterpret_cast<float2 *>(&sm.o[warp][nt * 8 + 2 * j + 1][d]) = make_float2(o[nt][b][u][1] * f[1], o[nt][b][u][3] * f[1]);
                }
            }
        }
        __syncthreads();
        const bool whole = sg.u0 == 0 && sg.u1 == sg.units;
        const int slot = 2 * blockIdx.x + (first ? 0 : 1);
        float *dst = part + (size_t)slot * attn_part_floats(R, DH);
        for (int e = tid; e < R * (DH / 4); e += DEC_THREADS) {
            const int r = e / (DH / 4), d = (e - r * (DH / 4)) * 4;
            float4 v = *reinterpret_cast<const float4 *>(&sm.o[0][r][d]);
#pragma unroll
            for (int w = 1; w < DEC_WARPS; w++) {
                const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][r][d]);
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            }
            if (!whole) *reinterpret_cast<float4 *>(dst + 2 * R + r * DH + d) = v;
            else attn_store(a, sg.t0, sg.n, sg.hk, sg.rt * R + r, d, v);
        }
        if (tid < R) {
            float ma = sm.m[0][tid], la = 0.f;
            for (int w = 1; w < DEC_WARPS; w++) ma = fmaxf(ma, sm.m[w][tid]);
            for (int w = 0; w < DEC_WARPS; w++) la += sm.l[w][tid] * ex2(sm.m[w][tid] - ma);
            if (!whole) { dst[2 * tid] = ma; dst[2 * tid + 1] = la; }
            else attn_store_lse(a, sg.t0, sg.n, sg.hk, sg.rt * R + tid, ma, la);
        }
        // the CTA that has a cut span's first piece says what belongs together
        if (tid == 0 && !whole && sg.u0 == 0) desc[blockIdx.x] = plan_parts(a, rule, sg, pos, slot);
        __syncthreads();
        first = false;
        plan_next(a, rule, sg, pos);
    }
}

template <int DH, int NT, bool F32>
static int run(const AttnArgs &a, int all, void *ws, cudaStream_t st) {
    static bool attr_done[MAX_DEVICES] = {false};
    static int occ[MAX_DEVICES] = {0};
    const int smem = sizeof(DecSmem<DH, NT, F32 ? 2 : 1>), dev = current_device();
    int rc;
    if (dev < 0) return Q36_MOE_EINVAL;
    if ((rc = ensure_smem_attr((const void *)k_attn_decode<DH, NT, F32>, smem, attr_done))) return rc;
    if (!occ[dev]) {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_attn_decode<DH, NT, F32>, DEC_THREADS, smem) != cudaSuccess || n < 1) return check_launch() ? Q36_MOE_ECUDA : Q36_MOE_EUNSUPPORTED;
        occ[dev] = min(n, DEC_MAX_OCC);
    }
    const int grid = sm_count() * occ[dev];
    AttnPart *desc = (AttnPart *)ws;
    float *part = (float *)((uint8_t *)ws + attn_desc_bytes(grid));
    launch_k(k_attn_decode<DH, NT, F32>, dim3(grid), dim3(DEC_THREADS), smem, st, a, all, desc, part);
    if ((rc = check_launch())) return rc;
    return launch_attn_join(a, 8 * NT, grid, desc, part, st);
}

// Rows per tile: 8, or 16 where that halves what is read and widened for no more instructions: 64-wide heads and f32 prompts, in calls
// that fill the GPU and without a tile that is half empty.  us with 8 / 16: 64 requests, 266,000 tokens, 16 query heads per kv head of 64
// 49 / 42, of 128 62 / 62, 20 query heads of 128 84 / 98; f32 prompt of 2048 394 / 336, of 8192 5690 / 4690; one request of 2000
// tokens 15 / 21.  256-wide heads have accumulators for 8.
static int decode_nt(const AttnArgs &a, int rows, int all) {
    const bool gains = a.kv.Dh == 64 || (a.kv.Dh == 128 && !a.q_bf16 && rows >= 64);
    return all && gains && (long long)a.T * a.G > 256 && (rows + 15) / 16 * 2 <= (rows + 7) / 8 ? 2 : 1;
}

uint64_t decode_ws_bytes(int Dh) {
    const int grid = sm_count() * DEC_MAX_OCC;
    return attn_desc_bytes(grid) + 2ull * grid * attn_part_floats(Dh == 256 ? 8 : 16, Dh) * 4;
}

// rows: of one request, at most; all: every request, not only those that the tile kernel leaves
int launch_decode(const AttnArgs &a, int rows, int all, void *ws, cudaStream_t st) {
    const bool f32 = !a.q_bf16;
    const int nt = decode_nt(a, rows, all);
    if (a.kv.Dh == 64) {
        if (nt == 1) return f32 ? run<64, 1, true>(a, all, ws, st) : run<64, 1, false>(a, all, ws, st);
        return f32 ? run<64, 2, true>(a, all, ws, st) : run<64, 2, false>(a, all, ws, st);
    }
    if (a.kv.Dh == 128) {
        if (!f32) return run<128, 1, false>(a, all, ws, st);
        return nt == 1 ? run<128, 1, true>(a, all, ws, st) : run<128, 2, true>(a, all, ws, st);
    }
    return f32 ? run<256, 1, true>(a, all, ws, st) : run<256, 1, false>(a, all, ws, st);
}

}  // namespace q36
