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
// to a reference per row and block of dims and rounds the weights of every block by themselves, which holds for any exponents.
// Blocks of zeros (scale byte 1) need no place in the window.
// The normaliser is the sum of the unrounded weights in f32.
// q enters as f16 after an exact power of two per row (bf16 and f16 fit); f32 activations enter as two f16 terms, and so do
// their weights, which leaves 2^-22.
//
// Work.  A unit is 16 tokens of one (request, kv head, row tile).  The units of all requests, in order, are cut into equal
// ranges, one per CTA, so that ragged lengths load every SM alike.  A range's first and last pieces may be parts of what a
// neighbour has the rest of: they go to the workspace and k_attn_join adds them up in a fixed order.
#include <math.h>

#include "attn_plan.cuh"

namespace q36 {

constexpr int DEC_WARPS = 4, DEC_THREADS = 32 * DEC_WARPS, DEC_UNIT = 16;
constexpr float DEC_NONE = -3.0e38f;      // "no token yet" of the running references: finite, so that differences stay defined
constexpr float DEC_TOP = 7.f, DEC_MAX = 11.f;        // log2 of the largest weight when the reference moves, and when it has to
constexpr int DEC_WIN_LO = 8, DEC_WIN_HI = 4;         // window of V exponents around the anchor
constexpr float DEC_WIDE_TOP = 11.f, DEC_WIDE_MAX = 15.f;   // the same with a reference per block of dims

// the four bytes of w, two E2M1 codes each (low nibble first), as f16x2
__device__ __forceinline__ void e2m1x8_to_f16x2(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
template <int W>
__device__ __forceinline__ void ld_words(const uint8_t *p, uint32_t (&r)[W]) {
    if constexpr (W == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        r[0] = v.x; r[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; i++) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i);
            r[4 * i] = v.x; r[4 * i + 1] = v.y; r[4 * i + 2] = v.z; r[4 * i + 3] = v.w;
        }
    }
}

// What a lane holds of 16 tokens.  Lane (g, j): g = lane / 4, j = lane % 4.
template <int DH>
struct DecFrag {
    static constexpr int NB = DH / 32, W = DH / 32, SW = (NB + 3) / 4, VB = NB >= 4 ? NB / 4 : 1;
    uint32_t k[2][W];      // K words of tokens g and g + 8: word b = dims 32b + 8j ..
    uint32_t v[2][W];      // V of token pairs j and j + 4, group g: first half token 2p, second half token 2p + 1
    uint32_t ks[2][SW];    // K scales of tokens g and g + 8
    uint32_t vs[2];        // V scales of tokens g and g + 8, blocks VB j .. (bytes)
    __device__ __forceinline__ void load(const uint8_t *reg, int bs, int tok, int g, int j) {
        const uint8_t *vc = reg + bs * (DH / 2), *ksp = reg + bs * DH, *vsp = ksp + bs * NB;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            ld_words<W>(reg + kv_k_off(tok + g + 8 * h, j, 0, DH), k[h]);
            ld_words<W>(vc + kv_v_off(tok + 2 * j + 8 * h, g, 0, DH), v[h]);
            const uint8_t *kp = ksp + (tok + g + 8 * h) * NB, *vp = vsp + (tok + g + 8 * h) * NB;
            if constexpr (NB == 2) ks[h][0] = __ldg(reinterpret_cast<const uint16_t *>(kp));
            else if constexpr (NB == 4) ks[h][0] = __ldg(reinterpret_cast<const uint32_t *>(kp));
            else { const uint2 u = __ldg(reinterpret_cast<const uint2 *>(kp)); ks[h][0] = u.x; ks[h][1] = u.y; }
            if constexpr (NB == 8) vs[h] = __ldg(reinterpret_cast<const uint16_t *>(vp) + j);
            else if constexpr (NB == 4) vs[h] = __ldg(vp + j);
            else vs[h] = __ldg(vp + (j & 1));
        }
    }
};

template <int DH, int NT>
struct DecSmem {
    static constexpr int R = 8 * NT, LD = DH + 4;
    alignas(16) float o[DEC_WARPS][R][LD];
    float m[DEC_WARPS][R], l[DEC_WARPS][R], M[DEC_WARPS][DH / 32][R];      // M: the wide form's references
    alignas(16) uint16_t sc[DEC_WARPS][4][DH / 32][4];     // f16 2^(vs - anchor): [j][block][tokens 2j, 2j+1, 2j+8, 2j+9]
    PlanSmem<DEC_THREADS> plan;
};

template <int DH, int NT, bool F32>
__global__ void __launch_bounds__(DEC_THREADS)
k_attn_decode(AttnArgs a, int all, AttnPart *__restrict__ desc, float *__restrict__ part) {
    constexpr int NB = DH / 32, R = 8 * NT, TERMS = F32 ? 2 : 1;
    using Frag = DecFrag<DH>;
    Q36_GDS();
    extern __shared__ __align__(16) uint8_t smem_raw[];
    DecSmem<DH, NT> &sm = *reinterpret_cast<DecSmem<DH, NT> *>(smem_raw);
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
        // ---- q: operand fragments of the row tile, lane = (row g, quarter j): dims 32b + 8j + 4s + 0..3
        uint32_t qf[TERMS][NT][NB][4];
        float fac[NT][2];       // scale * log2(e) / 2^(power of two of the row), of columns 2j, 2j + 1
        int hi[NT][2], lo[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = sg.rt * R + nt * 8 + g, rows = sg.n * a.G;
            const bool in = r < rows;
            const int i = in ? r / a.G : 0, hq = sg.hk * a.G + (in ? r - i * a.G : 0);
            float x[NB][8];
            float am = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const size_t e = (size_t)(sg.t0 + i) * a.q_stride + (size_t)hq * DH + 32 * b + 8 * j;
                if (!in) {
#pragma unroll
                    for (int c = 0; c < 8; c++) x[b][c] = 0.f;
                } else {
                    load8(a.q, e, !F32 || a.q_bf16, x[b]);
                }
#pragma unroll
                for (int c = 0; c < 8; c++) am = fmaxf(am, fabsf(x[b][c]));
            }
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
            const int ea = (int)(__float_as_uint(am) >> 23) - 127;                     // amax in [2^ea, 2^(ea+1))
            const int up = am > 0.f ? min(14 - ea, 126) : 0;
            const float f = __uint_as_float((uint32_t)(up + 127) << 23), inv = a.scale2 * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float x0 = x[b][2 * c] * f, x1 = x[b][2 * c + 1] * f;
                    qf[0][nt][b][c] = pack_f16(x0, x1);
                    if constexpr (F32) {
                        const float2 h = unpack_f16(qf[0][nt][b][c]);
                        qf[1][nt][b][c] = pack_f16(x0 - h.x, x1 - h.y);
                    }
                }
            const int p = sg.len - sg.n + i, l0 = a.window > 0 ? p - a.window + 1 : 0;
            const int ph = in ? p : -1;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                fac[nt][c] = __shfl_sync(0xffffffffu, inv, 8 * j + 4 * c);
                hi[nt][c] = __shfl_sync(0xffffffffu, ph, 8 * j + 4 * c);
                lo[nt][c] = __shfl_sync(0xffffffffu, l0, 8 * j + 4 * c);
            }
        }
        // tokens that every row of the tile sees (rows beyond the last one see none: their tile is never interior; its last rows'
        // results are not stored)
        const int i_first = sg.rt * R / a.G, i_last = min(sg.rt * R + R - 1, sg.n * a.G - 1) / a.G;
        const int any_hi = sg.len - sg.n + i_last, any_lo = a.window > 0 ? sg.len - sg.n + i_first - a.window + 1 : 0;
        const int all_hi = sg.len - sg.n + i_first, all_lo = a.window > 0 ? sg.len - sg.n + i_last - a.window + 1 : 0;

        float m[NT][2], l[NT][2], o[NT][NB][2][4];
        int anchor = 0;          // 0: no group read yet; -1: wide
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

        // ---- this warp's groups: every DEC_WARPS-th.  Block ids come 32 groups at a time, one per lane.
        const int *row = a.table + (size_t)sg.b * a.max_blocks;
        const int n_mine = (sg.u1 - sg.u0 - warp + DEC_WARPS - 1) / DEC_WARPS, unit0 = sg.u_first + sg.u0 + warp;
        int ids = -1;
        auto fetch_ids = [&](int k) {
            const int gi = k + lane;
            ids = -1;
            if (gi < n_mine) {
                const int col = ((unit0 + gi * DEC_WARPS) * DEC_UNIT) >> a.kv.log_bs;
                if (col < a.max_blocks) ids = __ldg(row + col);
            }
        };
        auto load_group = [&](int k, Frag &f) {
            if ((k & 31) == 0) fetch_ids(k);
            const int id = __shfl_sync(0xffffffffu, ids, k & 31);
            const bool ok = id >= 0 && id < a.kv.n_blocks;
            if (ok) f.load(a.kv.at(id, sg.hk), a.kv.bs, ((unit0 + k * DEC_WARPS) * DEC_UNIT) & (a.kv.bs - 1), g, j);
            return ok;
        };
        Frag cur, nxt;
        bool cur_ok = n_mine > 0 && load_group(0, cur);
        for (int k = 0; k < n_mine; k++) {
            const bool nxt_ok = k + 1 < n_mine && load_group(k + 1, nxt);
            if (cur_ok) {
                const int tok = (unit0 + k * DEC_WARPS) * DEC_UNIT;
                const bool inner = tok >= all_lo && tok + DEC_UNIT - 1 <= all_hi;
                // V exponents (own: tokens g, g + 8, blocks VB j ..): inside the window?
                if (anchor >= 0) {
                    int top = 0;
                    bool out = false;
                    const bool in0 = inner || (tok + g <= any_hi && tok + g >= any_lo), in1 = inner || (tok + g + 8 <= any_hi && tok + g + 8 >= any_lo);
                    if (anchor == 0) {
#pragma unroll
                        for (int c = 0; c < Frag::VB; c++)
                            top = max(top, max(in0 ? (int)(cur.vs[0] >> (8 * c)) & 0xff : 0, in1 ? (int)(cur.vs[1] >> (8 * c)) & 0xff : 0));
                        anchor = (int)__reduce_max_sync(0xffffffffu, (unsigned)top);
                    }
#pragma unroll
                    for (int c = 0; c < Frag::VB; c++) {
                        const int v0 = (int)(cur.vs[0] >> (8 * c)) & 0xff, v1 = (int)(cur.vs[1] >> (8 * c)) & 0xff;
                        out |= in0 && v0 > 1 && (unsigned)(v0 - anchor + DEC_WIN_LO) > (unsigned)(DEC_WIN_LO + DEC_WIN_HI);
                        out |= in1 && v1 > 1 && (unsigned)(v1 - anchor + DEC_WIN_LO) > (unsigned)(DEC_WIN_LO + DEC_WIN_HI);
                    }
                    __syncwarp();
                    if (__any_sync(0xffffffffu, out)) {
                        // the sums so far count 2^(m + anchor - 127)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int c = 0; c < 2; c++)
                                for (int b = g; b < NB; b += 8)
                                    sm.M[warp][b][nt * 8 + 2 * j + c] = m[nt][c] == DEC_NONE ? DEC_NONE : m[nt][c] + (float)(anchor - 127) + DEC_WIDE_TOP;
                        anchor = -1;
                        __syncwarp();
                    } else if (NB >= 4 || j < NB) {
#pragma unroll
                        for (int c = 0; c < Frag::VB; c++) {
                            const int b = Frag::VB * j + c;
                            const int e0 = ((int)(cur.vs[0] >> (8 * c)) & 0xff) - anchor + 15, e1 = ((int)(cur.vs[1] >> (8 * c)) & 0xff) - anchor + 15;
                            // (a block of zeros, or a token that no row sees: any finite factor)
                            sm.sc[warp][g >> 1][b][g & 1] = (uint16_t)(min(max(e0, 0), 30) << 10);
                            sm.sc[warp][g >> 1][b][2 + (g & 1)] = (uint16_t)(min(max(e1, 0), 30) << 10);
                        }
                    }
                }
                // scores
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) s[nt][c] = 0.f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t k0[4], k1[4];
                    e2m1x8_to_f16x2(cur.k[0][b], k0);
                    e2m1x8_to_f16x2(cur.k[1][b], k1);
                    const float sc0 = __uint_as_float(((cur.ks[0][b / 4] >> (8 * (b & 3))) & 0xff) << 23);
                    const float sc1 = __uint_as_float(((cur.ks[1][b / 4] >> (8 * (b & 3))) & 0xff) << 23);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int t = 0; t < TERMS; t++) {
                            mma_f16(c, k0[0], k1[0], k0[1], k1[1], qf[t][nt][b][0], qf[t][nt][b][1]);
                            mma_f16(c, k0[2], k1[2], k0[3], k1[3], qf[t][nt][b][2], qf[t][nt][b][3]);
                        }
                        s[nt][0] = fmaf(c[0], sc0, s[nt][0]);
                        s[nt][1] = fmaf(c[1], sc0, s[nt][1]);
                        s[nt][2] = fmaf(c[2], sc1, s[nt][2]);
                        s[nt][3] = fmaf(c[3], sc1, s[nt][3]);
                    }
                }
                bool move = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        float x = s[nt][c] * fac[nt][c & 1];
                        if (!inner) {
                            const int tt = tok + g + (c >> 1) * 8;
                            if (tt > hi[nt][c & 1] || tt < lo[nt][c & 1]) x = -INFINITY;
                        }
                        s[nt][c] = x;
                        move |= x > m[nt][c & 1] + DEC_MAX;
                    }
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const float mn = fmaxf(m[nt][c], column_max(fmaxf(s[nt][c], s[nt][c + 2])) - DEC_TOP), f = ex2(m[nt][c] - mn);
                            l[nt][c] *= f;
                            m[nt][c] = mn;
                            if (anchor >= 0) {
#pragma unroll
                                for (int b = 0; b < NB; b++)
#pragma unroll
                                    for (int u = 0; u < 2; u++) { o[nt][b][u][c] *= f; o[nt][b][u][c + 2] *= f; }
                            }
                        }
                }
                // weights, transposed into the narrow operand: (token 2j, 2j+1 | 2j+8, 2j+9) of row g
                uint32_t w[TERMS][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float p[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        p[c] = ex2(s[nt][c] - m[nt][c & 1]);
                        l[nt][c & 1] += p[c];
                    }
                    if (anchor >= 0) weights_f16<TERMS>(p, w, nt);
                }
                __syncwarp();
                // output: A = V codes, rows dims 4g + 2u (+1), columns tokens
#pragma unroll
                for (int b2 = 0; b2 < NB / 2; b2++) {
                    uint32_t ev[2][4], od[2][4];       // [token pair j, j + 4][byte: block 2 b2 codes 0/1, 2/3, block 2 b2 + 1 codes ...]
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t A = cur.v[h][b2], B = cur.v[h][NB / 2 + b2];
                        e2m1x8_to_f16x2((A & 0x0f0f0f0fu) | ((B << 4) & 0xf0f0f0f0u), ev[h]);
                        e2m1x8_to_f16x2(((A >> 4) & 0x0f0f0f0fu) | (B & 0xf0f0f0f0u), od[h]);
                    }
#pragma unroll
                    for (int bb = 0; bb < 2; bb++) {
                        const int b = 2 * b2 + bb;
                        uint2 sc = make_uint2(0x3c003c00u, 0x3c003c00u);
                        if (anchor >= 0) {
                            sc = *reinterpret_cast<const uint2 *>(sm.sc[warp][j][b]);
                        } else {
                            // weights of this block alone: 2^(S + vs - M), M per row and block
                            const float v0 = (float)__shfl_sync(0xffffffffu, (int)(cur.vs[0] >> (8 * (b % Frag::VB))) & 0xff, (lane & 28) | (b / Frag::VB)) - 127.f;
                            const float v1 = (float)__shfl_sync(0xffffffffu, (int)(cur.vs[1] >> (8 * (b % Frag::VB))) & 0xff, (lane & 28) | (b / Frag::VB)) - 127.f;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                float p[4];
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    float *Mp = &sm.M[warp][b][nt * 8 + 2 * j + c];
                                    const float x0 = s[nt][c] + v0, x1 = s[nt][c + 2] + v1, M0 = *Mp;
                                    float M = M0;
                                    const float t = column_max(fmaxf(x0, x1));
                                    if (t > M + (DEC_WIDE_MAX - DEC_WIDE_TOP)) {
                                        const float f = ex2(M - t);
                                        M = t;
                                        o[nt][b][0][c] *= f; o[nt][b][0][c + 2] *= f;
                                        o[nt][b][1][c] *= f; o[nt][b][1][c + 2] *= f;
                                    }
                                    __syncwarp();
                                    if (g == 0) *Mp = M;
                                    p[c] = ex2(x0 - (M - DEC_WIDE_TOP));
                                    p[c + 2] = ex2(x1 - (M - DEC_WIDE_TOP));
                                }
                                weights_f16<TERMS>(p, w, nt);
                            }
                        }
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
            cur = nxt;
            cur_ok = nxt_ok;
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
                // 2^reference / (2^ma la), the sum in the exponent: V may be as large or small as f32
                float f[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float ref = anchor >= 0 ? m[nt][c] : sm.M[warp][b][nt * 8 + 2 * j + c];
                    f[c] = exp2f((ref - ma2[c]) + ((anchor >= 0 ? (float)(anchor - 127) : -DEC_WIDE_TOP) - lg[c]));
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
    const int smem = sizeof(DecSmem<DH, NT>), dev = current_device();
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

// Rows per tile: 8 while a request's rows fit them, else 16 (halves what the cache is read); 256-wide heads keep 8, whose
// accumulators are what 16 rows of 128 are.
static int decode_nt(int Dh, int rows) { return Dh == 256 || rows <= 8 ? 1 : 2; }

uint64_t decode_ws_bytes(int Dh, int rows) {
    const int grid = sm_count() * DEC_MAX_OCC;
    return attn_desc_bytes(grid) + 2ull * grid * attn_part_floats(8 * decode_nt(Dh, rows), Dh) * 4;
}

int launch_decode(const AttnArgs &a, int rows, int all, void *ws, cudaStream_t st) {
    const bool f32 = !a.q_bf16;
    const int nt = decode_nt(a.kv.Dh, rows);
    if (a.kv.Dh == 64) {
        if (nt == 1) return f32 ? run<64, 1, true>(a, all, ws, st) : run<64, 1, false>(a, all, ws, st);
        return f32 ? run<64, 2, true>(a, all, ws, st) : run<64, 2, false>(a, all, ws, st);
    }
    if (a.kv.Dh == 128) {
        if (nt == 1) return f32 ? run<128, 1, true>(a, all, ws, st) : run<128, 1, false>(a, all, ws, st);
        return f32 ? run<128, 2, true>(a, all, ws, st) : run<128, 2, false>(a, all, ws, st);
    }
    return f32 ? run<256, 1, true>(a, all, ws, st) : run<256, 1, false>(a, all, ws, st);
}

}  // namespace q36
