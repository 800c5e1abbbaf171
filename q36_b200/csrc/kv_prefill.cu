// Attention of many rows per request over the paged 4-bit cache, bf16: prompts and prompt chunks.
//
// Rows are (new token, query head of the kv head's group): a tile of 256 rows (128 at 256-wide heads) shares K and V, so that the
// cache is read and widened to bf16 once for all of them.  E2M1 times a power of two is exact in bf16.
// One CTA, tiles of 64 cached tokens:
//   warps 0-3, 4-7     softmax of 128 rows each, a row per thread with its scores in registers: maximum, 2^(S - m) rounded to bf16
//                      once (half a step 2^-8, as the output's), the sum of the unrounded weights in f32
//   warps 8-11, 12-15  K, V: 4-bit rows -> bf16 operand tiles in shared memory (128-byte swizzle)
//   warps 16 - 19      S = Q K^T and O += P V of each row tile on tcgen05 (f32 in TMEM; P is read from TMEM, where it takes S's
//                      place), an issuing warp for each, since they wait for different things
// Every row tile has two S, so that the products of a tile run while the softmax is at the one before.
// m is a lagging maximum: O is rescaled (in TMEM) only when a row would pass 2^8.
//
// What bounds it: nothing alone.  A tile takes 2300 cycles (2048 tokens behind 32,768, 16 heads of 128 on 2: 589 us, 962 TFLOP/s; prompt of
// 8192 339 us, 811).  The tensor pipe needs 1320 of them (an MMA of 128 x 64 x 16 with both operands in shared memory takes 50 cycles,
// shared memory's rate, one of 128 x 128 x 16 with P in TMEM 65), the exponentials 1070, the ALU 1330, issue slots two thirds.  Without the
// exponentials the time stays, with twice the widening warps too, with both it falls by a tenth.  Tried without gain: a polynomial for
// some of the exponentials, turns between the two row tiles' exponentials, sleeping waits, other register splits.
//
// Work: the spans (kv head, row tile) of all long requests, measured in the tokens they see, are cut into equal ranges, one per CTA;
// cuts are moved down to tile boundaries.  Cut spans are joined as in the decode kernel.
#include <math.h>

#include "attn_plan.cuh"
#include "tc_ptx.cuh"

namespace q36 {

constexpr int PF_THREADS = 20 * 32;
// registers after the roles part: softmax, widening, issuers; 640 threads start with 96 each
constexpr int PF_REGS_SOFTMAX = 120, PF_REGS_WIDEN = 88, PF_REGS_ISSUE = 64;
static_assert(2 * PF_REGS_SOFTMAX + 2 * PF_REGS_WIDEN + PF_REGS_ISSUE <= 5 * 96, "the block's registers");

template <int DH>
struct PfCfg {
    static constexpr int NQ = DH == 256 ? 1 : 2, R = 128 * NQ, KT = 64, STAGES = DH == 256 ? 2 : 4;
    static constexpr int NB = DH / 32, BPT = NB / 2;                   // scale blocks, and those a widening thread has
    static constexpr int Q_BYTES = 128 * DH * 2, T_BYTES = KT * DH * 2;
    static constexpr int SMEM = NQ * Q_BYTES + 2 * STAGES * T_BYTES + 1024;
    static constexpr int TM_S = KT, TM_O0 = 2 * NQ * KT;               // columns: two S of each row tile, then O of each
    static constexpr int TMEM = 512;
};
constexpr float PF_NONE = -3.0e38f;      // "no token yet": finite, so that differences stay defined
constexpr float PF_GROW = 8.f;
constexpr float PF_LARGE = 1 << 20;
// V is widened 2^32 lower than it is, so that weights of up to 2^8 on as many tokens as memory holds stay in f32 at any of its exponents
// (infinities are stored as 6 * 2^125); what falls out is below 2^-92.
constexpr int PF_V_DOWN = 32;
// What a span costs beside its tokens (Q in, results out, the pipeline's start), in tokens.  us at 192 / 320 / 448 / 640 / 768: prompt of 8192,
// 128-wide heads (2 x 256 spans) 414 / 359 / 338 / 343 / 346, 64-wide 301 / 283 / 285 / 290 / 292; of 4096, 256-wide (2 x 256 spans of half the
// rows) 318 / 268 / 260 / 267 / 271.
constexpr int PF_SPAN = 448;
constexpr int PF_MIN = 1024;        // the smallest range of a CTA
// Places for the bad pages of a tile, which go from the group that widens K to the softmax without a barrier of their own.  K runs up to 9
// tiles ahead of a softmax: behind a span whose second row tile is empty, that tile's issuers pass the stages on, so only V holds K back.
// K's tile X + 10 needs S of X + 6, that the product of X + 4, that V of X + 4, that the second row tile's product of X, and that its softmax of X.
constexpr int PF_BAD_RING = 16;
__device__ int g_prefill_status;         // where a wait gave up (0: nowhere)

// ---------------------------------------------------------------- plan
// Span rt of a request: tokens c rt .. of the new ones (c whole tokens of G rows); it sees cached tokens [lo, hi).  Its size is
// hi - lo + PF_SPAN, which is piecewise linear in rt: prefix sums have a closed form.
struct PfSeq { int t0, n, len, c, tiles; };
__device__ __forceinline__ long long sum_pos(long long a, long long c, long long n) {      // sum over x < n of max(0, a + c x)
    long long x0 = a < 0 ? (-a + c - 1) / c : 0;
    if (x0 >= n) return 0;
    const long long k = n - x0, f = a + c * x0;
    return k * f + c * (k * (k - 1) / 2);
}
__device__ __forceinline__ PfSeq pf_seq(const AttnArgs &a, int R, int b) {
    PfSeq s;
    seq_span(a, b, s.t0, s.n, s.len);
    s.c = R / a.G;
    s.tiles = is_long(a, s.n * a.G, s.len) ? (s.n + s.c - 1) / s.c : 0;
    return s;
}
__device__ __forceinline__ void pf_range(const AttnArgs &a, const PfSeq &s, int rt, int &lo, int &hi) {
    const int base = s.len - s.n;
    hi = max(0, base + min((rt + 1) * s.c, s.n));
    lo = a.window > 0 ? min(max(0, base + rt * s.c - a.window + 1), hi) : 0;
}
// units of the row tiles before rt
__device__ __forceinline__ long long pf_prefix(const AttnArgs &a, const PfSeq &s, int rt) {
    const long long base = s.len - s.n;
    long long u = sum_pos(base + s.c, s.c, rt) + (long long)rt * PF_SPAN;
    if (rt > 0 && (long long)rt * s.c > s.n) u += max(0ll, base + s.n) - max(0ll, base + (long long)rt * s.c);     // the last tile is shorter
    if (a.window > 0) u -= sum_pos(base - a.window + 1, s.c, rt);
    return u;
}
struct PfPos { long long at, end, per, seq_base, span_base; int b, hk, rt; PfSeq s; };
__device__ __forceinline__ void pf_locate(const AttnArgs &a, int R, PfPos &p) {
    long long one;
    for (;;) {
        p.s = pf_seq(a, R, p.b);
        one = pf_prefix(a, p.s, p.s.tiles);
        if (p.at < p.seq_base + one * a.kv.Hkv) break;
        p.seq_base += one * a.kv.Hkv;
        p.b++;
    }
    const long long off = p.at - p.seq_base;
    p.hk = (int)(off / one);
    const long long in = off - p.hk * one;
    int lo = 0, hi = p.s.tiles;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (pf_prefix(a, p.s, m) <= in) lo = m; else hi = m;
    }
    p.rt = lo;
    p.span_base = p.seq_base + p.hk * one + pf_prefix(a, p.s, lo);
}
struct PfSeg { int lo, hi, j0, j1, whole, head; long long units; };     // key tiles [j0, j1); head: this is the span's first piece
__device__ __forceinline__ PfSeg pf_segment(const AttnArgs &a, int KT, const PfPos &p) {
    PfSeg g;
    pf_range(a, p.s, p.rt, g.lo, g.hi);
    g.units = (long long)(g.hi - g.lo) + PF_SPAN;
    const long long y0 = p.at - p.span_base, y1 = min(g.units, p.end - p.span_base);
    g.head = y0 == 0;
    g.whole = g.head && y1 == g.units;
    const int first = g.lo / KT, last = max((g.hi + KT - 1) / KT, first + 1);
    g.j0 = y0 == 0 ? first : min((int)((g.lo + y0) / KT), last);
    g.j1 = y1 == g.units ? last : min((int)((g.lo + y1) / KT), last);
    return g;
}
// The span behind this one (spans of a request: row tiles of one kv head after the other); false behind the range.
__device__ __forceinline__ bool pf_next(const AttnArgs &a, int R, const PfSeg &g, PfPos &p) {
    p.at = min(p.span_base + g.units, p.end);
    if (p.at >= p.end) return false;
    p.span_base = p.at;
    if (++p.rt < p.s.tiles) return true;
    p.rt = 0;
    if (++p.hk < a.kv.Hkv) return true;
    p.hk = 0;
    do p.s = pf_seq(a, R, ++p.b); while (p.s.tiles == 0);
    return true;
}

// ---------------------------------------------------------------- 4 bits -> bf16
// The eight magnitudes of a block as bf16, high and low bytes apart: eight bytes each, picked by the three magnitude bits of a code.
struct Lut { uint32_t ha, hb, la, lb; };
// `has` false: a token that is not there, all zeros.
__device__ __forceinline__ Lut make_lut(uint32_t s, bool has) {
    const uint32_t one = has ? 0x00800080u : 0u;
    const uint32_t p23 = s * one + (has ? 0x00400000u : 0u), p45 = p23 + one, p67 = p45 + one, p01 = has ? (s - 1) << 23 : 0u;
    return Lut{__byte_perm(p01, p23, 0x7531), __byte_perm(p45, p67, 0x7531), __byte_perm(p01, p23, 0x6420), __byte_perm(p45, p67, 0x6420)};
}
__device__ __forceinline__ void widen4(const Lut &t, uint32_t sel, uint32_t sign, uint32_t &x, uint32_t &y) {
    const uint32_t h = __byte_perm(t.ha, t.hb, sel) | (sign & 0x80808080u), l = __byte_perm(t.la, t.lb, sel);
    x = __byte_perm(l, h, 0x5140);
    y = __byte_perm(l, h, 0x7362);
}
__device__ __forceinline__ uint32_t prmt_sign(uint32_t a, uint32_t b, uint32_t sel) {      // bytes of 0xff / 0x00 by sign bits
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// eight codes (low nibble first) -> eight bf16
__device__ __forceinline__ uint4 widen8(const Lut &t, uint32_t w) {
    uint4 o;
    const uint32_t m = w & 0x77777777u, w4 = w << 4;
    widen4(t, m, prmt_sign(w4, w, 0xd9c8), o.x, o.y);
    widen4(t, m >> 16, prmt_sign(w4, w, 0xfbea), o.z, o.w);
    return o;
}

// ---------------------------------------------------------------- tcgen05
__device__ __forceinline__ void pf_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// operand whose contiguous direction is N (the dims): 64 of them per 128-byte row, rows (tokens) in groups of 8, panels of 64 dims
// `panel` bytes apart
__device__ __forceinline__ uint64_t desc_n_major(uint32_t saddr, uint32_t panel) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ float pf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&r);
}

// Every wait names a phase by its parity, so no barrier may be two phases on from one that is still to be awaited: the P / O barriers
// are one per place, whose next phase needs what follows the wait.
struct PfBars { uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2][2], p_full[2][2], o_done[2][2], o_last[2], q_full[2]; };      // o_done: product with the P in one of two places, o_last: a piece's last

// 1, 2 or 4 bytes
template <int BYTES>
__device__ __forceinline__ uint32_t ld_part(const uint8_t *p) {
    if constexpr (BYTES == 1) return *p;
    else if constexpr (BYTES == 2) return *reinterpret_cast<const uint16_t *>(p);
    else return *reinterpret_cast<const uint32_t *>(p);
}

template <int DH>
__global__ void __launch_bounds__(PF_THREADS, 1)
k_attn_prefill(AttnArgs a, AttnPart *__restrict__ desc, float *__restrict__ part) {
    using C = PfCfg<DH>;
    constexpr int NQ = C::NQ, R = C::R, KT = C::KT, NB = C::NB, BPT = C::BPT, ST = C::STAGES;
    constexpr uint32_t ID_QK = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(KT >> 3) << 17) | (8u << 24);
    constexpr uint32_t ID_PV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(DH >> 3) << 17) | (8u << 24);
    Q36_GDS();
    extern __shared__ uint8_t raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    __shared__ PfBars bars;
    __shared__ uint32_t tmem_s, bad_s[PF_BAD_RING][2];      // bad_s: tokens of a tile whose page is bad
    __shared__ volatile int abort_flag;
    __shared__ long long plan_sum[PF_THREADS / 32], plan_base;
    __shared__ int plan_b;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t q_s = smem_u32(smem), k_s = q_s + NQ * C::Q_BYTES, v_s = k_s + ST * C::T_BYTES;
    auto bar = [&](uint64_t &b) { return smem_u32(&b); };
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < ST; i++) {
            mbar_init(bar(bars.k_full[i]), 4);
            mbar_init(bar(bars.v_full[i]), 4);
            mbar_init(bar(bars.k_empty[i]), NQ);
            mbar_init(bar(bars.v_empty[i]), NQ);
        }
        for (int i = 0; i < 2; i++) {
            for (int x = 0; x < 2; x++) { mbar_init(bar(bars.s_full[i][x]), 1); mbar_init(bar(bars.p_full[i][x]), 4); mbar_init(bar(bars.o_done[i][x]), 1); }
            mbar_init(bar(bars.o_last[i]), 1);
            mbar_init(bar(bars.q_full[i]), 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        desc[blockIdx.x].parts = 0;
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(C::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    // ---- this CTA's range of the work
    PfPos pos;
    {
        const int per = (a.B + PF_THREADS - 1) / PF_THREADS, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
        long long mine = 0;
        for (int b = b0; b < b1; b++) {
            const PfSeq s = pf_seq(a, R, b);
            if (s.tiles) mine += pf_prefix(a, s, s.tiles) * a.kv.Hkv;
        }
        long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) plan_sum[warp] = inc;
        __syncthreads();
        long long total = 0, before = 0;
        for (int w = 0; w < PF_THREADS / 32; w++) {
            if (w == warp) before = total;
            total += plan_sum[w];
        }
        const long long excl = before + inc - mine;
        pos.per = max((total + gridDim.x - 1) / gridDim.x, (long long)PF_MIN);
        pos.at = min(pos.per * blockIdx.x, total);
        pos.end = min(pos.at + pos.per, total);
        if (pos.at < pos.end && pos.at >= excl && pos.at < excl + mine) { plan_base = excl; plan_b = b0; }
        __syncthreads();
        if (pos.at < pos.end) {
            pos.seq_base = plan_base;
            pos.b = plan_b;
            pf_locate(a, R, pos);
        }
    }
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    bool more = pos.at < pos.end;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PF_REGS_SOFTMAX));
        // ------------------------------------------------------------ softmax: a row per thread
        const int i = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        uint32_t sc = 0, kt = 0, pieces = 0;       // tiles of this row tile, K tiles before this piece, pieces
        // a negative scale goes to the signs of q: m follows the largest score
        const float scale2 = fmaxf(fabsf(a.scale2), 1e-37f);      // (not 0: a hidden score stays -infinity)
        const uint32_t flip = a.scale2 < 0.f ? 0x80008000u : 0u;
        // rows of Q, and of results on their way out, in shared memory: 16-byte chunks swizzled as the MMA reads them.  A warp moves 32 rows,
        // RPI of them at a time with CPR lanes on each.
        constexpr int CPR = DH / 8, RPI = 32 / CPR;
        auto chunk = [&](int rr, int c) { return smem + i * C::Q_BYTES + (c >> 3) * 16384 + ((warp & 3) * 32 + rr) * 128 + ((c ^ (rr & 7)) & 7) * 16; };
        bool first = true, ok = true;
        while (more && ok && i < NQ) {
            const PfSeg g = pf_segment(a, KT, pos);
            const int r_tile = i * 128 + row, rows = min(pos.s.c * a.G, pos.s.n * a.G - pos.rt * pos.s.c * a.G), r = pos.rt * pos.s.c * a.G + r_tile;
            const bool mine = r_tile < rows, active = i * 128 < rows && g.j0 < g.j1;
            const int tok_i = mine ? r / a.G : 0, hq = pos.hk * a.G + (mine ? r - tok_i * a.G : 0);
            const long long q_off = mine ? (long long)(pos.s.t0 + tok_i) * a.q_stride + (long long)hq * DH : -1;
            const long long q_first = (long long)pos.s.t0 * a.q_stride + (long long)pos.hk * a.G * DH;
            if (active) {
                // Q: this warp's 32 rows, neighbouring lanes on neighbouring 16 bytes (the MMAs that read the last rows are over:
                // their results were awaited)
                const uint16_t *q = reinterpret_cast<const uint16_t *>(a.q) + (lane % CPR) * 8;
#pragma unroll 1
                for (int k0 = 0; k0 < CPR; k0 += 8) {
                    // (all on their way before the first is stored; a row that is not there reads the tile's first)
                    long long off[8];
                    uint4 v[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) off[k] = __shfl_sync(0xffffffffu, q_off, (k0 + k) * RPI + lane / CPR);
#pragma unroll
                    for (int k = 0; k < 8; k++) v[k] = *reinterpret_cast<const uint4 *>(q + (off[k] < 0 ? q_first : off[k]));
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const uint32_t keep = off[k] < 0 ? 0u : ~0u;
                        *reinterpret_cast<uint4 *>(chunk((k0 + k) * RPI + lane / CPR, lane % CPR)) =
                            make_uint4((v[k].x ^ flip) & keep, (v[k].y ^ flip) & keep, (v[k].z ^ flip) & keep, (v[k].w ^ flip) & keep);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(bars.q_full[i]));
            }
            const int p = pos.s.len - pos.s.n + tok_i;              // position; the row sees [lo_r, p]
            const int hi_r = mine ? p : -1, lo_r = a.window > 0 ? p - a.window + 1 : 0;
            float m = PF_NONE, l = 0.f, limit = PF_NONE;       // limit: what a score must pass to move m
            if (active) {
                const int t_first = min((pos.rt * pos.s.c * a.G + i * 128) / a.G, pos.s.n - 1), t_last = min((pos.rt * pos.s.c * a.G + min(i * 128 + 127, rows - 1)) / a.G, pos.s.n - 1);
                const int all_hi = pos.s.len - pos.s.n + t_first, all_lo = a.window > 0 ? pos.s.len - pos.s.n + t_last - a.window + 1 : 0;
                for (int j = g.j0; j < g.j1; j++, sc++) {
                    const uint32_t x = sc & 1, ph = (sc >> 1) & 1;
                    if (!(ok = mbar_wait(bar(bars.s_full[i][x]), ph, &abort_flag, &g_prefill_status, 0x500 + x, TC_SPIN_LIMIT, 0))) break;
                    __syncwarp();
                    tc_fence_after();
                    const uint32_t s_col = tmem + lanes + (2 * i + x) * C::TM_S;
                    const uint32_t st = (kt + (j - g.j0)) % PF_BAD_RING;       // its place in bad_s
                    uint32_t bad = 0;
#pragma unroll
                    for (int w = 0; w < KT / 32; w++) bad |= bad_s[st][w];
                    const bool edge = bad || j * KT < all_lo || j * KT + KT - 1 > all_hi;
                    uint32_t v[KT / 32][32];
#pragma unroll
                    for (int c = 0; c < KT / 32; c++) tc_ld32(s_col + 32 * c, v[c]);
                    tc_ld_wait();
                    if (edge) {
#pragma unroll
                        for (int c = 0; c < KT / 32; c++) {
                            // bits of the tokens that the row does not see
                            const int t = j * KT + 32 * c, from = lo_r - t, to = hi_r - t;
                            uint32_t hide = bad_s[st][c];
                            hide |= from >= 32 ? 0xffffffffu : from > 0 ? (1u << from) - 1u : 0u;
                            hide |= to < 0 ? 0xffffffffu : to < 31 ? 0xfffffffeu << to : 0u;
#pragma unroll
                            for (int e = 0; e < 32; e++)
                                if (hide >> e & 1) v[c][e] = 0xff800000u;
                        }
                    }
                    float mc[KT / 32];
#pragma unroll
                    for (int c = 0; c < KT / 32; c++) {
                        mc[c] = fmaxf(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]));
#pragma unroll
                        for (int e = 2; e < 32; e += 2) mc[c] = max3(mc[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
                    }
                    float mx = mc[0];
#pragma unroll
                    for (int c = 1; c < KT / 32; c++) mx = fmaxf(mx, mc[c]);
                    const float top = mx == -INFINITY ? mx : mx * scale2;
                    float k1 = scale2, m1 = -m;
                    if (__any_sync(0xffffffffu, top > limit)) {
                        const float mn = top > m + PF_GROW ? top : m, f = pf_ex2(m - mn);
                        l *= f;
                        m = mn;
                        m1 = -m;
                        limit = m + PF_GROW;
                        // The multiply-add below rounds once where m has been rounded already: it is off by up to 2^-24 |m|.  So large scores are
                        // rounded first, like m, in every tile of these rows.
                        if (__any_sync(0xffffffffu, fabsf(m) >= PF_LARGE && m != PF_NONE)) {
                            limit = -INFINITY;
                            k1 = 1.f;
                            m1 = 0.f;
#pragma unroll
                            for (int c = 0; c < KT / 32; c++)
#pragma unroll
                                for (int e = 0; e < 32; e++) v[c][e] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(v[c][e]), scale2), m));
                        }
                        if (j > g.j0) {
                            // O holds the tiles before this one
                            if (!(ok = mbar_wait(bar(bars.o_done[i][x ^ 1]), ((sc - 1) >> 1) & 1, &abort_flag, &g_prefill_status, 0x600, TC_SPIN_LIMIT, 0))) break;
                            __syncwarp();
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < DH; c += 16) {
                                uint32_t v[16];
                                const uint32_t o_col = tmem + lanes + C::TM_O0 + i * DH + c;
                                tc_ld16(o_col, v);
                                tc_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                                tc_st16(o_col, v);
                            }
                        }
                    }
                    float2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
                    const float2 k2 = {k1, k1}, m2 = {m1, m1};
#pragma unroll
                    for (int c = 0; c < KT / 32; c++) {
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float2 x = fma2(make_float2(__uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1])), k2, m2);
                            x.x = pf_ex2(x.x);
                            x.y = pf_ex2(x.y);
                            sum[(e >> 1) & 3] = add2(sum[(e >> 1) & 3], x);
                            w[e / 2] = pack_bf16(x.x, x.y);
                        }
                        tc_st16(s_col + 16 * c, w);
                    }
                    sum[0] = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
                    l += sum[0].x + sum[0].y;
                    tc_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(bars.p_full[i][x]));
                }
                if (!ok) break;
                // ---- the piece's result
                if (!(ok = mbar_wait(bar(bars.o_last[i]), pieces++ & 1, &abort_flag, &g_prefill_status, 0x700 + i, TC_SPIN_LIMIT, TC_BACKOFF_NS))) break;
                __syncwarp();
                tc_fence_after();
            }
            float *dst = part + (size_t)(2 * blockIdx.x + (first ? 0 : 1)) * attn_part_floats(R, DH);
            const float inv = l == 0.f ? 0.f : 4294967296.f / l;      // (and 2^PF_V_DOWN)
            if (active) {
                // through Q's place, so that a row leaves as a whole: bf16 at once, f32 in halves
                const int n_pass = g.whole ? 1 : 2, dims = DH / n_pass;
#pragma unroll 1
                for (int pass = 0; pass < n_pass; pass++) {
#pragma unroll 1
                    for (int c = 0; c < dims; c += 32) {
                        uint32_t v[32];
                        tc_ld32(tmem + lanes + C::TM_O0 + i * DH + pass * dims + c, v);
                        tc_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * inv);
                        if (g.whole) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                uint32_t w[4];
#pragma unroll
                                for (int x = 0; x < 4; x++) w[x] = pack_bf16(__uint_as_float(v[8 * e + 2 * x]), __uint_as_float(v[8 * e + 2 * x + 1]));
                                *reinterpret_cast<uint4 *>(chunk(lane, c / 8 + e)) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; e++) *reinterpret_cast<uint4 *>(chunk(lane, c / 4 + e)) = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                        }
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int k = 0; k < CPR; k++) {
                        const int rr = k * RPI + lane / CPR, c = lane % CPR;
                        const long long off = __shfl_sync(0xffffffffu, mine ? (long long)(pos.s.t0 + tok_i) * a.o_stride + (long long)hq * DH : -1ll, rr);
                        const uint4 v = *reinterpret_cast<const uint4 *>(chunk(rr, c));
                        if (off < 0) continue;
                        if (g.whole) *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(a.out) + off + c * 8) = v;
                        else *reinterpret_cast<uint4 *>(dst + 2 * R + (size_t)(i * 128 + (warp & 3) * 32 + rr) * DH + pass * dims + c * 4) = v;
                    }
                    __syncwarp();
                }
                tc_fence_before();
            }
            if (mine) {
                if (g.whole) { if (a.lse) a.lse[(size_t)(pos.s.t0 + tok_i) * a.Hq + hq] = l > 0.f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY; }
                else { dst[2 * r_tile] = m; dst[2 * r_tile + 1] = l; }
            }
            if (tid == 0 && !g.whole && g.head) {
                AttnPart d;
                d.parts = (int)((pos.span_base + g.units - 1) / pos.per - blockIdx.x) + 1;
                d.slot = 2 * blockIdx.x + (first ? 0 : 1);
                d.t0 = pos.s.t0;
                d.n = pos.s.n;
                d.hk = pos.hk;
                d.row0 = pos.rt * pos.s.c * a.G;
                d.rows = rows;
                d.pad = 0;
                desc[blockIdx.x] = d;
            }
            first = false;
            kt += max(g.j1 - g.j0, 0);
            more = pf_next(a, R, g, pos);
        }
    } else if (warp < 16) {
        // ------------------------------------------------------------ widening: half a token of K or V per thread
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PF_REGS_WIDEN));
        const int th = tid & 127, tl = th % KT, half = th / KT;
        const bool is_v = warp >= 12;
        const int down = is_v ? PF_V_DOWN : 0;
        uint32_t kc = 0;
        bool ok = true;
        while (more && ok) {
            const PfSeg g = pf_segment(a, KT, pos);
            const int *row = a.table + (size_t)pos.b * a.max_blocks;
            auto page = [&](int j) {
                const int t = j * KT + tl, col = t >> a.kv.log_bs;
                return j < g.j1 && t < pos.s.len && col < a.max_blocks ? row[col] : -1;
            };
            constexpr int RAW = BPT == 1 ? 8 : 4 * BPT;
            struct Half { uint32_t w[RAW], scale; bool has; };
            auto fetch = [&](int j, int id, Half &f) {
                f.has = id >= 0 && id < a.kv.n_blocks;
                if (!f.has) {
                    f.scale = 0;
                    return;
                }
                const int t = (j * KT + tl) & (a.kv.bs - 1);
                const uint8_t *reg = a.kv.at(id, pos.hk);
                f.scale = ld_part<BPT>(reg + a.kv.bs * DH + (is_v ? a.kv.bs * NB : 0) + t * NB + half * BPT);
                if (!is_v) {
                    const uint8_t *src = reg + kv_k_off(t, 0, half * BPT, DH);
#pragma unroll
                    for (int q = 0; q < 4; q++) {       // word q of every block
                        if constexpr (BPT == 4) {
                            const uint4 u = *reinterpret_cast<const uint4 *>(src + q * (DH / 8));
                            f.w[4 * q] = u.x; f.w[4 * q + 1] = u.y; f.w[4 * q + 2] = u.z; f.w[4 * q + 3] = u.w;
                        } else if constexpr (BPT == 2) {
                            const uint2 u = *reinterpret_cast<const uint2 *>(src + q * (DH / 8));
                            f.w[2 * q] = u.x; f.w[2 * q + 1] = u.y;
                        } else {
                            f.w[q] = *reinterpret_cast<const uint32_t *>(src + q * (DH / 8));
                        }
                    }
                } else {
                    const uint8_t *src = reg + a.kv.bs * (DH / 2) + kv_v_off(t, 0, half * BPT, DH);
#pragma unroll
                    for (int q = 0; q < 8; q++) {       // four dims of every block
                        if constexpr (BPT == 4) {
                            const uint2 u = *reinterpret_cast<const uint2 *>(src + q * (DH / 8));
                            f.w[2 * q] = u.x; f.w[2 * q + 1] = u.y;
                        } else {
                            f.w[q] = ld_part<2 * BPT>(src + q * (DH / 8));
                        }
                    }
                }
            };
            // data two tiles ahead, page ids three
            Half cur = {}, nxt = {}, far = {};
            int id_next = page(g.j0 + 2);
            fetch(g.j0, page(g.j0), cur);
            fetch(g.j0 + 1, page(g.j0 + 1), nxt);
            for (int j = g.j0; j < g.j1; j++, kc++) {
                const uint32_t st = kc % ST, ph = (kc / ST) & 1;
                const int id = id_next;
                id_next = page(j + 3);
                fetch(j + 2, id, far);
                if (!(ok = mbar_wait(bar(is_v ? bars.v_empty[st] : bars.k_empty[st]), ph ^ 1, &abort_flag, &g_prefill_status, 0x800 + st, TC_SPIN_LIMIT, TC_BACKOFF_NS))) break;
                __syncwarp();
                uint8_t *dst = smem + NQ * C::Q_BYTES + ((is_v ? ST : 0) + st) * C::T_BYTES + tl * 128;
#pragma unroll
                for (int b = 0; b < BPT; b++) {
                    const int sc = (int)(cur.scale >> (8 * b) & 0xff) - down;
                    const Lut t = make_lut(sc, sc > 0);
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint32_t w;
                        if (!is_v) w = cur.w[BPT * q + b];
                        else if constexpr (BPT == 1) w = cur.w[2 * q] | cur.w[2 * q + 1] << 16;
                        else w = __byte_perm(cur.w[(BPT / 2) * (2 * q) + b / 2], cur.w[(BPT / 2) * (2 * q + 1) + b / 2], (b & 1) ? 0x7632 : 0x5410);
                        const int c = (half * BPT + b) * 4 + q;      // 16-byte chunk of the token's row: dims 8 c ..
                        *reinterpret_cast<uint4 *>(dst + (c >> 3) * (KT * 128) + (((c & 7) ^ (tl & 7)) << 4)) = widen8(t, w);
                    }
                }
                if (!is_v && half == 0) {
                    // tokens of the request whose page is bad
                    const uint32_t bad = __ballot_sync(0xffffffffu, !cur.has && j * KT + tl < pos.s.len);
                    if (lane == 0) bad_s[kc % PF_BAD_RING][tl >> 5] = bad;
                }
                cur = nxt;
                nxt = far;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(is_v ? bars.v_full[st] : bars.k_full[st]));
            }
            if (ok) more = pf_next(a, R, g, pos);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PF_REGS_ISSUE));
        const int i = (warp - 16) >> 1;
        if (i < NQ && elect_one()) {
            // ------------------------------------------------------------ products of row tile i: S (even warps) or P V (odd)
            const bool do_s = (warp & 1) == 0;
            uint32_t kv = 0, n_mine = 0, qn = 0;       // tiles passed, products of this issuer, pieces
            bool ok = true;
            auto wait = [&](uint64_t &b, uint32_t ph, int where) { ok = ok && mbar_wait(bar(b), ph, &abort_flag, &g_prefill_status, where); };
            const uint32_t qa = q_s + i * C::Q_BYTES;
            while (more && ok) {
                const PfSeg g = pf_segment(a, KT, pos);
                const int n = g.j1 - g.j0;
                // a tile without rows only passes the stages on
                const bool active = i * 128 < min(pos.s.c * a.G, pos.s.n * a.G - pos.rt * pos.s.c * a.G);
                if (n > 0 && active && do_s) wait(bars.q_full[i], qn++ & 1, 0x100);
                for (int j = 0; j < n && ok; j++, kv++) {
                    const uint32_t st = kv % ST, x = n_mine & 1;
                    uint64_t &full = do_s ? bars.k_full[st] : bars.v_full[st], &empty = do_s ? bars.k_empty[st] : bars.v_empty[st];
                    wait(full, (kv / ST) & 1, do_s ? 0x210 : 0x200);
                    if (!ok) break;
                    if (!active) {
                        mbar_arrive(bar(empty));
                        continue;
                    }
                    const uint32_t s_col = tmem + (2 * i + x) * C::TM_S;
                    if (do_s) {
                        // the place was P's of two tiles ago
                        if (n_mine >= 2) wait(bars.o_done[i][x], ((n_mine >> 1) & 1) ^ 1, 0x220);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t kb = k_s + st * C::T_BYTES;
#pragma unroll
                        for (int kk = 0; kk < DH / 16; kk++)
                            pf_mma_ss(s_col, desc_sw128(qa + (kk >> 2) * 16384 + (kk & 3) * 32), desc_sw128(kb + (kk >> 2) * (KT * 128) + (kk & 3) * 32), ID_QK, kk ? 1u : 0u);
                        tc_commit(bar(bars.s_full[i][x]));
                        tc_commit(bar(empty));
                    } else {
                        wait(bars.p_full[i][x], (n_mine >> 1) & 1, 0x300);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t vb = v_s + st * C::T_BYTES;
#pragma unroll
                        for (int kk = 0; kk < KT / 16; kk++)
                            pf_mma_ts(tmem + C::TM_O0 + i * DH, s_col + kk * 8, desc_n_major(vb + kk * 2048, KT * 128), ID_PV, (j > 0 || kk) ? 1u : 0u);
                        tc_commit(bar(bars.o_done[i][x]));
                        tc_commit(bar(empty));
                        if (j == n - 1) tc_commit(bar(bars.o_last[i]));
                    }
                    n_mine++;
                }
                if (ok) more = pf_next(a, R, g, pos);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        if (abort_flag)
#pragma unroll 1
            for (int i = 0; i < 200; i++) __nanosleep(1000);      // products and copies in flight land before the block gives its memory back
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
    }
}

template <int DH>
static int run_prefill(const AttnArgs &a, void *ws, cudaStream_t st) {
    using C = PfCfg<DH>;
    static bool attr_done[MAX_DEVICES] = {false};
    int rc;
    if ((rc = ensure_smem_attr((const void *)k_attn_prefill<DH>, C::SMEM, attr_done))) return rc;
    const int grid = min(sm_count(), 256);      // (the join keeps a weight per piece)
    AttnPart *desc = (AttnPart *)ws;
    float *part = (float *)((uint8_t *)ws + attn_desc_bytes(grid));
    launch_k(k_attn_prefill<DH>, dim3(grid), dim3(PF_THREADS), C::SMEM, st, a, desc, part);
    if ((rc = check_launch())) return rc;
    return launch_attn_join(a, C::R, grid, desc, part, st);
}

uint64_t prefill_ws_bytes(int Dh) {
    const int grid = sm_count(), rows = Dh == 256 ? 128 : 256;
    return attn_desc_bytes(grid) + 2ull * grid * attn_part_floats(rows, Dh) * 4;
}
int launch_prefill(const AttnArgs &a, void *ws, cudaStream_t st) {
    if (a.kv.Dh == 64) return run_prefill<64>(a, ws, st);
    return a.kv.Dh == 128 ? run_prefill<128>(a, ws, st) : run_prefill<256>(a, ws, st);
}

// Where a bounded wait gave up (0: nowhere) since this was last asked, on the current device; the stream has been synchronised.
int prefill_wait_status(int *out) {
    const int zero = 0;
    if (cudaMemcpyFromSymbol(out, g_prefill_status, sizeof(int)) != cudaSuccess) return check_launch();
    if (*out && cudaMemcpyToSymbol(g_prefill_status, &zero, sizeof(int)) != cudaSuccess) return check_launch();
    return Q36_MOE_OK;
}

// Waits for a barrier that nobody completes, 1024 polls, and records it as the roles above do.
__global__ void k_prefill_wait_timeout() {
    Q36_GDS();
    __shared__ uint64_t bar;
    __shared__ volatile int abort_flag;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        mbar_init(smem_u32(&bar), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (threadIdx.x == 0) mbar_wait(smem_u32(&bar), 0, &abort_flag, &g_prefill_status, 0xA00, 1024u);
    __syncthreads();
}
int launch_prefill_wait_timeout(cudaStream_t st) {
    launch_k(k_prefill_wait_timeout, dim3(1), dim3(32), 0, st);
    return check_launch();
}

}  // namespace q36
