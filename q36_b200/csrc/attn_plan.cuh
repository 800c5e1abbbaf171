// How the attention kernels share their work: the (request, kv head, row tile) spans of all requests, in order, cut into equal
// ranges of token units, one per CTA, from the lengths on the device.
#pragma once
#include "attn.cuh"

namespace q36 {

// rows: rows of a tile; unit: tokens of a unit; all: every request takes part, not only those that is_long leaves.
struct SpanRule { int rows, unit, all; };

// Which requests go to the tile kernel (bf16): those of 65 rows and more whose rows times cached tokens reach a.long_work.  It does 128
// or 256 rows at five times the rate of the other one, but begins and ends in 40 us.  A batch amortises that, a short continuation alone
// does not: 2^20 as a rule, 2^22 where the call has 1024 rows per kv head at most.  us of the few-row kernel / of the tile kernel, one
// request, 16 heads of 128 on 2: 32 new tokens (256 rows) on 4096 23 / 42, on 32,768 78 / 63; 64 on 4096 31 / 43, on 32,768 139 / 65;
// 128 on 512 20 / 25, on 4096 48 / 46, on 32,768 265 / 72.
constexpr int LONG_ROWS = 65, LONG_WORK = 1 << 20, LONG_WORK_FEW = 1 << 22, LONG_FEW_ROWS = 1024;
__device__ __forceinline__ bool is_long(const AttnArgs &a, int rows, int len) { return rows >= LONG_ROWS && (long long)rows * len >= a.long_work; }

struct SeqSpans { int t0, n, len, tiles, u_lo, u_hi; };   // units [u_lo, u_hi) of the cached tokens that any row sees

__device__ __forceinline__ SeqSpans seq_spans(const AttnArgs &a, const SpanRule &r, int b) {
    SeqSpans s;
    seq_span(a, b, s.t0, s.n, s.len);
    const int rows = s.n * a.G;
    s.tiles = rows > 0 && (r.all || !is_long(a, rows, s.len)) ? (rows + r.rows - 1) / r.rows : 0;
    const int lo = a.window > 0 ? max(0, s.len - s.n - a.window + 1) : 0;
    s.u_lo = lo / r.unit;
    s.u_hi = max((s.len + r.unit - 1) / r.unit, s.u_lo + 1);     // (at least one: rows that see nothing are written too)
    return s;
}
template <int THREADS>
struct PlanSmem { long long sum[THREADS / 32]; long long base; int b; };

struct PlanPos {
    long long at, end, per, seq_base;   // this CTA's range, units per CTA, first unit of request b
    int b;
    SeqSpans s;
    // inside request b: kv head, row tile, and the first unit of that span
    int hk, rt;
    long long span_base;
};

__device__ __forceinline__ long long seq_units(const AttnArgs &a, const SeqSpans &s) {
    return (long long)s.tiles * a.kv.Hkv * (s.u_hi - s.u_lo);
}

// (32 bits nearly always do)
__device__ __forceinline__ long long div64(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}

// Moves pos to the span that holds pos.at, from request pos.b (whose first unit is pos.seq_base) on.
__device__ __forceinline__ void plan_locate(const AttnArgs &a, const SpanRule &r, PlanPos &pos) {
    for (;;) {
        pos.s = seq_spans(a, r, pos.b);
        const long long n = seq_units(a, pos.s);
        if (pos.at < pos.seq_base + n) break;
        pos.seq_base += n;
        pos.b++;
    }
    const long long off = pos.at - pos.seq_base;
    const int u = pos.s.u_hi - pos.s.u_lo, span = (int)div64(off, u);
    pos.hk = span / pos.s.tiles;
    pos.rt = span - pos.hk * pos.s.tiles;
    pos.span_base = pos.seq_base + (long long)span * u;
}

// This CTA's range; false when it is empty.  All threads take part.
template <int THREADS>
__device__ __forceinline__ bool plan_start(const AttnArgs &a, const SpanRule &r, int min_units, PlanSmem<THREADS> &sm, PlanPos &pos) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.B + THREADS - 1) / THREADS, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    long long mine = 0;
    for (int b = b0; b < b1; b++) mine += seq_units(a, seq_spans(a, r, b));
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sm.sum[warp] = inc;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w == warp) before = total;
        total += sm.sum[w];
    }
    const long long excl = before + inc - mine;
    pos.per = max(div64(total + gridDim.x - 1, gridDim.x), (long long)min_units);
    pos.at = min(pos.per * blockIdx.x, total);
    pos.end = min(pos.at + pos.per, total);
    if (pos.at >= pos.end) return false;
    if (pos.at >= excl && pos.at < excl + mine) { sm.base = excl; sm.b = b0; }
    __syncthreads();
    pos.seq_base = sm.base;
    pos.b = sm.b;
    plan_locate(a, r, pos);
    return true;
}

// A piece of one span: units [u0, u1) of [0, units), the first of which holds token u_first * unit.
struct PlanSeg { int b, hk, rt, t0, n, len, u0, u1, units, u_first; long long span_base; };

__device__ __forceinline__ PlanSeg plan_segment(const PlanPos &pos) {
    PlanSeg g;
    g.b = pos.b; g.hk = pos.hk; g.rt = pos.rt;
    g.t0 = pos.s.t0; g.n = pos.s.n; g.len = pos.s.len;
    g.units = pos.s.u_hi - pos.s.u_lo;
    g.u_first = pos.s.u_lo;
    g.u0 = (int)(pos.at - pos.span_base);
    g.u1 = (int)min((long long)g.units, pos.end - pos.span_base);
    g.span_base = pos.span_base;
    return g;
}
__device__ __forceinline__ void plan_next(const AttnArgs &a, const SpanRule &r, const PlanSeg &g, PlanPos &pos) {
    pos.at += g.u1 - g.u0;
    if (pos.at >= pos.end) return;
    plan_locate(a, r, pos);
}

// A span that was cut: its first piece's slot and the number of pieces.  The next pieces are the first pieces of the CTAs
// that follow: slot 2 * CTA.
struct AttnPart { int parts, slot, t0, n, hk, row0, rows, pad; };

__device__ __forceinline__ AttnPart plan_parts(const AttnArgs &a, const SpanRule &r, const PlanSeg &g, const PlanPos &pos, int slot) {
    AttnPart p;
    p.parts = (int)(div64(g.span_base + g.units - 1, pos.per) - blockIdx.x) + 1;
    p.slot = slot;
    p.t0 = g.t0;
    p.n = g.n;
    p.hk = g.hk;
    p.row0 = g.rt * r.rows;
    p.rows = min(r.rows, g.n * a.G - p.row0);
    p.pad = 0;
    return p;
}

// A partial result: (m, l) of each row, then the rows divided by their l.
__host__ __device__ __forceinline__ int attn_part_floats(int rows, int Dh) { return rows * (Dh + 2); }
inline uint64_t attn_desc_bytes(int grid) { return ((uint64_t)grid * sizeof(AttnPart) + 255) & ~(uint64_t)255; }

// four dims of row r of a (request, kv head); rows behind the last one are not stored
__device__ __forceinline__ void attn_store(const AttnArgs &a, int t0, int n, int hk, int r, int d, float4 v) {
    if (r >= n * a.G) return;
    const int i = r / a.G, hq = hk * a.G + r - i * a.G;
    const size_t e = (size_t)(t0 + i) * a.o_stride + (size_t)hq * a.kv.Dh + d;
    if (a.o_bf16) {
        __nv_bfloat162 p[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
        *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + e) = *reinterpret_cast<const uint2 *>(p);
    } else {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + e) = v;
    }
}
__device__ __forceinline__ void attn_store_lse(const AttnArgs &a, int t0, int n, int hk, int r, float m, float l) {
    if (!a.lse || r >= n * a.G) return;
    const int i = r / a.G, hq = hk * a.G + r - i * a.G;
    a.lse[(size_t)(t0 + i) * a.Hq + hq] = l > 0.f || l != l ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

constexpr int DEC_MAX_OCC = 4;
int launch_decode(const AttnArgs &a, int rows, int all, void *ws, cudaStream_t st);
uint64_t decode_ws_bytes(int Dh);
int launch_prefill(const AttnArgs &a, void *ws, cudaStream_t st);
uint64_t prefill_ws_bytes(int Dh);
int prefill_wait_status(int *out);
int linear_wait_status(int *out);
int launch_prefill_wait_timeout(cudaStream_t st);
int launch_attn_join(const AttnArgs &a, int tile_rows, int grid, const AttnPart *desc, const float *part, cudaStream_t st);

}  // namespace q36
