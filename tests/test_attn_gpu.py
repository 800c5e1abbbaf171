"""The attention side of a layer against plain 64-bit forms: cache tables, 4-bit rows, attention over them, the projection,
and all of it together in front of a MoE block.

Bounds.  Half a step of bf16 is 2^-8 of the value, of f32 2^-24.  Attention works on the values that the cache holds, so
its reference does too.  With |q.k| the sum of |q_d k_d| and A the softmax-weighted mean of |v|:
  score: f32 sums of Dh products err by at most (Dh + 8) 2^-24 scale |q.k| =: d (q as two f16 terms: 2^-22 of it more, inside
  4 x that); weights: exp of it and the fast exponential (2^-21): a factor 1 +- (4d + 2^-20); their sums over n tokens:
  (n + 64) 2^-24; numerator and denominator both: twice that, times A.
  bf16 inputs: the weights are rounded once for the product with V (half a step of bf16: 2^-8 A, which covers f16's 2^-11),
  and the output is (2^-8 of the value).
  small weights: f16 has no step finer than 2^-24, so a weight w against a largest one of 2^7 is off by up to 2^-25 before and
  2^-25 after its factor f = 2^(exponent of v - anchor), 2^-8 <= f <= 2^4.  That is 2^-25 (1 + f) / f |v| <= 2^-24 2^7 |v| of a
  normaliser of at least 2^7: 2^-24 |v| for every token seen, which shows where the strong tokens' v are 0.
"""
import itertools

import numpy as np
import pytest

import attn_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn(moe):
    from q36_b200 import attn
    return attn


def dt(x):
    import torch
    return torch.bfloat16 if x == "bf16" else torch.float32


def cu(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def ints(a):
    return cu(np.asarray(a, np.int32))


# ------------------------------------------------------------------ tables
TABLE_CASES = {
    "one": dict(old=[0], new=[1], bs=16, free=4, width=2),
    "decode": dict(old=[15, 16, 17, 0, 31], new=[1] * 5, bs=16, free=8, width=4),
    "mixed": dict(old=[100, 0, 3, 64, 63, 0], new=[1, 700, 0, 1, 2, 65], bs=64, free=20, width=12, pad=7),
    "pool_short": dict(old=[10, 0, 5, 20, 16], new=[30, 40, 1, 3, 1], bs=16, free=4, width=8, pad=3),
    "narrow": dict(old=[10, 30, 200, 5], new=[1, 40, 1, 20], bs=16, free=9, width=4),
    "negative": dict(old=[-1, 5, 5, 0], new=[3, -2, 2, 4], bs=32, free=9, width=4),
    "rows_short": dict(old=[5, 5, 5, 5], new=[3, 4, 5, 0], bs=16, free=9, width=4, pad=-6),
    "nothing": dict(old=[0, 7], new=[0, 0], bs=16, free=0, width=1, pad=2),
    "huge": dict(old=[2**31 - 1, 5, 2**31 - 1], new=[2**31 - 1, 2**31 - 1, 1], bs=16, free=3, width=4, T=6),
    "bad_ids": dict(old=[10, 0, 16], new=[10, 20, 3], bs=16, free=6, width=3, n_blocks=4),
    "many": dict(many=5000, bs=16, free=40000, width=30, pad=11),
    "many_short": dict(many=3000, bs=32, free=900, width=20),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", TABLE_CASES)
def test_tables(attn, name, in_place):
    c = dict(TABLE_CASES[name])
    rng = np.random.default_rng(len(name))
    if "many" in c:
        c["old"] = rng.integers(0, 300, c["many"])
        c["new"] = np.where(rng.random(c["many"]) < 0.02, rng.integers(0, 150, c["many"]), 1)
    old, new, bs, width = np.asarray(c["old"], np.int64), np.asarray(c["new"], np.int64), c["bs"], c["width"]
    T = c.get("T", int(np.maximum(new, 0).sum()) + c.get("pad", 0))
    ids = rng.permutation(c["free"] + len(old) * width).astype(np.int32)
    head = min(1, c["free"])
    n_blocks = c.get("n_blocks", len(ids) + 1)
    free, table = ids[:c["free"]], ids[c["free"]:].reshape(len(old), width)
    want = R.tables(old.tolist(), new.tolist(), bs, free.tolist(), head, table, T, n_blocks)
    o, n, f, h, t = ints(old), ints(new), ints(free), ints([head]), ints(table)
    out = None
    if in_place:
        import torch
        e = lambda k: torch.empty(k, dtype=torch.int32, device="cuda")  # noqa: E731
        out = attn.Tables(e(len(old) + 1), o, e(T), e(T), h, e(1))
    g = attn.kv_tables(o, n, bs, f, h, t, T, n_blocks=n_blocks, out=out)
    for got, exp, what in zip((t, g.cu_q, g.kv_len, g.slots, g.positions, g.free_head, g.status), want,
                              ("table", "cu_q", "kv_len", "slots", "positions", "free_head", "status")):
        np.testing.assert_array_equal(got.cpu().numpy().reshape(np.shape(exp)), exp, err_msg=what)


# ------------------------------------------------------------------ rows in and out
def awkward_rows(rng, T, H, D):
    """Values at every corner of the format: ties, powers of two, tiny, huge, zero blocks, NaN, infinities."""
    x = rng.standard_normal((T, H, D)).astype(np.float32) * np.exp2(rng.integers(-20, 20, (T, H, D // 32))).astype(np.float32).repeat(32, -1)
    f = x.reshape(-1, 32)
    for i in range(len(f)):
        kind = i % 11
        if kind == 1:
            f[i] = np.array([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -6, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5] * 2) * 2.0 ** rng.integers(-30, 30)
        elif kind == 2:
            f[i] = 0.0
        elif kind == 3:
            f[i] *= np.float32(2.0 ** -130)
        elif kind == 4:
            f[i] = np.float32(3e38) * rng.uniform(-1, 1, 32)
        elif kind == 5:
            f[i, 3], f[i, 9] = np.nan, -np.nan
        elif kind == 6:
            f[i, 5], f[i, 7] = np.inf, -np.inf
        elif kind == 7:
            f[i] = 2.0 ** rng.integers(-126, 127) * rng.choice([-1, 1], 32)
        elif kind == 8:
            f[i] = np.nan
    return x


@pytest.mark.parametrize("Dh,H,bs,x", [(64, 1, 16, "f32"), (64, 3, 128, "bf16"), (128, 2, 64, "f32"), (128, 2, 16, "bf16"), (256, 2, 32, "bf16"),
                                       (256, 1, 64, "f32")])
@pytest.mark.parametrize("T", [1, 7, 61])
def test_rows_in_and_out(attn, Dh, H, bs, x, T):
    """Codes, scales and their places, byte for byte; slots outside the cache skipped; every other byte left alone."""
    import torch
    rng = np.random.default_rng(T + Dh)
    n_blocks = T // bs + 2
    fill = rng.integers(0, 256, (n_blocks, H, bs * Dh * 17 // 16)).astype(np.uint8)
    kv = attn.KVCache(n_blocks, bs, H, Dh, data=cu(fill))
    # rows of a wider buffer, as a fused projection leaves them
    buf = torch.zeros((T, 2, H + 1, Dh), dtype=dt(x), device="cuda")
    buf[:, :, :H] = cu(awkward_rows(rng, 2 * T, H, Dh).reshape(T, 2, H, Dh), dt(x))
    k, v = buf[:, 0, :H], buf[:, 1, :H]
    slots = rng.permutation(n_blocks * bs)[:T]
    if T > 3:
        slots[[1, 3]] = [-1, n_blocks * bs]
    kv.append(k, v, ints(slots))
    qk, qv = (R.quantise(t.float().cpu().numpy()) for t in (k, v))
    want = fill.copy()
    for h in range(H):
        for blk in range(n_blocks):
            mine = [(t, s % bs) for t, s in enumerate(slots) if 0 <= s < n_blocks * bs and s // bs == blk]
            if not mine:
                continue
            z = lambda *s: np.zeros(s, np.uint8)  # noqa: E731
            kc, vc, ks, vs = z(bs, Dh), z(bs, Dh), z(bs, Dh // 32), z(bs, Dh // 32)
            mask = [z(bs, Dh), z(bs, Dh // 32)]
            for t, off in mine:
                kc[off], ks[off], vc[off], vs[off] = qk[0][t, h], qk[1][t, h], qv[0][t, h], qv[1][t, h]
                mask[0][off], mask[1][off] = 15, 255
            touched = R.region_bytes(mask[0], mask[1], mask[0], mask[1])
            want[blk, h] = np.where(touched == 255, R.region_bytes(kc, ks, vc, vs), fill[blk, h])
    np.testing.assert_array_equal(kv.data.cpu().numpy(), want)
    gk, gv = kv.read(ints(slots), dt(x))
    ok = (slots >= 0) & (slots < n_blocks * bs)
    for g, q in ((gk, qk), (gv, qv)):
        np.testing.assert_array_equal(g.double().cpu().numpy(), np.where(ok[:, None, None], q[2], 0))
    none = kv.read(ints([]), dt(x))
    kv.append(k[:0], v[:0], ints([]))
    assert none[0].shape == (0, H, Dh)


# ------------------------------------------------------------------ attention
class Setup:
    """Requests with (new, cached) tokens in a shuffled paged cache whose unused bytes are garbage."""

    def __init__(self, attn, rng, lens, Hq, Hkv, Dh, bs, x, pad=0, wide=0, scale_k=1.0, outliers=False):
        import torch
        self.lens, self.Hq, self.Hkv, self.Dh, self.bs, self.x = lens, Hq, Hkv, Dh, bs, x
        nblk = [-(-kv // bs) for _, kv in lens]
        self.n_blocks = sum(nblk) + 2
        data = torch.randint(0, 256, (self.n_blocks, Hkv, bs * Dh * 17 // 16), dtype=torch.uint8, device="cuda",
                             generator=torch.Generator("cuda").manual_seed(int(rng.integers(1 << 30))))
        data[:, :, bs * Dh:] = 255                                              # scales that stand for no number
        self.kv = attn.KVCache(self.n_blocks, bs, Hkv, Dh, data=data)
        ids = rng.permutation(self.n_blocks)[:sum(nblk)]
        table = rng.integers(-(1 << 30), 1 << 30, (len(lens), max(nblk + [1]) + wide))      # ids behind a request's blocks: anything
        slots, at = [], 0
        for b, (_, kv) in enumerate(lens):
            table[b, :nblk[b]] = ids[at:at + nblk[b]]
            at += nblk[b]
            j = np.arange(kv)
            slots.append(table[b, j // bs] * bs + j % bs)
        self.table = ints(table)
        n = sum(kv for _, kv in lens)
        k, v = (rng.standard_normal((max(n, 1), Hkv, Dh), dtype=np.float32) for _ in range(2))
        k *= scale_k
        if outliers:
            v *= np.exp2(rng.integers(-12, 13, (len(v), Hkv, Dh // 32))).astype(np.float32).repeat(32, -1)
            k *= np.exp2(rng.integers(-3, 4, (1, Hkv, Dh // 32))).astype(np.float32).repeat(32, -1)
        if n:
            s = ints(np.concatenate(slots))
            self.kv.append(cu(k), cu(v), s)
            self.k, self.v = (t.double().cpu().numpy() for t in self.kv.read(s))
        else:
            self.k = self.v = np.zeros((0, Hkv, Dh))
        self.T = sum(q for q, _ in lens)
        self.cu_q = ints(np.concatenate([[0], np.cumsum([q for q, _ in lens])]))
        self.kv_len = ints([kv for _, kv in lens])
        self.q = cu(rng.standard_normal((self.T + pad, Hq, Dh), dtype=np.float32), dt(x))
        self.max_q = max([q for q, _ in lens] + [1])

    def run(self, window=0, scale=None, **kw):
        return self.kv.attention(self.q, self.table, self.cu_q, self.kv_len, self.max_q, scale=scale, window=window, want_lse=True, **kw)

    def check(self, got, window=0, scale=None, drop=None, rows=None):
        out, lse = (t.double().cpu().numpy() for t in got)
        q = self.q.double().cpu().numpy()
        scale = 1 / np.sqrt(self.Dh) if scale is None else scale
        t0 = j0 = 0
        for b, (n, kv) in enumerate(self.lens):
            if rows is None or b in rows:
                o, l, A, d, V = R.attention(q[t0:t0 + n], self.k[j0:j0 + kv], self.v[j0:j0 + kv], n, scale, window, None if drop is None else drop[b])
                d = abs(d) * abs(scale) * (self.Dh + 8) * 2.0 ** -24
                sums = (kv + 64) * 2.0 ** -24
                tol = A * (2 * (4 * d + 2.0 ** -20 + sums))[..., None] + 2.0 ** -24 * V + 1e-30
                tol += 2.0 ** -8 * (np.abs(o) + A) if self.x == "bf16" else 2.0 ** -24 * np.abs(o)
                err = np.abs(out[t0:t0 + n] - o)
                assert (err <= tol).all(), (b, n, kv, float((err / tol).max()))
                fin = np.isfinite(l)
                assert (lse[t0:t0 + n][~fin] == -np.inf).all() and (out[t0:t0 + n][~fin] == 0).all()
                e = np.abs(lse[t0:t0 + n][fin] - l[fin])
                assert (e <= 4 * d[fin] + 2.0 ** -20 + sums + 2.0 ** -22 * np.abs(l[fin])).all(), (b, "lse")
            t0, j0 = t0 + n, j0 + kv


HEADS = [(16, 2), (8, 8), (12, 4), (5, 1), (32, 2), (40, 2)]
DECODE = [(1, n) for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500)]


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
def test_single_tokens(attn, heads, Dh, x):
    rng = np.random.default_rng(Dh + heads[0])
    s = Setup(attn, rng, DECODE, *heads, Dh, 16, x)
    s.check(s.run())


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 1, 17, 130])
def test_prompts_mixed_with_single_tokens(attn, bs, x, window):
    """Prompts (from the first token, behind a cached prefix) among decoding requests and one without new tokens."""
    rng = np.random.default_rng(bs + window)
    s = Setup(attn, rng, [(1, 300), (150, 150), (0, 40), (70, 333), (3, 3), (1, 1), (130, 131), (17, 200)], 16, 2, 128, bs, x, pad=3)
    s.check(s.run(window=window), window=window)


@pytest.mark.parametrize("heads,Dh", [((4, 4), 64), ((6, 2), 128), ((16, 2), 256), ((5, 1), 64), ((48, 1), 128), ((128, 1), 64)])
@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_prompts_of_every_shape(attn, heads, Dh, x):
    rng = np.random.default_rng(Dh)
    s = Setup(attn, rng, [(257, 257), (1, 90), (64, 700)], *heads, Dh, 64, x)
    s.check(s.run(scale=0.2), scale=0.2)


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("q", [1, 200])
def test_long_context_is_split_and_joined(attn, x, q):
    rng = np.random.default_rng(q)
    s = Setup(attn, rng, [(q, 20000), (1, 5), (q, 9001)], 16, 2, 128, 64, x)
    s.check(s.run())
    s.check(s.run(window=3000), window=3000)


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
def test_scales_that_differ_widely(attn, Dh, x):
    """V blocks between 2^-12 and 2^12, strong K channels, sharp softmax: what the packed arithmetic has to keep apart."""
    rng = np.random.default_rng(Dh)
    s = Setup(attn, rng, [(1, 777), (40, 300), (1, 64)], 16, 2, Dh, 32, x, scale_k=3.0, outliers=True)
    s.check(s.run())


@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_rows_that_see_nothing(attn, x):
    """More new tokens than cached ones, empty requests, a negative and an overlong cached length."""
    import torch
    rng = np.random.default_rng(4)
    for nq in (7, 90):
        s = Setup(attn, rng, [(nq, 3), (1, 0), (nq, 0), (2, 50), (nq, 40)], 16, 2, 128, 16, x)
        s.check(s.run())
    s = Setup(attn, rng, [(1, 30), (1, 48)], 16, 2, 128, 16, x)
    s.kv_len = ints([-5, 1 << 30])
    out, lse = s.run()
    assert (out[0] == 0).all() and (lse[0] == -torch.inf).all()
    s.check((out, lse), rows=[1])                                                  # cut at the table's width: 48 tokens


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("q", [1, 100])
def test_bad_pages_are_left_out(attn, x, q):
    rng = np.random.default_rng(5)
    s = Setup(attn, rng, [(q, 200), (1, 70)], 16, 2, 128, 16, x)
    s.table[0, 2], s.table[0, 7], s.table[1, 0] = -1, s.n_blocks, 2**31 - 1
    drop = [np.zeros(200, bool), np.zeros(70, bool)]
    drop[0][32:48] = drop[0][112:128] = drop[1][:16] = True
    s.check(s.run(), drop=drop)


@pytest.mark.parametrize("q", [1, 100])
def test_rows_behind_the_last_request_are_left_alone(attn, q):
    import torch
    rng = np.random.default_rng(6)
    s = Setup(attn, rng, [(q, 200), (1, 70)], 16, 2, 128, 16, "bf16", pad=9)
    s.q[s.T:] = torch.nan
    out = torch.full_like(s.q, 7.0)
    got = s.run(out=out)
    s.check((out[:s.T], got[1][:s.T]))
    assert (out[s.T:] == 7.0).all()


@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_strided_rows(attn, x):
    """q inside a fused projection's rows, out inside a wider buffer."""
    import torch
    rng = np.random.default_rng(7)
    s = Setup(attn, rng, [(40, 100), (1, 33)], 16, 2, 64, 16, x)
    plain = s.run()
    wide = torch.zeros((s.T, 20, 64), dtype=s.q.dtype, device="cuda")
    wide[:, 2:18] = s.q
    s.q = wide[:, 2:18]
    buf = torch.full((s.T, 24, 64), 3.0, dtype=s.q.dtype, device="cuda")
    out, lse = s.run(out=buf[:, 4:20])
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    assert (buf[:, :4] == 3).all() and (buf[:, 20:] == 3).all()


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("heads,Dh", [((32, 2), 64), ((24, 2), 64), ((40, 2), 64), ((32, 2), 128)])
@pytest.mark.parametrize("q", [1, 9])
def test_many_requests_with_a_tile_of_16_rows(attn, heads, Dh, x, q):
    """Calls that fill the GPU: the wider tile, whole, with rows missing and with a second tile."""
    rng = np.random.default_rng(16)
    s = Setup(attn, rng, [(q, int(n)) for n in rng.integers(q, 700, 30)], *heads, Dh, 32, x)
    s.check(s.run())
    s.check(s.run(window=40), window=40)


@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_any_scale_and_any_window(attn, x):
    """Negative and zero scales; windows up to the largest integer, with fewer cached tokens than new ones."""
    rng = np.random.default_rng(13)
    s = Setup(attn, rng, [(1, 90), (200, 6000), (9, 4)], 16, 2, 128, 16, x)
    for scale in (-0.1, 0.0):
        s.check(s.run(scale=scale), scale=scale)
    for window in (2**30 - 1, 2**30, 2**31 - 2, 2**31 - 1):
        s.check(s.run(window=window), window=window)


@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_scores_of_any_size(attn, x):
    """Scores of -2^100 and below: the one token whose score is 2^100 above the others' has all the weight."""
    import torch
    rng = np.random.default_rng(14)
    s = Setup(attn, rng, [(1, 90), (200, 6000)], 16, 2, 128, 16, x)
    k = torch.zeros((6090, 2, 128), device="cuda")
    k[:, :, 0] = 2.0
    k[[33, 90 + 4567], :, 0] = 1.0
    slots = [int(s.table[b, j // 16]) * 16 + j % 16 for b, n in enumerate((90, 6000)) for j in range(n)]
    v = cu(s.v, torch.float32)
    s.kv.append(k, v, ints(slots))
    s.q.zero_()
    s.q[:, :, 0] = -(2.0 ** 100)
    out, lse = s.run(scale=1.0)
    want = torch.cat([v[33:34], v[90 + 4567:90 + 4568].expand(200, -1, -1)]).repeat_interleave(8, 1)
    assert torch.equal(out.float(), want.to(out.dtype).float())                                    # (a 4-bit value is exact in both types)
    assert (lse + 2.0 ** 100).abs().max() <= 2.0 ** 78                                             # 2^-22 of it


def test_offsets_past_32_bits(attn):
    """A cache of 9 GB whose pages lie on both sides of 2^31 and 2^32 bytes; rows of q, out, x, y and the residual 2^27 elements
    apart.  The numbers are those of the same requests with everything close together."""
    import torch
    rng = np.random.default_rng(15)
    for lens in ([(1, 1000), (1, 700)], [(70, 2500)]):
        s = Setup(attn, rng, lens, 16, 2, 128, 16, "bf16")
        want = s.run()
        pages = 9 * 10**9 // s.kv.data[0].numel()
        far = attn.KVCache(pages, 16, 2, 128, data=torch.empty((pages, 2, 16 * 128 * 17 // 16), dtype=torch.uint8, device="cuda"))
        near = s.table.cpu().numpy()
        ids = np.linspace(0, pages - 1, s.n_blocks).astype(np.int64)
        far.data[torch.from_numpy(ids).cuda()] = s.kv.data
        s.table = ints(np.where((near >= 0) & (near < s.n_blocks), ids[near.clip(0, s.n_blocks - 1)], -1))
        s.kv = far
        q = torch.empty((20, 1 << 27), dtype=torch.bfloat16, device="cuda")
        if s.T <= 20:
            wide = q[:s.T, :2048].unflatten(1, (16, 128))
            wide.copy_(s.q)
            s.q = wide
            out, lse = s.run(out=q[:s.T, 4096:4096 + 2048].unflatten(1, (16, 128)))
        else:
            out, lse = s.run()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        k = cu(rng.standard_normal((2, 2, 128), dtype=np.float32))
        last = ints([pages * 16 - 1, 5])
        far.append(k, -k, last)
        a, b = far.read(last)
        assert torch.equal(a, -b) and (a - k).abs().max() < 1
    x, w = q[:, :512].copy_(torch.randn(20, 512)), torch.randn(96, 512, device="cuda").bfloat16()
    res = q[:, 1024:1024 + 96].copy_(torch.randn(20, 96))
    want = attn.linear(x.contiguous(), w, residual=res.contiguous())
    assert torch.equal(attn.linear(x, w, residual=res, out=q[:, 2048:2048 + 96]), want)
    assert torch.equal(attn.linear(x[-3:], w, residual=res[-3:], out=q[-3:, 2048:2048 + 96]), attn.linear(x[-3:].contiguous(), w, residual=res[-3:].contiguous()))


def test_more_rows_than_one_launch_takes(attn):
    """Rows are written and read 2^30 eights at a time: those on both sides of the cut."""
    import torch
    H, Dh, T = 1024, 256, (1 << 30) // (1024 * 256 // 8) + 2
    kv = attn.KVCache(1, 16, H, Dh)
    k = torch.empty((T, H, Dh), dtype=torch.bfloat16, device="cuda")
    rows = [0, T - 3, T - 2, T - 1]
    slots = np.full(T, -1)
    slots[rows] = [3, 9, 0, 15]
    k[rows] = torch.randn((4, H, Dh), device="cuda").bfloat16()
    kv.append(k, k, ints(slots))
    del k
    got, _ = kv.read(ints(slots), torch.bfloat16)
    want, _ = kv.read(ints(slots[rows]), torch.bfloat16)
    assert torch.equal(got[rows], want) and (want != 0).any(-1).all() and not got[1].any() and not got[T // 2].any()


def test_max_q_chooses_kernels_only(attn):
    """Any stated largest number of new tokens gives right results."""
    rng = np.random.default_rng(8)
    s = Setup(attn, rng, [(300, 400), (1, 100), (20, 20)], 16, 2, 128, 16, "bf16")
    for s.max_q in (1, 8, 300, 100000):
        s.check(s.run())


@pytest.mark.parametrize("heads,Dh", [((16, 2), 128), ((16, 2), 256), ((12, 4), 64), ((24, 2), 128)])
def test_pieces_of_several_spans_on_one_cta(attn, heads, Dh):
    """Prompts long enough that every CTA goes through pieces of several row tiles, some of them with one half empty: no wait
    may give up, twice the same bits, and the rows of the request that the host can afford to check against 64 bits."""
    import torch
    rng = np.random.default_rng(10)
    s = Setup(attn, rng, [(2100, 2600), (130, 9000), (1400, 1400), (1, 600), (300, 4000)], *heads, Dh, 64, "bf16")
    a, b = s.run(), s.run()
    attn.check_device_status()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    s.check(a, rows=[1, 3, 4])


def test_a_wait_that_gives_up_is_reported_once(attn, moe):
    import torch
    st = torch.cuda.current_stream().cuda_stream
    assert attn.lib.q36_attn_status(st) == moe.OK
    assert attn.lib.q36_attn_selftest_wait_timeout(st) == moe.OK
    with pytest.raises(attn.MoEError):
        attn.check_device_status()
    attn.check_device_status()


def test_same_bits_twice_on_two_streams_and_from_a_graph(attn):
    """Two calls at once on two streams, a captured and replayed one, and the same call again: the same bits."""
    import torch
    rng = np.random.default_rng(9)
    s = Setup(attn, rng, [(1, 5000), (130, 900), (1, 77)], 16, 2, 128, 16, "bf16")
    want = s.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = []
    for _ in range(3):
        for st in streams:
            both.append(s.run(stream=st))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both.append(s.run())
        graphs.append(g)
    for _ in range(2):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for out, lse in both:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


# ------------------------------------------------------------------ linear
def act64(v, act):
    from math import erf, sqrt
    with np.errstate(over="ignore"):
        return {"none": lambda: v, "relu": lambda: np.maximum(v, 0), "silu": lambda: v / (1 + np.exp(-v)),
                "gelu": lambda: 0.5 * v * (1 + np.vectorize(erf)(v / sqrt(2))),
                "gelu_tanh": lambda: 0.5 * v * (1 + np.tanh(sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))}[act]()


def linear_case(attn, T, N, K, act, bias, res, y, strided=False, inplace=False, rows=None, seed=0):
    """Bound: f32 sums of K products err by at most (K + 8) 2^-24 sum|x||w|; no activation here is steeper than 1.13; its own
    evaluation errs by at most 2^-20 of max(1, |v|); then one rounding of the result."""
    import torch
    g = torch.Generator("cuda").manual_seed(seed + T + N + K)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    pad = 8 if strided else 0
    x = r(T, K + pad).bfloat16()[:, :K]
    w = (r(N, K) * K ** -0.5).bfloat16()
    b = r(N) if bias else None
    rr = None if res is None else r(T, N + pad // 2).to(dt(res))[:, :N]
    out = None
    if inplace:
        out = rr
    elif strided or rows is not None:
        out = torch.full((T, N + pad), 5.0, dtype=dt(y), device="cuda")[:, :N]
    before = None if out is None else out.clone()
    keep = None if rr is None else rr.double().cpu().numpy()
    got = attn.linear(x, w, bias=b, act=act, residual=rr, out=out, out_dtype=None if out is not None else dt(y),
                      rows_used=None if rows is None else ints([rows]))
    xd, wd = x.double(), w.double()
    v = xd @ wd.t()
    mag = (xd.abs() @ wd.abs().t()).cpu().numpy()
    v = v.cpu().numpy() + (0 if b is None else b.double().cpu().numpy())
    want = act64(v, act) + (0 if keep is None else keep)
    tol = 1.13 * ((K + 8) * 2.0 ** -24 * mag + 2.0 ** -24 * np.abs(v)) + 2.0 ** -23 * np.abs(want)
    tol += 0 if act == "none" else 2.0 ** -20 * np.maximum(1, np.abs(v))
    tol += 2.0 ** -8 * np.abs(want) if got.dtype == torch.bfloat16 else 0
    n = T if rows is None else min(max(rows, 0), T)
    err = np.abs(got.double().cpu().numpy() - want)[:n]
    assert (err <= tol[:n]).all(), float((err / tol[:n]).max())
    if n < T:
        assert torch.equal(got[n:], before[n:])
    if strided and not inplace:
        wide = torch.as_strided(got, (T, N + pad), (N + pad, 1))
        assert (wide[:, N:] == 5.0).all()


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 33, 64, 100, 129, 300, 1000])
@pytest.mark.parametrize("N,K", [(1, 8), (63, 72), (64, 64), (129, 256), (1000, 1000), (2048, 2048)])
def test_linear_sizes(attn, T, N, K):
    linear_case(attn, T, N, K, "none", False, None, "f32")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("T", [1, 30, 260])
@pytest.mark.parametrize("res,y", [(None, "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
def test_linear_epilogue(attn, act, T, res, y):
    linear_case(attn, T, 200, 136, act, True, res, y)


@pytest.mark.parametrize("T", [1, 12, 40, 300])
@pytest.mark.parametrize("rows", [None, 0, 1, 11, 1000, -3])
@pytest.mark.parametrize("inplace", [False, True])
def test_linear_strides_in_place_and_rows_used(attn, T, rows, inplace):
    linear_case(attn, T, 130, 264, "silu", True, "f32", "f32", strided=True, inplace=inplace, rows=rows)


@pytest.mark.parametrize("T", [1, 70])
def test_linear_passes_infinities_and_nan_of_a_row_to_that_row_only(attn, T):
    import torch
    x = torch.ones((T, 64), device="cuda").bfloat16()
    w = torch.ones((40, 64), device="cuda").bfloat16()
    x[0, 3] = torch.inf
    w[7, 5] = torch.nan
    y = attn.linear(x, w, out_dtype=torch.float32)
    assert torch.isnan(y[:, 7]).all()
    others = [i for i in range(40) if i != 7]
    assert (y[0, others] == torch.inf).all() and (T == 1 or (y[1:, others] == 64).all())


# ------------------------------------------------------------------ together
def test_decoding_steps_of_a_layer(attn, moe):
    """Prompt, then single tokens, through tables -> block -> MoE block: every step against the 64-bit chain, in one captured
    graph per shape that is replayed on growing lengths with padding rows at the end."""
    import torch
    rng = np.random.default_rng(11)
    D, Hq, Hkv, Dh, bs, E, B = 512, 8, 2, 64, 16, 32, 3
    layer = moe.MoELayer(n_expert=E, k=4, D=D, FF=512).random_planes(3)
    kv = attn.KVCache(40, bs, Hkv, Dh)
    w_o = cu(rng.standard_normal((D, Hq * Dh), dtype=np.float32) / 20, torch.bfloat16)
    norm_w, next_w = torch.ones(D, device="cuda"), torch.ones(D, device="cuda")
    router = cu(rng.standard_normal((E + 1, D), dtype=np.float32) * 0.1)
    free, head, table = ints(rng.permutation(40)), ints([0]), ints(np.full((B, 8), -1))
    lens = ints(np.zeros(B))
    keys = [[] for _ in range(B)]
    steps = [[20, 0, 33], [1, 7, 1]] + [[1, 1, 1]] * 5
    graphs = {}
    for si, new in enumerate(steps):
        T = 56 if si == 0 else 12 if si == 1 else 5            # padded
        if T not in graphs:
            bufs = dict(q=torch.zeros((T, Hq, Dh), device="cuda").bfloat16(), k=torch.zeros((T, Hkv, Dh), device="cuda").bfloat16(),
                        v=torch.zeros((T, Hkv, Dh), device="cuda").bfloat16(), h=torch.zeros((T, D), device="cuda"), new=ints(np.zeros(B)))
            e = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
            out = attn.Tables(e(B + 1), lens, e(T), e(T), head, e(1))

            def step(bufs=bufs, out=out, T=T):
                attn.kv_tables(lens, bufs["new"], bs, free, head, table, T, n_blocks=40, out=out)
                kv.block(bufs["q"], bufs["k"], bufs["v"], out.slots, table, out.cu_q, out.kv_len, 33, w_o, bufs["h"])
                return layer.block(bufs["h"].clone(), None, norm_w, router, next_w)

            layer.block(torch.zeros((T, D), device="cuda"), None, norm_w, router, next_w)      # (its workspace, before the capture)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                res = step()
            graphs[T] = (g, bufs, out, res)
        g, bufs, out, res = graphs[T]
        n = sum(new)
        for name in ("q", "k", "v", "h"):
            bufs[name].copy_(cu(rng.standard_normal(tuple(bufs[name].shape), dtype=np.float32)))
        bufs["new"].copy_(ints(new))
        h0 = bufs["h"].clone()
        g.replay()
        torch.cuda.synchronize()
        assert int(out.status) == 0
        t0 = 0
        want = h0.double().cpu().numpy()
        tol = np.zeros_like(want)
        for b, nb in enumerate(new):
            r = slice(t0, t0 + nb)
            keys[b].append([R.quantise(bufs[x][r].float().cpu().numpy())[2] for x in ("k", "v")])
            k, v = (np.concatenate([p[i] for p in keys[b]]) for i in (0, 1))
            assert int(out.kv_len[b]) == len(k)
            o, _, A, _, _ = R.attention(bufs["q"][r].double().cpu().numpy(), k, v, nb, Dh ** -0.5)
            w = w_o.double().cpu().numpy()
            want[r] += o.reshape(nb, Hq * Dh) @ w.T
            tol[r] = (2.0 ** -8 * (np.abs(o) + A) * 1.02).reshape(nb, Hq * Dh) @ np.abs(w).T + 1e-5 * (1 + np.abs(want[r]))
            t0 += nb
        err = np.abs(bufs["h"].double().cpu().numpy() - want)
        assert (err <= tol).all() and (err[n:] == 0).all(), (si, float(err.max()))
        hx = bufs["h"].clone()
        x_next, moe_out = layer.block(hx, None, norm_w, router, next_w)
        assert torch.equal(x_next[:n], res[0][:n]) and torch.equal(moe_out[:n], res[1][:n])


def test_block_is_its_parts(attn):
    import torch
    rng = np.random.default_rng(12)
    for x, q in itertools.product(("bf16", "f32"), (1, 50)):
        s = Setup(attn, rng, [(q, 100 + q), (1, 40)], 16, 2, 128, 16, x)
        new = cu(rng.standard_normal((2, s.T, 2, 128), dtype=np.float32), s.q.dtype)
        j = [np.arange(kv - n, kv) for n, kv in s.lens]
        tab = s.table.cpu().numpy()
        slots = ints(np.concatenate([tab[b, p // 16] * 16 + p % 16 for b, p in enumerate(j)]))
        w_o, bias = cu(rng.standard_normal((96, 2048), dtype=np.float32) / 40, torch.bfloat16), cu(rng.standard_normal(96, dtype=np.float32))
        h = cu(rng.standard_normal((s.T, 96), dtype=np.float32))
        h1 = h.clone()
        s.kv.block(s.q, new[0], new[1], slots, s.table, s.cu_q, s.kv_len, s.max_q, w_o, h1, bias_o=bias)
        s.kv.append(new[0], new[1], slots)
        a = s.run()[0].to(torch.bfloat16).flatten(1)
        assert torch.equal(h1, attn.linear(a, w_o, bias=bias, residual=h, out_dtype=torch.float32))
