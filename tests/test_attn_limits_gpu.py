"""The attention side of a layer at the limits of what it takes, against plain 64-bit forms; bounds as in test_attn_gpu.py."""
import numpy as np
import pytest

import attn_ref as R
from test_attn_gpu import Setup, cu, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn(moe):
    from q36_b200 import attn
    return attn


def own_rows(s, k, v):
    """The cached rows of a Setup's requests, all of them, replaced."""
    tab = s.table.cpu().numpy()
    slots = ints(np.concatenate([tab[b, np.arange(n) // s.bs] * s.bs + np.arange(n) % s.bs for b, (_, n) in enumerate(s.lens)]))
    s.kv.append(cu(np.asarray(k, np.float32)), cu(np.asarray(v, np.float32)), slots)
    s.k, s.v = (t.double().cpu().numpy() for t in s.kv.read(slots))


@pytest.mark.parametrize("Dh", [64, 128])
def test_bad_pages_behind_a_half_empty_row_tile(attn, Dh):
    """Requests of 32 + 16 new tokens of 8 heads: a row tile of 256 rows, then one whose second half has none, on the same CTA.  The second
    half of the first one is slow (its rows' scores grow by 2^9 a tile or so, so that the sums move with every tile), and pages of its
    last tiles and of the next row tile's first ones are bad, each tile in a pattern of its own."""
    import torch
    rng = np.random.default_rng(17)
    s = Setup(attn, rng, [(48, int(n)) for n in rng.integers(2740, 3400, 40)], 16, 2, Dh, 16, "bf16")
    half = Dh // 2
    k, v = rng.standard_normal((len(s.k), 2, Dh)), rng.standard_normal((len(s.k), 2, Dh))
    tile = np.concatenate([np.arange(n) // 64 * half / (n // 64 + 1) for _, n in s.lens])
    k[:, :, :half] = np.arange(half) < tile[:, None, None]
    own_rows(s, k, v)
    grows = torch.arange(s.T, device="cuda") % 48
    s.q[:, :, :half] = torch.where((grows >= 16) & (grows < 32), 1.0, -1.0)[:, None, None] * 6.5 * Dh ** 0.5
    drop = []
    for b, (_, n) in enumerate(s.lens):
        pages = -(-n // 16)
        bad = np.zeros(pages, bool)
        bad[1:48], bad[-24:-1] = rng.random(47) < 0.4, rng.random(23) < 0.4
        s.table[b, :pages][torch.from_numpy(bad).cuda()] = int(rng.choice([-1, s.n_blocks, 2**31 - 1]))
        drop.append(bad.repeat(16)[:n])
    first = s.run()
    s.check(first, drop=drop)
    for _ in range(50):
        out, lse = s.run()
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    attn.check_device_status()


def test_two_threads_on_one_stream(attn):
    """Different requests on the same cache and the same (default) stream from two host threads: the bits of one thread alone."""
    import threading
    import torch
    rng = np.random.default_rng(18)
    a = Setup(attn, rng, [(1, int(n)) for n in rng.integers(500, 3000, 40)], 16, 2, 128, 16, "bf16")
    b = Setup(attn, rng, [(1, 9000), (3, 20), (300, 4000)], 16, 2, 128, 16, "bf16")
    both = attn.KVCache(a.n_blocks + b.n_blocks, 16, 2, 128, data=torch.cat([a.kv.data, b.kv.data]))
    b.table = torch.where((b.table >= 0) & (b.table < b.n_blocks), b.table + a.n_blocks, -1)
    a.table = torch.where(a.table < a.n_blocks, a.table, -1)
    a.kv = b.kv = both
    want = [s.run() for s in (a, b)]
    a.check(want[0])
    got = [[], []]
    start = threading.Barrier(2)

    def work(i, s):
        start.wait()
        for _ in range(200):
            got[i].append(s.run())

    threads = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate((a, b))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 200
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])


def tables_of(attn, B):
    """Tables of B requests, every entry."""
    import torch
    rng = np.random.default_rng(B)
    old, new = rng.integers(0, 60, B), np.where(rng.random(B) < 0.02, rng.integers(0, 40, B), 1)
    T, width, free = int(new.sum()) + 3, 8, 3 * B
    ids = rng.permutation(free + B * width).astype(np.int32)
    table = ids[free:].reshape(B, width)
    want = R.tables(old.tolist(), new.tolist(), 16, ids[:free].tolist(), 2, table, T, len(ids))
    t = ints(table)
    g = attn.kv_tables(ints(old), ints(new), 16, ints(ids[:free]), ints([2]), t, T, n_blocks=len(ids))
    for got, exp in zip((t, g.cu_q, g.kv_len, g.slots, g.positions, g.free_head, g.status), want):
        np.testing.assert_array_equal(got.cpu().numpy().reshape(np.shape(exp)), exp)
    torch.cuda.synchronize()


@pytest.mark.parametrize("B", [6127, 6143, 6144, 16384])
def test_tables_of_many_requests_as_a_process_first_call(B):
    """Sizes around 48 KB of shared memory, the limit of a launch that has not asked for more, and the largest."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = f"import sys; sys.path[:0] = {[here, os.path.dirname(here)]!r}; from test_attn_limits_gpu import tables_of; from q36_b200 import attn; tables_of(attn, {B})"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
def test_tiny_values_beside_ordinary_ones(attn, Dh, x):
    """V blocks of about 1e-38, whose scale byte is that of a block of zeros, and blocks of zeros among blocks of about 1: token by token, in
    all tokens of a block of dims, and in a request's first tokens."""
    rng = np.random.default_rng(19)
    s = Setup(attn, rng, [(1, 777), (40, 300), (1, 64), (1, 500), (200, 6000)], 16, 2, Dh, 32, x)
    n, nb = len(s.k), Dh // 32
    size = rng.choice([1.0, 1.0, 1e-38, 0.0], (n, 2, nb))
    size[:, 0, 0] = 1e-38
    size[777:1077] = np.where(size[777:1077] == 1.0, 1.0, 1e-38)
    size[1141:1141 + 40] = np.where(np.arange(40) % 2, 1e-38, 0.0)[:, None, None]
    size[1141 + 40:1641] = 1.0
    own_rows(s, rng.standard_normal((n, 2, Dh)), rng.standard_normal((n, 2, Dh)) * size.repeat(32, -1))
    assert 0 < np.abs(s.v[:1077, 0, :32]).max() < 1e-36
    got = s.run()
    s.check(got)
    tiny = got[0].float().cpu().numpy()[:41, :8, :32]                            # kv head 0, block 0: tiny in every token of requests 0 and 1
    assert np.abs(tiny).max() < 1e-36


def act64(v, act):
    """The activations in 64 bits, without cancellation; their limit at -infinity."""
    from math import erfc
    with np.errstate(over="ignore", invalid="ignore"):
        u = 2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
        y = {"none": lambda: v, "relu": lambda: np.maximum(v, 0), "silu": lambda: v / (1 + np.exp(-v)), "gelu_tanh": lambda: v / (1 + np.exp(-u)),
             "gelu": lambda: 0.5 * v * np.vectorize(erfc)(-v / np.sqrt(2))}[act]()
    return np.where((v == -np.inf) & (act != "none"), 0.0, y), v if act == "silu" else u


@pytest.mark.parametrize("y", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 260])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_activations_of_sums_of_any_size(attn, act, T, y):
    """Relative to the result.  silu and gelu_tanh, in half steps 2^-24: the argument of the exponential has six roundings (gelu_tanh), its
    base-2 form two, of |u| each, which count as they stand in a result that goes as e^u; the exponentials 2^-22 twice, the quotient
    and the products: 20; and the last steps of the smallest numbers, 2^-149.  gelu below 0: 1 + erf in f32, 2^-20 in all."""
    import torch
    v = torch.tensor([-75, -100, -87.5, -95, -103, -104.5, -130, -1e4, -1e13, -1e31, -3e38, -torch.inf, -10, -6, -4, -1, -1e-30, 0, 1e-30, 0.5, 3, 12,
                      20, 90, 130, 1e13, 1e31, 3e38, torch.inf, torch.nan]).bfloat16().cuda()
    w = torch.zeros((len(v), 8), dtype=torch.bfloat16, device="cuda")
    w[:, 0] = 1
    x = torch.zeros((T, 8), dtype=torch.bfloat16, device="cuda")
    got = np.zeros((len(v), len(v)))
    for i in range(len(v)):                                                       # one at a time: 0 times infinity is no number
        x[:, 0] = v[i]
        out = attn.linear(x, w, act=act, out_dtype=torch.bfloat16 if y == "bf16" else torch.float32)
        assert torch.equal(out.nan_to_num(7.0), out[:1].expand_as(out).nan_to_num(7.0))
        got[i] = out[0].double().cpu().numpy()
    vd = v.double().cpu().numpy()
    want, u = act64(vd, act)
    assert np.isnan(got[-1]).all()
    for i in range(len(v) - 1):
        if np.isinf(want[i]):
            assert (got[i] == want[i]).all(), vd[i]
            continue
        rel = {"silu": 20 + 2 * abs(u[i]), "gelu_tanh": 20 + 8 * abs(u[i])}.get(act, 4) * 2.0 ** -24 if want[i] else 0.0
        tol = rel * abs(want[i]) + 4 * 2.0 ** -149 + (2.0 ** -20 if act == "gelu" and vd[i] < 0 else 0.0)
        tol += (2.0 ** -8 * abs(want[i]) + 2.0 ** -134) if y == "bf16" else 0.0
        assert (np.abs(got[i] - want[i]) <= tol).all(), (vd[i], got[i][0], want[i], tol)


OUTLIERS = [False, True]         # V blocks between 2^-12 and 2^12 of what they are (and K's dims apart): the few-row kernel's second form


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
@pytest.mark.parametrize("e", [18, 24, 32, 45, 100])
@pytest.mark.parametrize("outliers", OUTLIERS)
def test_scores_of_2_to_the_e(attn, outliers, Dh, x, e):
    """Scores of either sign that differ by far more than f32's steps at their size: the token with the largest has all the weight.  A
    score errs by (Dh + 8) 2^-24 of the sum of |q||k| (test_attn_gpu.py); rows whose best two are closer than eight times that are left out."""
    rng = np.random.default_rng(21 + e)
    s = Setup(attn, rng, [(1, 300), (150, 3500), (70, 4000)], 16, 2, Dh, 32, x, outliers=outliers)
    s.q *= 2.0 ** e
    out, lse = (t.double().cpu().numpy() for t in s.run())
    q, scale, t0, j0, clear = s.q.double().cpu().numpy(), Dh ** -0.5, 0, 0, []
    for n, kv in s.lens:
        for h in range(16):
            k, v, qq = s.k[j0:j0 + kv, h // 8], s.v[j0:j0 + kv, h // 8], q[t0:t0 + n, h]
            seen = np.arange(kv) <= kv - n + np.arange(n)[:, None]
            sc = np.where(seen, qq @ k.T * scale, -np.inf)
            err = np.where(seen, np.abs(qq) @ np.abs(k).T * scale, 0).max(-1) * (Dh + 8) * 2.0 ** -24
            best = sc.argmax(-1)
            top, second = np.partition(sc, -2, -1)[:, -1], np.partition(sc, -2, -1)[:, -2]
            ok = top - second > 8 * err + 60
            # A 4-bit value is exact in both types.  (Below 2^20 a weight need not be a power of two: its rounding to bf16, and the output's.
            # The other tokens' weights are below e^-60 each, which shows where the value is 0.)
            near = np.where(np.abs(top) * 1.4427 < 1.01 * 2 ** 20, 2.0 ** -7, 0)[ok, None] * np.abs(v[best[ok]])
            assert (np.abs(out[t0:t0 + n, h][ok] - v[best[ok]]) <= near + kv * np.exp(-60.0) * np.abs(v).max()).all()
            assert (np.abs(lse[t0:t0 + n, h] - top) <= err + 2.0 ** -22 * np.abs(top) + np.log(kv)).all()
            clear.append(ok.mean())
        t0, j0 = t0 + n, j0 + kv
    assert np.mean(clear) > 0.8


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
def test_keys_and_queries_of_opposite_sizes(attn, Dh, x):
    """K of 2^e, q of 2^-e and scores of about 1, up to where K's scales end; some tokens' K far below the others'.  (One more rounding than the
    bounds count, that of scale * 2^-126 to f32's smallest numbers: 2^-21 of a score, where they have (Dh + 8) 2^-24.)"""
    rng = np.random.default_rng(20)
    sizes = [(1, 400, 115), (1, 90, 122), (1, 300, -115), (1, 70, -122), (3, 200, 100), (1, 500, 64), (70, 4000, 115), (70, 4000, -115)]
    s = Setup(attn, rng, [(n, kv) for n, kv, _ in sizes], 16, 2, Dh, 32, x)
    e = np.concatenate([np.full(kv, e) for _, kv, e in sizes])
    e = np.where(rng.random(len(e)) < 0.3, np.where(rng.random(len(e)) < 0.5, e - 20, 0), e).clip(-122)
    own_rows(s, rng.standard_normal((len(s.k), 2, Dh)) * 2.0 ** e[:, None, None], rng.standard_normal((len(s.k), 2, Dh)))
    at = 0
    for n, _, e in sizes:
        s.q[at:at + n] *= 2.0 ** -e
        at += n
    if x == "f32":
        s.q = s.q.bfloat16().float() + s.q.bfloat16().float() * 2.0 ** -12
    s.check(s.run())


VALUE_LENS = [[(1, 30000), (3, 400)], [(70, 4000), (200, 9000)]]


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
@pytest.mark.parametrize("e", [105, 124])
@pytest.mark.parametrize("lens", VALUE_LENS)
def test_values_up_to_the_largest(attn, lens, Dh, x, e):
    """V of 2^e and some infinities (stored as 6 * 2^125), in spans that are cut and joined and in whole ones: sums of tens of thousands
    of them times their weights, which have to be divided before they leave f32."""
    rng = np.random.default_rng(22 + e)
    s = Setup(attn, rng, lens, 16, 2, Dh, 64, x)
    v = np.clip(rng.standard_normal((len(s.k), 2, Dh)) + 2, -2, 4) * 2.0 ** e
    if e == 124:
        v[rng.random(v.shape) < 0.01] = np.inf
    own_rows(s, rng.standard_normal((len(s.k), 2, Dh)), v)
    assert np.abs(s.v).max() >= 2.0 ** e and (e < 124 or np.abs(s.v).max() == 6 * 2.0 ** 125)
    s.check(s.run())


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [64, 128, 256])
def test_blocks_of_dims_far_apart_in_turn(attn, Dh, x):
    """V in one block of dims at 2^12 (one token of 16, then 16 without any), in another at 2^-20 (those 16), zeros everywhere else: what
    the first one is must not set the precision of the second.  Requests so many that a warp goes through several groups of 16."""
    rng = np.random.default_rng(23)
    s = Setup(attn, rng, [(1, int(n)) for n in rng.integers(1500, 2500, 64)], 16, 2, Dh, 32, x)
    v = np.zeros((len(s.k), 2, Dh))
    t = np.concatenate([np.arange(n) for _, n in s.lens])
    odd = t // 16 % 2 == 1
    v[t % 32 == 3, :, 32:64] = rng.standard_normal(((t % 32 == 3).sum(), 2, 32)) * 2.0 ** 12
    v[odd, :, :32] = rng.standard_normal((odd.sum(), 2, 32)) * 2.0 ** -20
    own_rows(s, s.k, v)
    s.check(s.run())
