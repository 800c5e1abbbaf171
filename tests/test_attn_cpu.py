"""CPU tests of the attention side's boundary: symbols, sizes, and every refusal before the device is touched."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = C.c_void_p(4096)          # never dereferenced: every call here is refused
ODD = C.c_void_p(4096 + 4)
BIG = 1 << 40


@pytest.fixture(scope="module")
def attn(moe):
    from q36_b200 import attn
    return attn


def test_every_declared_symbol_is_exported_and_bound(attn):
    txt = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "q36_attn.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(q36_\w+)\s*\(", txt))
    assert names == set(attn._SIGS)
    assert all(hasattr(attn.lib, n) for n in names)


def test_header_is_plain_c99(tmp_path):
    src = tmp_path / "u.c"
    src.write_text('#include "q36_attn.h"\nint main(void) { return (int)(sizeof(&q36_linear) == 0); }\n')
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), "-fsyntax-only", str(src)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_sizes(attn):
    L = attn.lib
    assert L.q36_kv_block_bytes(64, 2, 128) == 64 * 2 * 2 * (128 // 2 + 128 // 32)
    for bs, h, d in ((8, 2, 128), (48, 2, 128), (64, 0, 128), (64, 2, 96), (64, 2, 512), (256, 2, 64)):
        assert L.q36_kv_block_bytes(bs, h, d) == 0
    assert L.q36_kv_attention_workspace_bytes(16, 2, 128, 1) > 0
    for hq, hk, d, q in ((15, 2, 128, 1), (0, 2, 128, 1), (16, 2, 100, 1), (16, 2, 128, 0), (129, 1, 64, 1)):
        assert L.q36_kv_attention_workspace_bytes(hq, hk, d, q) == 0
        assert L.q36_attn_block_workspace_bytes(4, hq, hk, d, q) == 0
    assert L.q36_attn_block_workspace_bytes(4, 16, 2, 128, 1) >= L.q36_kv_attention_workspace_bytes(16, 2, 128, 1) + 4 * 16 * 128 * 2


def _change(good, i, v):
    a = list(good)
    a[i] = v
    return a


def test_tables_refusals(attn, moe):
    f = attn.lib.q36_kv_tables
    good = [P, P, 4, 64, 100, P, 10, P, P, 8, P, P, P, P, 16, P, P, None]
    for i, v in [(0, None), (1, None), (5, None), (7, None), (8, None), (10, None), (11, None), (12, None), (13, None), (15, None), (16, None),
                 (2, 0), (2, 16385), (3, 24), (3, 0), (4, 0), (4, 1 << 25), (6, -1), (9, 0), (9, 1 << 25), (14, -1)]:
        assert f(*_change(good, i, v)) == moe.EINVAL, (i, v)


def test_append_and_read_refusals(attn, moe):
    f = attn.lib.q36_kv_append
    good = [P, P, 1, 256, 256, P, P, 100, 64, 2, 128, 4, None]
    for i, v in [(0, None), (1, None), (5, None), (6, None), (0, ODD), (1, ODD), (6, ODD), (3, 255), (4, 248), (3, 260), (7, 0), (7, 1 << 25), (8, 20),
                 (9, 0), (10, 80), (11, -1)]:
        assert f(*_change(good, i, v)) == moe.EINVAL, (i, v)
    f = attn.lib.q36_kv_read
    good = [P, 100, 64, 2, 128, P, P, P, 1, 4, None]
    for i, v in [(0, None), (5, None), (6, None), (7, None), (0, ODD), (6, ODD), (7, ODD), (1, 0), (2, 20), (3, 0), (4, 80), (9, -1)]:
        assert f(*_change(good, i, v)) == moe.EINVAL, (i, v)


#        q  bf st    cache nb  bs  Hq  Hk  Dh   tab mb cu len B  scale win out ostr  lse   T  mq ws wsb  stream
ATTN = [P, 1, 2048, P, 100, 64, 16, 2, 128, P, 8, P, P, 4, 0.1, 0, P, 2048, None, 4, 1, P, BIG, None]


def test_attention_refusals(attn, moe):
    f = attn.lib.q36_kv_attention
    for i, v in [(0, None), (3, None), (9, None), (11, None), (12, None), (16, None), (21, None), (0, ODD), (3, ODD), (16, ODD), (21, ODD),
                 (2, 2040), (2, 2052), (17, 2040), (17, 2052), (4, 0), (4, 1 << 25), (5, 20), (6, 15), (6, 0), (7, 0), (8, 96), (10, 0), (10, 1 << 25),
                 (13, 0), (13, 16385), (14, float("nan")), (14, float("inf")), (15, -1), (19, -1), (20, 0)]:
        assert f(*_change(ATTN, i, v)) == moe.EINVAL, (i, v)
    a = _change(ATTN, 6, 2 * 129)
    a[2] = a[17] = 2 * 129 * 128
    assert f(*a) == moe.EINVAL                                              # more than 128 query heads per kv head
    assert f(*_change(ATTN, 22, 16)) == moe.ENOSPACE
    assert f(*_change(ATTN, 19, 0)) == moe.OK                               # nothing to do: nothing launched


def test_linear_refusals(attn, moe):
    f = attn.lib.q36_linear
    #       x  xs   w  bias act res rbf rs  y  ybf ys  T  N   K   rows stream
    good = [P, 256, P, None, 0, None, 0, 0, P, 1, 64, 4, 64, 256, None, None]
    for i, v in [(0, None), (2, None), (8, None), (0, ODD), (2, ODD), (1, 248), (1, 260), (4, -1), (4, 5), (10, 63), (11, -1), (12, 0), (13, 0), (13, 250)]:
        assert f(*_change(good, i, v)) == moe.EINVAL, (i, v)
    assert f(*_change(good, 8, C.c_void_p(4097))) == moe.EINVAL
    with_res = _change(good, 5, P)
    assert f(*_change(with_res, 7, 63)) == moe.EINVAL
    with_res[7] = 64
    assert f(*with_res) == moe.EINVAL                                       # residual is y, with another type
    with_res[6], with_res[7] = 1, 128
    assert f(*with_res) == moe.EINVAL                                       # residual is y, with another stride
    assert f(*_change(good, 11, 0)) == moe.OK


def test_block_refusals(attn, moe):
    f = attn.lib.q36_attn_block
    #       q  k  v bf qs    ks   vs   slots cache nb  bs  Hq  Hk Dh   tab mb cu len B  scale win wo bias h  D    T mq ws wsb  stream
    good = [P, P, P, 1, 2048, 256, 256, P, P, 100, 64, 16, 2, 128, P, 8, P, P, 4, 0.1, 0, P, None, P, 512, 4, 1, P, BIG, None]
    for i, v in [(0, None), (1, None), (2, None), (7, None), (8, None), (14, None), (16, None), (17, None), (21, None), (23, None), (27, None),
                 (1, ODD), (2, ODD), (21, ODD), (27, ODD), (4, 2040), (5, 248), (6, 250), (10, 20), (11, 15), (13, 96), (24, 0), (25, -1), (26, 0)]:
        assert f(*_change(good, i, v)) == moe.EINVAL, (i, v)
    assert f(*_change(good, 28, 16)) == moe.ENOSPACE
    assert f(*_change(good, 25, 0)) == moe.OK


def test_binding_refuses_what_the_library_cannot_see(attn):
    """Types, shapes and devices: the C side gets bare pointers."""
    import torch
    z = lambda *s, **k: torch.zeros(*s, **k)  # noqa: E731
    i32 = torch.int32
    with pytest.raises(attn.MoEError):
        attn.KVCache(4, 24, 2, 128, device="cpu")
    with pytest.raises(attn.MoEError):
        attn.KVCache(4, 16, 2, 128, data=z((4, 2, 16), dtype=torch.uint8))
    kv = attn.KVCache(4, 16, 2, 64, device="cpu")
    k = z((3, 2, 64))
    for kk, vv, ss in ((k, k[:2], z(3, dtype=i32)), (k, k.bfloat16(), z(3, dtype=i32)), (k, k, z(3, dtype=torch.int64)), (k, k, z(2, dtype=i32)),
                       (k.double(), k.double(), z(3, dtype=i32)), (z((3, 64, 2)).transpose(1, 2), k, z(3, dtype=i32)),
                       (z((3, 2, 32)), z((3, 2, 32)), z(3, dtype=i32))):
        with pytest.raises(attn.MoEError):
            kv.append(kk, vv, ss)
    q, tab, cu, ln = z((3, 4, 64)), z((1, 2), dtype=i32), z(2, dtype=i32), z(1, dtype=i32)
    for args in ((q[0], tab, cu, ln), (q, tab[0], cu, ln), (q, tab, cu[:1], ln), (q, tab.long(), cu, ln), (q.half(), tab, cu, ln)):
        with pytest.raises(attn.MoEError):
            kv.attention(*args, 1, out=None if args[0].dtype != torch.float16 else q)
    x, w = z((2, 64), dtype=torch.bfloat16), z((8, 64), dtype=torch.bfloat16)
    for kw in (dict(x=x.float()), dict(w=w.t()), dict(w=w[:, :32]), dict(act="tanh"), dict(bias=z(7)), dict(bias=z(8).bfloat16()),
               dict(residual=z((2, 7))), dict(out=z((3, 8))), dict(rows_used=z(1, dtype=torch.int64))):
        with pytest.raises(attn.MoEError):
            attn.linear(**{**dict(x=x, w=w), **kw})


def test_binding_refuses_numbers_that_would_wrap(attn):
    """ctypes cuts integers to 32 bits without a word."""
    import torch
    i32 = torch.int32
    kv = attn.KVCache(4, 16, 2, 64, device="cpu")
    q, tab, cu, ln = torch.zeros((3, 4, 64)), torch.zeros((1, 2), dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32)
    for window in (-1, 2**31, 2**32 + 5):
        with pytest.raises(attn.MoEError, match="window"):
            kv.attention(q, tab, cu, ln, 1, window=window)
    with pytest.raises(AttributeError):
        kv.data = torch.zeros(1)                                            # its address is the library's


def test_sizes_whose_sums_would_pass_32_bits_are_refused(attn, moe):
    f = attn.lib.q36_kv_attention
    for i, v in [(19, (1 << 30) // 16 + 1), (14, 3e38), (18, C.c_void_p(4098))]:
        assert f(*_change(ATTN, i, v)) == moe.EINVAL, (i, v)
    f = attn.lib.q36_linear
    good = [P, 256, P, None, 0, None, 0, 0, P, 1, 64, 4, 64, 256, None, None]
    for i, v in [(11, (1 << 30) + 1), (3, C.c_void_p(4098))]:
        assert f(*_change(good, i, v)) == moe.EINVAL, (i, v)
    big = _change(good, 12, (1 << 30) + 1)
    big[10] = 1 << 31
    assert f(*big) == moe.EINVAL
