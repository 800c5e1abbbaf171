"""What the binding of the attention side has to refuse itself: numbers beyond 32 bits, which ctypes cuts without a word, and an empty
tensor where the library takes a null address for something else."""
import pytest


@pytest.fixture
def attn(moe, monkeypatch):
    """The binding with a library that takes every call, so that only the binding's own checks can refuse."""
    import torch
    from q36_b200 import attn
    monkeypatch.setattr(attn, "_call", lambda dev, st=None: attn._Here(0))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for name in ("_attention_ws", "_block_ws"):
        monkeypatch.setattr(attn, name, lambda *a: 256)
    for name in ("q36_kv_tables", "q36_kv_append", "q36_kv_read", "q36_kv_attention", "q36_linear", "q36_attn_block"):
        monkeypatch.setattr(attn.lib, name, lambda *a: 0)
    return attn


def i32(*shape):
    import torch
    return torch.zeros(shape, dtype=torch.int32)


def test_tables(attn):
    good = dict(kv_old=i32(2), q_len=i32(2), block_size=16, free_blocks=i32(4), free_head=i32(1), block_table=i32(2, 3), T=5, n_blocks=9)
    attn.kv_tables(**good)
    attn.kv_tables(**{**good, "n_blocks": None})
    for change in (dict(n_blocks=2**32 + 5), dict(n_blocks=2**31), dict(block_size=2**32 + 16), dict(T=-1)):
        with pytest.raises(attn.MoEError):
            attn.kv_tables(**{**good, **change})


def test_tables_with_more_than_32_bits_of_entries(attn):
    """(On the meta device: sizes without memory.)"""
    import torch
    m = lambda *shape: torch.empty(shape, dtype=torch.int32, device="meta")  # noqa: E731
    good = dict(kv_old=m(1), q_len=m(1), block_size=16, free_blocks=m(4), free_head=m(1), block_table=m(1, 3), T=5, n_blocks=9)
    attn.kv_tables(**good)
    for change in (dict(block_table=m(1, 2**32 + 3)), dict(free_blocks=m(2**32 + 4)), dict(T=2**32 + 5),
                   dict(kv_old=m(2**32 + 2), q_len=m(2**32 + 2), block_table=m(2**32 + 2, 1))):
        with pytest.raises(attn.MoEError, match="32 bits"):
            attn.kv_tables(**{**good, **change})


def test_cache(attn):
    import torch
    for args in ((2**32 + 4, 16, 2, 64), (4, 2**32 + 16, 2, 64), (4, 16, 2**32 + 2, 64), (4, 16, 2, 2**32 + 64)):
        with pytest.raises(attn.MoEError):
            attn.KVCache(*args, device="meta")
    kv = attn.KVCache(4, 16, 2, 64, device="cpu")
    q, k, w, h = torch.zeros((3, 4, 64)), torch.zeros((3, 2, 64)), torch.zeros((8, 256), dtype=torch.bfloat16), torch.zeros((3, 8))
    kv.attention(q, i32(1, 2), i32(2), i32(1), 3)
    kv.block(q, k, k, i32(3), i32(1, 2), i32(2), i32(1), 3, w, h)
    for max_q in (2**31, 2**32 + 1, -2**31 - 1):
        with pytest.raises(attn.MoEError):
            kv.attention(q, i32(1, 2), i32(2), i32(1), max_q)
        with pytest.raises(attn.MoEError):
            kv.block(q, k, k, i32(3), i32(1, 2), i32(2), i32(1), max_q, w, h)


def test_linear(attn):
    import torch
    x, w = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((8, 64), dtype=torch.bfloat16)
    attn.linear(x, w, rows_used=i32(1))
    attn.linear(x, w, rows_used=torch.tensor(1, dtype=torch.int32))
    for rows in (i32(0), i32(2)):                                                 # (the address of none is null: all rows)
        with pytest.raises(attn.MoEError, match="rows_used"):
            attn.linear(x, w, rows_used=rows)
    big = torch.empty((2**32 + 8, 64), dtype=torch.bfloat16, device="meta")
    with pytest.raises(attn.MoEError, match="32 bits"):
        attn.linear(torch.empty((2, 64), dtype=torch.bfloat16, device="meta"), big)


def test_a_stream_of_another_device(moe):
    """Its device would become the current one, and the launch would be that device's with this one's addresses."""
    import types
    import torch
    from q36_b200 import attn
    for dev, index in ((0, 1), (3, 0)):
        with pytest.raises(attn.MoEError, match="different devices"):
            attn._call(dev, types.SimpleNamespace(device=torch.device("cuda", index)))
