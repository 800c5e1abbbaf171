"""The binding's scratch when several host threads use one cache: a call's launches hand partial results over in it, so no other call may
be given it until the last of them is in the stream."""
import threading
import time

import pytest


@pytest.fixture
def cache(moe, monkeypatch):
    """A cache on the host and a library whose launches only note who has which workspace."""
    import torch
    from q36_b200 import attn
    stream = threading.local()
    kv = attn.KVCache(4, 16, 2, 64, device="cpu")
    busy, seen, clash = {}, set(), []

    def launches(*args):
        ws = args[-3]
        clash.append(busy.get(ws, 0))
        busy[ws] = busy.get(ws, 0) + 1
        seen.add((stream.st, ws))
        time.sleep(0.002)                       # (the library runs without the interpreter's lock)
        busy[ws] -= 1
        return 0

    monkeypatch.setattr(attn, "_call", lambda dev, st=None: attn._Here(stream.st))
    monkeypatch.setattr(attn, "_attention_ws", lambda *a: 256)
    monkeypatch.setattr(attn, "_block_ws", lambda *a: 256)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for name in ("q36_kv_attention", "q36_attn_block"):
        monkeypatch.setattr(attn.lib, name, launches)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    q, k, w, h = torch.zeros((3, 4, 64)), torch.zeros((3, 2, 64)), torch.zeros((8, 256), dtype=torch.bfloat16), torch.zeros((3, 8))

    def work(st, n=12):
        stream.st = st
        for i in range(n):
            if i % 2:
                kv.attention(q, torch.zeros((1, 2), dtype=torch.int32), i32(2), i32(1), 1)
            else:
                kv.block(q, k, k, i32(3), torch.zeros((1, 2), dtype=torch.int32), i32(2), i32(1), 1, w, h)

    return work, seen, clash


@pytest.mark.parametrize("streams", [(7, 7), (7, 7, 9, 9)])
def test_no_two_calls_have_one_scratch_at_a_time(cache, streams):
    work, seen, clash = cache
    threads = [threading.Thread(target=work, args=(st,)) for st in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(clash) == 12 * len(streams) and not any(clash)
    by_stream = {st: {ws for s, ws in seen if s == st} for st in streams}
    assert not set.intersection(*by_stream.values()) if len(by_stream) > 1 else True      # two streams may run at the same time
