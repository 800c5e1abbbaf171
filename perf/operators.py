"""The attention side of a layer, as cases that can be timed: the tables of a paged cache made from request lengths, the
cache's writer and reader (4-bit MXFP4 rows), attention over that cache from one new token per request to whole prompts,
and the matrix product with bias, activation and residual that leads back into the residual stream.

`own` chooses between the library's entry points (q36_b200.attn) and plain torch operations on the same inputs.

  kind     one pass
  -------  ---------------------------------------------------------------------------------------------
  tables   block tables, row starts, cache slots and positions of a step's new tokens
  append   K and V rows into the cache as MXFP4, and the rows read back as the values they stand for
  attn     attention of the step's new tokens over the cached ones (causal, optionally a window)
  linear   y = act(x W^T + bias) + residual

The cache, as a program holds it: uint8 [blocks, kv heads, bytes], each (block, head) laid out as K codes, V codes,
K scales, V scales.  A scale byte s stands for 2^(s-127) and covers 32 consecutive dims; codes are E2M1 nibbles.
  K codes: token t, word j*(Dh/32) + b of Dh/8 words holds dims 32b + 8j .. + 7 (low nibble first)
  V codes: token pair t/2, group g of 8, token t%2: halfword b of Dh/32 holds dims 32b + 4g .. + 3
"""
import math

import torch

own = False


def _kv(name, kind, **kw):
    c = {"kind": kind, "Hq": 16, "Hkv": 2, "Dh": 128, "bs": 64, "x": "bf16", "window": 0, "lse": False}
    c.update(kw)
    return dict({"name": name}, **c) if name else c


def _lin(name, T, N, K, act="none", bias=False, res="none", y="bf16"):
    c = {"kind": "linear", "T": T, "N": N, "K": K, "act": act, "bias": bias, "res": res, "y": y}
    return dict({"name": name}, **c) if name else c


def listed():
    return [
        # the tables of a decoding step: a few users, one token each
        {"name": "tables_8", "kind": "tables", "B": 8, "ctx": 4096, "q": 1, "prompts": 0, "bs": 64},
        # those of a large mixed step: two thousand requests, most decode, sixteen bring prompts
        {"name": "tables_2000", "kind": "tables", "B": 2000, "ctx": 8192, "q": 1201, "prompts": 16, "bs": 16},
        # a decoding step's rows into the cache
        _kv("append_8", "append", T=8, x="f32"),
        # a long prompt's rows into the cache
        _kv("append_32768", "append", T=32768),
        # one user, a short context: latency
        _kv("attn_decode_1", "attn", B=1, ctx=700, q=1, prompts=0),
        # many users, contexts of all lengths up to 8192
        _kv("attn_decode_64", "attn", B=64, ctx=8192, q=1, prompts=0, Dh=128, bs=16),
        # two users with very long contexts, wide heads
        _kv("attn_decode_long", "attn", B=2, ctx=131072, q=1, prompts=0, Dh=256),
        # decoding with f32 activations, an odd group of heads, a window and the statistics asked for
        _kv("attn_decode_f32", "attn", B=33, ctx=3001, q=1, prompts=0, Hq=12, Hkv=4, Dh=64, bs=32, x="f32", window=1024, lse=True),
        # a step that mixes prompt chunks with decoding users
        _kv("attn_mixed", "attn", B=40, ctx=6000, q=777, prompts=3),
        # a prompt from its first token
        _kv("attn_prompt_8192", "attn", B=1, ctx=8192, q=8192, prompts=1),
        # the projection back into the residual stream, one token
        _lin("linear_1", 1, 2048, 2048, res="f32", y="f32"),
        # a prompt through a wide projection with everything in the epilogue
        _lin("linear_8000", 8000, 4100, 2048, act="gelu_tanh", bias=True, res="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attn", "attn", "attn", "linear", "linear"])
    if kind == "tables":
        B = _log_int(rng, 1, 2000)
        prompts = rng.choice([0, 0, 1, min(B, 16)])
        return {"kind": "tables", "B": B, "ctx": _log_int(rng, 64, 8192), "q": _log_int(rng, 2, 1201) if prompts else 1,
                "prompts": prompts, "bs": rng.choice([16, 32, 64, 128])}
    heads = rng.choice([(16, 2), (16, 2), (12, 4), (8, 8), (32, 8), (16, 1), (5, 1)])
    geo = {"Hq": heads[0], "Hkv": heads[1], "bs": rng.choice([16, 32, 64, 128]), "x": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "append":
        Dh = rng.choice([64, 128, 256])
        return _kv("", "append", Dh=Dh, T=_log_int(rng, 1, 32768 * 256 // (heads[1] * Dh)), **geo)
    if kind == "linear":
        return _lin("", _log_int(rng, 1, 8000), _log_int(rng, 64, 4100), 8 * _log_int(rng, 8, 256),
                    act=rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]), bias=rng.random() < 0.5,
                    res=rng.choice(["none", "f32", "bf16"]), y=rng.choice(["f32", "bf16"]))
    form = rng.choice(["decode", "decode", "long", "mixed", "prompt"])
    win = rng.choice([0, 0, 0, rng.randint(1, 2000)])
    lse = rng.random() < 0.3
    if form == "long":
        return _kv("", "attn", B=rng.randint(1, 2), ctx=_log_int(rng, 8192, 131072), q=1, prompts=0, Dh=rng.choice([64, 128]),
                   window=0, lse=lse, **geo)
    if form == "decode":
        return _kv("", "attn", B=_log_int(rng, 1, 64), ctx=_log_int(rng, 1, 8192), q=1, prompts=0, Dh=rng.choice([64, 128, 256]),
                   window=win, lse=lse, **geo)
    if geo["x"] == "f32":
        geo["Hq"], geo["Hkv"] = 16, 2
    if form == "mixed":
        B = _log_int(rng, 2, 40)
        return _kv("", "attn", B=B, ctx=_log_int(rng, 200, 6000), q=_log_int(rng, 2, 200 if geo["x"] == "f32" else 777),
                   prompts=rng.randint(1, min(B, 3)), Dh=rng.choice([64, 128]), window=win, lse=lse, **geo)
    q = _log_int(rng, 16, 700 if geo["x"] == "f32" else 4000)
    return _kv("", "attn", B=1, ctx=q + rng.choice([0, 0, rng.randint(1, 4000)]), q=q, prompts=1, Dh=rng.choice([64, 128]),
               window=win, lse=lse, **geo)


def _lens(case):
    """(new tokens, cached tokens with the new ones) of each request: contexts spread evenly over 1..ctx, the first ones prompts."""
    out = []
    for b in range(case["B"]):
        n = case["q"] if b < case["prompts"] else 1
        part = 1.0 if case["B"] == 1 else math.fmod((b + 1) * 0.6180339887498949, 1.0)
        out.append((n, n + int(max(case["ctx"] - n, 0) * part)))
    return out


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dtype(x):
    return torch.bfloat16 if x == "bf16" else torch.float32


# ------------------------------------------------------------------ the cache's format, in plain operations
def _positions(bs, Dh, dev):
    """Byte offset and shift inside a (block, head) region of every K code and V code [bs, Dh]."""
    t = torch.arange(bs, device=dev)[:, None]
    d = torch.arange(Dh, device=dev)[None, :]
    b, r, nb = d // 32, d % 32, Dh // 32
    k = t * (Dh // 2) + (r // 8) * (Dh // 8) + b * 4 + (r % 8) // 2
    v = bs * (Dh // 2) + (t // 2) * Dh + (r // 4) * (Dh // 8) + (t % 2) * (Dh // 16) + b * 2 + (r % 4) // 2
    shift = (4 * (d % 2)).expand(bs, Dh)
    ks = bs * Dh + t * nb + b
    return k, v, shift, ks, ks + bs * nb


def _quant(x):
    """MXFP4 codes (0..15) and scale bytes of rows whose length is a multiple of 32."""
    xb = torch.nan_to_num(x.float(), nan=0.0, posinf=math.inf, neginf=-math.inf).unflatten(-1, (-1, 32))
    amax = xb.abs().amax(-1, keepdim=True)
    bits = amax.contiguous().view(torch.int32)
    e = ((bits >> 23) - 129 + ((bits & 0x7FFFFF) > 0x400000).int()).clamp(-126, 125)
    scale = ((127 - e) << 23).view(torch.float32)
    m = (xb.abs() * scale).clamp(max=6.0)
    # steps between neighbouring values of 0 .5 1 1.5 2 3 4 6, a tie to the even code
    code = (m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int() + (m >= 3.5).int() + (m > 5.0).int()
    code = code + 8 * torch.signbit(xb).int()
    return code.flatten(-2), (e + 127).squeeze(-1)


def _values(code, scale):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    table = torch.cat([table, -table])
    return (table[code.long()].unflatten(-1, (-1, 32)) * torch.ldexp(torch.ones_like(scale, dtype=torch.float32), scale.int() - 127)[..., None]).flatten(-2)


def _pack(kc, ks, vc, vs):
    """Codes [n, bs, Dh] and scale bytes [n, bs, Dh/32] -> regions [n, bytes]."""
    n, bs, Dh = kc.shape
    ko, vo, shift, kso, vso = _positions(bs, Dh, kc.device)
    reg = torch.zeros((n, bs * Dh * 17 // 16), dtype=torch.int32, device=kc.device)
    for code, off in ((kc, ko), (vc, vo)):
        for s in (0, 1):      # the two nibbles of a byte
            reg[:, off[:, s::2].reshape(-1)] += code[:, :, s::2].reshape(n, -1).int() << (4 * s)
    reg[:, kso[:, ::32].reshape(-1)] = ks.reshape(n, -1).int()
    reg[:, vso[:, ::32].reshape(-1)] = vs.reshape(n, -1).int()
    return reg.to(torch.uint8)


def _unpack(regions, bs, Dh):
    """Regions [n, bytes] -> K and V values [n, bs, Dh] in 32 bits."""
    ko, vo, shift, kso, vso = _positions(bs, Dh, regions.device)
    take = lambda off: regions[:, off.reshape(-1)].unflatten(-1, off.shape)  # noqa: E731
    out = []
    for off, so in ((ko, kso), (vo, vso)):
        out.append(_values((take(off) >> shift.to(torch.uint8)) & 15, take(so[:, ::32]).int()))
    return out


def _make_cache(case, n_blocks, g):
    """A cache that earlier steps filled: rows as an attention layer makes them (a few strong K channels, V of one scale)."""
    Hkv, bs, Dh = case["Hkv"], case["bs"], case["Dh"]
    cache = torch.empty((n_blocks, Hkv, bs * Dh * 17 // 16), dtype=torch.uint8, device="cuda")
    gain = torch.exp(0.7 * torch.randn((1, Hkv, 1, Dh), device="cuda", generator=g))
    step = max(1, (1 << 24) // (Hkv * bs * Dh))
    for i in range(0, n_blocks, step):
        n = min(step, n_blocks - i)
        k = torch.randn((n, Hkv, bs, Dh), device="cuda", generator=g) * gain
        v = torch.randn((n, Hkv, bs, Dh), device="cuda", generator=g)
        kc, ks = _quant(k.flatten(0, 1))
        vc, vs = _quant(v.flatten(0, 1))
        cache[i:i + n] = _pack(kc, ks, vc, vs).unflatten(0, (n, Hkv))
    return cache


# ------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    kind = case["kind"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if kind == "tables":
        lens, bs = _lens(case), case["bs"]
        old, new = i32([kv - q for q, kv in lens]), i32([q for q, kv in lens])
        held = (old + bs - 1) // bs
        need = (old + new + bs - 1) // bs - held
        width, used, fresh = int((held + need).max()), int(held.sum()), int(need.sum())
        perm = torch.randperm(used + fresh + 64, device="cuda", generator=g).int()
        table = torch.full((case["B"], width), -1, dtype=torch.int32, device="cuda")
        own_rows = torch.arange(width, device="cuda")[None, :] < held[:, None]
        table[own_rows] = perm[:used]
        st.update(old=old, new=new, table=table, free=perm[used:].contiguous(), head=i32([3]), T=sum(q for q, _ in lens), n_blocks=used + fresh + 64)
    elif kind == "append":
        T, Hkv, Dh, bs = case["T"], case["Hkv"], case["Dh"], case["bs"]
        n_blocks = T // bs + 2
        st["cache"] = torch.zeros((n_blocks, Hkv, bs * Dh * 17 // 16), dtype=torch.uint8, device="cuda")
        kv = torch.randn((2, T, Hkv, Dh), device="cuda", generator=g)
        kv[0] *= torch.exp(0.7 * torch.randn((Hkv, Dh), device="cuda", generator=g))
        st["k"], st["v"] = kv.to(_dtype(case["x"])).unbind(0)
        # a run of tokens over shuffled blocks, starting inside one
        pos = torch.arange(T, device="cuda") + int(torch.randint(0, bs, (1,), device="cuda", generator=g))
        blocks = torch.randperm(n_blocks, device="cuda", generator=g)
        st["slots"] = (blocks[pos // bs] * bs + pos % bs).int()
    elif kind == "attn":
        lens, Hq, Dh, bs = _lens(case), case["Hq"], case["Dh"], case["bs"]
        nblk = [(kv + bs - 1) // bs for _, kv in lens]
        n_blocks, width = sum(nblk) + 1, max(nblk)
        st["cache"] = _make_cache(case, n_blocks, g)
        perm = torch.randperm(n_blocks, device="cuda", generator=g).int()
        cnt = torch.tensor(nblk, device="cuda")
        st["table"] = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        st["table"][torch.arange(width, device="cuda")[None, :] < cnt[:, None]] = perm[:sum(nblk)]
        T = sum(q for q, _ in lens)
        st["q"] = torch.randn((T, Hq, Dh), device="cuda", generator=g).to(_dtype(case["x"]))
        st["cu_q"] = torch.cat([i32([0]), torch.cumsum(i32([q for q, _ in lens]), 0).int()])
        st["kv_len"] = i32([kv for _, kv in lens])
        st["lens"] = lens
    else:
        T, N, K = case["T"], case["N"], case["K"]
        st["x"] = torch.randn((T, K), device="cuda", generator=g).to(torch.bfloat16)
        st["w"] = (torch.randn((N, K), device="cuda", generator=g) / math.sqrt(K)).to(torch.bfloat16)
        st["b"] = torch.randn((N,), device="cuda", generator=g) if case["bias"] else None
        st["r"] = None if case["res"] == "none" else torch.randn((T, N), device="cuda", generator=g).to(_dtype(case["res"]))
    if own and kind in ("append", "attn"):
        from q36_b200 import attn
        st["kv"] = attn.KVCache(st["cache"].shape[0], case["bs"], case["Hkv"], case["Dh"], data=st["cache"])
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from q36_b200 import attn
        if kind == "tables":
            t = attn.kv_tables(st["old"], st["new"], case["bs"], st["free"], st["head"], st["table"], st["T"])
            return {"table": st["table"], "cu_q": t.cu_q, "kv_len": t.kv_len, "slots": t.slots, "positions": t.positions, "head": t.free_head}
        if kind == "append":
            st["kv"].append(st["k"], st["v"], st["slots"])
            return st["kv"].read(st["slots"], st["k"].dtype)
        if kind == "attn":
            return st["kv"].attention(st["q"], st["table"], st["cu_q"], st["kv_len"], max(q for q, _ in st["lens"]),
                                      window=case["window"], want_lse=case["lse"])
        return attn.linear(st["x"], st["w"], bias=st["b"], act=case["act"], residual=st["r"], out_dtype=_dtype(case["y"]))
    return {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attn, "linear": _plain_linear}[kind](st)


def _plain_tables(st):
    bs, old, new, table = st["case"]["bs"], st["old"], st["new"], st["table"]
    held = (old + bs - 1) // bs
    need = (old + new + bs - 1) // bs - held
    start = torch.cumsum(need, 0) - need + st["head"]
    col = torch.arange(table.shape[1], device="cuda")[None, :] - held[:, None]
    fresh = (col >= 0) & (col < need[:, None])
    table = torch.where(fresh, st["free"][torch.where(fresh, start[:, None] + col, 0).long()], table)
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0).int()])
    t = torch.arange(st["T"], dtype=torch.int32, device="cuda")
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = old[b] + t - cu[b]
    slots = table[b, (pos // bs).long()] * bs + pos % bs
    return {"table": table, "cu_q": cu, "kv_len": old + new, "slots": slots, "positions": pos, "head": st["head"] + need.sum().int()}


def _plain_append(st):
    case, cache = st["case"], st["cache"]
    bs, Dh, Hkv = case["bs"], case["Dh"], case["Hkv"]
    ko, vo, _, kso, vso = _positions(bs, Dh, cache.device)
    slots = st["slots"].long()
    blk, tok = (slots // bs)[:, None, None], slots % bs
    head = torch.arange(Hkv, device=cache.device)[None, :, None]
    for x, off, so in ((st["k"], ko, kso), (st["v"], vo, vso)):
        code, scale = _quant(x)
        byte = (code[..., 0::2] + code[..., 1::2] * 16).to(torch.uint8)
        cache[blk, head, off[:, ::2][tok][:, None, :]] = byte
        cache[blk, head, so[:, ::32][tok][:, None, :]] = scale.to(torch.uint8)
    out = []
    for off, so in ((ko, kso), (vo, vso)):
        byte = cache[blk, head, off[:, ::2][tok][:, None, :]].int()
        code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
        out.append(_values(code, cache[blk, head, so[:, ::32][tok][:, None, :]].int()).to(st["k"].dtype))
    return tuple(out)


def _plain_attn(st):
    case, q = st["case"], st["q"]
    Hq, Hkv, Dh, bs, win = case["Hq"], case["Hkv"], case["Dh"], case["bs"], case["window"]
    G, scale = Hq // Hkv, 1.0 / math.sqrt(Dh)
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if case["lse"] else None
    t0 = 0
    for b, (n, kv) in enumerate(st["lens"]):
        blocks = st["table"][b, :(kv + bs - 1) // bs].long()
        pos = torch.arange(kv - n, kv, device=q.device)
        j = torch.arange(kv, device=q.device)
        hide = j[None, :] > pos[:, None]
        if win:
            hide = hide | (j[None, :] <= pos[:, None] - win)
        for h in range(Hkv):
            k, v = _unpack(st["cache"][blocks, h], bs, Dh)
            k, v = k.reshape(-1, Dh)[:kv], v.reshape(-1, Dh)[:kv]
            qq = q[t0:t0 + n, h * G:(h + 1) * G].float()
            step = max(1, (1 << 28) // (kv * G))
            for i in range(0, n, step):
                s = (qq[i:i + step] @ k.t()) * scale
                s = s.masked_fill(hide[i:i + step, None, :], -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.exp(s - m)
                l = p.sum(-1, keepdim=True)
                out[t0 + i:t0 + min(i + step, n), h * G:(h + 1) * G] = (p @ v / l).to(q.dtype)
                if lse is not None:
                    lse[t0 + i:t0 + min(i + step, n), h * G:(h + 1) * G] = (m + torch.log(l)).squeeze(-1)
        t0 += n
    return (out, lse) if case["lse"] else out


def _act(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(st):
    case = st["case"]
    y = st["x"].float() @ st["w"].float().t()
    if st["b"] is not None:
        y = y + st["b"]
    y = _act(y, case["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    return y.to(_dtype(case["y"]))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "linear":
        T, N, K = case["T"], case["N"], case["K"]
        size = {"f32": 4, "bf16": 2, "none": 0}
        return {"bytes": 2 * T * K + 2 * N * K + (4 * N if case["bias"] else 0) + T * N * (size[case["res"]] + size[case["y"]]),
                "flops": 2 * T * N * K}
    if kind == "append":
        n = 2 * case["T"] * case["Hkv"] * case["Dh"]
        x = 2 if case["x"] == "bf16" else 4
        return {"bytes": n * x + n * 17 // 32 + n * 17 // 32 + n * x + 4 * case["T"], "flops": 4 * n}
    lens, bs = _lens(case), case["bs"]
    T = sum(q for q, _ in lens)
    if kind == "tables":
        fresh = sum((kv + bs - 1) // bs - (kv - q + bs - 1) // bs for q, kv in lens)
        return {"bytes": 8 * len(lens) + 8 * fresh + 8 * len(lens) + 8 * T + 8, "flops": 4 * T}
    Hq, Hkv, Dh, win = case["Hq"], case["Hkv"], case["Dh"], case["window"]
    x = 2 if case["x"] == "bf16" else 4
    rows, pairs = 0, 0
    for q, kv in lens:
        rows += min(kv, win + q - 1) if win else kv
        # visible pairs: position p sees min(p + 1, window) tokens
        lo, hi = kv - q + 1, kv
        if win and lo < win < hi:
            pairs += (win - lo) * (lo + win - 1) // 2 + (hi - win + 1) * win
        elif win and win <= lo:
            pairs += q * win
        else:
            pairs += q * (lo + hi) // 2
    return {"bytes": rows * Hkv * Dh * 17 // 16 + 2 * T * Hq * Dh * x + 4 * sum((kv + bs - 1) // bs for _, kv in lens) + 8 * len(lens)
            + (4 * T * Hq if case["lse"] else 0), "flops": 4 * pairs * Hq * Dh}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rows(regions, bs, Dh, which):
    """Rows of K (0) or V (1) of regions [n, bytes], code by code from the layout, in 64 bits."""
    n, nb = regions.shape[0], Dh // 32
    half = bs * Dh // 2
    raw = regions[:, which * half:(which + 1) * half].long()
    nib = torch.stack([raw % 16, raw // 16], -1)
    if which == 0:      # [bs][4 groups][blocks][8 codes]
        code = nib.reshape(n, bs, 4, nb, 8).permute(0, 1, 3, 2, 4)
    else:               # [bs/2][8 groups][2 tokens][blocks][4 codes]
        code = nib.reshape(n, bs // 2, 8, 2, nb, 4).permute(0, 1, 3, 4, 2, 5)
    code = code.reshape(n, bs, nb, 32)
    mag, ex = (code % 8) % 2, (code % 8) // 2
    val = torch.where(ex == 0, 0.5 * mag.double(), (1 + 0.5 * mag.double()) * torch.exp2((ex - 1).double()))
    val = torch.where(code >= 8, -val, val)
    s = regions[:, 2 * half + which * bs * nb:2 * half + (which + 1) * bs * nb].reshape(n, bs, nb, 1).double()
    return (val * torch.exp2(s - 127)).reshape(n, bs, Dh)


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None
    st = prepare(case, seed)
    if kind == "append":
        out = []
        for x in (st["k"], st["v"]):
            y = x.double().reshape(*x.shape[:-1], -1, 32)
            top = y.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(top / 6))
            e = torch.where(top <= 6 * torch.exp2(e - 1), e - 1, torch.where(top > 6 * torch.exp2(e), e + 1, e)).clamp(-126, 125)
            grid = torch.tensor([0.0, 1.0, 2.0, 3.0, 4.0, 6.0, 8.0, 12.0], dtype=torch.float64, device="cuda") / 2
            z = y / torch.exp2(e)
            near = (z.abs().unsqueeze(-1) - grid).abs()
            even = torch.tensor([0, 1, 0, 1, 0, 1, 0, 1], device="cuda")
            # the nearest value, of two equally near ones that with the even code
            best = near.amin(-1, keepdim=True)
            pick = torch.where(near == best, even, 2).argmin(-1)
            out.append((torch.copysign(grid[pick], z) * torch.exp2(e)).reshape(x.shape))
        return tuple(out)
    if kind == "linear":
        y = st["x"].double() @ st["w"].double().t()
        if case["bias"]:
            y = y + st["b"].double()
        act = case["act"]
        if act == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif act == "silu":
            y = y * torch.special.expit(y)
        elif act == "gelu":
            y = y * torch.special.ndtr(y)
        elif act == "gelu_tanh":
            y = y * torch.special.expit(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return y if st["r"] is None else y + st["r"].double()
    Hq, Hkv, Dh, bs, win = case["Hq"], case["Hkv"], case["Dh"], case["bs"], case["window"]
    G = Hq // Hkv
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (n, kv) in enumerate(_lens(case)):
        ids = st["table"][b, :-(-kv // bs)].long()
        for h in range(Hkv):
            reg = st["cache"][ids, h]
            k = _exact_rows(reg, bs, Dh, 0).reshape(-1, Dh)[:kv]
            v = _exact_rows(reg, bs, Dh, 1).reshape(-1, Dh)[:kv]
            for i in range(0, n, 1024):
                m = min(1024, n - i)
                p = torch.arange(m, device="cuda")[:, None] + (kv - n + i)
                j = torch.arange(kv, device="cuda")[None, :]
                seen = (j <= p) & (j > p - win) if win else j <= p
                for a in range(h * G, h * G + G):
                    s = st["q"][t0 + i:t0 + i + m, a].double() @ k.t() / math.sqrt(Dh)
                    s = torch.where(seen, s, torch.full_like(s, -math.inf))
                    lse[t0 + i:t0 + i + m, a] = torch.logsumexp(s, -1)
                    out[t0 + i:t0 + i + m, a] = torch.softmax(s, -1) @ v
        t0 += n
    return (out, lse) if case["lse"] else out
