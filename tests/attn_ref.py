"""Plain 64-bit forms of the attention side of a layer, for its tests (numpy, no code of the library)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """MXFP4 of rows: (codes 0..15, scale bytes, the values they stand for in 64 bits)."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = np.abs(x).max(-1)
    e = np.full(amax.shape, -126)
    for k in range(-126, 126):                          # smallest e with amax <= 6 * 2^e; 125 when there is none
        e = np.where(amax > 6 * 2.0 ** k, min(k + 1, 125), e)
    with np.errstate(invalid="ignore"):
        z = np.clip(x / 2.0 ** e[..., None], -6, 6)
    d = np.abs(np.abs(z)[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = np.arange(8) % 2 == 0
    mag = np.where((near & even).any(-1), (near & even).argmax(-1), near.argmax(-1))
    codes = mag + 8 * np.signbit(x)
    val = np.copysign(GRID[mag], x) * 2.0 ** e[..., None]
    flat = (*x.shape[:-2], 32 * x.shape[-2])
    return codes.reshape(flat), (e + 127).astype(np.uint8), val.reshape(flat)


def region_bytes(kc, ks, vc, vs):
    """One (block, kv head) region from codes [bs, Dh] and scale bytes [bs, Dh/32], nibble by nibble."""
    bs, Dh = kc.shape
    nb, half = Dh // 32, bs * Dh // 2
    out = np.zeros(bs * Dh * 17 // 16, np.uint8)
    for t in range(bs):
        for d in range(Dh):
            b, r = divmod(d, 32)
            word = 4 * (t * (Dh // 8) + (r // 8) * nb + b)
            out[word + r % 8 // 2] |= kc[t, d] << (4 * (r % 2))
            halfword = 2 * (((t // 2) * 8 + r // 4) * 2 * nb + (t % 2) * nb + b)
            out[half + halfword + r % 4 // 2] |= vc[t, d] << (4 * (r % 2))
    out[2 * half:2 * half + bs * nb] = ks.reshape(-1)
    out[2 * half + bs * nb:] = vs.reshape(-1)
    return out


def attention(q, k, v, n, scale, window=0, drop=None):
    """Rows q [n, Hq, Dh] over k, v [len, Hkv, Dh] -> (out, lse, A, delta, V) with A = softmax-weighted |v|, delta = the largest
    sum of |q||k| of a row, V = the sum of |v| over the tokens a row sees: what the error bounds are made of.  drop [len]: tokens left out."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    L, Hkv = k.shape[:2]
    Hq, Dh = q.shape[1:]
    G = Hq // Hkv
    pos = L - n + np.arange(n)
    j = np.arange(L)
    seen = j[None] <= pos[:, None]
    if window:
        seen &= j[None] > pos[:, None] - window
    if drop is not None:
        seen &= ~drop[None]
    out, lse = np.zeros((n, Hq, Dh)), np.full((n, Hq), -np.inf)
    A, delta, V = np.zeros((n, Hq, Dh)), np.zeros((n, Hq)), np.zeros((n, Hq, Dh))
    for h in range(Hq):
        kk, vv = k[:, h // G], v[:, h // G]
        s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
        m = s.max(-1, initial=-np.inf)
        ok = np.isfinite(m)
        p = np.exp(s[ok] - m[ok, None])
        l = p.sum(-1, keepdims=True)
        out[ok, h], A[ok, h] = p @ vv / l, p @ np.abs(vv) / l
        lse[ok, h] = m[ok] + np.log(l[:, 0])
        V[:, h] = seen @ np.abs(vv)
        delta[:, h] = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T * scale, 0).max(-1, initial=0)
    return out, lse, A, delta, V


def tables(old, new, bs, free, head, table, T, n_blocks):
    """The tables of a step, request by request."""
    table = table.copy()
    width = table.shape[1]
    cu, kv, slots, pos, flags, used, pre, rows = [0], [], [-1] * T, [-1] * T, 0, head, 0, 0
    for b, (o, q) in enumerate(zip(old, new)):
        ok, held, need = True, 0, 0
        first = rows
        rows += max(q, 0)
        if o < 0 or q < 0:
            flags, ok = flags | 4, False
        else:
            held = -(-o // bs)
            need = -(-(o + q) // bs) - held
            if held + need > width:
                flags, ok, need = flags | 2, False, 0
        if q > 0 and rows > T:
            flags |= 8
        if ok and need and head + pre + need > len(free):
            flags |= 1
        serve = ok and (need == 0 or head + pre + need <= len(free)) and (max(q, 0) == 0 or rows <= T)
        if serve:
            for i in range(need):
                table[b, held + i] = free[head + pre + i]
            if need:
                used = max(used, head + pre + need)
            for i in range(q):
                blk = table[b, (o + i) // bs]
                pos[first + i] = o + i
                slots[first + i] = blk * bs + (o + i) % bs if 0 <= blk < n_blocks else -1
        pre += need
        cu.append(min(rows, T))
        kv.append(o + q if serve else 0)
    return table, np.array(cu), np.array(kv), np.array(slots), np.array(pos), used, flags
