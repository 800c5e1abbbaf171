"""Host-side binding of the attention side of a layer (the C ABI in include/q36_attn.h): the paged 4-bit cache and its
tables, attention over it, and the matrix product back into the residual stream.

As in q36_b200.moe, torch is used for device memory and streams only.  Tensors live on the device of the cache (or of
their first operand), which is made current for the call; the stream is that device's current one unless given.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import NamedTuple

import torch

from . import moe
from .moe import MoEError, check, f32, i32, lib, ptr, u64, vp  # noqa: F401

i64 = C.c_int64

_SIGS = {
    "q36_kv_block_bytes": (u64, [i32, i32, i32]),
    "q36_kv_tables": (i32, [vp, vp, i32, i32, i32, vp, i32, vp, vp, i32, vp, vp, vp, vp, i32, vp, vp, vp]),
    "q36_kv_append": (i32, [vp, vp, i32, i64, i64, vp, vp, i32, i32, i32, i32, i32, vp]),
    "q36_kv_read": (i32, [vp, i32, i32, i32, i32, vp, vp, vp, i32, i32, vp]),
    "q36_kv_attention_workspace_bytes": (u64, [i32, i32, i32, i32]),
    "q36_kv_attention": (i32, [vp, i32, i64, vp, i32, i32, i32, i32, i32, vp, i32, vp, vp, i32, f32, i32, vp, i64, vp, i32, i32, vp, u64, vp]),
    "q36_linear": (i32, [vp, i64, vp, vp, i32, vp, i32, i64, vp, i32, i64, i32, i32, i32, vp, vp]),
    "q36_attn_block_workspace_bytes": (u64, [i32, i32, i32, i32, i32]),
    "q36_attn_block": (i32, [vp, vp, vp, i32, i64, i64, i64, vp, vp, i32, i32, i32, i32, i32, vp, i32, vp, vp, i32, f32, i32, vp, vp, vp, i32,
                             i32, i32, vp, u64, vp]),
}
for _n, (_r, _a) in _SIGS.items():
    _f = getattr(lib, _n)
    _f.restype, _f.argtypes = _r, _a

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _need(cond, what):
    if not cond:
        raise MoEError(f"{what}: {lib.q36_moe_strerror(moe.EINVAL).decode()}")


def _on(t: torch.Tensor, *others, what="") -> None:
    for o in others:
        _need(o is None or o.device == t.device, f"{what} (operands on different devices)")


def _ints(what, *ts):
    for t in ts:
        _need(t.dtype == torch.int32 and t.is_contiguous(), f"{what} (int32, contiguous)")


def _is_bf16(t, what) -> int:
    _need(t.dtype in (torch.bfloat16, torch.float32), f"{what} (bf16 or f32)")
    return int(t.dtype == torch.bfloat16)


@contextlib.contextmanager
def _on_device(dev, stream):
    with torch.cuda.device(dev), torch.cuda.stream(stream):
        yield torch.cuda.current_stream(dev).cuda_stream


def _call(dev, stream=None):
    """Makes the operands' device, and the stream asked for, current (what a call allocates belongs to that stream)."""
    _need(dev.type == "cuda", "operands not on a CUDA device")
    if stream is None and dev.index == torch.cuda.current_device():
        return contextlib.nullcontext(torch.cuda.current_stream().cuda_stream)
    return _on_device(dev, stream)


def _rows(t, inner, what) -> int:
    """Elements between the rows of t [T, *inner], whose rows are contiguous."""
    _need(tuple(t.shape[1:]) == tuple(inner), f"{what} (shape {tuple(t.shape)}, rows of {tuple(inner)})")
    n = 1
    for size, stride in zip(reversed(inner), reversed(t.stride()[1:])):
        _need(size == 1 or stride == n, f"{what} (rows not contiguous)")
        n *= size
    return t.stride(0) if t.shape[0] > 1 else n


def kv_block_bytes(block_size: int, n_kv_head: int, head_dim: int) -> int:
    return int(lib.q36_kv_block_bytes(block_size, n_kv_head, head_dim))


class Tables(NamedTuple):
    cu_q: torch.Tensor
    kv_len: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    free_head: torch.Tensor
    status: torch.Tensor


def kv_tables(kv_old, q_len, block_size, free_blocks, free_head, block_table, T, n_blocks=None, out: Tables | None = None, stream=None) -> Tables:
    """q36_kv_tables: block_table [B, width] gets its new entries in place; the rest comes back (in `out` when given,
    whose free_head and kv_len may be the ones passed in)."""
    dev, B = kv_old.device, kv_old.numel()
    _ints("kv_tables", kv_old, q_len, free_blocks, free_head, block_table)
    _on(kv_old, q_len, free_blocks, free_head, block_table, what="kv_tables")
    _need(q_len.numel() == B and block_table.shape[0] == B and free_head.numel() == 1, "kv_tables (shapes)")
    if out is None:
        with _call(dev, stream):
            out = Tables(*(torch.empty(n, dtype=torch.int32, device=dev) for n in (B + 1, B, T, T, 1, 1)))
    _ints("kv_tables", *out)
    _on(kv_old, *out, what="kv_tables")
    _need(all(t.numel() == n for t, n in zip(out, (B + 1, B, T, T, 1, 1))), "kv_tables (out)")
    with _call(dev, stream) as st:
        check(lib.q36_kv_tables(kv_old.data_ptr(), q_len.data_ptr(), B, block_size, n_blocks or (2**31 - 1) // block_size, free_blocks.data_ptr(),
                                free_blocks.numel(), free_head.data_ptr(), block_table.data_ptr(), block_table.shape[1], out.cu_q.data_ptr(),
                                out.kv_len.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(), T, out.free_head.data_ptr(),
                                out.status.data_ptr(), st), "kv_tables")
    return out


class KVCache:
    """The paged 4-bit cache of one layer: uint8 [n_blocks, n_kv_head, bytes]."""

    def __init__(self, n_blocks: int, block_size: int, n_kv_head: int, head_dim: int, device="cuda", data: torch.Tensor | None = None):
        nbytes = kv_block_bytes(block_size, n_kv_head, head_dim)
        _need(nbytes > 0 and n_blocks > 0, "KVCache (geometry)")
        shape = (n_blocks, n_kv_head, nbytes // n_kv_head)
        if data is None:
            data = torch.zeros(shape, dtype=torch.uint8, device=device)
        _need(data.shape == shape and data.dtype == torch.uint8 and data.is_contiguous(), "KVCache (data)")
        self.data, self.device = data, data.device
        self.n_blocks, self.block_size, self.n_kv_head, self.head_dim = n_blocks, block_size, n_kv_head, head_dim
        self._ws = {}

    def _geom(self):
        return self.data.data_ptr(), self.n_blocks, self.block_size

    def workspace(self, nbytes: int, stream: int) -> torch.Tensor:
        """Scratch of a call; one per stream, since calls on two streams may run at the same time.  Under capture a graph
        gets one of its own, which it keeps: replays of two graphs may run at the same time too."""
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        ws = self._ws.get(stream)
        if ws is None or ws.numel() < nbytes:
            ws = self._ws[stream] = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return ws

    def append(self, k, v, slots, stream=None) -> None:
        """k, v [T, n_kv_head, head_dim] into the cache at slots [T] (-1: skipped)."""
        _ints("kv_append", slots)
        _on(self.data, k, v, slots, what="kv_append")
        _need(k.dtype == v.dtype and k.shape == v.shape and slots.numel() == k.shape[0], "kv_append (k, v, slots)")
        inner = (self.n_kv_head, self.head_dim)
        bf, ks, vs = _is_bf16(k, "kv_append"), _rows(k, inner, "kv_append"), _rows(v, inner, "kv_append")
        with _call(self.device, stream) as st:
            check(lib.q36_kv_append(k.data_ptr(), v.data_ptr(), bf, ks, vs, slots.data_ptr(), *self._geom(), self.n_kv_head, self.head_dim, k.shape[0], st), "kv_append")

    def read(self, slots, dtype=torch.float32, stream=None):
        """(k, v) [T, n_kv_head, head_dim]: the values at slots [T]; zeros for -1."""
        _ints("kv_read", slots)
        _on(self.data, slots, what="kv_read")
        _need(dtype in (torch.bfloat16, torch.float32), "kv_read (bf16 or f32)")
        with _call(self.device, stream) as st:
            k, v = (torch.empty((slots.numel(), self.n_kv_head, self.head_dim), dtype=dtype, device=self.device) for _ in range(2))
            check(lib.q36_kv_read(*self._geom(), self.n_kv_head, self.head_dim, slots.data_ptr(), k.data_ptr(), v.data_ptr(), int(dtype == torch.bfloat16),
                                  slots.numel(), st), "kv_read")
        return k, v

    def _attn_args(self, q, block_table, cu_q, kv_len, scale, window, what):
        _ints(what, block_table, cu_q, kv_len)
        _on(self.data, q, block_table, cu_q, kv_len, what=what)
        _need(q.dim() == 3, f"{what} (q [T, n_head, head_dim])")
        B, n_head = kv_len.numel(), q.shape[1]
        _need(cu_q.numel() == B + 1 and block_table.dim() == 2 and block_table.shape[0] == B, f"{what} (tables)")
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        return (n_head, self.n_kv_head, self.head_dim, block_table.data_ptr(), block_table.shape[1], cu_q.data_ptr(), kv_len.data_ptr(), B, scale,
                window)

    def attention(self, q, block_table, cu_q, kv_len, max_q, scale=None, window=0, out=None, want_lse=False, ws=None, stream=None):
        """q [T, n_head, head_dim] -> out of the same type (and the log-sum-exp [T, n_head] when want_lse)."""
        T = q.shape[0]
        args = self._attn_args(q, block_table, cu_q, kv_len, scale, window, "kv_attention")
        inner = (q.shape[1], self.head_dim)
        _need(out is None or (out.dtype == q.dtype and out.shape == q.shape), "kv_attention (out)")
        _on(self.data, out, ws, what="kv_attention")
        bf, qs = _is_bf16(q, "kv_attention"), _rows(q, inner, "kv_attention")
        os_ = 0 if out is None else _rows(out, inner, "kv_attention")
        with _call(self.device, stream) as st:
            if out is None:
                out = torch.empty((T, *inner), dtype=q.dtype, device=self.device)
                os_ = inner[0] * inner[1]
            lse = torch.empty((T, q.shape[1]), dtype=torch.float32, device=self.device) if want_lse else None
            if ws is None:
                ws = self.workspace(int(lib.q36_kv_attention_workspace_bytes(q.shape[1], self.n_kv_head, self.head_dim, max(max_q, 1))), st)
            check(lib.q36_kv_attention(q.data_ptr(), bf, qs, *self._geom(), *args, out.data_ptr(), os_, ptr(lse), T, max_q, ws.data_ptr(), ws.numel(), st), "kv_attention")
        return (out, lse) if want_lse else out

    def block(self, q, k, v, slots, block_table, cu_q, kv_len, max_q, w_o, h, bias_o=None, scale=None, window=0, ws=None, stream=None):
        """q36_attn_block: append k, v; attention; h [T, D] f32 += attention W_o^T + bias_o, in place."""
        T = q.shape[0]
        what = "attn_block"
        args = self._attn_args(q, block_table, cu_q, kv_len, scale, window, what)
        _ints(what, slots)
        _on(self.data, k, v, slots, w_o, h, bias_o, ws, what=what)
        _need(k.dtype == q.dtype and v.dtype == q.dtype and k.shape[0] == T and v.shape[0] == T and slots.numel() == T, f"{what} (q, k, v, slots)")
        _need(w_o.dtype == torch.bfloat16 and w_o.is_contiguous() and w_o.dim() == 2 and w_o.shape[1] == q.shape[1] * self.head_dim, f"{what} (w_o)")
        _need(h.dtype == torch.float32 and h.is_contiguous() and h.shape == (T, w_o.shape[0]), f"{what} (h)")
        _need(bias_o is None or (bias_o.dtype == torch.float32 and bias_o.is_contiguous() and bias_o.numel() == w_o.shape[0]), f"{what} (bias_o)")
        inner, kv_inner = (q.shape[1], self.head_dim), (self.n_kv_head, self.head_dim)
        strides = _rows(q, inner, what), _rows(k, kv_inner, what), _rows(v, kv_inner, what)
        bf = _is_bf16(q, what)
        with _call(self.device, stream) as st:
            if ws is None:
                ws = self.workspace(int(lib.q36_attn_block_workspace_bytes(T, q.shape[1], self.n_kv_head, self.head_dim, max(max_q, 1))), st)
            check(lib.q36_attn_block(q.data_ptr(), k.data_ptr(), v.data_ptr(), bf, *strides, slots.data_ptr(), *self._geom(), *args, w_o.data_ptr(), ptr(bias_o), h.data_ptr(),
                                     w_o.shape[0], T, max_q, ws.data_ptr(), ws.numel(), st), what)
        return h


def linear(x, w, bias=None, act="none", residual=None, out=None, out_dtype=None, rows_used=None, stream=None):
    """act(x W^T + bias) + residual: x [T, K] bf16 (rows may be strided), w [N, K] bf16, bias [N] f32, residual [T, N] f32 or
    bf16 (may be `out`), out [T, N] f32 or bf16.  rows_used: int32 device scalar; rows from it on are not written."""
    _need(x.dim() == 2 and w.dim() == 2 and x.dtype == torch.bfloat16 and w.dtype == torch.bfloat16 and w.is_contiguous(), "linear (x, w bf16)")
    (T, K), N, dev = x.shape, w.shape[0], x.device
    _need(w.shape[1] == K and act in ACTS, "linear (shapes, act)")
    _on(x, w, bias, residual, out, rows_used, what="linear")
    _need(bias is None or (bias.dtype == torch.float32 and bias.is_contiguous() and bias.shape == (N,)), "linear (bias)")
    _need(residual is None or residual.shape == (T, N), "linear (residual)")
    _need(out is None or (out.shape == (T, N) and (out_dtype is None or out.dtype == out_dtype)), "linear (out)")
    if rows_used is not None:
        _ints("linear", rows_used)
    xs = _rows(x, (K,), "linear")
    rbf, rs = (0, 0) if residual is None else (_is_bf16(residual, "linear"), _rows(residual, (N,), "linear"))
    ys = N if out is None else _rows(out, (N,), "linear")
    ybf = int(out_dtype in (None, torch.bfloat16)) if out is None else _is_bf16(out, "linear")
    _need(out_dtype in (None, torch.bfloat16, torch.float32), "linear (out_dtype)")
    with _call(dev, stream) as st:
        if out is None:
            out = torch.empty((T, N), dtype=out_dtype or torch.bfloat16, device=dev)
        check(lib.q36_linear(x.data_ptr(), xs, w.data_ptr(), ptr(bias), ACTS[act], ptr(residual), rbf, rs, out.data_ptr(), ybf, ys, T, N, K, ptr(rows_used), st), "linear")
    return out
