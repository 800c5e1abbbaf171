"""Host-side binding of the attention side of a layer (the C ABI in include/q36_attn.h): the paged 4-bit cache and its
tables, attention over it, and the matrix product back into the residual stream.

As in q36_b200.moe, torch is used for device memory and streams only.  Tensors live on the device of the cache (or of
their first operand), which is made current for the call; the stream is that device's current one unless given.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
import threading
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
_SIGS["q36_attn_status"] = _SIGS["q36_attn_selftest_wait_timeout"] = (i32, [vp])
for _n, (_r, _a) in _SIGS.items():
    _f = getattr(lib, _n)
    _f.restype, _f.argtypes = _r, _a

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


_I32, _BF16, _F32, _U8 = torch.int32, torch.bfloat16, torch.float32, torch.uint8


def _refuse(what):
    raise MoEError(f"{what}: {lib.q36_moe_strerror(moe.EINVAL).decode()}")


def _need(cond, what):
    if not cond:
        _refuse(what)


# The checks below run on every call of a decoding step, next to kernels of a few microseconds: they look at attributes only.
def _ints(what, dev, *ts):
    """int32, contiguous, on device `dev` (an index; -1: the host, refused when the call is made)."""
    for t in ts:
        if t.dtype is not _I32 or not t.is_contiguous() or t.get_device() != dev:
            _refuse(f"{what} (int32, contiguous, on the operands' device)")


# ctypes cuts integers to 32 bits without a word.  (Sizes whose tensors would not fit the GPU's memory are not looked at.)
_INT_MAX = 2**31 - 1


def _on(what, dev, *ts):
    for t in ts:
        if t is not None and t.get_device() != dev:
            _refuse(f"{what} (operands on different devices)")


def _is_bf16(t, what) -> int:
    if t.dtype is _BF16:
        return 1
    if t.dtype is not _F32:
        _refuse(f"{what} (bf16 or f32)")
    return 0


# the current stream's handle without a Stream object around it (3 us of a call that takes 10)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


@contextlib.contextmanager
def _on_device(dev, stream):
    with torch.cuda.device(dev), torch.cuda.stream(stream):
        yield _raw_stream(dev)


class _Here:
    """The operands' device is current already, and so is the stream."""

    __slots__ = ("st",)

    def __init__(self, st):
        self.st = st

    def __enter__(self):
        return self.st

    def __exit__(self, *a):
        return False


def _call(dev: int, stream=None):
    """Makes the operands' device, and the stream asked for, current (what a call allocates belongs to that stream)."""
    if dev < 0:
        _refuse("operands not on a CUDA device")
    if stream is None and dev == torch.cuda.current_device():
        return _Here(_raw_stream(dev))
    if stream is not None and stream.device.index != dev:
        _refuse("operands and stream on different devices")
    return _on_device(dev, stream)


def _rows2(t, n, what) -> int:
    """Elements between the rows of t [T, n], whose rows are contiguous."""
    T, m = t.shape
    s = t.stride()
    if m != n or (n > 1 and s[1] != 1):
        _refuse(f"{what} (shape {tuple(t.shape)}, rows of {n}, contiguous)")
    return s[0] if T > 1 else n


def _rows3(t, h, d, what) -> int:
    """Elements between the rows of t [T, h, d], whose rows are contiguous."""
    if t.dim() != 3 or t.shape[1] != h or t.shape[2] != d:
        _refuse(f"{what} (shape {tuple(t.shape)}, rows of {h} x {d})")
    s = t.stride()
    if s[2] != 1 or (h > 1 and s[1] != d):
        _refuse(f"{what} (rows not contiguous)")
    return s[0] if t.shape[0] > 1 else h * d


# (strides given: a microsecond less than torch.empty)
def _rows(T, h, d, dtype, device):
    return torch.empty_strided((T, h, d), (h * d, d, 1), dtype=dtype, device=device)


def kv_block_bytes(block_size: int, n_kv_head: int, head_dim: int) -> int:
    _need(max(block_size, n_kv_head, head_dim) <= _INT_MAX, "kv_block_bytes (32 bits)")
    return int(lib.q36_kv_block_bytes(block_size, n_kv_head, head_dim))


def check_device_status(device=None) -> None:
    """Raises when a bounded wait of the attention or product kernels gave up on the device since the last check (by anyone: for one
    checking thread per device)."""
    with torch.cuda.device(device):
        check(lib.q36_attn_status(torch.cuda.current_stream().cuda_stream), "attn device status")


# Workspace sizes by device (which is current) and sizes: a call of the library costs a microsecond.
@functools.lru_cache(maxsize=1024)
def _attention_ws(dev, n_head, n_kv_head, head_dim, max_q) -> int:
    return int(lib.q36_kv_attention_workspace_bytes(n_head, n_kv_head, head_dim, max_q))


@functools.lru_cache(maxsize=1024)
def _block_ws(dev, T, n_head, n_kv_head, head_dim, max_q) -> int:
    return int(lib.q36_attn_block_workspace_bytes(T, n_head, n_kv_head, head_dim, max_q))


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
    dev, B = kv_old.get_device(), kv_old.numel()
    _ints("kv_tables", dev, kv_old, q_len, free_blocks, free_head, block_table)
    if q_len.numel() != B or block_table.dim() != 2 or block_table.shape[0] != B or free_head.numel() != 1:
        _refuse("kv_tables (shapes)")
    if n_blocks is None:
        n_blocks = _INT_MAX // max(block_size, 1)
    if T < 0 or B > _INT_MAX or T > _INT_MAX or block_size > _INT_MAX or n_blocks > _INT_MAX or free_blocks.numel() > _INT_MAX or block_table.shape[1] > _INT_MAX:
        _refuse("kv_tables (sizes below 0 or beyond 32 bits)")
    sizes = (B + 1, B, T, T, 1, 1)
    if out is not None:
        _ints("kv_tables", dev, *out)
        _need(all(t.numel() == n for t, n in zip(out, sizes)), "kv_tables (out)")
    with _call(dev, stream) as st:
        if out is None:
            out = Tables(*torch.unsafe_split_with_sizes(torch.empty(2 * (B + T) + 3, dtype=_I32, device=kv_old.device), sizes))
        rc = lib.q36_kv_tables(kv_old.data_ptr(), q_len.data_ptr(), B, block_size, n_blocks, free_blocks.data_ptr(),
                               free_blocks.numel(), free_head.data_ptr(), block_table.data_ptr(), block_table.shape[1], out.cu_q.data_ptr(),
                               out.kv_len.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(), T, out.free_head.data_ptr(),
                               out.status.data_ptr(), st)
        if rc:
            check(rc, "kv_tables")
    return out


_NO_LOCK = contextlib.nullcontext()      # (a caller with a workspace of its own)


class KVCache:
    """The paged 4-bit cache of one layer: uint8 [n_blocks, n_kv_head, bytes]."""

    def __init__(self, n_blocks: int, block_size: int, n_kv_head: int, head_dim: int, device="cuda", data: torch.Tensor | None = None):
        nbytes = kv_block_bytes(block_size, n_kv_head, head_dim)
        _need(nbytes > 0 and 0 < n_blocks <= _INT_MAX, "KVCache (geometry)")
        shape = (n_blocks, n_kv_head, nbytes // n_kv_head)
        if data is None:
            data = torch.zeros(shape, dtype=_U8, device=device)
        _need(data.shape == shape and data.dtype is _U8 and data.is_contiguous(), "KVCache (data)")
        self._data, self.device, self._dev = data, data.device, data.get_device()
        self.n_blocks, self.block_size, self.n_kv_head, self.head_dim = n_blocks, block_size, n_kv_head, head_dim
        self._geom = (data.data_ptr(), n_blocks, block_size)
        self._ws, self._lock = {}, threading.Lock()

    @property
    def data(self) -> torch.Tensor:
        return self._data

    def _scratch(self, nbytes: int, st: int) -> torch.Tensor:
        """Scratch of a call; one per stream, since calls on two streams may run at the same time.  Calls of two threads on one
        stream hold the lock from here to their last launch: a call's launches hand its parts over in here, and another call's may not
        come between them.  Under capture a graph gets one of its own, which it keeps: replays of two graphs may run at the same time too."""
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(nbytes, dtype=_U8, device=self.device)
        ws = self._ws.get(st)
        if ws is None or ws.numel() < nbytes:
            ws = self._ws[st] = torch.empty(nbytes, dtype=_U8, device=self.device)
        return ws

    def append(self, k, v, slots, stream=None) -> None:
        """k, v [T, n_kv_head, head_dim] into the cache at slots [T] (-1: skipped)."""
        dev, T = self._dev, slots.numel()
        _ints("kv_append", dev, slots)
        _on("kv_append", dev, k, v)
        if k.dtype is not v.dtype or k.shape != v.shape or T != k.shape[0]:
            _refuse("kv_append (k, v, slots)")
        bf = _is_bf16(k, "kv_append")
        ks, vs = (_rows3(t, self.n_kv_head, self.head_dim, "kv_append") for t in (k, v))
        with _call(dev, stream) as st:
            rc = lib.q36_kv_append(k.data_ptr(), v.data_ptr(), bf, ks, vs, slots.data_ptr(), *self._geom, self.n_kv_head, self.head_dim, T, st)
            if rc:
                check(rc, "kv_append")

    def read(self, slots, dtype=torch.float32, stream=None):
        """(k, v) [T, n_kv_head, head_dim]: the values at slots [T]; zeros for -1."""
        dev, T = self._dev, slots.numel()
        _ints("kv_read", dev, slots)
        if dtype is not _BF16 and dtype is not _F32:
            _refuse("kv_read (bf16 or f32)")
        with _call(dev, stream) as st:
            k, v = _rows(T, self.n_kv_head, self.head_dim, dtype, self.device), _rows(T, self.n_kv_head, self.head_dim, dtype, self.device)
            rc = lib.q36_kv_read(*self._geom, self.n_kv_head, self.head_dim, slots.data_ptr(), k.data_ptr(), v.data_ptr(), int(dtype is _BF16), T, st)
            if rc:
                check(rc, "kv_read")
        return k, v

    def _attn_args(self, q, block_table, cu_q, kv_len, max_q, scale, window, what):
        _ints(what, self._dev, block_table, cu_q, kv_len)
        _on(what, self._dev, q)
        B = kv_len.numel()
        if q.dim() != 3 or cu_q.numel() != B + 1 or block_table.dim() != 2 or block_table.shape[0] != B:
            _refuse(f"{what} (q [T, n_head, head_dim], tables)")
        if not 0 <= window < 2**31:
            _refuse(f"{what} (window)")
        if not 0 < max_q <= _INT_MAX or block_table.shape[1] > _INT_MAX:
            _refuse(f"{what} (max_q, table: 1 to 2^31 - 1)")
        scale = self.head_dim ** -0.5 if scale is None else scale
        return (*self._geom, q.shape[1], self.n_kv_head, self.head_dim, block_table.data_ptr(), block_table.shape[1], cu_q.data_ptr(),
                kv_len.data_ptr(), B, scale, window)

    def attention(self, q, block_table, cu_q, kv_len, max_q, scale=None, window=0, out=None, want_lse=False, ws=None, stream=None):
        """q [T, n_head, head_dim] -> out of the same type (and the log-sum-exp [T, n_head] when want_lse).  max_q: the largest
        number of new tokens of a request, as far as known; it chooses kernels only."""
        what = "kv_attention"
        args = self._attn_args(q, block_table, cu_q, kv_len, max_q, scale, window, what)
        T, h, d = q.shape
        bf, qs = _is_bf16(q, what), _rows3(q, h, self.head_dim, what)
        os_ = h * d
        if out is not None:
            if out.dtype is not q.dtype or out.shape != q.shape:
                _refuse(f"{what} (out)")
            os_ = _rows3(out, h, d, what)
        _on(what, self._dev, out, ws)
        if ws is not None and not ws.is_contiguous():
            _refuse(f"{what} (ws)")
        with _call(self._dev, stream) as st:
            if out is None:
                out = _rows(T, h, d, q.dtype, self.device)
            lse = torch.empty((T, h), dtype=_F32, device=self.device) if want_lse else None
            with self._lock if ws is None else _NO_LOCK:
                if ws is None:
                    ws = self._scratch(_attention_ws(self._dev, h, self.n_kv_head, d, max_q), st)
                rc = lib.q36_kv_attention(q.data_ptr(), bf, qs, *args, out.data_ptr(), os_, ptr(lse), T, max_q, ws.data_ptr(), ws.numel(), st)
            if rc:
                check(rc, what)
        return (out, lse) if want_lse else out

    def block(self, q, k, v, slots, block_table, cu_q, kv_len, max_q, w_o, h, bias_o=None, scale=None, window=0, ws=None, stream=None):
        """q36_attn_block: append k, v; attention; h [T, D] f32 += attention W_o^T + bias_o, in place."""
        what = "attn_block"
        args = self._attn_args(q, block_table, cu_q, kv_len, max_q, scale, window, what)
        dev, (T, n_head, _) = self._dev, q.shape
        _ints(what, dev, slots)
        _on(what, dev, k, v, w_o, h, bias_o, ws)
        _need(k.dtype is q.dtype and v.dtype is q.dtype and k.shape[0] == T and v.shape[0] == T and slots.numel() == T, f"{what} (q, k, v, slots)")
        _need(w_o.dtype is _BF16 and w_o.is_contiguous() and w_o.dim() == 2 and w_o.shape[1] == n_head * self.head_dim, f"{what} (w_o)")
        D = w_o.shape[0]
        _need(ws is None or ws.is_contiguous(), f"{what} (ws)")
        _need(h.dtype is _F32 and h.is_contiguous() and h.shape == (T, D), f"{what} (h)")
        _need(bias_o is None or (bias_o.dtype is _F32 and bias_o.is_contiguous() and bias_o.shape == (D,)), f"{what} (bias_o)")
        bf, qs = _is_bf16(q, what), _rows3(q, n_head, self.head_dim, what)
        ks, vs = (_rows3(t, self.n_kv_head, self.head_dim, what) for t in (k, v))
        with _call(dev, stream) as st:
            with self._lock if ws is None else _NO_LOCK:
                if ws is None:
                    ws = self._scratch(_block_ws(dev, T, n_head, self.n_kv_head, self.head_dim, max_q), st)
                rc = lib.q36_attn_block(q.data_ptr(), k.data_ptr(), v.data_ptr(), bf, qs, ks, vs, slots.data_ptr(), *args, w_o.data_ptr(), ptr(bias_o),
                                        h.data_ptr(), D, T, max_q, ws.data_ptr(), ws.numel(), st)
            if rc:
                check(rc, what)
        return h


def linear(x, w, bias=None, act="none", residual=None, out=None, out_dtype=None, rows_used=None, stream=None):
    """act(x W^T + bias) + residual: x [T, K] bf16 (rows may be strided), w [N, K] bf16, bias [N] f32, residual [T, N] f32 or
    bf16 (may be `out`), out [T, N] f32 or bf16 (bf16 unless asked for).  rows_used: int32 device scalar; rows from it on are
    not written."""
    if x.dim() != 2 or w.dim() != 2 or x.dtype is not _BF16 or w.dtype is not _BF16 or not w.is_contiguous():
        _refuse("linear (x [T, K], w [N, K], bf16)")
    (T, K), N, dev = x.shape, w.shape[0], x.get_device()
    if w.shape[1] != K or act not in ACTS:
        _refuse("linear (shapes, act)")
    if T > _INT_MAX or N > _INT_MAX or K > _INT_MAX:
        _refuse("linear (sizes beyond 32 bits)")
    _on("linear", dev, w, bias, residual, out)
    if bias is not None and (bias.dtype is not _F32 or not bias.is_contiguous() or bias.shape != (N,)):
        _refuse("linear (bias)")
    xs, rbf, rs, ys = _rows2(x, K, "linear"), 0, 0, N
    if residual is not None:
        if residual.shape != (T, N):
            _refuse("linear (residual)")
        rbf, rs = _is_bf16(residual, "linear"), _rows2(residual, N, "linear")
    if out is not None:
        if out.shape != (T, N) or (out_dtype is not None and out.dtype is not out_dtype):
            _refuse("linear (out)")
        ys = _rows2(out, N, "linear")
    elif out_dtype is None:
        out_dtype = _BF16
    elif out_dtype is not _BF16 and out_dtype is not _F32:
        _refuse("linear (out_dtype)")
    if rows_used is not None:
        _ints("linear", dev, rows_used)
        _need(rows_used.numel() == 1, "linear (rows_used: one number)")
    with _call(dev, stream) as st:
        if out is None:
            out = torch.empty_strided((T, N), (N, 1), dtype=out_dtype, device=x.device)
        rc = lib.q36_linear(x.data_ptr(), xs, w.data_ptr(), ptr(bias), ACTS[act], ptr(residual), rbf, rs, out.data_ptr(), _is_bf16(out, "linear"), ys,
                            T, N, K, ptr(rows_used), st)
        if rc:
            check(rc, "linear")
    return out
