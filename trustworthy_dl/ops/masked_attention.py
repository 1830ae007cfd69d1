"""Attention under document, prefix and length masks, with capped scores and a distance bias.

``causal_attention`` is GPT-2's dense training attention on packed qkv.  The ops here take separate
query / key / value heads (shared KV heads included) and the masks that packed fine-tuning batches and
caches need, for whole sequences (forward and backward) and for single tokens against a cache:

    mask = attention_mask(B, Tq, Tk, documents=ids)          # once per batch, for every layer
    out  = masked_attention(q, k, v, mask, softcap=50.0, slopes=slopes)

``documents``, ``prefix``, ``lengths`` and ``causal`` leave each query one interval of visible keys; the
mask object holds those intervals and the tables that let the kernels skip whole tiles.  GPU tensors run
csrc/masked_attention_fwd.hip / _bwd.hip (bf16 and fp16, head dims up to 128); CPU tensors run the same
definition in PyTorch.  Results and gradients are the same bits in every run (no atomics).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ptr

_Q_TILE, _K_TILE = 32, 128     # csrc/masked_attention.h QT, KT
MIN_SOFTCAP, MAX_SOFTCAP = 1e-6, 1000.0
MIN_SCALE, MAX_SCALE = 1e-30, 1e30      # (with any softcap, the products of them that the kernels take stay in fp32's range)


# ============================================================== the mask
class AttentionMask:
    """Which keys each query of a batch sees: ``lo[b, i] <= j < hi[b, i]`` (``attention_mask``).

    Made from its inputs once; later changes of those tensors are not seen.  Like any tensor, a mask
    built on one stream is used on another only after that stream has waited for the first, and is told of it
    (``record_stream``) where it may be dropped before the other stream's work is done."""

    def __init__(self, batch: int, q_len: int, k_len: int, memory: torch.Tensor, nq: int, nk: int):
        self.batch, self.q_len, self.k_len = batch, q_len, k_len
        # One tensor of 32-bit words (a version for autograd to watch, an allocation per batch).  Tables first: they are
        # read 16 and 8 bytes at a time
        self.memory = memory
        self._tiles = nq, nk
        k_table = 4 * batch * nq
        lo = k_table + 2 * batch * nk
        self._at = lo, lo + batch * q_len, lo + 2 * batch * q_len, 0, k_table     # words: lo, hi, pos, q_table, k_table

    def _part(self, i: int, *shape: int) -> torch.Tensor:
        return self.memory[self._at[i]:self._at[i] + math.prod(shape)].view(shape)

    lo = property(lambda self: self._part(0, self.batch, self.q_len), doc="int32 [batch, q_len]")
    hi = property(lambda self: self._part(1, self.batch, self.q_len), doc="int32 [batch, q_len]")
    pos = property(lambda self: self._part(2, self.batch), doc="int32 [batch]: position of the first query")
    # what lets the kernels skip tiles (on the GPU; csrc/masked_attention.h qtab, ktab)
    q_table = property(lambda self: self._part(3, self.batch, self._tiles[0], 4), doc="int32 [batch, tiles of 32 queries, 4]")
    k_table = property(lambda self: self._part(4, self.batch, self._tiles[1], 2), doc="int32 [batch, blocks of 128 keys, 2]")

    @property
    def device(self) -> torch.device:
        return self.memory.device

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """``Tensor.record_stream`` for the mask's memory: it is not used again before ``stream``'s work so far is done."""
        self.memory.record_stream(stream)

    def dense(self) -> torch.Tensor:
        """[batch, q_len, k_len] booleans (for inspection and the CPU path)."""
        j = torch.arange(self.k_len, device=self.device)
        return (j >= self.lo[..., None]) & (j < self.hi[..., None])


def _int_input(name: str, t: Optional[torch.Tensor], shape, device, dtypes=(torch.int32, torch.int64)):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}, got "
                         f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the mask on {device}")
    return t.contiguous()


def attention_mask(batch: int, q_len: int, k_len: Optional[int] = None, *, causal: bool = True,
                   documents: Optional[torch.Tensor] = None, prefix: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, q_start: Optional[torch.Tensor] = None,
                   device=None) -> AttentionMask:
    """The mask of ``batch`` rows of ``q_len`` queries over ``k_len`` keys (default: as many).

    ``causal``     a query at position p sees the keys at positions <= p (else all of its row / document)
    ``documents``  int [batch, k_len]: document id of every position.  A document is a run of equal ids;
                   positions see their own document only.  A negative id marks padding: it sees nothing
                   and is seen by nothing.
    ``prefix``     positions that are seen both ways under ``causal``: int [batch] = the row's first
                   prefix[b] positions (without ``documents``), or bool [batch, k_len] marking the
                   positions with which each document (or row) begins.
    ``lengths``    int [batch]: valid positions of each row; keys behind them are never seen and queries
                   behind them see nothing.
    ``q_start``    int [batch]: position of each row's first query.  Default: the queries are the last
                   ``q_len`` valid positions of the row (a cache), or with q_len == k_len start at 0.
    ``device``     where the mask is used (default: that of the tensors above, or the CPU).
    """
    k_len = q_len if k_len is None else k_len
    if batch < 0 or q_len < 0 or k_len < q_len:
        raise ValueError(f"attention_mask needs 0 <= q_len <= k_len, got batch {batch}, q_len {q_len}, k_len {k_len}")
    if max(q_len, k_len) >= 1 << 30 or batch >= 1 << 22:
        raise ValueError("attention_mask: at most 2^30 - 1 positions and 2^22 - 1 rows")
    if device is None:
        device = next((t.device for t in (documents, prefix, lengths, q_start) if isinstance(t, torch.Tensor)), torch.device("cpu"))
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    documents = _int_input("documents", documents, (batch, k_len), device)
    lengths = _int_input("lengths", lengths, (batch,), device)
    q_start = _int_input("q_start", q_start, (batch,), device)
    rows = marks = None
    if prefix is not None:
        if not causal:
            raise ValueError("prefix needs causal=True (without it every position is seen both ways already)")
        if isinstance(prefix, torch.Tensor) and prefix.dim() == 2:
            marks = _int_input("prefix", prefix, (batch, k_len), device, (torch.bool, torch.uint8))
        else:
            rows = _int_input("prefix", prefix, (batch,), device)
            if documents is not None:
                raise ValueError("with documents the prefix is given per position: bool [batch, k_len]")
    small = [None if t is None else t.clamp(-(1 << 30), 1 << 30).to(torch.int32) if t.dtype == torch.int64 else t
             for t in (lengths, q_start, rows)]
    lengths, q_start, rows = small
    if device.type != "cuda":
        return _mask_reference(batch, q_len, k_len, causal, documents, rows, marks, lengths, q_start, device)

    nq, nk = -(-q_len // _Q_TILE), -(-k_len // _K_TILE)
    with torch.inference_mode(False):     # (a mask may be kept for training: autograd saves its tensor)
        memory = torch.empty(batch * (4 * nq + 2 * nk + 2 * q_len + 1), dtype=torch.int32, device=device)
    m = AttentionMask(batch, q_len, k_len, memory, nq, nk)
    if batch == 0 or q_len == 0:
        return m
    ws = torch.empty(batch * 3 * k_len, dtype=torch.int32, device=device) if documents is not None or marks is not None else None
    _lib.call_on(device, "tdl_attn_mask", ptr(documents), int(documents is not None and documents.dtype == torch.int64), ptr(rows),
                 ptr(marks), ptr(lengths), ptr(q_start), batch, q_len, k_len, int(causal), ptr(ws), *_pointers(memory, m._at))
    return m


def _pointers(memory: torch.Tensor, at) -> list:
    base = memory.data_ptr()
    return [base + 4 * x for x in at]


def _mask_reference(B, Tq, Tk, causal, documents, rows, marks, lengths, q_start, device) -> AttentionMask:
    j = torch.arange(Tk, device=device).expand(B, Tk)
    length = (lengths.clamp(0, Tk) if lengths is not None else torch.full((B,), Tk, device=device)).long()
    start, end = torch.zeros(B, Tk, dtype=torch.long, device=device), torch.full((B, Tk), Tk, device=device)
    if documents is not None and Tk:
        edge = torch.ones(B, Tk + 1, dtype=torch.bool, device=device)
        edge[:, 1:Tk] = documents[:, 1:] != documents[:, :-1]
        start = torch.cummax(torch.where(edge[:, :Tk], j, 0), 1)[0]
        end = torch.flip(torch.cummin(torch.flip(torch.where(edge[:, 1:], j + 1, Tk), [1]), 1)[0], [1])
    p0 = q_start.long() if q_start is not None else (length - Tq if Tq < Tk else torch.zeros_like(length))
    p = p0[:, None] + torch.arange(Tq, device=device)
    ok = (p >= 0) & (p < length[:, None])
    pc = p.clamp(0, max(Tk - 1, 0))
    if Tk and documents is not None:
        ok &= documents.gather(1, pc) >= 0
    if Tk == 0 or B == 0 or Tq == 0:
        none = torch.zeros(2 * B * Tq, dtype=torch.int32, device=device)
        return AttentionMask(B, Tq, Tk, torch.cat([none, p0.int()]), 0, 0)
    e = torch.minimum(end.gather(1, pc), length[:, None])
    lo, hi = start.gather(1, pc), e
    if causal:
        pe = torch.zeros_like(e)
        if marks is not None:
            free = torch.flip(torch.cummin(torch.flip(torch.where(marks == 0, j, Tk), [1]), 1)[0], [1])
            pe = free.gather(1, lo)
        elif rows is not None:
            pe = rows.long()[:, None].expand_as(e)
        hi = torch.maximum(p + 1, torch.minimum(pe, e))
    zero = torch.zeros_like(lo)
    lo, hi = torch.where(ok, lo, zero), torch.where(ok, hi, zero)
    return AttentionMask(B, Tq, Tk, torch.cat([lo.flatten(), hi.flatten(), p0]).int(), 0, 0)


# ============================================================== launches
class _Args(ctypes.Structure):
    """csrc/masked_attention.h mattn::Args (strides: batch, token, head of each tensor)"""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "dout", "o", "dq", "dk", "dv", "lse", "delta", "ws", "rest", "slopes",
                                                "lo", "hi", "pos", "qtab", "ktab")]
                + [(n + i, ctypes.c_int64) for n in ("qs", "ks", "vs", "os", "dos", "dqs", "dks", "dvs") for i in "012"]
                + [(n, ctypes.c_int) for n in ("B", "Tq", "Tk", "H", "Hk", "D", "dtype", "nsplit")]
                + [("scale", ctypes.c_float), ("cap", ctypes.c_float)])


_UNUSED = (0, 0, 0)


def _strides(t: torch.Tensor):
    # a dimension of one element is never stepped over
    (b, n, h, _), (sb, sn, sh, _) = t.shape, t.stride()
    return sb if b > 1 else 0, sn if n > 1 else 0, sh if h > 1 else 0


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, T, heads, D] with unit column stride and rows that start at 16 bytes (64 of which span less
    than 2 GiB): as it is, or a contiguous copy."""
    s = t.stride()
    if s[3] == 1 and t.data_ptr() % 16 == 0 and s[1] < 1 << 24:
        if not (s[0] | s[1] | s[2]) % 8 or all(s[i] % 8 == 0 for i in range(3) if t.shape[i] > 1):
            return t
    return _lib.dense(t)


def few_queries(batch: int, kv_heads: int, group: int, q_len: int, k_len: int) -> int:
    """0: the tiled kernel (32 queries of one head per wave).  Else the number of key ranges of the
    few-queries kernel, which reads K / V once for the rows (heads of a group x queries) of a tile of 32.

    Two workgroups a CU where the keys allow it, at least 4 ranges so that ragged caches even out, 512 keys
    or more in each (a range costs a workgroup's start and its part of the join).  48 x 8 tiles of up to 8191 keys:
    1 range 370 us, 2 317, 4 293, 8 294, 16 307; 16 tiles of 5003: 4 31 us, 8 23, 10 22, 20 27, 40 39; 12 tiles
    of 1000: 1 12 us, 4 10 and a second launch.
    Up to 32 queries it is the faster one (16 x 16 heads of 64, 4096 keys: 16 queries 63 against 96 us, 32 68
    against 83, 64 125 against 87; 4 x 2 groups of 8 heads of 128, 5003 keys: 32 queries 42 against 148 us)."""
    if q_len > 32:
        return 0
    tiles = batch * kv_heads * -(-(group * q_len) // 32)
    return max(1, min(max(-(-512 // tiles), 4), k_len // 512, 64))


MAX_GROUPS = (1 << 24) - 1     # workgroups of 256 threads in a launch (csrc/masked_attention.h MAX_GRID)


def largest_launch(B: int, Tq: int, Tk: int, H: int, Hk: int, D: int) -> int:
    """Workgroups of the largest launch of a forward or backward pass."""
    n = few_queries(B, Hk, H // Hk, Tq, Tk)
    fwd = max(B * Hk * n * -(-(H // Hk * Tq) // 32), -(-(B * H * Tq) // (16 if D <= 64 else 8))) if n else 0
    return max(fwd, B * H * -(-Tq // 128), B * Hk * -(-Tk // 128))


def _forward(q, k, v, mask, scale, cap, slopes, want_lse: bool, want_rest: bool):
    """(out, lse or None, out's rounding remainder for the backward pass or None, the call's arguments)"""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    dev = q.device
    out = torch.empty(B, Tq, H, D, dtype=q.dtype, device=dev)
    lse = torch.empty(B, H, Tq, dtype=torch.float32, device=dev) if want_lse else None
    rest = torch.empty(B, Tq, H, D, dtype=torch.uint8, device=dev) if want_rest else None
    if out.numel() == 0:
        return out, lse, rest, None
    nsplit = few_queries(B, Hk, H // Hk, Tq, Tk)
    ws = None
    if nsplit > 1:
        ws = torch.empty(B * H * Tq * nsplit * ((64 if D <= 64 else 128) + 2), dtype=torch.float32, device=dev)
    a = _Args(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, out.data_ptr(), 0, 0, 0, 0 if lse is None else lse.data_ptr(), 0,
              0 if ws is None else ws.data_ptr(), 0 if rest is None else rest.data_ptr(), 0 if slopes is None else slopes.data_ptr(),
              *_pointers(mask.memory, mask._at), *_strides(q), *_strides(k), *_strides(v), *_strides(out), *_UNUSED, *_UNUSED, *_UNUSED,
              *_UNUSED, B, Tq, Tk, H, Hk, D, _lib.DTYPE_CODE[q.dtype], nsplit, scale, cap)
    _lib.call_on(dev, "tdl_masked_attn_fwd", ctypes.addressof(a))
    return out, lse, rest, a


def _set(a: _Args, prefix: str, t: torch.Tensor):
    s = _strides(t)
    setattr(a, prefix + "0", s[0])
    setattr(a, prefix + "1", s[1])
    setattr(a, prefix + "2", s[2])


def _backward(ctx, q, k, v, out, lse, rest, slopes, mask, moved, dout, dq, dk, dv):
    """Writes dq and, unless both are None, dk and dv.  ``out``, ``lse``, ``rest``, ``slopes`` and the mask's memory: dense.
    The forward's arguments serve again; ``moved``: the operands' strides are others."""
    if q.numel() == 0:
        for g in (dk, dv):
            if g is not None:
                g.zero_()
        return
    B, Tq, H, D = q.shape
    # 512 words of scratch, then the rows' statistics, padded to whole tiles: lse log2(e) and -rowsum(dout out)
    ws = torch.empty(512 + B * H * 2 * (-(-Tq // _Q_TILE) * _Q_TILE), dtype=torch.float32, device=q.device)
    a = _Args.from_buffer_copy(ctx.args)
    a.q, a.k, a.v, a.o, a.dout = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr()
    a.lse, a.rest, a.slopes = lse.data_ptr(), rest.data_ptr(), 0 if slopes is None else slopes.data_ptr()
    a.lo, a.hi, a.pos, a.qtab, a.ktab = _pointers(mask, ctx.mask_at)
    a.ws, a.delta, a.dq = ws.data_ptr(), ws.data_ptr() + 2048, dq.data_ptr()
    _set(a, "dos", dout)
    _set(a, "dqs", dq)
    if dk is not None:
        a.dk, a.dv = dk.data_ptr(), dv.data_ptr()
        _set(a, "dks", dk)
        _set(a, "dvs", dv)
    if moved:
        for prefix, t in (("qs", q), ("ks", k), ("vs", v)):
            _set(a, prefix, t)
    _lib.call_on(q.device, "tdl_masked_attn_bwd", ctypes.addressof(a))


def _saved(name, ctx, dout, inputs):
    """The saved tensors as the kernels take them, whatever hooks made of them: operands (``inputs``: their shapes) with
    strides of their own, the rest dense; and whether an operand is another.  (The mask's memory is one of them: a
    change of it is noticed like one of an operand's.)"""
    B, T, H, D = shape = dout.shape
    n, moved = len(inputs), []

    def was(i):
        if i < n:
            return inputs[i], dout.dtype
        return ((shape, dout.dtype), ((B, H, T), torch.float32), (shape, torch.uint8), ((H,), torch.float32), (ctx.words, torch.int32))[i - n]

    def layout(i, t):
        if i >= n:
            return _lib.dense(t)
        moved.append(i)
        return _aligned(t)
    return (*_lib.came_back(name, ctx, dout.device, was, layout), bool(moved))


class _MaskedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, scale, cap, slopes, want_lse):
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        grad = any(ctx.needs_input_grad[:3])
        out, lse, rest, ctx.args = _forward(q, k, v, mask, scale, cap, slopes, want_lse or grad, grad)
        ctx.keys, ctx.mask_at, ctx.words = k.shape, mask._at, mask.memory.shape
        _lib.keep(ctx, q, k, v, out, lse, rest, slopes, mask.memory)
        ctx.set_materialize_grads(False)   # (no zeros for the statistics)
        if lse is not None:
            ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dlse):
        if dout is None:
            return (None,) * 8
        q, k, v, *rest = _saved("masked_attention", ctx, dout, (dout.shape, ctx.keys, ctx.keys))
        keys = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device) if keys else None
        dv = torch.empty(v.shape, dtype=v.dtype, device=v.device) if keys else None
        _backward(ctx, q, k, v, *rest, _aligned(dout), dq, dk, dv)
        return dq, dk, dv, None, None, None, None, None


class _MaskedAttentionPacked(torch.autograd.Function):
    """The gradients of q, k and v are written straight into one packed gradient."""

    @staticmethod
    def forward(ctx, qkv, n_head, n_kv_head, mask, scale, cap, slopes, grad):
        qkv = _aligned(qkv)
        q, k, v = qkv.split((n_head, n_kv_head, n_kv_head), dim=2)
        out, lse, rest, ctx.args = _forward(q, k, v, mask, scale, cap, slopes, grad, grad)
        ctx.heads, ctx.mask_at, ctx.words = (n_head, n_kv_head, n_kv_head), mask._at, mask.memory.shape
        _lib.keep(ctx, qkv, out, lse, rest, slopes, mask.memory)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        B, T, _, D = dout.shape
        qkv, *rest = _saved("masked_attention_packed", ctx, dout, ((B, T, sum(ctx.heads), D),))
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _backward(ctx, *qkv.split(ctx.heads, dim=2), *rest, _aligned(dout), *dqkv.split(ctx.heads, dim=2))
        return (dqkv,) + (None,) * 7


# ============================================================== CPU definition
def _reference(q, k, v, mask, scale, cap, slopes):
    """The definition with differentiable torch operations, in 32 bits (64 for double inputs)."""
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    B, Tq, H, D = q.shape
    G = H // k.shape[2]
    seen = mask.dense()
    # a key that no query of its row sees takes no part, nor does a query that sees nothing or its upstream gradient,
    # whatever stands there
    used = seen.any(1)[:, :, None, None] if Tq else torch.zeros(B, k.shape[1], 1, 1, dtype=torch.bool, device=k.device)
    sees, none = seen.any(-1)[:, :, None, None], torch.zeros((), dtype=wide, device=q.device)
    qf = torch.where(sees, q.to(wide), none).transpose(1, 2)
    kf, vf = (torch.where(used, t.to(wide), none).transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    s = (qf @ kf.transpose(-1, -2)) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        p = mask.pos.long()[:, None] + torch.arange(Tq, device=q.device)
        dist = (p[:, :, None] - torch.arange(mask.k_len, device=q.device)).abs()
        s = s - slopes.to(wide).view(1, H, 1, 1) * dist[:, None].to(wide)
    s = s.masked_fill(~seen[:, None], float("-inf"))
    top = s.detach().amax(-1, keepdim=True) if mask.k_len else s.new_zeros(B, H, Tq, 1)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(s - top)
    z = e.sum(-1, keepdim=True)
    out = (e / torch.where(z == 0, torch.ones_like(z), z)) @ vf
    lse = torch.where(z == 0, torch.full_like(z, float("-inf")), top + torch.log(z))[..., 0].detach().float()
    return torch.where(sees, out.transpose(1, 2), none).to(q.dtype), lse


# ============================================================== entry points
def _check(name: str, q, k, v, mask, scale, softcap, slopes):
    if not isinstance(mask, AttentionMask):
        raise ValueError(f"{name} needs a mask made by attention_mask, got {type(mask).__name__}")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{name}: q [B, Tq, H, D], k and v [B, Tk, Hk, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D or Hk == 0 or H == 0 or H % Hk:
        raise ValueError(f"{name}: {H} query heads of {tuple(q.shape)} do not share the KV heads of {tuple(k.shape)}")
    if (mask.batch, mask.q_len, mask.k_len) != (B, Tq, Tk):
        raise ValueError(f"{name}: the mask is for (batch, q_len, k_len) = {(mask.batch, mask.q_len, mask.k_len)}, the tensors have "
                         f"{(B, Tq, Tk)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"{name}: q, k and v differ in type ({q.dtype}, {k.dtype}, {v.dtype})")
    if not (q.device == k.device == v.device == mask.device):
        raise ValueError(f"{name}: q, k, v and the mask are on {q.device}, {k.device}, {v.device}, {mask.device}")
    if q.is_cuda:
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"native {name} supports bfloat16 and float16 (got {q.dtype})")
        if D % 8 or not 8 <= D <= 128:
            raise ValueError(f"native {name} supports head dims that are multiples of 8 up to 128 (got {D})")
        if (H + 2 * Hk) * D >= 1 << 24:    # (64 rows have to span less than 2 GiB, packed ones too)
            raise ValueError(f"native {name} supports tokens of less than 2^24 elements (got {H} + 2 x {Hk} heads of {D})")
        if B * H * (Tq + Tk) > MAX_GROUPS and largest_launch(B, Tq, Tk, H, Hk, D) > MAX_GROUPS:
            raise ValueError(f"native {name}: {B} x {Tq} queries of {H} heads over {Tk} keys are more than one launch takes; split the batch")
    elif not q.dtype.is_floating_point:
        raise ValueError(f"{name}: floating-point inputs, got {q.dtype}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not MIN_SCALE <= scale <= MAX_SCALE:
        raise ValueError(f"{name}: scale must lie in [{MIN_SCALE:g}, {MAX_SCALE:g}], got {scale}")
    cap = 0.0 if softcap is None else float(softcap)
    if softcap is not None and not MIN_SOFTCAP <= cap <= MAX_SOFTCAP:
        # cap tanh(x / cap) is evaluated to cap x 2^-21: beyond this the cap's own rounding would show (and
        # below it scale / cap would leave fp32's range)
        raise ValueError(f"{name}: softcap must lie in [{MIN_SOFTCAP:g}, {MAX_SOFTCAP:g}], got {softcap}")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor):
            raise ValueError(f"{name}: slopes must be a [{H}] tensor, got {type(slopes).__name__}")
        if slopes.shape != (H,) or slopes.device != q.device:
            raise ValueError(f"{name}: slopes must be a [{H}] tensor on {q.device}, got {tuple(slopes.shape)} on {slopes.device}")
        if slopes.requires_grad:
            raise ValueError(f"{name}: slopes are constants (no gradient is computed for them); pass slopes.detach()")
        slopes = slopes.to(torch.float32).contiguous()
    if q.is_cuda and forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v, slopes)):
        raise NotImplementedError(f"native {name} has no forward-mode derivative; use reverse mode")
    return scale, cap, slopes


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: AttentionMask, *, scale: Optional[float] = None,
                     softcap: Optional[float] = None, slopes: Optional[torch.Tensor] = None, return_lse: bool = False):
    """softmax(s) v over the keys each query sees, ``s = cap tanh(scale q.k / cap) - slopes[h] |p - j|``.

    q [B, Tq, H, D], k and v [B, Tk, Hk, D] with H a multiple of Hk (query head h reads KV head
    h // (H / Hk)); any batch / token / head strides.  ``scale`` defaults to 1 / sqrt(D); without
    ``softcap`` the scores are not capped, without ``slopes`` (fp32 [H], finite, of
    either sign) there is no distance bias (p, j: positions of query and key).  Returns [B, Tq, H, D] in q's type; a query that sees nothing
    gives zeros, and keys it does not see have no effect on it, whatever they hold (on the CPU: keys that no
    query of the row sees).  Scores are kept in 32 bits: at a size of S their weights are known to S 2^-21 (past
    2^21: not at all).  With
    ``return_lse`` also the fp32 log-sum-exp of each query's scores [B, H, Tq] (-inf where it sees
    nothing; not differentiable)."""
    scale, cap, slopes = _check("masked_attention", q, k, v, mask, scale, softcap, slopes)
    if q.is_cuda and torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _MaskedAttention.apply(q, k, v, mask, scale, cap, slopes, return_lse)
    elif q.is_cuda:   # (a single token's call is bound by the host: no autograd node)
        out, lse, _, _ = _forward(_aligned(q), _aligned(k), _aligned(v), mask, scale, cap, slopes, return_lse, False)
    else:
        out, lse = _reference(q, k, v, mask, scale, cap, slopes)
    return (out, lse) if return_lse else out


def masked_attention_packed(qkv: torch.Tensor, n_head: int, mask: AttentionMask, *, n_kv_head: Optional[int] = None,
                            scale: Optional[float] = None, softcap: Optional[float] = None,
                            slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``masked_attention`` on a projection's packed output [B, T, (H + 2 Hk) D] -> [B, T, H D]: query
    heads, then key heads, then value heads, as ``causal_attention`` takes them.  The gradient comes
    back packed too."""
    hk = n_head if n_kv_head is None else n_kv_head
    if qkv.dim() != 3 or n_head < 1 or hk < 1 or qkv.shape[2] % (n_head + 2 * hk):
        raise ValueError(f"masked_attention_packed: {tuple(qkv.shape)} does not hold {n_head} + 2 x {hk} heads")
    B, T, C = qkv.shape
    x = qkv.reshape(B, T, n_head + 2 * hk, C // (n_head + 2 * hk))
    q, k, v = x.split((n_head, hk, hk), dim=2)
    scale, cap, slopes = _check("masked_attention_packed", q, k, v, mask, scale, softcap, slopes)
    if qkv.is_cuda:
        # (under no_grad an input that requires a gradient still counts as one that needs it)
        out = _MaskedAttentionPacked.apply(x, n_head, hk, mask, scale, cap, slopes, x.requires_grad and torch.is_grad_enabled())
    else:
        out, _ = _reference(q, k, v, mask, scale, cap, slopes)
    return out.reshape(B, T, -1)
