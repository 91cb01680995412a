"""Operators of a dense transformer over packed batches: several sequences (bags, slides) of different lengths lie one
behind the other in token-major tensors, without padding.

  packed_attention : softmax attention of every token over its own sequence, optionally causal, grouped heads,
                     forward and backward; a ``PackedPlan`` holds the work tables of the batch's lengths
  rope_axes        : rotary positions with up to eight axes (for example level, row and column of a patch)
  layer_norm       : layer norm over the last dimension

All of them are differentiable once (in reverse mode; dual tensors of ``torch.autograd.forward_ad`` are refused), run on the
current CUDA stream of the inputs' device and raise ``SwvError`` for calls that the kernels do not serve.  The reference's dense ViT-5 has the same pieces for one slide at a time
(src/sparse_wsi_vit/models/vit_5/models_vit5.py:72-115, rope.py:72-97).
"""
from __future__ import annotations

import ctypes
import functools

import numpy as np
import torch
from torch.autograd import forward_ad

from ._lib import SwvError, check, lib
from .ops import _CHECK, _require_cuda, check_status, status_word

_POS_CODES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_DIM = 1 << 29                                       # of the dimensions that the library takes as 32-bit numbers
_I3 = ctypes.c_int64 * 3
_raw_stream = torch._C._cuda_getCurrentRawStream        # (torch.cuda.current_stream builds an object: 2 us a call)


def _call(fn, what, dev, *args):
    """One call of the library on the current stream of ``dev`` (its last argument), whichever device is current."""
    i = dev.index
    if torch._C._cuda_getDevice() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(i))
    if rc != 0:
        check(rc, what)
    if _CHECK:
        check_status(dev, what)


def _same_device(first, *ts):
    dev = first.device
    _require_cuda(first)
    for t in ts:
        if t is not None and t.device != dev:
            raise SwvError("all tensors of a call must be on one device")


def _no_tangent(*ts):
    """A dual tensor asks for a derivative without ``requires_grad``: the result would silently have none."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise SwvError("forward-mode differentiation is not supported: the operators have reverse-mode gradients only")


def _reach(shape, strides):
    """Elements from the first to behind the last one."""
    return 1 + sum((n - 1) * s for n, s in zip(shape, strides)) if all(shape) else 0


def _apart(a, b):
    """No byte of the two is shared: one ends before the other begins, or their rows (first dimension) are equally far apart and
    they lie in different columns, as the heads of one projection do."""
    a0, b0 = a.data_ptr(), b.data_ptr()
    if a0 + _reach(a.shape, a.stride()) * a.itemsize <= b0 or b0 + _reach(b.shape, b.stride()) * b.itemsize <= a0:
        return True
    row = a.stride(0) * a.itemsize
    if row == 0 or row != b.stride(0) * b.itemsize:
        return False
    between = (b0 - a0) % row
    return (_reach(a.shape[1:], a.stride()[1:]) * a.itemsize <= between and
            between + _reach(b.shape[1:], b.stride()[1:]) * b.itemsize <= row)


def _check_out(out, like, inputs, same=None):
    """An output buffer of the caller: no part of an autograd graph, no element twice, and no memory of the inputs (``same``: or
    exactly that one)."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise SwvError("out must have the result's shape, type and device")
    if out.requires_grad:
        raise SwvError("out must not require a gradient")
    if not out.is_contiguous():
        reach = 1                                         # elements that the dimensions inside span
        for n, s in sorted(zip(out.shape, out.stride()), key=lambda d: d[1]):
            if n > 1 and s < reach:
                raise SwvError("out must not hold an element twice")
            reach += (n - 1) * s
    for t in inputs:
        if not (t is same and out.data_ptr() == t.data_ptr() and out.stride() == t.stride()) and not _apart(out, t):
            raise SwvError("out must not share memory with the inputs")


# --------------------------------------------------------------------------- #
# layer norm
# --------------------------------------------------------------------------- #
def _ptr(t):
    return None if t is None else t.data_ptr()


def _code(t):
    return 0 if t is None else _DTYPES[t.dtype]


def _rows2d(t):
    """``t`` as rows of its last dimension: a view where the rows are evenly spaced, else a copy."""
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    return t.reshape(-1, t.shape[-1])


def _norm_fwd(x, weight, bias, eps, out_dtype, want_stats):
    E, dev = x.shape[-1], x.device
    x2 = _rows2d(x)
    N = x2.shape[0]
    y = x.new_empty(x.shape, dtype=out_dtype)
    stats = mean = rstd = None
    if want_stats:
        stats = x.new_empty(2 * N, dtype=torch.float32)      # mean, rstd
        mean = stats.data_ptr()
        rstd = mean + 4 * N
    _call(lib.swv_layer_norm_fwd, "swv_layer_norm_fwd", dev, x2.data_ptr(), x2.stride(0), _DTYPES[x.dtype], _ptr(weight),
          _code(weight), _ptr(bias), _code(bias), y.data_ptr(), E, _DTYPES[out_dtype], mean, rstd, N, E, eps)
    return y, stats


@functools.lru_cache(maxsize=1024)
def _norm_bwd_bytes(N, E):
    n = ctypes.c_size_t()
    check(lib.swv_layer_norm_bwd_bytes(N, E, ctypes.byref(n)), "swv_layer_norm_bwd_bytes")
    return n.value


class LayerNormFunction(torch.autograd.Function):
    """``layer_norm`` with its gradients; the sums over the rows are added up in a fixed order."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, stats = _norm_fwd(x, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_tangent(dy)
        x, weight, stats = ctx.saved_tensors
        E, dev = x.shape[-1], x.device
        x2, dy2 = _rows2d(x), _rows2d(dy)
        N = x2.shape[0]
        dx = x.new_empty(x.shape)
        _, want_w, want_b, _, _ = ctx.needs_input_grad
        dw = weight.new_empty(E) if want_w else None
        db = x.new_empty(E, dtype=ctx.bias_dtype) if want_b else None
        ws, nws = None, 0
        if want_w or want_b:
            nws = _norm_bwd_bytes(N, E)
            ws = x.new_empty(nws, dtype=torch.uint8)
        mean = stats.data_ptr()
        _call(lib.swv_layer_norm_bwd, "swv_layer_norm_bwd", dev, dy2.data_ptr(), dy2.stride(0), _DTYPES[dy.dtype],
              x2.data_ptr(), x2.stride(0), _DTYPES[x.dtype], _ptr(weight), _code(weight), mean, mean + 4 * N, dx.data_ptr(), E,
              _ptr(dw), _code(dw), _ptr(db), _code(db), N, E, _ptr(ws), nws)
        return dx, dw, db, None, None


def _norm_param(t, name, x):
    if t.dim() != 1 or t.shape[0] != x.shape[-1]:
        raise SwvError(f"{name} has shape {tuple(t.shape)}, expected {(x.shape[-1],)}")
    if t.dtype not in _DTYPES:
        raise SwvError(f"{name} is float32, bfloat16 or float16, not {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """Layer norm over the last dimension of ``x (..., E)``, as ``torch.nn.functional.layer_norm(x, (E,), weight, bias)``.

    ``x`` fp32, bf16 or fp16; ``weight`` and ``bias`` (E,) of any of the three types, or None.  The statistics and all
    sums are fp32.  ``out_dtype``: x's type (the default) or fp32, for an fp32 ``x`` any of the three.  Rows may be evenly
    spaced views; other layouts are copied."""
    _same_device(x, weight, bias)
    _no_tangent(x, weight, bias)
    dt = x.dtype
    out_dtype = out_dtype or dt
    if dt not in _DTYPES or out_dtype not in _DTYPES:
        raise SwvError(f"layer_norm takes float32, bfloat16 and float16, not {dt} -> {out_dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise SwvError("layer_norm needs a last dimension of one value or more")
    if x.shape[-1] > _MAX_DIM:
        raise SwvError(f"layer_norm takes rows of up to {_MAX_DIM} values, not {x.shape[-1]}")
    if out_dtype != dt and dt != torch.float32 and out_dtype != torch.float32:
        raise SwvError(f"layer_norm of {dt} gives {dt} or float32, not {out_dtype}")
    grad = x.requires_grad
    if weight is not None:
        weight = _norm_param(weight, "weight", x)
        grad = grad or weight.requires_grad
    if bias is not None:
        bias = _norm_param(bias, "bias", x)
        grad = grad or bias.requires_grad
    if grad and torch.is_grad_enabled():
        return LayerNormFunction.apply(x, weight, bias, float(eps), out_dtype)
    return _norm_fwd(x, weight, bias, float(eps), out_dtype, False)[0]


# --------------------------------------------------------------------------- #
# rotary positions with several axes
# --------------------------------------------------------------------------- #
class RopeAxes:
    """How the channel pairs of a head turn: which axis of the position each pair follows, and how fast.

    ``sections``: the number of pairs of each axis, in channel order; pairs beyond their sum are not rotated.
    ``ladder``: "axis" -- every axis has frequencies theta^(-i / n) of its own, i = 0 .. n - 1 over its n pairs (with
    two equal sections and scales 1 / coord_high this is ``rope2d``); "head" -- one ladder theta^(-p / R) over all R
    rotated pairs p, of which every axis has its section.
    ``pairing``: "adjacent" -- pair p is channels (2p, 2p + 1); "halves" -- channels (p, R + p).
    ``scales``: a factor for the positions of each axis (default 1)."""

    def __init__(self, head_dim, sections, theta=10000.0, scales=None, ladder="axis", pairing="adjacent"):
        sections = [int(n) for n in sections]
        scales = [1.0] * len(sections) if scales is None else [float(s) for s in scales]
        R = sum(sections)
        if not 1 <= len(sections) <= 8 or min(sections) < 0 or R < 1 or 2 * R > head_dim or R > 128:
            raise SwvError(f"sections {sections}: one to eight axes and 1 to min(head_dim / 2, 128) pairs (head_dim {head_dim})")
        if len(scales) != len(sections):
            raise SwvError(f"{len(scales)} scales for {len(sections)} axes")
        if ladder not in ("axis", "head") or pairing not in ("adjacent", "halves"):
            raise SwvError(f"ladder is 'axis' or 'head', pairing 'adjacent' or 'halves'; got {ladder!r}, {pairing!r}")
        if not 0 < theta < float("inf") or not np.isfinite(scales).all():
            raise SwvError("theta must be positive, and it and the scales finite")
        self.head_dim, self.sections, self.pairs, self.halves = int(head_dim), tuple(sections), R, pairing == "halves"
        power = [(sum(sections[:a]) + i) / R if ladder == "head" else i / n for a, n in enumerate(sections) for i in range(n)]
        self._axis = np.repeat(np.arange(len(sections)), sections).astype(np.uint8)
        with np.errstate(over="ignore"):
            self._freq = np.asarray(scales)[self._axis] * np.float64(theta) ** -np.asarray(power, dtype=np.float64)
        if not np.isfinite(self._freq).all():
            raise SwvError(f"the frequencies pass the range of 64 bits: theta {theta}, scales {scales}")
        self._bind()

    def _bind(self):
        """The library's arguments: addresses of this object's own arrays."""
        self._call = (self._freq.ctypes.data, self._axis.ctypes.data, self.pairs, len(self.sections), int(self.halves))

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_call"}

    def __setstate__(self, state):                        # (a copied or unpickled object has arrays of its own)
        self.__dict__.update(state)
        self._bind()


def _rope_apply(x, positions, rope, inverse, out=None):
    T, H, hd = x.shape
    if x.stride(2) != 1:
        x = x.contiguous()
    y = x.new_empty((T, H, hd)) if out is None else out
    _call(lib.swv_rope_axes_apply, "swv_rope_axes_apply", x.device, x.data_ptr(), _I3(*x.stride()), y.data_ptr(),
          _I3(*y.stride()), _DTYPES[x.dtype], positions.data_ptr(), _POS_CODES[positions.dtype], positions.stride(0),
          *rope._call, inverse, T, H, hd)
    return y


class RopeAxesFunction(torch.autograd.Function):
    """``rope_axes`` with its gradient: the upstream gradient turned by the opposite angles."""

    @staticmethod
    def forward(ctx, x, positions, rope):
        ctx.save_for_backward(positions)
        ctx.rope = rope
        return _rope_apply(x, positions, rope, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        _no_tangent(g)
        return _rope_apply(g, ctx.saved_tensors[0], ctx.rope, True), None, None


def rope_axes(x, positions, rope, out=None):
    """Turns the heads ``x (T, H, head_dim)`` (fp32, bf16 or fp16) by ``positions (T, axes)`` (fp32, int32 or int64) as
    ``rope`` (a ``RopeAxes``) says.  The queries and keys of a fused projection turn in one call as its leading heads.
    ``out``: where to write (inference only), exactly ``x`` or elements that no input holds; those of a row may lie beside the inputs'
    in one buffer."""
    _same_device(x, positions)
    _no_tangent(x, positions, out)
    if x.dim() != 3 or x.shape[2] != rope.head_dim:
        raise SwvError(f"x has shape {tuple(x.shape)}, expected (tokens, heads, {rope.head_dim})")
    if not 1 <= x.shape[1] <= _MAX_DIM or x.shape[2] > _MAX_DIM:
        raise SwvError(f"rope_axes takes one to {_MAX_DIM} heads and channels, not {tuple(x.shape[1:])}")
    if x.dtype not in _DTYPES:
        raise SwvError(f"rope_axes takes float32, bfloat16 and float16, not {x.dtype}")
    if positions.dtype not in _POS_CODES:
        raise SwvError(f"positions are float32, int32 or int64, not {positions.dtype}")
    if tuple(positions.shape) != (x.shape[0], len(rope.sections)):
        raise SwvError(f"positions have shape {tuple(positions.shape)}, expected {(x.shape[0], len(rope.sections))}")
    if positions.requires_grad and torch.is_grad_enabled():
        raise SwvError("positions have no gradient: detach them")
    if positions.stride(1) != 1 and positions.shape[1] > 1:
        positions = positions.contiguous()
    grad = torch.is_grad_enabled() and x.requires_grad
    if out is not None:
        if grad:
            raise SwvError("rope_axes writes into `out` only where no gradient is asked for")
        _check_out(out, x, (x, positions), same=x)
        if out.stride(2) != 1:
            raise SwvError("out must have unit inner stride")
        torch.autograd.graph.increment_version(out)       # (a graph that has saved it notices)
    return RopeAxesFunction.apply(x, positions, rope) if grad else _rope_apply(x, positions, rope, False, out)


# --------------------------------------------------------------------------- #
# packed attention
# --------------------------------------------------------------------------- #
def _lengths(x):
    a = np.asarray(x).reshape(-1)
    if a.size and a.dtype.kind not in "iu":
        raise SwvError(f"lengths are whole numbers, not {a.dtype}")
    return np.ascontiguousarray(a, dtype=np.int64)


class PackedPlan:
    """The work tables of one packed batch, for any number of calls with its lengths (all layers of an encoder).

    ``q_lengths`` / ``k_lengths``: tokens of every sequence (k_lengths None: the same); ``heads`` query heads share
    ``kv_heads`` key / value heads evenly.  ``causal``: query i of a sequence sees the keys j <= i + lk - lq.
    Made on the host and copied to ``device`` once; a captured CUDA graph keeps using the plan it was captured with, so
    the plan must outlive it.  (Before a backward pass is captured, let go of eager graphs of the same leaves, as for any torch
    operator: their gradient nodes belong to another stream.)"""

    def __init__(self, q_lengths, k_lengths=None, *, heads, kv_heads=None, causal=False, device="cuda"):
        ql = _lengths(q_lengths)
        kl = ql if k_lengths is None else _lengths(k_lengths)
        if len(ql) != len(kl):
            raise SwvError(f"{len(ql)} query lengths and {len(kl)} key lengths")
        self.heads, self.kv_heads, self.causal = int(heads), int(heads if kv_heads is None else kv_heads), bool(causal)
        if self.heads > _MAX_DIM or self.kv_heads > 65535:
            raise SwvError(f"up to 65535 key / value heads of up to 128 query heads each, not {self.heads} and {self.kv_heads}")
        device = torch.device(device)
        self._not_captured(device)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device
        self.q_tokens, self.k_tokens = int(ql.sum()), int(kl.sum())
        size = ctypes.c_size_t()
        words = np.empty(1 << 14, dtype=np.int32)
        for _ in range(2):
            rc = lib.swv_packed_plan(len(ql), ql.ctypes.data, kl.ctypes.data, self.heads, self.kv_heads, int(self.causal),
                                     words.ctypes.data, words.nbytes, ctypes.byref(size))
            if rc != -5:                                  # (the tables need a larger array)
                break
            words = np.empty(size.value // 4, dtype=np.int32)
        check(rc, "swv_packed_plan")
        self._host = words[: size.value // 4].copy()
        self._upload()

    @staticmethod
    def _not_captured(device):
        if device.type == "cuda" and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise SwvError("make the plan before the capture: its tables are copied from the host")

    def _upload(self):
        self._table = torch.from_numpy(self._host).to(self.device)      # (waits for the copy: any stream may use it)
        self._call = (self._host.ctypes.data, self._table.data_ptr())
        self._stream = _raw_stream(self.device.index) if self.device.type == "cuda" else 0
        self._bytes = {}
        if self.device.type == "cuda":
            status_word(self.device)                      # (made in a capture, it would be the graph's: zeroed by every replay)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_table", "_call", "_stream", "_bytes")}

    def __setstate__(self, state):                        # (a copied or unpickled plan has tables of its own)
        self.__dict__.update(state)
        self._not_captured(self.device)
        self._upload()

    def _used(self):
        """The tables are read on the current stream: their memory is not given to others before that is through."""
        if _raw_stream(self.device.index) != self._stream and not torch.cuda.is_current_stream_capturing():
            self._table.record_stream(torch.cuda.current_stream(self.device))
        return self._call

    def _workspace_bytes(self, D, Tq=None):
        """Forward (Tq None) or backward workspace for head dimension D and buffers of Tq query rows."""
        if (D, Tq) not in self._bytes:
            n = ctypes.c_size_t()
            if Tq is None:
                check(lib.swv_packed_attn_bytes(self._call[0], D, ctypes.byref(n)), "swv_packed_attn_bytes")
            else:
                check(lib.swv_packed_attn_bwd_bytes(self._call[0], Tq, D, ctypes.byref(n)), "swv_packed_attn_bwd_bytes")
            self._bytes[D, Tq] = n.value
        return self._bytes[D, Tq]


def _rows_ok(t):
    a, b, c = t.stride()
    return c == 1 and a > 0 and b > 0 and not ((a | b) & 7 or t.data_ptr() & 15)


def _aligned(t):
    """A layout that the copy engines take: rows on 16 bytes."""
    return t if _rows_ok(t) else torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _attn_check(q, k, v, plan):
    _same_device(q, k, v)
    if not isinstance(plan, PackedPlan):
        raise SwvError("packed_attention needs a PackedPlan")
    if plan.device != q.device:
        raise SwvError(f"the plan is on {plan.device}, the tensors on {q.device}")
    bf16 = torch.bfloat16
    if q.dtype != bf16 or k.dtype != bf16 or v.dtype != bf16:
        raise SwvError("packed_attention needs bf16 q, k and v")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise SwvError("packed_attention takes q (Tq, heads, D) and k, v (Tk, kv_heads, D)")
    Tq, H, D = q.shape
    if H != plan.heads or k.shape[1] != plan.kv_heads:
        raise SwvError(f"{H} and {k.shape[1]} heads, the plan is for {plan.heads} and {plan.kv_heads}")
    if Tq < plan.q_tokens or k.shape[0] < plan.k_tokens:
        raise SwvError(f"{Tq} query and {k.shape[0]} key tokens, the plan's sequences have {plan.q_tokens} and "
                       f"{plan.k_tokens}")
    if D % 8 or not 8 <= D <= 128:
        raise SwvError(f"packed_attention supports head dimensions that are multiples of 8 up to 128, not {D}")


def _attn_fwd(q, k, v, plan, scale, want_lse, out=None):
    dev = q.device
    Tq, H, D = q.shape
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    o = out
    if o is None:
        o = q.new_empty((Tq, H, D))
        if plan.q_tokens < Tq:
            o[plan.q_tokens:].zero_()                     # rows behind the last sequence
    lse = None
    if want_lse:
        lse = q.new_empty((H, Tq), dtype=torch.float32)
        if plan.q_tokens < Tq:
            lse[:, plan.q_tokens:].fill_(-float("inf"))
    nws = plan._workspace_bytes(D)
    ws = q.new_empty(nws, dtype=torch.uint8) if nws else None
    _call(lib.swv_packed_attn_fwd, "swv_packed_attn_fwd", dev, q.data_ptr(), _I3(*q.stride()), k.data_ptr(),
          _I3(*k.stride()), v.data_ptr(), _I3(*v.stride()), o.data_ptr(), _I3(*o.stride()), _ptr(lse), *plan._used(), Tq,
          k.shape[0], D, scale, _ptr(ws), nws, status_word(dev).data_ptr())
    return o, lse


class PackedAttentionFunction(torch.autograd.Function):
    """``packed_attention`` with its gradients (no atomics: the same bits every time); the log-sum-exp of the rows is
    kept for the backward pass."""

    @staticmethod
    def forward(ctx, q, k, v, plan, scale):
        o, lse = _attn_fwd(q, k, v, plan, scale, True)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.plan, ctx.scale = plan, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)                  # (no (heads, Tq) zeros for lse in every backward pass)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, _):
        if d_out is None:
            return None, None, None, None, None
        _no_tangent(d_out)
        q, k, v, o, lse = ctx.saved_tensors
        plan, dev, D = ctx.plan, q.device, q.shape[2]
        q, k, v, d_out = _aligned(q), _aligned(k), _aligned(v), _aligned(d_out)
        Tq, Tk = q.shape[0], k.shape[0]
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        if plan.q_tokens < Tq:                            # rows behind the last sequence
            dq[plan.q_tokens:].zero_()
        if plan.k_tokens < Tk:
            dk[plan.k_tokens:].zero_()
            dv[plan.k_tokens:].zero_()
        nws = plan._workspace_bytes(D, Tq)
        ws = q.new_empty(nws, dtype=torch.uint8)
        dqs, dks = _I3(*dq.stride()), _I3(*dk.stride())
        _call(lib.swv_packed_attn_bwd, "swv_packed_attn_bwd", dev, d_out.data_ptr(), _I3(*d_out.stride()), q.data_ptr(),
              _I3(*q.stride()), k.data_ptr(), _I3(*k.stride()), v.data_ptr(), _I3(*v.stride()), o.data_ptr(), dqs,
              lse.data_ptr(), dq.data_ptr(), dqs, dk.data_ptr(), dks, dv.data_ptr(), dks, *plan._used(), Tq, Tk, D, ctx.scale,
              ws.data_ptr(), nws, status_word(dev).data_ptr())
        return dq, dk, dv, None, None


def packed_attention(q, k, v, plan, scale=None, return_lse=False, out=None):
    """Softmax attention inside each sequence of a packed batch.

    ``q (Tq, heads, D)``, ``k, v (Tk, kv_heads, D)`` bf16, D a multiple of 8 up to 128, any strides (views of a fused
    projection are read as they are if their rows lie on 16 bytes); ``plan``: the batch's ``PackedPlan``; ``scale``
    defaults to 1 / sqrt(D).  Returns ``(Tq, heads, D)`` bf16, with ``return_lse`` also the rows' log-sum-exp (heads, Tq)
    fp32, which has no gradient.  A row that sees no key is zero (lse -inf), and so are rows behind the last
    sequence; with ``out`` (inference only; elements that no input holds, for example other heads of one buffer) those are left as
    they were.  A NaN or an infinity never leaves its sequence;
    inside a causal one it can reach rows that do not see it (a masked pair is multiplied with zero): from a value row
    the results, from any input the gradients."""
    _attn_check(q, k, v, plan)
    _no_tangent(q, k, v, out)
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -60 <= scale <= 2.0 ** 60:
        raise SwvError("scale must be positive, between 2^-60 and 2^60")
    grad = (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled()
    if out is not None:
        if grad:
            raise SwvError("packed_attention writes into `out` only where no gradient is asked for")
        _check_out(out, q, (q, k, v))
        if not _rows_ok(out):
            raise SwvError("out must have rows on 16 bytes")
        torch.autograd.graph.increment_version(out)
    o, lse = PackedAttentionFunction.apply(q, k, v, plan, scale) if grad else _attn_fwd(q, k, v, plan, scale, return_lse, out)
    return (o, lse) if return_lse else o
