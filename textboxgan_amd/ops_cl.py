"""Channels-last layers ([N, ..., C], channels contiguous) in fp32, bf16 and fp16: group norm with an activation, and 8-bit activation
checkpoints with the backward passes that read them (include/tbg.h "CHANNELS-LAST LAYERS").

What a layer keeps of its input between forward and backward is most of a training step's memory.  Here it can be kept in 8 bits
(``Act8``: blocks of 32 channels, one power-of-two scale each, amax / 127 or better; 33 / 32 bytes a value) and the kernels of the backward
pass read that form directly:

* ``act8_pack`` / ``act8_unpack``       rows of channels to 8 bits and back
* ``group_norm_act``                    group norm + affine + activation; ``save="act8"`` keeps the centred input in 8 bits, ``sink=True``
                                        also returns the output's own checkpoint, written by the same launch, for the layer that follows
* ``dense_act8``                        dense (1x1) layer whose input is kept in 8 bits only
* ``act8_wgrad``                        its weight and bias gradients, straight from the checkpoint

Parameters and their gradients are fp32 in every mode, as in ``ops``.  First order, reverse mode: the backward passes are not themselves
differentiable, and dual tensors of forward-mode differentiation are refused (``dense_act8`` without reverse-mode gradients takes them).
Everything is enqueued on the current stream and can be captured into a graph; a backward pass is captured where no graph made on the default
stream from the same leaves is alive (these functions refuse the leaves of one that they have seen).
Inputs whose rows are not evenly spaced with contiguous channels are copied once (``contiguous()``); slices of wider tensors are not.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import native as N

ACTS = {"linear": 0, "lrelu": 1, "silu": 2}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 32
MAX_CHANNELS, MAX_POSITIONS, MAX_SAMPLES, MAX_DENSE = 1 << 24, 1 << 30, 1 << 30, 1 << 20


class Act8(NamedTuple):
    """8-bit checkpoint of a tensor of ``shape`` and ``dtype``, its rows (all axes but the last) laid end to end: q int8
    [rows, 32 * blocks] (padding zero) and the scale codes e uint8 [rows, blocks] = exponent + 127, 255 for a block that was not finite."""
    q: torch.Tensor
    e: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype

    @property
    def rows(self) -> int:
        return self.q.shape[0]

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.e.numel()


_raw_stream = torch._C._cuda_getCurrentRawStream


def _call(name: str, t: torch.Tensor, *args):
    """One C entry, on the device of ``t`` (the current one as a rule: then nothing is switched) and its current stream."""
    fn = getattr(N.lib(), name)
    idx, cur = t.device.index, torch.cuda.current_device()
    if idx == cur:
        rc = fn(*args, _raw_stream(idx))
    else:
        torch.cuda.set_device(idx)
        try:
            rc = fn(*args, _raw_stream(idx))
        finally:
            torch.cuda.set_device(cur)
    if rc:
        N.check(rc, name)


def _check(t, what: str, dtypes):
    if not isinstance(t, torch.Tensor):
        raise N.TbgError(f"{what}: a tensor is wanted, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise N.TbgError(f"{what}: unsupported dtype {t.dtype}")


def _no_tangents(what: str, *ts):
    """no operand is a dual tensor of forward-mode differentiation: the kernels would drop its tangent without a word"""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise N.TbgError(f"{what}: forward-mode derivatives are not implemented (an operand is a dual tensor)")


def _most(what: str, size: int, limit: int, name: str):
    """sizes within what the C entries take (their integers are narrower than a tensor's sizes)"""
    if size > limit:
        raise N.TbgError(f"{what}: {size} {name}, at most {limit} are taken")


def _placed(what: str, *ts):
    """every operand on one device that the kernels run on (checked last: what a call asks for is looked at first)"""
    for t in ts:
        if not t.is_cuda:
            raise N.TbgError(f"{what}: libtbg_hip kernels need device tensors (no CPU path in the product)")
        if t.device != ts[0].device:
            raise N.TbgError(f"{what}: operands on {ts[0].device} and {t.device}")


def _rows(x: torch.Tensor):
    """x [..., C] as rows of contiguous channels an even pitch apart: (tensor that owns the memory, rows, pitch)."""
    ch = x.shape[-1]
    if x.is_contiguous():
        return x, x.numel() // ch, ch
    if x.stride(-1) == 1 or ch == 1:
        pitch, span, even = None, 1, True
        for n, s in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if n == 1:
                continue
            if pitch is None:
                pitch = s
            elif s != pitch * span:
                even = False
                break
            span *= n
        if even and pitch is not None and pitch >= ch:
            return x, x.numel() // ch, pitch
    x = x.contiguous()
    return x, x.numel() // ch, ch


def _samples(x: torch.Tensor):
    """x [N, ..., C] as samples of evenly spaced rows: (tensor, sample pitch, row pitch, positions)."""
    n, ch = x.shape[0], x.shape[-1]
    pos = x.numel() // (n * ch)
    if x.is_contiguous():
        return x, pos * ch, ch, pos
    if n > 0 and x.stride(0) >= 0:
        t, _, pitch = _rows(x[0])
        if t.data_ptr() == x.data_ptr():
            return x, x.stride(0), pitch, pos
    x = x.contiguous()
    return x, pos * ch, ch, pos


def _alloc8(rows: int, ch: int, device):
    nb = (ch + BLOCK - 1) // BLOCK
    return torch.empty((rows, nb * BLOCK), device=device, dtype=torch.int8), torch.empty((rows, nb), device=device, dtype=torch.uint8)


def _check8(a: Act8):
    if not isinstance(a, Act8):
        raise N.TbgError(f"an Act8 checkpoint is wanted, got {type(a).__name__}")
    _check(a.q, "checkpoint values", (torch.int8,))
    _check(a.e, "checkpoint scales", (torch.uint8,))
    ch = a.shape[-1] if len(a.shape) else 0
    if ch < 1:
        raise N.TbgError(f"a checkpoint of [..., channels] is wanted, got one of {tuple(a.shape)}")
    _most("checkpoint", ch, MAX_CHANNELS, "channels")
    nb = (ch + BLOCK - 1) // BLOCK
    rows = 1
    for v in a.shape[:-1]:
        rows *= v
    if tuple(a.q.shape) != (rows, nb * BLOCK) or tuple(a.e.shape) != (rows, nb) or not a.q.is_contiguous() or not a.e.is_contiguous():
        raise N.TbgError(f"checkpoint of {tuple(a.shape)}: values {tuple(a.q.shape)}, scales {tuple(a.e.shape)} do not fit (or are not contiguous)")


# ----------------------------------------------------------------------------------------
# 8-bit checkpoints
# ----------------------------------------------------------------------------------------
def act8_pack(x: torch.Tensor) -> Act8:
    """x [..., C] -> its 8-bit checkpoint."""
    _check(x, "act8_pack", _DTYPES)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise N.TbgError(f"act8_pack: [..., channels] is wanted, got {tuple(x.shape)}")
    _most("act8_pack", x.shape[-1], MAX_CHANNELS, "channels")
    _placed("act8_pack", x)
    shape = tuple(x.shape)
    rows = x.numel() // shape[-1]
    q, e = _alloc8(rows, shape[-1], x.device)
    if rows:
        x, _, pitch = _rows(x.detach() if x.requires_grad else x)
        _call("tbg_act8_pack", x, x.data_ptr(), _DTYPES[x.dtype], rows, shape[-1], pitch, q.data_ptr(), e.data_ptr())
    return Act8(q, e, shape, x.dtype)


def act8_unpack(a: Act8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values a checkpoint stands for, in the checkpointed tensor's shape and (unless ``dtype`` says otherwise) type.  In fp16, values that
    lie beyond the type's range by no more than half a step come back as its end (what fp16 holds from 65280 on is kept as 65536)."""
    _check8(a)
    dtype = a.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise N.TbgError(f"act8_unpack: unsupported dtype {dtype}")
    _placed("act8_unpack", a.q, a.e)
    x = torch.empty(a.shape, device=a.q.device, dtype=dtype)
    if a.rows:
        _call("tbg_act8_unpack", x, a.q.data_ptr(), a.e.data_ptr(), a.rows, a.shape[-1], x.data_ptr(), _DTYPES[dtype], a.shape[-1])
    return x


def act8_wgrad(a: Act8, dy: torch.Tensor, coef: float = 1.0, want_db: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dw [cin, cout], db [cout] | None) of y = coef * x @ w + b, from the checkpoint of x [..., cin] and dy [..., cout]; fp32."""
    _check8(a)
    _check(dy, "act8_wgrad", _DTYPES)
    cin = a.shape[-1]
    if dy.dim() < 1 or dy.shape[-1] < 1 or tuple(dy.shape[:-1]) != tuple(a.shape[:-1]):
        raise N.TbgError(f"act8_wgrad: a gradient {tuple(dy.shape)} does not belong to a checkpoint of {tuple(a.shape)}")
    _most("act8_wgrad", max(cin, dy.shape[-1]), MAX_DENSE, "channels")
    _no_tangents("act8_wgrad", dy)
    _placed("act8_wgrad", a.q, a.e, dy)
    cout, dev = dy.shape[-1], dy.device
    if not a.rows:
        return torch.zeros((cin, cout), device=dev), torch.zeros(cout, device=dev) if want_db else None
    dw = torch.empty((cin, cout), device=dev, dtype=torch.float32)
    db = torch.empty(cout, device=dev, dtype=torch.float32) if want_db else None
    dy, rows, pitch = _rows(dy.detach() if dy.requires_grad else dy)
    dt = _DTYPES[dy.dtype]
    nbytes = N.lib().tbg_act8_wgrad_workspace_bytes(rows, cin, cout, dt)
    N.check(min(nbytes, 0), "tbg_act8_wgrad_workspace_bytes")
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    _call("tbg_act8_wgrad", dy, a.q.data_ptr(), a.e.data_ptr(), dy.data_ptr(), dt, rows, cin, cout, pitch, float(coef), dw.data_ptr(),
          None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return dw, db


# ----------------------------------------------------------------------------------------
# group norm + activation
# ----------------------------------------------------------------------------------------
_ptr = lambda t: None if t is None else t.data_ptr()
_PLANS = {}  # arguments of a group norm call that follow from sizes, pitches and options alone: (reference to the descriptor, workspace bytes)


def _gn_plan(backward: int, *fields):
    key = (backward, fields)
    plan = _PLANS.get(key)
    if plan is None:
        d = C.byref(N.GnDesc(*fields))
        nbytes = N.lib().tbg_group_norm_workspace_bytes(d, backward)
        N.check(min(nbytes, 0), "tbg_group_norm_workspace_bytes")
        if len(_PLANS) >= 1024:
            _PLANS.clear()
        plan = _PLANS[key] = (d, nbytes)
    return plan


def _gn_fwd(x, gamma, beta, cfg, want_stats, save8, sink):
    groups, act, eps = cfg
    shape, dev, dtype = x.shape, x.device, x.dtype
    n, ch = shape[0], shape[-1]
    x, xn, xs, pos = _samples(x)
    rows = n * pos
    d, nbytes = _gn_plan(0, xn, xs, xn, xs, n, pos, ch, groups, _DTYPES[dtype], act, gamma.dim() - 1, eps)
    y = torch.empty(shape, device=dev, dtype=dtype)
    stats = torch.empty((n, groups, 2), device=dev, dtype=torch.float64) if want_stats else None
    q, e = _alloc8(rows, ch, dev) if save8 else (None, None)
    yq, ye = _alloc8(rows, ch, dev) if sink else (None, None)
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    _call("tbg_group_norm_fwd", x, d, x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), _ptr(stats), _ptr(q), _ptr(e), _ptr(yq),
          _ptr(ye), _ptr(ws), nbytes)
    return y, stats, q, e, Act8(yq, ye, tuple(shape), dtype) if sink else None


def _gn_bwd(x, q, e, dy, gamma, beta, stats, cfg):
    groups, act, eps = cfg
    shape, dev, dtype = dy.shape, dy.device, dy.dtype
    n, ch = shape[0], shape[-1]
    dy, dn, ds, pos = _samples(dy)
    xn, xs = dn, ds
    if x is not None:
        x, xn, xs, _ = _samples(x)
    d, nbytes = _gn_plan(1, xn, xs, dn, ds, n, pos, ch, groups, _DTYPES[dtype], act, gamma.dim() - 1, eps)
    dx = torch.empty(shape, device=dev, dtype=dtype)
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    _call("tbg_group_norm_bwd", dy, d, _ptr(x), _ptr(q), _ptr(e), dy.data_ptr(), gamma.data_ptr(), beta.data_ptr(), stats.data_ptr(), dx.data_ptr(),
          dgamma.data_ptr(), dbeta.data_ptr(), _ptr(ws), nbytes)
    return dx, dgamma, dbeta


def _leaves(what: str, y: torch.Tensor) -> torch.Tensor:
    """y, an output just made.  The accumulation node of a leaf belongs to the stream of the graph that first used the leaf, for as long as that
    graph lives.  A captured backward pass that reaches one of the default stream would end the capture, and the process, from the autograd
    engine's thread: such a leaf is refused while its forward pass is captured."""
    fn = y.grad_fn
    if fn is not None:
        for node, _ in fn.next_functions:
            if type(node).__name__ == "AccumulateGrad":
                idx = node.variable.device.index
                if node.metadata.setdefault("tbg_stream", _raw_stream(idx)) == 0 and _raw_stream(idx) and torch.cuda.is_current_stream_capturing():
                    raise N.TbgError(f"{what}: a graph that was made on the default stream from the same leaf {tuple(node.variable.shape)} is alive; "
                                     "release its outputs before the backward pass is captured")
    return y


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, cfg, save8, sink, box):
        y, stats, q, e, y8 = _gn_fwd(x, gamma, beta, cfg, True, save8, sink)
        if save8:
            ctx.save_for_backward(gamma, beta, stats, q, e)
        else:
            ctx.save_for_backward(gamma, beta, stats, x)
        ctx.cfg = cfg
        if sink:
            box.append(y8)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_tangents("group_norm_act backward", dy)
        gamma, beta, stats, *kept = ctx.saved_tensors
        x, q, e = (None, *kept) if len(kept) == 2 else (kept[0], None, None)
        dx, dgamma, dbeta = _gn_bwd(x, q, e, dy, gamma, beta, stats, ctx.cfg)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dgamma if need[1] else None, dbeta if need[2] else None, None, None, None, None


def group_norm_act(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, groups: int, act: str = "linear", eps: float = 1e-5,
                   save: str = "input", sink: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, Act8]]:
    """y = act(gamma * (x - mean) * rstd + beta), statistics over the positions and the channels of each of ``groups`` groups.

    x [N, ..., C] fp32 / bf16 / fp16; gamma, beta fp32, [C] or [N, C] (a scale and shift per sample, as styles give); act "linear",
    "lrelu" (slope 0.2, gain sqrt2, as the other layers of this package) or "silu".
    save: what the backward pass keeps of x -- "input" (x itself) or "act8" (8 bits of x - mean).
    sink: return (y, Act8 of y); pass the checkpoint to the layer that consumes y (``dense_act8(y, ..., x8=...)``)."""
    _check(x, "group_norm_act", _DTYPES)
    if x.dim() < 2 or x.shape[-1] < 1:
        raise N.TbgError(f"group_norm_act: [N, ..., channels] is wanted, got {tuple(x.shape)}")
    n, ch = x.shape[0], x.shape[-1]
    _most("group_norm_act", n, MAX_SAMPLES, "samples")
    _most("group_norm_act", ch, MAX_CHANNELS, "channels")
    _most("group_norm_act", x.numel() // max(n * ch, 1), MAX_POSITIONS, "positions")
    if not isinstance(groups, int) or isinstance(groups, bool) or groups < 1 or ch % groups:
        raise N.TbgError(f"group_norm_act: {ch} channels do not divide into {groups} groups")
    if act not in ACTS:
        raise N.TbgError(f"group_norm_act: unknown activation {act!r} (one of {', '.join(ACTS)})")
    if save not in ("input", "act8"):
        raise N.TbgError(f"group_norm_act: save is \"input\" or \"act8\", got {save!r}")
    if not eps > 0:
        raise N.TbgError(f"group_norm_act: eps has to be positive, got {eps}")
    _check(gamma, "group_norm_act: gamma", (torch.float32,))
    _check(beta, "group_norm_act: beta", (torch.float32,))
    if tuple(gamma.shape) not in ((ch,), (n, ch)) or gamma.shape != beta.shape:
        raise N.TbgError(f"group_norm_act: gamma {tuple(gamma.shape)} and beta {tuple(beta.shape)} have to be ({ch},) or ({n}, {ch}) alike")
    _no_tangents("group_norm_act", x, gamma, beta)
    _placed("group_norm_act", x, gamma, beta)
    grad = torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad)
    if x.numel() == 0:
        y = x * gamma.sum() * beta.sum() if grad else torch.empty(x.shape, device=x.device, dtype=x.dtype)
        y = y.to(x.dtype)
        return (y, Act8(*_alloc8(0, ch, x.device), tuple(x.shape), x.dtype)) if sink else y
    gamma, beta, cfg = gamma.contiguous(), beta.contiguous(), (groups, ACTS[act], float(eps))
    if not grad:
        y, *_, y8 = _gn_fwd(x, gamma, beta, cfg, False, False, sink)
        return (y, y8) if sink else y
    box = []
    y = _leaves("group_norm_act", _GroupNormAct.apply(x, gamma, beta, cfg, save == "act8", sink, box))
    return (y, box[0]) if sink else y


# ----------------------------------------------------------------------------------------
# dense (1x1) layer on an 8-bit checkpoint
# ----------------------------------------------------------------------------------------
def _own_types(fn):
    """fn(tensor, ...) outside the caller's autocast: its products run in the types of its operands"""
    @functools.wraps(fn)
    def call(t, *args):
        kind = t.device.type
        if not torch.is_autocast_enabled(kind):
            return fn(t, *args)
        with torch.autocast(kind, enabled=False):
            return fn(t, *args)
    return call


@_own_types
def _dense_fwd(x, w, b, coef):
    y = x.reshape(-1, w.shape[0]) @ (w * coef).to(x.dtype)
    if b is not None:
        y = y + b.to(x.dtype)
    return y.reshape(*x.shape[:-1], w.shape[1])


@_own_types
def _dense_dx(dy, w, coef, shape, dtype):
    return (dy.reshape(-1, w.shape[1]) @ (w * coef).to(dtype).t()).reshape(shape)


def _column_sums(dy):
    """db [cout] = sum of dy's rows, in fp32.  (torch's sum over many rows clears its counters by a memset, which a captured graph does not replay
    reliably.)"""
    cout, dev = dy.shape[-1], dy.device
    db = torch.empty(cout, device=dev, dtype=torch.float32)
    if not dy.numel():
        return db.zero_()
    dy, rows, pitch = _rows(dy)
    dt = _DTYPES[dy.dtype]
    nbytes = N.lib().tbg_column_sums_workspace_bytes(rows, cout, dt)
    N.check(min(nbytes, 0), "tbg_column_sums_workspace_bytes")
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    _call("tbg_column_sums", dy, dy.data_ptr(), dt, rows, cout, pitch, db.data_ptr(), _ptr(ws), nbytes)
    return db


class _DenseAct8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, coef, q, e):
        y = _dense_fwd(x, w, b, coef)
        if q is None and ctx.needs_input_grad[1]:
            a = act8_pack(x)
            q, e = a.q, a.e
        ctx.save_for_backward(q, e, w)
        ctx.cfgv = (tuple(x.shape), x.dtype, coef)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_tangents("dense_act8 backward", dy)
        q, e, w = ctx.saved_tensors
        shape, dtype, coef = ctx.cfgv
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0]:
            dx = _dense_dx(dy, w, coef, shape, dtype)
        if need[1]:
            dw, db = act8_wgrad(Act8(q, e, shape, dtype), dy, coef, need[2])
        elif need[2]:
            db = _column_sums(dy)
        return dx, dw, db, None, None, None


def dense_act8(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None, coef: float = 1.0, x8: Optional[Act8] = None) -> torch.Tensor:
    """y = coef * x @ w + b over the channels of x [..., cin] (a dense layer, or a 1x1 convolution of channels-last maps), with x kept for
    the weight gradient in 8 bits only.  w [cin, cout], b [cout] fp32 (rounded to x's type for the products, which are plain library GEMMs);
    y in x's type.  x8: the checkpoint of x where its producer has written it (``group_norm_act(..., sink=True)``), else it is packed here."""
    _check(x, "dense_act8", _DTYPES)
    _check(w, "dense_act8: w", (torch.float32,))
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[0] or w.shape[0] < 1 or w.shape[1] < 1:
        raise N.TbgError(f"dense_act8: input {tuple(x.shape)} and weight {tuple(w.shape)} do not fit")
    if b is not None:
        _check(b, "dense_act8: b", (torch.float32,))
        if tuple(b.shape) != (w.shape[1],):
            raise N.TbgError(f"dense_act8: bias {tuple(b.shape)}, ({w.shape[1]},) is wanted")
    if x8 is not None:
        _check8(x8)
        if tuple(x8.shape) != tuple(x.shape) or x8.dtype != x.dtype:
            raise N.TbgError(f"dense_act8: a checkpoint of {tuple(x8.shape)} {x8.dtype} is not one of the input {tuple(x.shape)} {x.dtype}")
    _placed("dense_act8", x, w, *(() if b is None else (b,)), *(() if x8 is None else (x8.q, x8.e)))
    coef = float(coef)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, b)):
        return _leaves("dense_act8", _DenseAct8.apply(x, w, b, coef, None if x8 is None else x8.q, None if x8 is None else x8.e))
    return _dense_fwd(x, w, b, coef)
