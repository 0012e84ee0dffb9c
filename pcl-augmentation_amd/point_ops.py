"""What a training step on the points of resident scenes needs beside the scenes themselves (``scene_pool``): rotary positions
over the axes of a point or a pixel, and the softmax cross entropy of a linear head over the labels, with their gradients.
Tensors on the GPU in and out, on the current stream; no CPU fallback (include/real3daug_hip.h, r3d_rotary, r3d_linear_ce_*).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools

from . import _lib

_REDUCTIONS = {"none": _lib.CE_NONE, "sum": _lib.CE_SUM, "mean": _lib.CE_MEAN}


_HERE = contextlib.nullcontext()


@functools.lru_cache(maxsize=None)
def _types():
    import torch
    return ({torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16},
            {torch.int32: _lib.T_I32, torch.int64: _lib.T_I64, torch.float32: _lib.T_F32, torch.float64: _lib.T_F64})


def on_device_of(what, *tensors):
    """The device of these tensors made current (a null context where it is already); refuses tensors that are not on one GPU."""
    import torch
    index = tensors[0].get_device()
    if index < 0:
        _lib.require_gpu()
        raise _lib.R3DError(f"{what}: the tensors must be on a GPU, got {tensors[0].device}")
    for t in tensors[1:]:
        if t.get_device() != index:
            raise ValueError(f"{what}: tensors on {tensors[0].device} and {t.device}")
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


@functools.lru_cache(maxsize=None)
def _forward_ad():
    import torch
    return torch.autograd.forward_ad


def forward_mode():
    """Inside of a level of forward-mode differentiation (``torch.autograd.forward_ad``, ``torch.func.jvp``)?"""
    return _forward_ad()._current_level >= 0


def not_as_read(what):
    """What stands in memory is not what the tensor reads as (the kernels read memory)."""
    return ValueError(f"{what}: a tensor that is negated or conjugated when it is read (resolve_neg, resolve_conj)")


def _value_type(what, t):
    kind = _types()[0].get(t.dtype)
    if kind is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16, got {t.dtype}")
    return kind


@functools.lru_cache(maxsize=None)
def _once():
    """Decorator of a backward pass that has none of its own: under ``create_graph`` its results raise where they are differentiated
    (torch's own lets them pass as constants where the incoming gradient needs none)."""
    import torch

    class Once(torch.autograd.Function):
        @staticmethod
        def forward(ctx, gradient, _):
            return gradient.view_as(gradient)

        @staticmethod
        def backward(ctx, *_):
            raise RuntimeError("rotary_positions and linear_cross_entropy are differentiable once")

    def decorate(backward):
        def run(ctx, *gradients):
            if forward_mode() and any(g is not None and torch.autograd.forward_ad.unpack_dual(g).tangent is not None for g in gradients):
                raise RuntimeError("rotary_positions and linear_cross_entropy have no forward-mode derivative of their gradients")
            if not torch.is_grad_enabled():
                return backward(ctx, *gradients)
            with torch.no_grad():
                got = backward(ctx, *gradients)
            return tuple(None if g is None else Once.apply(g, torch.empty(0, requires_grad=True)) for g in got)
        return run

    return decorate


# ---- rotary positions -------------------------------------------------------------------------------------------------
def _turn(tensors, positions, sections, base, interleaved, backward):
    """One launch over up to two [tokens, heads, dim] tensors (None: none), on the current device; returns dense ones."""
    import torch
    values, whole = _types()
    first = tensors[0] if tensors[0] is not None else tensors[1]
    if first is None:
        return [None, None]
    tokens, _, dim = first.shape
    outs, x, y, token_stride, head_stride, heads = [], [0, 0], [0, 0], [0, 0], [0, 0], [0, 0]
    kept = []
    for w, t in enumerate(tensors):
        if t is None:
            outs.append(None)
            continue
        out = torch.empty_like(t, memory_format=torch.contiguous_format)
        outs.append(out)
        strides = t.stride()
        if strides[2] != 1 or (backward and t.is_neg()):      # (a gradient may come in so)
            t = t.resolve_neg().contiguous()
            kept.append(t)      # (until the launch)
            strides = t.stride()
        x[w], y[w], heads[w] = t.data_ptr(), out.data_ptr(), t.shape[1]
        token_stride[w], head_stride[w], _ = strides
    if heads == [0, 0] or tokens == 0:
        return outs
    d = _lib.Rotary(tuple(x), tuple(y), tuple(token_stride), tuple(head_stride), tokens, tuple(heads), dim, values[first.dtype], interleaved, backward,
                    len(sections), sections, whole[positions.dtype], positions.data_ptr(), *positions.stride(), base)
    _lib.check(_lib.load().r3d_rotary(C.byref(d), _lib.raw_stream(positions.get_device())), "r3d_rotary")
    return outs


@functools.lru_cache(maxsize=None)
def _rotary_function():
    import torch

    class RotaryPositions(torch.autograd.Function):
        @staticmethod
        def forward(ctx, query, key, positions, sections, base, interleaved):
            ctx.save_for_backward(positions)
            ctx.how = sections, base, interleaved
            return tuple(_turn((query, key), positions, sections, base, interleaved, False))

        @staticmethod
        @_once()
        def backward(ctx, grad_query, grad_key):
            # a rotation: the gradient is turned back
            positions, = ctx.saved_tensors
            need = ctx.needs_input_grad
            with on_device_of("rotary_positions", positions):
                got = _turn((grad_query if need[0] else None, grad_key if need[1] else None), positions, *ctx.how, True)
            return got[0], got[1], None, None, None, None

    return RotaryPositions


def rotary_positions(query, positions, sections, key=None, base=10000.0, style="half"):
    """Rotary positions with several axes: ``query`` [tokens, heads, dim] (and ``key`` with heads of its own) turned by the
    positions of their tokens.

    positions [tokens, axes]: whole numbers (scan, row, column of a pixel) or floats (x, y, z of a point, in the units the base
    is meant for; a slice of packed rows, ``xyzi[:, :3]``, is taken as it lies); sections: pairs of every axis.  Pair j of an
    axis with s pairs turns by ``position * base ** (-j / s)``; the pairs of the axes stand one after the other, R in all
    (at most 256, 2 R <= dim): pair i is the elements (i, i + R) of a head (``style="half"``) or (2i, 2i + 1)
    (``"interleaved"``), elements from 2 R on stay.  Angles are taken in double, products in 32 bits, one rounding.
    Returns (query, key), key None where none was given; differentiable in both, once and backwards (forward mode raises)."""
    import torch
    shape, like, where = query.shape, None if key is None else key.shape, positions.shape
    if len(shape) != 3 or (like is not None and len(like) != 3):
        raise ValueError("rotary_positions: query and key must be [tokens, heads, dim]")
    if style not in ("half", "interleaved"):
        raise ValueError("rotary_positions: style is 'half' or 'interleaved'")
    sections = tuple([int(s) for s in sections])
    axes, pairs = len(sections), sum(sections)
    if not 1 <= axes <= _lib.ROTARY_MAX_AXES or min(sections) < 0:
        raise ValueError(f"rotary_positions: 1 to {_lib.ROTARY_MAX_AXES} sections of zero or more pairs")
    tokens, heads, dim = shape
    if len(where) != 2 or where[0] != tokens or where[1] != axes:
        raise ValueError(f"rotary_positions: positions must be [{tokens}, {axes}], got {tuple(where)}")
    if positions.dtype not in _types()[1]:
        raise TypeError(f"rotary_positions: positions are int32, int64, float32 or float64, got {positions.dtype}")
    if positions.requires_grad:
        raise ValueError("rotary_positions: positions have no gradient here (detach them)")
    _value_type("rotary_positions", query)
    if query.is_neg() or positions.is_neg() or (like is not None and key.is_neg()):
        raise not_as_read("rotary_positions")
    if like is not None and (key.dtype is not query.dtype or like[0] != tokens or like[2] != dim):
        raise ValueError("rotary_positions: key must have query's tokens, dim and type")
    if pairs > _lib.ROTARY_MAX_PAIRS or 2 * pairs > dim:
        raise ValueError(f"rotary_positions: {pairs} pairs do not fit a head of {dim} (at most {_lib.ROTARY_MAX_PAIRS} pairs)")
    if dim % 2 or dim > 4096:
        raise ValueError("rotary_positions: the size of a head must be even and at most 4096")
    if heads > 65536 or (like is not None and like[1] > 65536):
        raise ValueError("rotary_positions: at most 65536 heads")
    base = float(base)
    if not base > 0.0 or base == float("inf"):
        raise ValueError("rotary_positions: base must be positive and finite")
    with on_device_of("rotary_positions", query, positions, *(() if key is None else (key,))):
        # (a tangent of forward-mode differentiation shows in no flag of its tensor: inside of a level torch looks, and raises)
        if forward_mode() or (torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))):
            return _rotary_function().apply(query, key, positions, sections, base, style == "interleaved")
        return tuple(_turn((query, key), positions, sections, base, style == "interleaved", False))


# ---- softmax cross entropy of a linear head ------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _loss_function():
    import torch

    # Every line here is on the way of each step, forward on the caller's thread and backward on the engine's: what a small call
    # costs beyond its kernels is these lines (and the engine itself, 70 us).
    empty, f32, u8 = torch.empty, torch.float32, torch.uint8
    values, targets = _types()

    def follow(d, x, weight, bias, target, state):
        """The descriptor's tensors (in the backward pass: as they come back from where they were kept)."""
        d.x, d.w, d.bias, d.target = x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), target.data_ptr()
        # (the stride of a single row means nothing)
        d.ld_x, d.ld_w = (t.stride(0) if t.shape[0] > 1 else t.shape[1] for t in (x, weight))
        d.state = state.data_ptr()

    def space(lib, d, which, device):
        size = lib.r3d_linear_ce_bytes(C.byref(d), which)
        if size == 0:
            _lib.check(_lib.E_ARG, "r3d_linear_ce_bytes")
        return empty(size, dtype=u8, device=device)

    class LinearCrossEntropy(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, target, how):      # (the tensors' device is the current one)
            lib, device = _lib.load(), x.device
            (n, width), (v, _) = x.shape, weight.shape
            loss = empty(n if how[1] == _lib.CE_NONE else (), dtype=f32, device=device)
            d = _lib.LinearCE(x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), target.data_ptr(),
                              x.stride(0) if n > 1 else width, weight.stride(0) if v > 1 else width, n, v, width, how[0], how[2],
                              values[x.dtype], targets[target.dtype], how[1], 0, 0, loss.data_ptr())
            state = space(lib, d, _lib.CE_BYTES_STATE, device)
            d.state = state.data_ptr()
            ws = space(lib, d, _lib.CE_BYTES_FORWARD, device)
            _lib.check(lib.r3d_linear_ce_forward(C.byref(d), ws.data_ptr(), ws.numel(), _lib.raw_stream(x.get_device())), "r3d_linear_ce_forward")
            ctx.save_for_backward(x, weight, bias, target, state)
            ctx.descriptor, ctx.strides = d, (x.stride(), weight.stride())
            return loss

        @staticmethod
        @_once()
        def backward(ctx, grad):
            x, weight, bias, target, state = ctx.saved_tensors
            with on_device_of("linear_cross_entropy", x):
                lib, device = _lib.load(), x.device
                d = _lib.LinearCE.from_buffer_copy(ctx.descriptor)      # (two backward passes may run at once)
                if (x.data_ptr(), weight.data_ptr(), target.data_ptr(), state.data_ptr(), x.stride(), weight.stride()) != (d.x, d.w, d.target, d.state, *ctx.strides) \
                        or (bias is not None and bias.data_ptr() != d.bias):
                    # what was multiplied in place still has to be fit for it, wherever and however it was kept in the meantime
                    x, weight = (t if t.stride() == ctx.strides[i] else t.contiguous() for i, t in enumerate((x, weight)))
                    x, weight = (t.clone() if t.data_ptr() % 16 and not at % 16 else t for t, at in ((x, d.x), (weight, d.w)))
                    bias, target = None if bias is None else bias.contiguous(), target.contiguous()
                    follow(d, x, weight, bias, target, state)
                if grad.dtype is not f32 or not grad.is_contiguous() or grad.is_neg():
                    grad = grad.to(f32).resolve_neg().contiguous()
                d.grad = grad.data_ptr()
                need_x, need_w, need_b, _, _ = ctx.needs_input_grad
                dx = dw = db = None
                if need_x:
                    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
                    d.dx = dx.data_ptr()
                if need_w:
                    dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
                    d.dw = dw.data_ptr()
                if need_b:
                    db = torch.empty_like(bias, memory_format=torch.contiguous_format)
                    d.db = db.data_ptr()
                ws = space(lib, d, _lib.CE_BYTES_BACKWARD, device)
                _lib.check(lib.r3d_linear_ce_backward(C.byref(d), ws.data_ptr(), ws.numel(), _lib.raw_stream(x.get_device())), "r3d_linear_ce_backward")
            return dx, dw, db, None, None

    return LinearCrossEntropy


def _rows_dense(t):
    """[n, d] with the last axis dense and rows that do not overlap."""
    return t if t.stride(1) == 1 and (t.shape[0] == 1 or t.shape[1] <= t.stride(0) < 2 ** 31) else t.contiguous()


def linear_cross_entropy(x, weight, target, bias=None, ignore_index=-100, reduction="mean", piece=0):
    """Softmax cross entropy of the logits ``x @ weight.T + bias`` without ever holding them: x [..., features] (float32,
    bfloat16 or float16), weight [classes, features] and bias [classes] of the same type, target [...] int32 / int64.

    Points whose target is ``ignore_index`` have loss and gradient 0, whatever their features are; a target that is no class makes
    the loss NaN.  reduction: "mean" over the points that count (0 where none does), "sum" or "none" ([...]); the loss is
    float32.  Differentiable once in x, weight and bias (forward mode raises).  The same inputs give the same bits.  Sums are in 32
    bits; in the 16-bit types the logits' gradients are rounded to the type before the two products with them (half a step of
    each, beside half a step of the result), with weights of single points (reduction "none") float16 holds them relative to the
    largest one; float32 multiplies three planes of 8 bits, all that reaches beyond 2^-24.  A bias past 2.3e38 counts as infinite:
    the lowest float32 or bfloat16 masks a class as -inf does.

    Memory beside inputs, outputs and gradients: the backward pass holds the logits' gradients of ``piece`` classes at a time, 2 bytes
    a point and class (float32: 6), at least 128 classes; 0: what 512 MB take, at least 256 classes (none with few classes or few
    features), and 32-bit sums of dx and dweight where they are made in parts.  From forward to backward it keeps 20 bytes a
    point and, for float32 and for rows that are no multiples of 64 features, a packed copy of x and weight (6 and 2 bytes a value)."""
    import torch
    shape, dtype, wide = x.shape, x.dtype, weight.shape
    if len(shape) < 1 or len(wide) != 2 or shape[-1] != wide[1] or wide[0] < 1 or wide[1] < 1:
        raise ValueError(f"linear_cross_entropy: x [..., features] and weight [classes, features], got {tuple(shape)} and {tuple(wide)}")
    _value_type("linear_cross_entropy", x)
    if x.is_neg() or weight.is_neg() or (bias is not None and bias.is_neg()):
        raise not_as_read("linear_cross_entropy")
    if weight.dtype != dtype or (bias is not None and bias.dtype != dtype):
        raise TypeError("linear_cross_entropy: x, weight and bias must have one type")
    if bias is not None and bias.shape != wide[:1]:
        raise ValueError(f"linear_cross_entropy: bias must be [{wide[0]}], got {tuple(bias.shape)}")
    if target.shape != shape[:-1]:
        raise ValueError(f"linear_cross_entropy: target must be {tuple(shape[:-1])}, got {tuple(target.shape)}")
    if target.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"linear_cross_entropy: target is int32 or int64, got {target.dtype}")
    if reduction not in _REDUCTIONS:
        raise ValueError("linear_cross_entropy: reduction is 'none', 'sum' or 'mean'")
    if int(piece) < 0:
        raise ValueError("linear_cross_entropy: piece must not be negative")
    points = target.numel()
    if points > 2 ** 31 - 1025 or wide[0] > 2 ** 31 - 1025 or wide[1] > 1 << 20:
        raise ValueError("linear_cross_entropy: too large (2^31 points, 2^31 classes, 2^20 features)")
    here = on_device_of("linear_cross_entropy", x, weight, target, *(() if bias is None else (bias,)))
    if points == 0:      # nothing to sum, whatever the head holds; the gradients are zeros
        none = (x.sum() + weight[:0].sum() + (0 if bias is None else bias[:0].sum())).float()
        return none if reduction != "none" else none.expand(target.shape) + torch.zeros(target.shape, device=x.device)
    with here:
        loss = _loss_function().apply(_rows_dense(x if len(shape) == 2 else x.reshape(-1, shape[-1])), _rows_dense(weight),
                                      None if bias is None else bias.contiguous(),
                                      (target if len(shape) == 2 else target.reshape(-1)).contiguous(), (int(ignore_index), _REDUCTIONS[reduction], int(piece)))
    return loss.reshape(target.shape) if reduction == "none" and len(shape) != 2 else loss
