"""Feature-map operators beside the correlation: group normalisation with an
activation, and dropout from a counter-based generator.

The maps the correlation reads come out of an encoder as convolution ->
normalisation -> activation -> dropout. The reference leaves that encoder to
torch; these operators are its memory-bound part for channels-last maps
``[B, ..., C]`` (the layout of ``nchw_to_nhwc``; a torch ``channels_last`` map
``t`` is passed as ``t.permute(0, 2, 3, 1)``, without a copy), float32, float16
or bfloat16, forward and backward.

:func:`group_norm` and :func:`dropout` are the calls a model makes. Eagerly
they run the kernels behind one autograd Function; under ``torch.compile`` they
are ``torch.ops.localcorr.group_norm`` / ``.dropout`` (torch_ops.py).
"""

from __future__ import annotations

import contextlib
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _require_cuda, _timed

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_MODES = ("element", "channel")


_HERE = contextlib.nullcontext()


def _on_device(index):
    """``torch.cuda.device`` that costs nothing when the device is current."""
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


def _stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


# ---------------------------------------------------------------------------
# argument checks
# ---------------------------------------------------------------------------

def _check_map(x, what, name="x"):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a tensor, but got {type(x).__name__}")
    _require_cuda(x, what=what)
    if x.dtype not in _DTYPES:
        raise RuntimeError(
            f"{what} requires float32, float16 or bfloat16 maps, but got {x.dtype}.")
    if x.dim() < 2 or x.shape[-1] < 1:
        raise ValueError(f"{what} requires a channels-last map [B, ..., C] with C >= 1, but got "
                         f"shape {tuple(x.shape)}")


def _check_dropout(p, rng, mode, x, what):
    """The probability as a float, after checking it with its stream and mode."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: the dropout probability must be in [0, 1], but got {p}")
    if mode not in _MODES:
        raise ValueError(f"{what}: unknown dropout mode {mode!r} (expected one of {_MODES})")
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != x.device:
            raise ValueError(f"{what}: an rng tensor holds (seed, offset), int64 of shape [2] on "
                             f"{x.device}, but got {rng.dtype} {tuple(rng.shape)} on {rng.device}")
    elif rng is not None:
        if len(rng) != 2 or not all(isinstance(v, int) and 0 <= v < 2 ** 63 for v in rng):
            raise ValueError(f"{what}: rng is (seed, offset), two integers in [0, 2**63), but got "
                             f"{rng!r}")
    elif p > 0:
        raise ValueError(f"{what}: dropout with p > 0 needs rng, the (seed, offset) of its draws")
    return p


def _split_rng(rng):
    """(tensor or None, seed, offset) of an rng argument."""
    if isinstance(rng, torch.Tensor):
        return rng, 0, 0
    return (None, 0, 0) if rng is None else (None, int(rng[0]), int(rng[1]))


def _check_norm(x, num_groups, weight, bias, eps, activation, negative_slope):
    what = "group_norm"
    c = x.shape[-1]
    if not isinstance(num_groups, int) or num_groups < 1 or c % num_groups:
        raise ValueError(f"{what}: num_groups must be a positive divisor of C = {c}, but got "
                         f"{num_groups}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (c,):
            raise ValueError(f"{what}: {name} must have shape [{c}], but got {tuple(t.shape)}")
        if t.device != x.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the map on {x.device}")
        if t.dtype not in (torch.float32, x.dtype):
            raise RuntimeError(f"{what}: {name} must be float32 or {x.dtype}, but got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"{what}: weight and bias must have one dtype, but got {weight.dtype} "
                           f"and {bias.dtype}")
    if activation not in _lib.ACT_CODES:
        raise ValueError(f"{what}: unknown activation {activation!r} (expected one of "
                         f"{tuple(_lib.ACT_CODES)})")
    if not 0.0 <= eps <= 1e30:
        raise ValueError(f"{what}: eps must be finite and not negative, but got {eps}")
    if not abs(negative_slope) <= 1e30:
        raise ValueError(f"{what}: negative_slope must be finite, but got {negative_slope}")


def _check_residual(x, residual):
    if residual is None:
        return
    _check_map(residual, "dropout", "residual")
    if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
        raise ValueError(
            f"dropout: the residual must be like x, {x.dtype} {tuple(x.shape)} on {x.device}, "
            f"but got {residual.dtype} {tuple(residual.shape)} on {residual.device}")


def _check_tangents(what, *tensors):
    """Refuses forward-mode differentiation: a launch would drop the tangents without a word."""
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative (jvp)")


def _check_used(used, p, grad, what):
    """The stream a forward left for its backward; one with p = 0 may leave none."""
    if used is None or used.numel() == 0:
        if p > 0:
            raise ValueError(f"{what}: dropout with p > 0 needs the stream that the forward used")
        return
    _check_dropout(p, used, "element", grad, what)
    if not used.is_contiguous():
        raise ValueError(f"{what}: the stream used must be contiguous")


def _check_norm_backward(grad_y, x, stats, num_groups):
    what = "group_norm backward"
    if grad_y.shape != x.shape or grad_y.device != x.device:
        raise ValueError(f"{what}: the output gradient must be like x, {tuple(x.shape)} on "
                         f"{x.device}, but got {tuple(grad_y.shape)} on {grad_y.device}")
    if (stats.shape != (x.shape[0], num_groups, 2) or stats.dtype != torch.float64
            or stats.device != x.device or not stats.is_contiguous()):
        raise ValueError(f"{what}: the statistics must be the forward's, float64 "
                         f"{(x.shape[0], num_groups, 2)} on {x.device}, but got {stats.dtype} "
                         f"{tuple(stats.shape)} on {stats.device}")


# ---------------------------------------------------------------------------
# raw launchers (no autograd)
# ---------------------------------------------------------------------------

def _rows(x):
    b, c = x.shape[0], x.shape[-1]
    return b, x.numel() // (b * c) if b else 0, c


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _by_product(x, shape, dtype):
    """What a launch writes beside its map; an empty map's call writes nothing."""
    make = torch.empty if x.numel() else torch.zeros
    return make(shape, dtype=dtype, device=x.device)


def dropout_forward(x, residual, p, channel, rng, seed, offset):
    """(residual + dropout(x), the stream used [2]) of contiguous-or-copied maps."""
    lib = _lib.require_library()
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    if rng is not None:
        rng = rng.contiguous()
    b, rows, c = _rows(x)
    y = torch.empty_like(x)
    used = _by_product(x, 2, torch.int64)
    dev = x.get_device()
    with _on_device(dev):
        ok = _timed("dropout", lambda: lib.launchLocalCorrB200Dropout(
            x.data_ptr(), _ptr(residual), y.data_ptr(), b, rows, c, _DTYPES[x.dtype], p, channel,
            seed, offset, _ptr(rng), used.data_ptr(), _stream(dev)),
            x.nbytes * (3 if residual is not None else 2))
    _lib.check(ok, "dropout", lib)
    return y, used


def dropout_backward(grad, used, p, channel):
    """The gradient of dropout's x for the stream ``used`` of the forward."""
    lib = _lib.require_library()
    grad = grad.contiguous()
    b, rows, c = _rows(grad)
    gx = torch.empty_like(grad)
    dev = grad.get_device()
    with _on_device(dev):
        ok = _timed("dropout", lambda: lib.launchLocalCorrB200Dropout(
            grad.data_ptr(), None, gx.data_ptr(), b, rows, c, _DTYPES[grad.dtype], p, channel, 0,
            0, used.data_ptr(), None, _stream(dev)), 2 * grad.nbytes)
    _lib.check(ok, "dropout backward", lib)
    return gx


@functools.lru_cache(maxsize=256)
def _norm_workspace_bytes(device, b, rows, c, groups, dtype, backward):
    with torch.cuda.device(device):
        return int(_lib.require_library().localCorrB200GroupNormWorkspaceBytes(
            b, rows, c, groups, _DTYPES[dtype], backward))


def _norm_workspace(x, b, rows, c, groups, backward):
    n = _norm_workspace_bytes(x.get_device(), b, rows, c, groups, x.dtype, backward)
    return torch.empty(n, dtype=torch.uint8, device=x.device)


def _params_f32(x, weight, bias):
    t = weight if weight is not None else bias
    return t is None or t.dtype == torch.float32


def group_norm_forward(x, weight, bias, num_groups, eps, activation, negative_slope, p, channel,
                       rng, seed, offset):
    """(y, statistics float64 [B, G, 2], the stream used: int64 [2], None with p = 0)."""
    lib = _lib.require_library()
    x = x.contiguous()
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    if rng is not None:
        rng = rng.contiguous()
    b, rows, c = _rows(x)
    y = torch.empty_like(x)
    stats = _by_product(x, (b, num_groups, 2), torch.float64)
    used = _by_product(x, 2, torch.int64) if p > 0 else None
    ws = _norm_workspace(x, b, rows, c, num_groups, False)
    dev = x.get_device()
    with _on_device(dev):
        ok = _timed("group_norm_fwd", lambda: lib.launchLocalCorrB200GroupNormForward(
            x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), stats.data_ptr(), b, rows, c,
            num_groups, _DTYPES[x.dtype], _params_f32(x, weight, bias), eps,
            _lib.ACT_CODES[activation], negative_slope, p, channel, seed, offset, _ptr(rng),
            _ptr(used), ws.data_ptr(), ws.numel(), _stream(dev)), 2 * x.nbytes)
    _lib.check(ok, "group norm", lib)
    return y, stats, used


def group_norm_backward(grad_y, x, weight, bias, stats, used, num_groups, activation,
                        negative_slope, p, channel, need_x=True, need_weight=True,
                        need_bias=True):
    """(grad_x, grad_weight, grad_bias), None where not needed (or without the parameter)."""
    lib = _lib.require_library()
    grad_y, x = grad_y.contiguous(), x.contiguous()
    if grad_y.dtype != x.dtype:
        grad_y = grad_y.to(x.dtype)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    b, rows, c = _rows(x)
    gx = torch.empty_like(x) if need_x else None
    gw = torch.empty_like(weight) if need_weight and weight is not None else None
    gb = torch.empty_like(bias) if need_bias and bias is not None else None
    ws = _norm_workspace(x, b, rows, c, num_groups, True)
    dev = x.get_device()
    with _on_device(dev):
        ok = _timed("group_norm_bwd", lambda: lib.launchLocalCorrB200GroupNormBackward(
            grad_y.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias), stats.data_ptr(),
            _ptr(gx), _ptr(gw), _ptr(gb), b, rows, c, num_groups, _DTYPES[x.dtype],
            _params_f32(x, weight, bias), _lib.ACT_CODES[activation], negative_slope, p, channel,
            0, 0, _ptr(used), ws.data_ptr(), ws.numel(), _stream(dev)), 3 * x.nbytes)
    _lib.check(ok, "group norm backward", lib)
    return gx, gw, gb


# ---------------------------------------------------------------------------
# autograd Functions
# ---------------------------------------------------------------------------

def _once_differentiable(backward):
    """torch's once_differentiable, whose bookkeeping (4 us of a small step's 140) is only
    taken where a graph of the backward is being built."""
    guarded = once_differentiable(backward)

    def run(ctx, grad_y):
        return guarded(ctx, grad_y) if torch.is_grad_enabled() else backward(ctx, grad_y)

    return run


class GroupNormFunction(torch.autograd.Function):
    """group_norm with its gradients; saves x and the float64 statistics. ``params``: the
    arguments of :func:`group_norm_forward` between bias and rng."""

    @staticmethod
    def forward(ctx, x, weight, bias, params, rng, seed, offset):
        x = x.contiguous()
        y, stats, used = group_norm_forward(x, weight, bias, *params, rng, seed, offset)
        ctx.save_for_backward(x, weight, bias, stats, used)
        ctx.params = params
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, grad_y):
        num_groups, _, activation, negative_slope, p, channel = ctx.params
        nx, nw, nb = ctx.needs_input_grad[:3]
        return (*group_norm_backward(grad_y, *ctx.saved_tensors, num_groups, activation,
                                     negative_slope, p, channel, nx, nw, nb),
                None, None, None, None)


class DropoutFunction(torch.autograd.Function):
    """residual + dropout(x); the backward draws the mask again."""

    @staticmethod
    def forward(ctx, x, residual, p, channel, rng, seed, offset):
        y, used = dropout_forward(x, residual, p, channel, rng, seed, offset)
        ctx.save_for_backward(used)
        ctx.params = (p, channel)
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, grad_y):
        gx = (dropout_backward(grad_y, *ctx.saved_tensors, *ctx.params)
              if ctx.needs_input_grad[0] else None)
        gr = grad_y if ctx.needs_input_grad[1] else None
        return gx, gr, None, None, None, None, None


# ---------------------------------------------------------------------------
# public operators
# ---------------------------------------------------------------------------

def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation="none",
               negative_slope=0.01, p=0.0, rng=None, dropout_mode="element"):
    """dropout(act(group_norm(x))) of a channels-last map, one call.

    ``x`` [B, ..., C] is normalised per sample over groups of C / num_groups
    consecutive channels and all positions (``num_groups = C``: instance norm),
    with the biased variance, then scaled by ``weight`` and shifted by ``bias``
    ([C], either may be None; float32 or x's dtype, both the same). ``activation`` is "none", "relu",
    "silu" or "leaky_relu" (with ``negative_slope``). With ``p`` > 0 the result
    is dropped out as :func:`dropout` does with ``rng`` and ``dropout_mode``.
    Statistics are float64, also of maps far from zero; the result is rounded to
    x's dtype once; results repeat bit for bit for equal sizes and alignment. A
    group of equal values gives ``bias`` (NaN with ``eps`` = 0). Inputs that
    are not contiguous are copied. Gradients for x, weight and bias (once
    differentiable).
    """
    _check_map(x, "group_norm")
    _check_norm(x, num_groups, weight, bias, eps, activation, negative_slope)
    p = _check_dropout(p, rng, dropout_mode, x, "group_norm")
    tensor, seed, offset = _split_rng(rng)
    params = (num_groups, float(eps), activation, float(negative_slope), p,
              dropout_mode == "channel")
    if torch.compiler.is_compiling():
        return torch.ops.localcorr.group_norm(x, weight, bias, *params, tensor, seed, offset)[0]
    _check_tangents("group_norm", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return GroupNormFunction.apply(x, weight, bias, params, tensor, seed, offset)
    return group_norm_forward(x, weight, bias, *params, tensor, seed, offset)[0]


def dropout(x, p, rng, residual=None, mode="element"):
    """Dropout of a channels-last map [B, ..., C], optionally added to ``residual``.

    An element drops (becomes 0, whatever it held) with probability ``p``
    rounded to a multiple of 2**-16, and what stays is scaled by 1 / (1 - that
    probability); ``mode="channel"`` drops whole channels of a sample. The draws
    are a function of ``rng``, the position and nothing else: ``rng`` is
    ``(seed, offset)``, a call number under a seed, as two integers or as an
    int64 tensor [2] on x's device, which a captured CUDA graph can advance
    between replays. Equal (seed, offset) give equal masks, so every dropout of
    a step takes an offset of its own. No mask is stored: the backward
    pass draws it again from a copy of the stream that the forward kept. Call it
    in training only (``p = 0`` copies x). Gradients as for :func:`group_norm`.
    """
    _check_map(x, "dropout")
    p = _check_dropout(p, rng, mode, x, "dropout")
    _check_residual(x, residual)
    tensor, seed, offset = _split_rng(rng)
    args = (x, residual, p, mode == "channel", tensor, seed, offset)
    if torch.compiler.is_compiling():
        return torch.ops.localcorr.dropout(*args)[0]
    _check_tangents("dropout", x, residual)
    if torch.is_grad_enabled() and (x.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return DropoutFunction.apply(*args)
    return dropout_forward(*args)[0]
