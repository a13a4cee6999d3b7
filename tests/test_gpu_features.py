"""group_norm and dropout on the GPU against the 64-bit oracle.

Tolerances. u = eps(dtype) / 2 is the final rounding. The statistics are float64 sums,
off by 2^-45 at most here. z = (x - mu) a + c takes a handful of float32 roundings, below
2^-21 |gamma| (|xhat| + 1) + 2^-22 |z| with the exp and quotient of 2 ulp each. The
backward's sums are float32 over at most 256 rows of a thread and float64 beyond, so
they carry 2^-16 of the sum of their terms' magnitudes. z's tolerance is taken as
2^-16 |gamma| (|xhat| + 1) + 2^-22 |z| throughout, which covers both; the activations
have slope at most 1.1. A rectifier's gradient may take either side where |z| is below
z's tolerance here; that it takes float64's is test_rectifiers_take_the_float64_side.
"""

import math

import numpy as np
import pytest
import torch
from torch.library import opcheck

import localcorr_b200 as lc
from localcorr_b200 import _lib, features
from oracle import feature_maps as oracle
from oracle import oracle as corr_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("none", "relu", "silu", "leaky_relu")
SLOPE = 0.1


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    assert _lib.load_library() is not None


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(shape, seed, dtype=torch.float32, shift=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype)


def _norm_case(shape, dtype, seed=0, shift=0.0, param_dtype=torch.float32):
    c = shape[-1]
    x = (_rand(shape, seed) * torch.exp(0.5 * _rand((c,), seed + 1)) + _rand((c,), seed + 2)
         + shift).to(dtype)
    w = (1 + 0.2 * _rand((c,), seed + 3)).to(param_dtype)
    b = (0.2 * _rand((c,), seed + 4)).to(param_dtype)
    return x, w, b, _rand(shape, seed + 5, dtype)


def _check_norm(x, w, b, dy, groups, act, p=0.0, stream=(7, 3), mode="element", eps=1e-5,
                spread=1.0):
    """Forward and gradients of the GPU call against the oracle; spread scales the
    statistics' tolerance where the inputs' offset exceeds their spread."""
    gx, gw, gb = (t.to(DEV).requires_grad_(True) if t is not None else None for t in (x, w, b))
    kw = dict(p=p, rng=stream, dropout_mode=mode) if p > 0 else {}
    y = lc.group_norm(gx, groups, gw, gb, eps=eps, activation=act, negative_slope=SLOPE, **kw)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    leaves = [t for t in (gx, gw, gb) if t is not None]
    grads = iter(torch.autograd.grad(y, leaves, dy.to(DEV)))

    u = _u(x.dtype)
    x64, dy64 = x.double(), dy.double()
    w64 = w.double() if w is not None else torch.ones(x.shape[-1], dtype=torch.float64)
    b64 = b.double() if b is not None else torch.zeros(x.shape[-1], dtype=torch.float64)
    f = oracle.drop_factors(x.shape, p, *stream, mode == "channel") if p > 0 else \
        torch.ones((), dtype=torch.float64)
    xhat, rstd = oracle.normalised(x64, groups, eps)
    z = xhat * w64 + b64
    e = 2.0 ** -16 * spread
    z_tol = e * w64.abs() * (xhat.abs() + 1) + 2.0 ** -22 * z.abs()
    ref = oracle.activated(z, act, SLOPE) * f
    tiny = torch.finfo(x.dtype).tiny
    tol = 1.1 * f * z_tol + u * ref.abs() + tiny
    got = y.detach().double().cpu()
    assert bool(((got - ref).abs() <= tol).all()), float(((got - ref).abs() - tol).max())
    if p > 0:
        assert bool((got[(f == 0).expand(x.shape)] == 0).all())

    zl = z.clone().requires_grad_(True)
    (da,) = torch.autograd.grad(oracle.activated(zl, act, SLOPE).sum(), zl)
    dz = dy64 * f * da
    corner = (z.abs() <= z_tol) & torch.tensor(act in ("relu", "leaky_relu"))
    # dz itself: either side of the corner, z's error through a second derivative <= 0.5
    dz_tol = (dy64 * f).abs() * (torch.where(corner, 1.0, 0.5 * z_tol + 2.0 ** -20))
    shape4 = (x.shape[0], -1, groups, x.shape[-1] // groups)

    def mean(t):
        return t.reshape(shape4).mean((1, 3), keepdim=True).expand(
            x.reshape(shape4).shape).reshape(x.shape)

    g = dz * w64
    g_tol = dz_tol * w64.abs()
    dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
    size = g.abs() + mean(g.abs()) + xhat.abs() * mean((g * xhat).abs()) + \
        mean(g.abs()) * xhat.abs() + mean(g.abs() * xhat.abs())
    dx_tol = rstd * (2 * e * size + g_tol + mean(g_tol) + xhat.abs() * mean(g_tol * xhat.abs()))
    got = next(grads).double().cpu()
    tol = dx_tol + u * dx.abs() + tiny
    assert bool(((got - dx).abs() <= tol).all()), float(((got - dx).abs() - tol).max())
    over = tuple(range(x.dim() - 1))
    for t, ref, part, part_tol in (
            (w, dz * xhat, (dz * xhat).abs() + dz.abs(), dz_tol * (xhat.abs() + e)),
            (b, dz, dz.abs(), dz_tol)):
        if t is None:
            continue
        got = next(grads)
        assert got.dtype == t.dtype
        ref = ref.sum(over)
        tol = (2 * e * part + part_tol).sum(over) + _u(t.dtype) * ref.abs() + tiny
        assert bool(((got.double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [
    ((1, 1, 1, 256), 32),      # one token
    ((2, 64), 4),              # no spatial axis
    ((3, 47, 61, 96), 8),      # odd sizes, slices of unequal length
    ((2, 5, 7, 24), 3),        # groups that no 16-byte vector fits evenly
    ((2, 9, 33), 11),          # odd C: element by element
    ((5, 3, 3, 12), 12),       # instance norm
    ((1, 17, 4104), 8),        # wider than a CTA, groups cut by its column blocks
    ((2, 2, 2100), 1),         # one group across column blocks
    ((2, 3000, 33), 11),       # divided, element by element
    ((1, 90, 4104), 8),        # divided, wider than a CTA
    ((3, 41, 53, 64), 8),      # divided, streamed
    ((2, 37, 2048), 16),       # streamed in 16 bits, too wide in 32
    ((3, 65, 1032), 3),        # rows no thread tiling fits evenly
    ((2, 150, 512), 512),      # the most groups that are streamed
    ((2, 150, 520), 520),      # one vector more
    ((3, 50, 1), 1),           # a single channel
    ((2, 90000, 1), 1),        # the same, divided
])
def test_norm_against_oracle(dtype, act, shape, groups):
    x, w, b, dy = _norm_case(shape, DTYPES[dtype])
    _check_norm(x, w, b, dy, groups, act)


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 32, 33, 127, 1000, 4099])
def test_norm_lengths(rows):
    x, w, b, dy = _norm_case((2, rows, 40), torch.float16, seed=rows)
    _check_norm(x, w, b, dy, 5, "silu")


@pytest.mark.parametrize("groups", [1, 2, 5, 10, 50, 100])
@pytest.mark.parametrize("batch", [1, 3, 700])
def test_norm_groups_and_batches(groups, batch):
    x, w, b, dy = _norm_case((batch, 13, 100), torch.bfloat16, seed=groups)
    _check_norm(x, w, b, dy, groups, "leaky_relu")


@pytest.mark.parametrize("mode", ["element", "channel"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape,groups", [((2, 19, 23, 64), 8), ((3, 7, 33), 3), ((2, 5, 12), 2),
                                          ((2, 5, 6), 1), ((3, 41, 53, 64), 8),
                                          ((2, 1500, 100), 20), ((2, 2500, 33), 3)])
def test_norm_with_dropout(mode, dtype, shape, groups):
    x, w, b, dy = _norm_case(shape, DTYPES[dtype], seed=4)
    _check_norm(x, w, b, dy, groups, "relu", p=0.3, stream=(2 ** 62 + 12345, 2 ** 40 + 9),
                mode=mode)


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_norm_without_parameters(which):
    x, w, b, dy = _norm_case((2, 11, 48), torch.float16)
    _check_norm(x, w if which == "weight" else None, b if which == "bias" else None, dy, 6, "silu")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_norm_parameters_of_the_maps_type(dtype):
    x, w, b, dy = _norm_case((2, 50, 64), DTYPES[dtype], param_dtype=DTYPES[dtype])
    _check_norm(x, w, b, dy, 8, "relu")


def test_norm_offset_far_above_spread():
    # mean 1000, spread ~1: the difference to the mean is taken before anything is scaled
    x, w, b, dy = _norm_case((2, 40, 40, 32), torch.float32, shift=1000.0)
    _check_norm(x, w, b, dy, 4, "silu")


def test_norm_constant_group_and_eps():
    x = torch.full((2, 30, 16), 3.25, dtype=torch.float16, device=DEV)
    b = torch.linspace(-1, 1, 16, device=DEV)
    y = lc.group_norm(x, 4, None, b)
    # the variance cancels to below 2^-40 of x^2, and x - mean is 0
    torch.testing.assert_close(y.float(), b.half().float().expand(2, 30, 16), rtol=0,
                               atol=2.0 ** -11)
    y = lc.group_norm(x[:, :1, :4].contiguous(), 4, None, b[:4])  # groups of one value
    torch.testing.assert_close(y.float(), b[:4].half().float().expand(2, 1, 4), rtol=0,
                               atol=2.0 ** -11)


@pytest.mark.parametrize("rows", [21, 2100])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_norm_keeps_what_is_not_finite_in_its_group(bad, rows):
    x, w, b, dy = _norm_case((2, rows, 24), torch.float32)
    clean = lc.group_norm(x.to(DEV), 3, w.to(DEV), b.to(DEV), activation="relu").cpu()
    x[1, 7, 9] = bad
    xg = x.to(DEV).requires_grad_(True)
    y = lc.group_norm(xg, 3, w.to(DEV), b.to(DEV), activation="relu")
    assert bool(y[1, :, 8:16].isnan().all())
    y = y.detach().cpu()
    y[1, :, 8:16] = clean[1, :, 8:16]
    assert torch.equal(y, clean)
    (g,) = torch.autograd.grad(lc.group_norm(xg, 3), xg, dy.to(DEV))
    assert bool(g[0].isfinite().all() and g[1, :, :8].isfinite().all()
                and g[1, :, 16:].isfinite().all())


@pytest.mark.parametrize("shape,groups", [((4, 9000, 64), 64), ((3, 20000, 128), 16),
                                          ((2, 5000, 35), 5), ((6, 60, 96), 12)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rectifiers_take_the_float64_side(dtype, shape, groups):
    # with an output gradient of ones the bias's gradient counts the elements above the
    # corner: whole numbers, to be met exactly. float64 itself decides where |z| > 2^-40.
    x, w, b, dy = _norm_case(shape, DTYPES[dtype], seed=31)
    xhat, _ = oracle.normalised(x.double(), groups, 1e-5)
    z = xhat * w.double() + b.double()
    assert float(z.abs().min()) > 2.0 ** -40
    gb = b.to(DEV).requires_grad_(True)
    y = lc.group_norm(x.to(DEV), groups, w.to(DEV), gb, activation="relu")
    (count,) = torch.autograd.grad(y, gb, torch.ones_like(y))
    assert torch.equal(count.double().cpu(), (z > 0).sum((0, 1)).double())


@pytest.mark.parametrize("rows", [100, 4000])
def test_norm_statistics_are_float64(rows):
    x, w, b, dy = _norm_case((3, rows, 64), torch.bfloat16, seed=32, shift=50.0)
    _, stats, _ = features.group_norm_forward(x.to(DEV), None, None, 64, 1e-5, "none", 0.0, 0.0,
                                              False, None, 0, 0)
    v = x.double()
    mean, var = v.mean(1), v.var(1, correction=0)
    # n 2^-53 of the sums; mean^2 / var is below 2^13, which the cancellation costs
    torch.testing.assert_close(stats[..., 0].cpu(), mean, rtol=2.0 ** -40, atol=0)
    torch.testing.assert_close(stats[..., 1].cpu(), 1 / torch.sqrt(var + 1e-5), rtol=2.0 ** -26,
                               atol=0)


@pytest.mark.parametrize("shape", [(1, 20, 64), (2, 2000, 64), (2, 3000, 33)])
def test_relu_gradient_of_what_is_not_finite(shape):
    # an infinite output gradient behind a closed rectifier does not reach the bias
    x, w, b, dy = (t.to(DEV) for t in _norm_case(shape, torch.float32, seed=41))
    gb = b.clone().requires_grad_(True)
    y = lc.group_norm(x, 1, w, gb, activation="relu")
    closed = y.detach() == 0
    assert bool(closed.any())
    (g,) = torch.autograd.grad(y, gb, torch.where(closed, float("inf"), dy))
    (want,) = torch.autograd.grad(lc.group_norm(x, 1, w, gb, activation="relu"), gb,
                                  torch.where(closed, 0.0, dy))
    assert torch.equal(g, want)


def test_norm_large_float16_values():
    # squares far beyond float16's range
    x, w, b, dy = _norm_case((1, 100, 16), torch.float32, seed=8)
    _check_norm((x * 8000).half(), w, b, dy.half(), 2, "none")


def test_norm_gradient_against_differences():
    x, w, b, dy = _norm_case((2, 6, 7, 16), torch.float32, seed=11)
    x, w, b, dy = (t.to(DEV) for t in (x, w, b, dy))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = lc.group_norm(leaves[0], 4, leaves[1], leaves[2], activation="silu")
    grads = torch.autograd.grad(y, leaves, dy)

    def loss(*args):
        out = lc.group_norm(args[0], 4, args[1], args[2], activation="silu")
        return float((out.double() * dy.double()).sum())

    # a y off by 2^-22 (|y| + 1) each makes a loss off by noise
    noise = float((dy.abs() * (y.detach().abs() + 1)).sum()) * 2.0 ** -22
    for i, t in enumerate((x, w, b)):
        v = _rand(tuple(t.shape), 100 + i).to(DEV)
        diff = []
        for h in (2.0 ** -6, 2.0 ** -5):
            moved = [[x, w, b], [x, w, b]]
            moved[0][i], moved[1][i] = t + h * v, t - h * v
            diff.append((loss(*moved[0]) - loss(*moved[1])) / (2 * h))
        want = float((grads[i].double() * v.double()).sum())
        # truncation is h^2: the two steps differ by three times the smaller one's
        tol = abs(diff[1] - diff[0]) + 2 * noise / 2.0 ** -6
        assert abs(diff[0] - want) <= tol, (i, diff, want, tol)


@pytest.mark.parametrize("size", [(10, 12), (50, 60)])
def test_norm_strides_alignment_and_expanded_gradients(size):
    x, w, b, dy = _norm_case((2, *size, 40), torch.float16)
    want = lc.group_norm(x.to(DEV), 5, w.to(DEV), b.to(DEV), activation="relu")
    nchw = x.to(DEV).permute(0, 3, 1, 2).contiguous()                  # NCHW: copied
    assert torch.equal(lc.group_norm(nchw.permute(0, 2, 3, 1), 5, w.to(DEV), b.to(DEV),
                                     activation="relu"), want)
    last = nchw.contiguous(memory_format=torch.channels_last)          # no copy
    assert last.permute(0, 2, 3, 1).is_contiguous()
    assert torch.equal(lc.group_norm(last.permute(0, 2, 3, 1), 5, w.to(DEV), b.to(DEV),
                                     activation="relu"), want)
    for shift in (1, 2, 4):                                            # 2, 4, 8 bytes off
        flat = torch.empty(x.numel() + shift, dtype=x.dtype, device=DEV)[shift:]
        flat.copy_(x.reshape(-1))
        got = lc.group_norm(flat.view(x.shape), 5, w.to(DEV), b.to(DEV), activation="relu")
        torch.testing.assert_close(got, want, rtol=2 * _u(x.dtype), atol=2.0 ** -14)
    xg = x.to(DEV).requires_grad_(True)
    y = lc.group_norm(xg, 5, w.to(DEV), b.to(DEV), activation="silu")
    g0, = torch.autograd.grad(y, xg, torch.ones_like(y), retain_graph=True)
    g1, = torch.autograd.grad(y.sum(), xg)                             # stride 0 gradient
    assert torch.equal(g0, g1)


@pytest.mark.parametrize("shape", [(2, 10, 40), (3, 2000, 40), (2, 3000, 35)])
def test_norm_one_needed_gradient(shape):
    x, w, b, dy = (t.to(DEV) for t in _norm_case(shape, torch.float16))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(lc.group_norm(full[0], 5, full[1], full[2], activation="silu"),
                               full, dy)
    for i in range(3):
        args = [x, w, b]
        args[i] = full[i]
        got, = torch.autograd.grad(lc.group_norm(args[0], 5, args[1], args[2], activation="silu"),
                                   full[i], dy)
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("c", [64, 72, 56, 60])
def test_norm_repeats_bit_for_bit(c):
    x, w, b, dy = (t.to(DEV) for t in _norm_case((4, 60, 70, c), torch.float16))
    out = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = lc.group_norm(leaves[0], 4, leaves[1], leaves[2], activation="relu", p=0.2,
                          rng=(1, 5))
        out.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    for other in out[1:]:
        assert all(torch.equal(a, o) for a, o in zip(out[0], other))


def test_empty_maps():
    for shape in ((0, 5, 8), (3, 0, 8), (2, 4, 0, 8)):
        x = torch.zeros(shape, dtype=torch.float16, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        b = torch.ones(8, device=DEV, requires_grad=True)
        y = lc.group_norm(x, 2, w, b, p=0.5, rng=(1, 1))
        grads = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert y.shape == shape and grads[0].shape == shape
        assert bool((grads[1] == 0).all() and (grads[2] == 0).all())
        assert lc.dropout(x, 0.5, (1, 2), residual=x).shape == shape
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------

def _check_dropout(x, p, stream, mode, residual=None, rng=None):
    f = oracle.drop_factors(x.shape, p, *stream, mode == "channel").expand(x.shape)
    xg = x.to(DEV).requires_grad_(True)
    rg = residual.to(DEV).requires_grad_(True) if residual is not None else None
    y = lc.dropout(xg, p, rng if rng is not None else stream, residual=rg, mode=mode)
    dy = _rand(tuple(x.shape), 77, x.dtype)
    grads = torch.autograd.grad(y, (xg, rg) if rg is not None else (xg,), dy.to(DEV))
    u = _u(x.dtype)
    tiny = torch.finfo(x.dtype).tiny
    # the factor, a product and a sum in float32, then the rounding
    r64 = residual.double() if residual is not None else torch.zeros((), dtype=torch.float64)
    part = x.double() * f
    ref = part + r64
    tol = u * ref.abs() + 3 * 2.0 ** -24 * (part.abs() + r64.abs()) + tiny
    got = y.detach().double().cpu()
    assert bool(((got - ref).abs() <= tol).all())
    if residual is None:
        assert torch.equal(got == 0, (f == 0) | (got == 0)) and bool((got[f == 0] == 0).all())
    else:
        assert bool((got[f == 0] == r64[f == 0]).all())
        assert torch.equal(grads[1].cpu(), dy)
    ref = dy.double() * f
    got = grads[0].double().cpu()
    assert bool(((got - ref).abs() <= (u + 2 * 2.0 ** -24) * ref.abs() + tiny).all())
    assert bool((got[f == 0] == 0).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("mode", ["element", "channel"])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("shape", [(1, 256), (1, 1), (2, 3, 5), (3, 47, 61, 24), (2, 5, 7, 33),
                                   (4, 9, 100), (1, 3, 2056), (2, 11, 1030)])
def test_dropout_against_oracle(dtype, mode, with_residual, shape):
    # ones: an element that should stay and does not shows
    x = _rand(shape, 1, DTYPES[dtype]) + 4
    r = _rand(shape, 2, DTYPES[dtype]) if with_residual else None
    _check_dropout(x, 0.3, (2 ** 63 - 1, 2 ** 33 + 1), mode, r)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1.0])
@pytest.mark.parametrize("mode", ["element", "channel"])
def test_dropout_probabilities(p, mode):
    _check_dropout(_rand((2, 100, 72), 3, torch.float16) + 4, p, (11, 12), mode)


def test_dropout_share():
    # 2^22 draws: the share is within five standard deviations of p
    p, n = 0.1, 1 << 22
    y = lc.dropout(torch.ones(1, n // 64, 64, device=DEV, dtype=torch.bfloat16), p, (123, 456))
    share = float((y == 0).double().mean())
    assert abs(share - round(p * 65536) / 65536) < 5 * math.sqrt(p * (1 - p) / n)


def test_dropout_of_what_is_not_finite():
    x = torch.full((1, 64, 8), float("nan"), device=DEV)
    y = lc.dropout(x, 0.5, (1, 2))
    f = oracle.drop_factors(x.shape, 0.5, 1, 2)
    assert torch.equal(y.cpu().isnan(), f > 0) and bool((y.cpu()[f == 0] == 0).all())


def test_dropout_of_an_unaligned_map():
    for dtype in DTYPES.values():
        for shift in (1, 3):
            x = _rand((2, 31, 24), 5, dtype) + 4
            flat = torch.empty(x.numel() + shift, dtype=dtype, device=DEV)[shift:]
            flat.copy_(x.reshape(-1))
            for mode in ("element", "channel"):
                assert torch.equal(lc.dropout(flat.view(x.shape), 0.4, (1, 2), mode=mode),
                                   lc.dropout(x.to(DEV), 0.4, (1, 2), mode=mode))


def test_dropout_beyond_32_bit_offsets():
    n = (1 << 31) + 4104
    x = torch.ones(1, n // 8, 8, dtype=torch.float16, device=DEV)
    y = lc.dropout(x, 0.5, (3, 4)).view(-1)
    for start in (0, (1 << 31) - 64, n - 4096):
        kept = oracle.draws(3, 4, start, 64) >= 32768
        assert np.array_equal((y[start:start + 64] != 0).cpu().numpy(), kept)


def test_norm_beyond_32_bit_offsets():
    # 2^31 elements and more: the last sample equals the same sample alone
    b, rows, c = 5, (1 << 21) + 3, 208
    x = torch.empty(b, rows, c, dtype=torch.float16, device=DEV)
    for i in range(b):
        x[i].normal_()
    assert x.numel() > 1 << 31
    y = lc.group_norm(x, 13, activation="silu")[b - 1]
    alone = lc.group_norm(x[b - 1:].contiguous(), 13, activation="silu")[0]
    # other runs: the same statistics but for 2^-45, then the rounding of either
    torch.testing.assert_close(y, alone, rtol=2.0 ** -10, atol=2.0 ** -13)


# ---------------------------------------------------------------------------
# streams of draws, CUDA streams, graphs
# ---------------------------------------------------------------------------

def test_rng_tensor_equals_integers_and_may_advance_before_the_backward():
    x = _rand((2, 30, 40), 6, torch.float16).to(DEV).requires_grad_(True)
    dy = _rand((2, 30, 40), 7, torch.float16).to(DEV)
    rng = torch.tensor([17, 5], device=DEV)
    for call in (lambda r: lc.dropout(x, 0.4, r),
                 lambda r: lc.group_norm(x, 4, activation="silu", p=0.4, rng=r)):
        want = call((17, 5))
        wg, = torch.autograd.grad(want, x, dy)
        rng[1] = 5
        y = call(rng)
        rng[1] += 1
        g, = torch.autograd.grad(y, x, dy)
        assert torch.equal(y, want) and torch.equal(g, wg)
        assert not torch.equal(call(rng), want)


def test_every_element_and_offset_draws_its_own():
    x = torch.ones(1, 1000, 64, device=DEV)
    masks = [lc.dropout(x, 0.5, (9, i)) != 0 for i in range(4)]
    for i in range(4):
        for j in range(i):
            agree = float((masks[i] == masks[j]).double().mean())
            assert abs(agree - 0.5) < 5 * 0.5 / math.sqrt(64000)


def test_large_maps_of_many_chunks():
    # several chunks a team, runs that end inside samples: the same sample alone agrees
    x = torch.empty(13, 61, 1031, 256, dtype=torch.bfloat16, device=DEV).normal_()  # 419 MB
    w, b = (torch.linspace(0.5, 1.5, 256, device=DEV).requires_grad_(True) for _ in range(2))
    dy = torch.empty_like(x).normal_()
    xg = x.requires_grad_(True)
    y = lc.group_norm(xg, 16, w, b, activation="silu")
    gx, gw, gb = torch.autograd.grad(y, (xg, w, b), dy)
    sw = sb = 0
    for i in range(13):
        one = x[i:i + 1].detach().requires_grad_(True)
        yi = lc.group_norm(one, 16, w, b, activation="silu")
        gi, gwi, gbi = torch.autograd.grad(yi, (one, w, b), dy[i:i + 1])
        # other runs: the backward's sums to 2^-16, then the rounding of either to 2^-8
        torch.testing.assert_close(y[i:i + 1], yi, rtol=2.0 ** -7, atol=2.0 ** -12)
        torch.testing.assert_close(gx[i:i + 1], gi, rtol=2.0 ** -7, atol=2.0 ** -12)
        sw, sb = sw + gwi.double(), sb + gbi.double()
    # sums of 817,583 terms of about 1 in float32 pieces of at most a few hundred
    torch.testing.assert_close(gw.double(), sw, rtol=2.0 ** -16, atol=0.5)
    torch.testing.assert_close(gb.double(), sb, rtol=2.0 ** -16, atol=0.5)


def _train_step(x, w, b, dy, rng):
    y = lc.group_norm(x, 8, w, b, activation="relu", p=0.25, rng=rng)
    y2 = lc.dropout(y, 0.5, rng, residual=y, mode="channel")
    return (y2, *torch.autograd.grad(y2, (x, w, b), dy))


@pytest.mark.parametrize("shape", [(3, 7, 9, 64), (3, 66, 42, 64), (2, 50, 60, 40)])
def test_captured_training_steps_replay_with_new_draws(shape):
    x, w, b, dy = (t.to(DEV) for t in _norm_case(shape, torch.float16))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    rng = torch.tensor([31, 0], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _train_step(x, w, b, dy, rng)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _train_step(x, w, b, dy, rng)
            rng[1] += 1
        graphs.append(g)
        outs.append(out)
    seen = []
    for i in range(4):
        rng[1] = i
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = _train_step(x, w, b, dy, (31, i))
        got = outs[i % 2]
        assert int(rng[1]) == i + 1
        assert all(torch.equal(a, o) for a, o in zip(want, got))
        seen.append(got[0].detach().clone())
    assert not torch.equal(seen[0], seen[1])
    with torch.no_grad():  # new inputs in the captured buffers
        x.add_(0.5)
    rng[1] = 2
    graphs[0].replay()
    torch.cuda.synchronize()
    want = _train_step(x, w, b, dy, (31, 2))
    assert all(torch.equal(a, o) for a, o in zip(want, outs[0]))


def test_side_streams_at_once():
    cases = [[t.to(DEV) for t in _norm_case((2, 50 + i, 40, 64), torch.float16, seed=i)]
             for i in range(4)]
    want = []
    for x, w, b, dy in cases:
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        want.append(_train_step(*leaves, dy, (1, 2)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for s, (x, w, b, dy) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(_train_step(x, w, b, dy, (1, 2)))
        torch.cuda.synchronize()
        for a, o in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, o))


# ---------------------------------------------------------------------------
# registered operators, refusals, the run of a step
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("p", [0.0, 0.5])
def test_opcheck(p):
    x, w, b, dy = (t.to(DEV) for t in _norm_case((2, 6, 24), torch.float32))
    rng = torch.tensor([1, 2], device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    opcheck(torch.ops.localcorr.group_norm.default,
            (*leaves, 3, 1e-5, "silu", 0.0, p, True, rng if p else None, 0, 0))
    opcheck(torch.ops.localcorr.group_norm.default,
            (x, None, None, 3, 1e-5, "none", 0.0, p, False, None, 4, 5))
    opcheck(torch.ops.localcorr.dropout.default, (x, dy.requires_grad_(True), p, False, rng, 0, 0))
    opcheck(torch.ops.localcorr.dropout.default, (x, None, p, True, None, 4, 5))
    _, stats, used = features.group_norm_forward(x.detach(), w.detach(), b.detach(), 3, 1e-5,
                                                 "silu", 0.0, p, True, rng, 0, 0)
    opcheck(torch.ops.localcorr.group_norm_backward.default,
            (dy.detach(), x.detach(), w.detach(), b.detach(), stats, used, 3, "silu", 0.0, p, True))
    opcheck(torch.ops.localcorr.dropout_backward.default, (dy.detach(), rng, p, True))


def test_compiled_step_equals_eager():
    x, w, b, dy = (t.to(DEV) for t in _norm_case((2, 12, 10, 32), torch.float16))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    rng = torch.tensor([3, 4], device=DEV)

    def step(x, w, b):
        y = lc.group_norm(x, 4, w, b, activation="leaky_relu", negative_slope=0.1, p=0.1, rng=rng)
        return lc.dropout(y, 0.2, rng, residual=y, mode="channel")

    want = step(x, w, b)
    got = torch.compile(step, fullgraph=True)(x, w, b)
    assert torch.equal(want, got)
    for a, o in zip(torch.autograd.grad(want, (x, w, b), dy),
                    torch.autograd.grad(got, (x, w, b), dy)):
        # the residual's and the dropout's gradients may be added in another order
        torch.testing.assert_close(a, o, rtol=2.0 ** -9, atol=2.0 ** -9)


def test_parameters_of_other_strides_and_shared_leaves():
    x, w, b, dy = (t.to(DEV) for t in _norm_case((2, 30, 40), torch.float16))
    one = torch.full((1,), 1.25, device=DEV, requires_grad=True)
    pair = torch.stack([w, b], dim=1).requires_grad_(True)      # columns: stride 2
    y = lc.group_norm(x, 5, one.expand(40), None, activation="silu")
    (g,) = torch.autograd.grad(y, one, dy)
    full = torch.full((40,), 1.25, device=DEV, requires_grad=True)
    (want,) = torch.autograd.grad(lc.group_norm(x, 5, full, None, activation="silu"), full, dy)
    torch.testing.assert_close(g, want.sum(0, keepdim=True))
    (gp,) = torch.autograd.grad(lc.group_norm(x, 5, pair[:, 0], pair[:, 1]), pair, dy)
    lw, lb = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    gw, gb = torch.autograd.grad(lc.group_norm(x, 5, lw, lb), (lw, lb), dy)
    assert torch.equal(gp, torch.stack([gw, gb], dim=1))


def test_same_graph_twice():
    x, w, b, dy = (t.to(DEV) for t in _norm_case((2, 300, 64), torch.float16))
    xg = x.requires_grad_(True)
    y = lc.dropout(lc.group_norm(xg, 8, w, b, activation="relu", p=0.2, rng=(1, 2)), 0.5, (1, 3))
    first, = torch.autograd.grad(y, xg, dy, retain_graph=True)
    again, = torch.autograd.grad(y, xg, dy)
    assert torch.equal(first, again)


def test_refusals():
    x = torch.zeros(2, 5, 8, device=DEV, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        lc.group_norm(x.double(), 2)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        lc.dropout(x.int(), 0.5, (1, 2))
    with pytest.raises(ValueError, match="channels-last"):
        lc.group_norm(x[0, 0], 2)
    with pytest.raises(RuntimeError, match="weight is on cpu"):
        lc.group_norm(x, 2, torch.ones(8))
    with pytest.raises(ValueError, match="on cuda"):
        lc.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="like x"):
        lc.dropout(x, 0.5, (1, 2), residual=x[:1])
    with pytest.raises(ValueError, match="like x"):
        lc.dropout(x, 0.5, (1, 2), residual=x.float())
    with pytest.raises(ValueError, match="needs rng"):
        lc.group_norm(x, 2, p=0.5)
    y = lc.group_norm(x.float().requires_grad_(True), 2)
    (g,) = torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable,
                               create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_registered_operators_refuse_what_the_functions_refuse():
    op = torch.ops.localcorr
    x = torch.zeros(2, 5, 8, device=DEV)
    used = torch.zeros(2, dtype=torch.int64, device=DEV)
    stats = torch.ones(2, 4, 2, dtype=torch.float64, device=DEV)

    def norm(x=x, w=None, groups=4, act="relu", p=0.0, rng=None, seed=1):
        return op.group_norm(x, w, None, groups, 1e-5, act, 0.0, p, False, rng, seed, 0)

    def back(dy=x, w=None, stats=stats, used=used, p=0.0):
        return op.group_norm_backward(dy, x, w, None, stats, used, 4, "relu", 0.0, p, False)

    norm(), back(), back(used=None)
    for call, err in [
            (lambda: norm(w=torch.ones(7, device=DEV)), ValueError),
            (lambda: norm(w=torch.ones(8)), RuntimeError),
            (lambda: norm(x.double()), RuntimeError),
            (lambda: norm(groups=3), ValueError),
            (lambda: norm(act="gelu"), ValueError),
            (lambda: norm(p=0.5, rng=used[:1]), ValueError),
            (lambda: norm(p=0.5, rng=used.cpu()), ValueError),
            (lambda: norm(p=0.5, seed=-1), ValueError),
            (lambda: back(x[:1]), ValueError),
            (lambda: back(w=torch.ones(7, device=DEV)), ValueError),
            (lambda: back(stats=stats[:1]), ValueError),
            (lambda: back(stats=stats.float()), ValueError),
            (lambda: back(used=None, p=0.5), ValueError),
            (lambda: op.dropout(x, x[:1], 0.5, False, None, 1, 2), ValueError),
            (lambda: op.dropout(x, None, 0.5, False, used[:1], 0, 0), ValueError),
            (lambda: op.dropout(x, None, 2.0, False, None, 1, 2), ValueError),
            (lambda: op.dropout_backward(x, used[:1], 0.5, False), ValueError),
            (lambda: op.dropout_backward(x.int(), used, 0.5, False), RuntimeError)]:
        with pytest.raises(err):
            call()


def test_run_of_an_encoders_tail_into_the_correlation():
    """norm + ReLU + channel dropout on both maps, a dropped branch added to it, the pyramid
    lookup, and the gradients of everything, against the 64-bit oracle."""
    b, h, w, c, levels, radius = 2, 16, 24, 64, 2, 3
    x, gamma, beta, _ = _norm_case((2 * b, h, w, c), torch.float32, seed=21)
    coords = corr_oracle.make_coords_uniform(b, h, w, 4.0, seed=22)
    gout = _rand((b, levels * 49, h, w), 23)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gamma, beta)]

    y = lc.group_norm(leaves[0], 8, leaves[1], leaves[2], activation="silu", p=0.2, rng=(5, 0),
                      dropout_mode="channel")
    y = lc.dropout(y, 0.3, (5, 1), residual=y)
    maps = y.permute(0, 3, 1, 2)
    out = lc.get_localcorr_block(maps[:b], maps[b:], num_levels=levels, radius=radius,
                                 corr_mode="localcorr_cuda")(coords.to(DEV))
    grads = torch.autograd.grad(out, leaves, gout.to(DEV))

    ref = [t.double().requires_grad_(True) for t in (x, gamma, beta)]
    v = ref[0].reshape(2 * b, -1, 8, c // 8)
    mean = v.mean((1, 3), keepdim=True)
    xhat = ((v - mean) / torch.sqrt(((v - mean) ** 2).mean((1, 3), keepdim=True) + 1e-5))
    y64 = oracle.activated(xhat.reshape(x.shape) * ref[1] + ref[2], "silu")
    y64 = y64 * oracle.drop_factors(x.shape, 0.2, 5, 0, True)
    y64 = y64 + y64 * oracle.drop_factors(x.shape, 0.3, 5, 1)
    m = y64.permute(0, 3, 1, 2)
    want, g1, g2 = corr_oracle.block_grads(m[:b].detach(), m[b:].detach(), coords, levels, radius,
                                           gout)
    # the correlation's own tolerance in float32
    torch.testing.assert_close(out.detach().double().cpu(), want, rtol=1e-5, atol=1e-4)
    gm = torch.cat([g1, g2]).permute(0, 2, 3, 1)
    for a, o in zip(grads, torch.autograd.grad(y64, ref, gm)):
        scale = float(o.abs().max())
        torch.testing.assert_close(a.double().cpu(), o, rtol=1e-4, atol=1e-4 * max(1.0, scale))
