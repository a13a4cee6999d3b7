"""How exact the feature-map operators are, against 64-bit values on the GPU.

Every tolerance is derived beside its use from the roundings the kernels make: float32's is
2^-24, float64's 2^-53, relative to the rounded value.
"""

import pytest
import torch

import localcorr_b200 as lc
from localcorr_b200 import _lib, features
from oracle import feature_maps as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    assert _lib.load_library() is not None


def _randn(shape, seed, dtype=torch.float64):
    return torch.randn(shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV,
                       dtype=dtype)


def _by_group(x, groups):
    return x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def _statistics(x, groups, eps):
    """Mean and 1/std [B, G] in float64, centred before they are squared."""
    v = _by_group(x, groups)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    shape = (x.shape[0], groups)
    return mean.reshape(shape), (1 / (var + eps).sqrt()).reshape(shape)


def _kernel_statistics(x, groups, eps):
    stats = features.group_norm_forward(x, None, None, groups, eps, "none", 0.0, 0.0, False, None,
                                        0, 0)[1]
    return stats[..., 0], stats[..., 1]


# whole samples; streamed, groups of whole vectors and of single channels; plain, twice
SIZES = [((2, 100, 64), 8), ((3, 4000, 64), 8), ((2, 2000, 64), 64), ((2, 3000, 33), 3),
         ((1, 90, 4104), 8)]


@pytest.mark.parametrize("eps", [1e-5, 0.0])
@pytest.mark.parametrize("mean,std", [(0.0, 1.0), (1e4, 1.0), (1e5, 1.0), (1e6, 1.0),
                                      (3000.0, 0.002), (-2e7, 10.0)])
@pytest.mark.parametrize("shape,groups", SIZES)
def test_statistics_of_maps_far_from_zero(shape, groups, mean, std, eps):
    x = (_randn(shape, 1) * std + mean).float()
    want_mean, want_rstd = _statistics(x, groups, eps)
    got_mean, got_rstd = _kernel_statistics(x, groups, eps)
    # float64 sums of at most 2^18 terms around a value of the group, which lies less than 6
    # spreads from the mean: var is off by 37 * 2^18 * 2^-53 < 2^-29 of itself at the very worst
    # (every rounding of one sign); 2^-34 allows for 2^13 of them, 1/std halves it
    assert bool(((got_rstd - want_rstd).abs() <= 2.0 ** -35 * want_rstd).all())
    assert bool(((got_mean - want_mean).abs()
                 <= 2.0 ** -51 * abs(mean) + 2.0 ** -35 / want_rstd).all())


@pytest.mark.parametrize("shape,groups", SIZES)
def test_statistics_around_a_value_far_off(shape, groups):
    # the first value of each group is 1000 spreads of the others away
    x = _randn(shape, 2).float()
    first = x.reshape(shape[0], -1, groups, shape[-1] // groups)
    first[:, 0, :, 0] += 1000.0
    want_mean, want_rstd = _statistics(x, groups, 1e-5)
    got_mean, got_rstd = _kernel_statistics(x, groups, 1e-5)
    # the cancellation costs (1000 spreads)^2 / var < 2^20 of 2^13 roundings of 2^-53
    assert bool(((got_rstd - want_rstd).abs() <= 2.0 ** -20 * want_rstd).all())
    assert bool(((got_mean - want_mean).abs() <= 2.0 ** -30).all())


@pytest.mark.parametrize("shape,groups", SIZES)
def test_small_variance_far_from_zero_without_eps(shape, groups):
    # one value in a hundred is a float32 step (1/16) above 10^6
    x = torch.full(shape, 1e6, device=DEV)
    x.view(-1)[::99] += 0.0625
    want_mean, want_rstd = _statistics(x, groups, 0.0)
    # (33 channels in 3 groups: the values all lie in the first; a group without any has no
    # variance, 1/std is infinite and the outputs are 0 / 0)
    assert bool(want_rstd[:, 0].isfinite().all())
    got_mean, got_rstd = _kernel_statistics(x, groups, 0.0)
    # every x - K is a multiple of 1/16 and its sums are exact; the rest is a few roundings
    torch.testing.assert_close(got_rstd, want_rstd, rtol=2.0 ** -45, atol=0)
    y = lc.group_norm(x, groups, eps=0.0)
    want = ((_by_group(x, groups) - want_mean[:, None, :, None])
            * want_rstd[:, None, :, None]).reshape(shape)
    # x - mu is exact but for mu's part below float32, whose product with 1/std (at most
    # 1/30 * 10) is rounded; then 1/std, the product and the sum
    assert torch.equal(y.isnan(), want.isnan())
    off = ((y.double() - want).abs() - 2.0 ** -22 * (want.abs() + 1))[~want.isnan()]
    assert bool((off <= 0).all())


@pytest.mark.parametrize("eps", [1e-5, 0.0])
@pytest.mark.parametrize("dtype,mean,std", [
    (torch.float16, 1000.0, 1.0), (torch.float16, 30000.0, 20.0), (torch.float16, -2048.0, 0.6),
    (torch.float16, 0.01, 1e-4), (torch.bfloat16, 300.0, 1.0), (torch.bfloat16, 1e4, 40.0),
    (torch.bfloat16, -3e4, 1000.0), (torch.bfloat16, 1e18, 1e17)])
@pytest.mark.parametrize("shape,groups", SIZES)
def test_statistics_of_16_bit_maps_far_from_zero(shape, groups, dtype, mean, std, eps):
    x = (_randn(shape, 16) * std + mean).to(dtype)
    want_mean, want_rstd = _statistics(x, groups, eps)
    got_mean, got_rstd = _kernel_statistics(x, groups, eps)
    # nearly all values lie in two binades: their sums are exact. What is rounded (2^13 sums at
    # most) is weighed with 1 + mean^2 / var, which rounding to the type keeps below 2^22
    assert bool(want_rstd.isfinite().all())
    torch.testing.assert_close(got_rstd, want_rstd, rtol=2.0 ** -36, atol=0)
    torch.testing.assert_close(got_mean, want_mean, rtol=2.0 ** -45, atol=0)


@pytest.mark.parametrize("shape,groups", SIZES)
@pytest.mark.parametrize("dtype,level", [(torch.float16, 1000.0), (torch.bfloat16, 1000.0)])
def test_small_variance_of_16_bit_maps_without_eps(shape, groups, dtype, level):
    # one value in a hundred is a step above the others, one in a thousand is 0
    x = torch.full(shape, level, dtype=dtype, device=DEV)
    x.view(-1)[::97] = level + (0.5 if dtype == torch.float16 else 4.0)
    x.view(-1)[::997] = 0.0
    want_mean, want_rstd = _statistics(x, groups, 0.0)
    got_mean, got_rstd = _kernel_statistics(x, groups, 0.0)
    # multiples of one step throughout: exact sums, a few roundings behind them
    assert bool(want_rstd.isfinite().all())
    torch.testing.assert_close(got_rstd, want_rstd, rtol=2.0 ** -45, atol=0)
    torch.testing.assert_close(got_mean, want_mean, rtol=2.0 ** -48, atol=0)


@pytest.mark.parametrize("shape,groups", SIZES)
def test_constant_groups_give_the_bias(shape, groups):
    x = torch.full(shape, 1234567.0, device=DEV)
    b = torch.linspace(-1, 1, shape[-1], device=DEV)
    assert torch.equal(lc.group_norm(x, groups, None, b), b.expand(shape))


def test_groups_whose_vectors_pass_32_bits():
    # 268435460 channels a group, no whole number of vectors: eight times that passes 2^31
    c = 2 * 268_435_460
    x = torch.empty(1, c, dtype=torch.float16, device=DEV).normal_(
        generator=torch.Generator(DEV).manual_seed(7))
    x[0, c // 2:] += 2.0
    got_mean, got_rstd = _kernel_statistics(x, 2, 1e-5)
    want_mean, want_rstd = _statistics(x, 2, 1e-5)
    # 2^20 sequential float64 sums of a thread, 6 spreads from the group's first value at most
    torch.testing.assert_close(got_mean, want_mean, rtol=0, atol=2.0 ** -28)
    torch.testing.assert_close(got_rstd, want_rstd, rtol=2.0 ** -28, atol=0)
    y = lc.group_norm(x, 2)
    for lo in (0, c // 2 - 2048, c // 2, c - 2048):  # both ends of both groups
        g = lo // (c // 2)
        part = slice(lo, lo + 2048)
        want = (x[0, part].double() - want_mean[0, g]) * want_rstd[0, g]
        assert bool(((y[0, part].double() - want).abs()
                     <= 2.0 ** -11 * want.abs() + 2.0 ** -20).all())


# one streamed sample with 1024 and 2100 rows a thread; streamed with many rows of threads and
# several chunks; plain kernels, one to four bytes a thread; whole samples
LONG = [((1, 296 * 1024, 1024), 8, torch.float32), ((1, 296 * 2100, 1024), 8, torch.float32),
        ((6, 200_000, 64), 64, torch.float32),
        ((1, 296 * 1100, 1000), 8, torch.bfloat16), ((1, 400_000, 33), 3, torch.float32),
        ((2, 500_000, 1), 1, torch.float16), ((1, 8192, 1), 1, torch.float32)]


@pytest.mark.parametrize("value", [1.1, 1.7, 1 / 303104])
@pytest.mark.parametrize("shape,groups,dtype", LONG)
def test_equal_gradients_of_many_rows(shape, groups, dtype, value):
    # the gradient of a mean: equal terms, whose float32 sums all round the same way
    x = _randn(shape, 4, torch.float32).to(dtype).requires_grad_(True)
    b = torch.zeros(shape[-1], device=DEV, requires_grad=True)
    dy = torch.full((), value, dtype=dtype, device=DEV).expand(shape).contiguous()
    term = float(dy.view(-1)[0])
    y = lc.group_norm(x, groups, None, b)
    gx, gb = torch.autograd.grad(y, (x, b), dy)
    # 32 equal terms: partial sums k t, k = 2 ... 32, rounded by 2^-24 of themselves, 16.5 2^-24
    # of the sum; again for 32 such sums; a thread's, a slice's and the result's own rounding
    e = (2 * 16.5 + 3) * 2.0 ** -24
    want = term * (x.numel() // shape[-1])
    assert float((gb.double() - want).abs().max()) <= e * want
    # dx = r (dz - mean dz - xhat mean(dz xhat)) is 0 but for xhat's mean (and that of its
    # square over n); dz, the mean's error and the products are 1 + e + 4 2^-24 of r dz
    v = _by_group(x.detach(), groups)
    var = v.var((1, 3), correction=0, keepdim=True)
    r = 1 / (var + 1e-5).sqrt()
    xhat = ((v - v.mean((1, 3), keepdim=True)) * r).abs()
    # sum dz (x - mu): the terms are not equal; e of the sum of their magnitudes
    m2 = e * xhat.mean((1, 3), keepdim=True)
    tol = r * term * (e + 4 * 2.0 ** -24 + xhat * (m2 + 4 * 2.0 ** -24))
    got = _by_group(gx, groups).abs()
    assert bool((got <= tol * (1 + torch.finfo(dtype).eps)
                 + torch.finfo(dtype).smallest_normal).all())

# ---------------------------------------------------------------------------
# the forward's roundings, the parameters' gradients row by row, what dropout keeps
# ---------------------------------------------------------------------------

FORWARD = [((2, 46, 62, 256), 32), ((3, 47, 61, 96), 96), ((2, 3000, 33), 11), ((2, 37, 2048), 16),
           ((5, 3, 3, 12), 4), ((1, 17, 4104), 8), ((1, 1, 256), 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "leaky_relu"])
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("shape,groups", FORWARD)
def test_forward_to_its_roundings(shape, groups, p, act, dtype):
    c = shape[-1]
    x = (_randn(shape, 8) * (0.5 * _randn((c,), 9)).exp() + 3 * _randn((c,), 10)).to(dtype)
    w = (1 + 0.3 * _randn((c,), 11)).float()
    b = _randn((c,), 12).float()
    y = lc.group_norm(x, groups, w, b, activation=act, negative_slope=0.1, p=p, rng=(3, 4))

    mean, rstd = _statistics(x, groups, 1e-5)
    mean, rstd = (t[:, None, :, None] for t in (mean, rstd))
    grouped = _by_group(x, groups).shape
    xhat = ((_by_group(x, groups) - mean) * rstd).reshape(shape)
    shift = (mean.abs() * rstd).expand(grouped).reshape(shape)
    z = xhat * w.double() + b.double()
    e = 2.0 ** -24
    # z = (x - mu) a + c: x - mu; 1/std and its product with the weight; c, which holds what
    # mu loses in float32 (2^-24 of it); the sum
    z_err = e * (3 * (xhat * w).abs() + b.abs() + e * shift * w.abs() + z.abs())
    slope = 1.0
    if act == "none":
        want, err = z, 0.0
    elif act == "relu":
        want, err = z.clamp_min(0.0), 0.0
    elif act == "leaky_relu":
        slope32 = float(torch.tensor(0.1))
        want = torch.where(z > 0, z, slope32 * z)
        err = e * want.abs()
    else:
        # z sigma(z): exp within (2 + 1.173 |z|) ulp, which sigma takes on times 1 - sigma; the
        # sum; a quotient within 2 ulp; the product. A ulp is 2^-23 at most
        sigma = torch.sigmoid(z)
        want, slope = z * sigma, 1.1
        err = want.abs() * ((1 - sigma) * (2 + 1.173 * z.abs()) * 2 * e + e + 4 * e + e)
    err = slope * z_err + err
    if p > 0:
        kept = lc.dropout(torch.ones_like(x, dtype=torch.float32), p, (3, 4)) != 0
        t = int(p * 65536 + 0.5)
        factor = 65536 / (65536 - t)  # and its rounding, and the product's
        want, err = want * factor, err * factor + 2 * e * (want * factor).abs()
        assert bool((y[~kept] == 0).all())
        want, err = torch.where(kept, want, 0.0), torch.where(kept, err, 0.0)
    u = torch.finfo(dtype).eps / 2
    tol = (1 + 2 * u) * err + u * want.abs() + torch.finfo(dtype).smallest_normal * 2 * u
    off = (y.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((3, 2852, 64), 8), ((2, 8192, 128), 128),
                                          ((2, 3000, 33), 11), ((5, 20, 48), 4),
                                          ((1, 90, 4104), 8)])
def test_gradients_of_single_rows(shape, groups, dtype):
    # an output gradient of one row: what any row adds to the sums shows, and only that
    b, rows, c = shape
    x = _randn(shape, 13, torch.float32).to(dtype).requires_grad_(True)
    w = (1 + 0.3 * _randn((c,), 14)).float().requires_grad_(True)
    bias = torch.zeros(c, device=DEV, requires_grad=True)
    y = lc.group_norm(x, groups, w, bias)
    mean, rstd = _statistics(x.detach(), groups, 1e-5)
    r = rstd[:, None, :, None]
    v = (_by_group(x.detach(), groups) - mean[:, None, :, None]) * r  # xhat by group
    e = 2.0 ** -24
    u = torch.finfo(dtype).eps / 2
    n = rows * (c // groups)
    # ends of samples, of runs of rows a CTA has (whatever their length), and in between
    for i, row in enumerate([0, 1, rows - 1] + [k * rows // 7 + k % 3 for k in range(1, 7)]):
        sample, g = i % b, _randn((c,), 20 + i).to(dtype)
        dy = torch.zeros_like(x)
        dy[sample, row] = g
        gx, gw, gb = torch.autograd.grad(y, (x, w, bias), dy, retain_graph=True)
        assert torch.equal(gb, g.float())
        xhat = v[sample, row].reshape(c)
        want = g.double() * xhat
        # x - mu, its product with dy, the result; mu's part below float32 is added in float64
        assert bool(((gw.double() - want).abs() <= 4 * e * want.abs() + e * e * g.abs()).all())
        wg = (w.detach().double() * g.double()).reshape(groups, -1)
        vr = v[sample, row]
        m1 = (wg.sum(1) / n)[None, :, None]
        m2 = ((wg * vr).sum(1) / n)[None, :, None]
        size1 = (wg.abs().sum(1) / n)[None, :, None]
        size2 = ((wg * vr).abs().sum(1) / n)[None, :, None]
        dz = torch.zeros_like(v[sample])
        dz[row] = wg
        want = r[sample] * (dz - m1 - v[sample] * m2)
        # dx = a dz + (k2 (x - mu) + k3): the terms and two sums are rounded, a twice
        tol = r[sample] * (4 * e * dz.abs() + 4 * e * size1 + 6 * e * v[sample].abs() * size2)
        got = gx[sample].double().reshape(want.shape)
        assert bool(((got - want).abs() <= tol + u * (want.abs() + tol) + 2.0 ** -140).all())
        others = [k for k in range(b) if k != sample]
        assert bool((gx[others] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mode", ["element", "channel"])
@pytest.mark.parametrize("shape", [(2, 31, 24), (2, 31, 33), (1, 7, 2056), (3, 1)])
def test_dropout_drops_what_is_drawn_and_nothing_else(shape, mode, dtype):
    # every value is far from 0: an element is 0 exactly where the draw says so
    x = (_randn(shape, 15, torch.float32).sign() * 2 + 1).to(dtype)
    f = oracle.drop_factors(shape, 0.4, 5, 6, mode == "channel").expand(shape)
    y = lc.dropout(x, 0.4, (5, 6), mode=mode).cpu()
    assert torch.equal(y == 0, f == 0)
    r = torch.full_like(x, 0.5)
    z = lc.dropout(x, 0.4, (5, 6), residual=r, mode=mode).cpu()
    assert torch.equal(z == 0.5, f == 0)


# ---------------------------------------------------------------------------
# what autograd is told
# ---------------------------------------------------------------------------

def test_by_products_of_registered_operators_are_not_differentiable():
    x = _randn((2, 30, 16), 3).float().requires_grad_(True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    op = torch.ops.localcorr
    y, stats, used = op.group_norm(x, w, None, 4, 1e-5, "silu", 0.0, 0.5, False, None, 1, 2)
    assert not stats.requires_grad and not used.requires_grad
    want = lc.group_norm(x, 4, w, activation="silu", p=0.5, rng=(1, 2))
    for a, b in zip(torch.autograd.grad(y.sum(), (x, w)), torch.autograd.grad(want.sum(), (x, w))):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="does not require grad"):
        stats.sum().backward()
    y, used = op.dropout(x, x, 0.5, True, None, 1, 2)
    assert y.requires_grad and not used.requires_grad


def test_other_kinds_of_differentiation_are_refused():
    x = _randn((2, 30, 16), 5).float()
    w = torch.ones(16, device=DEV)
    calls = (lambda t: lc.group_norm(t, 4), lambda t: lc.group_norm(x, 4, w, t[0, 0]),
             lambda t: lc.dropout(t, 0.5, (1, 2)), lambda t: lc.dropout(x, 0.5, (1, 2), residual=t))
    for call in calls:
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x.expand(3, 2, 30, 16))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(x)


def test_hooks_see_all_that_is_saved():
    # what the backward needs lives where the graph's hooks (offloading) can move it
    x = _randn((2, 30, 16), 6).float().requires_grad_(True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    seen = []

    def pack(t):
        seen.append((tuple(t.shape), t.dtype))
        return t.cpu()

    for call, kept in (
            (lambda: lc.group_norm(x, 4, w, activation="silu", p=0.5, rng=(1, 2)),
             [((2, 30, 16), torch.float32), ((16,), torch.float32), ((2, 4, 2), torch.float64),
              ((2,), torch.int64)]),
            (lambda: lc.dropout(x, 0.5, (1, 2), residual=x), [((2,), torch.int64)])):
        seen.clear()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
            y = call()
        assert seen == kept
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0],
                           torch.autograd.grad(call().sum(), x)[0])
        # and is gone after the backward, unless it is asked to stay
        y = call()
        torch.autograd.grad(y.sum(), x)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("shape,groups,dtype", [((3, 4000, 64), 8, torch.float16),
                                                ((2, 2000, 64), 64, torch.float32)])
def test_context_with_a_part_of_the_multiprocessors(shape, groups, dtype):
    # the streamed kernels' CTAs do not fit all at once: the plain kernels take the call
    green = pytest.importorskip("torch.cuda.green_contexts")
    if not green.SUPPORTED:
        pytest.skip("green contexts not supported")
    x, dy = (_randn(shape, 30 + i, torch.float32).to(dtype) for i in range(2))
    w = torch.linspace(0.5, 1.5, shape[-1], device=DEV)

    def call():
        y, stats, _ = features.group_norm_forward(x, w, None, groups, 1e-5, "silu", 0.0, 0.0, False,
                                                  None, 0, 0)
        return y, *features.group_norm_backward(dy, x, w, None, stats, None, groups, "silu", 0.0,
                                                0.0, False)[:2]

    want = call()
    torch.cuda.synchronize()
    context = green.GreenContext.create(num_sms=16, device_id=torch.cuda.current_device())
    context.set_context()
    try:
        got = call()
        torch.cuda.synchronize()
    finally:
        context.pop_context()
    # float32 roundings of two orders of summation, 2^-18 at most, then the rounding of either
    u = torch.finfo(dtype).eps / 2
    for a, b in zip(got, want):
        e = u if a.dtype == dtype else 2.0 ** -24
        scale = b.double().abs().max()
        assert bool(((a.double() - b.double()).abs()
                     <= 2 * e * b.double().abs() + 2.0 ** -18 * scale).all())


def test_by_products_of_empty_maps_are_zero():
    torch.full((4096,), 7.0, dtype=torch.float64, device=DEV)  # what freed memory may hold
    x = torch.zeros(3, 0, 8, device=DEV)
    y, stats, used = torch.ops.localcorr.group_norm(x, None, None, 2, 1e-5, "none", 0.0, 0.5,
                                                    False, None, 1, 2)
    assert y.shape == x.shape and bool((stats == 0).all()) and bool((used == 0).all())
    assert bool((torch.ops.localcorr.dropout(x, None, 0.5, False, None, 1, 2)[1] == 0).all())
