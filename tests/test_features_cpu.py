"""Feature-map operators without a GPU: the oracle's generator against its
published known answers, argument checks of the Python calls and of the C entry
points (which validate before any CUDA call)."""

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import localcorr_b200 as lc
from localcorr_b200 import _lib, features
from oracle import feature_maps


def test_philox_known_answers():
    # Random123's published vectors of Philox4x32-10
    zero = feature_maps.philox4x32_10([0] * 4, (0, 0))
    assert [int(v) for v in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = feature_maps.philox4x32_10([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(v) for v in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_draws_are_pieces_of_blocks():
    d = feature_maps.draws(0, 0, 0, 16)
    assert list(d[:4]) == [0xE8D5, 0x6627, 0xC58D, 0xE169]
    assert np.array_equal(feature_maps.draws(5, 9, 11, 30), feature_maps.draws(5, 9, 0, 64)[11:41])


def test_exported():
    assert lc.group_norm is features.group_norm and lc.dropout is features.dropout
    for op in ("group_norm", "group_norm_backward", "dropout", "dropout_backward"):
        assert hasattr(torch.ops.localcorr, op)


def test_cpu_maps_are_refused():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(RuntimeError, match="CUDA device"):
        lc.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="CUDA device"):
        lc.dropout(x, 0.5, (1, 2))
    with pytest.raises(TypeError, match="must be a tensor"):
        lc.group_norm(x.numpy(), 2)


@pytest.mark.parametrize("kw,err,match", [
    (dict(num_groups=3), ValueError, "divisor"),
    (dict(num_groups=0), ValueError, "divisor"),
    (dict(num_groups=2.0), ValueError, "divisor"),
    (dict(weight=torch.zeros(7)), ValueError, "shape"),
    (dict(bias=torch.zeros(1, 8)), ValueError, "shape"),
    (dict(weight=torch.zeros(8, dtype=torch.float64)), RuntimeError, "must be float32"),
    (dict(weight=torch.zeros(8, dtype=torch.float16), bias=torch.zeros(8)), RuntimeError,
     "one dtype"),
    (dict(activation="swish"), ValueError, "unknown activation"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(negative_slope=float("inf")), ValueError, "negative_slope"),
])
def test_norm_arguments(kw, err, match):
    args = dict(num_groups=2, weight=None, bias=None, eps=1e-5, activation="none",
                negative_slope=0.01)
    x = torch.zeros(2, 5, 8, dtype=torch.float16)
    features._check_norm(x, **args)
    with pytest.raises(err, match=match):
        features._check_norm(x, **{**args, **kw})


@pytest.mark.parametrize("p,rng,mode,match", [
    (-0.1, (1, 2), "element", "probability"),
    (1.1, (1, 2), "element", "probability"),
    (float("nan"), (1, 2), "element", "probability"),
    (0.5, None, "element", "needs rng"),
    (0.5, (1, 2), "row", "unknown dropout mode"),
    (0.5, (1,), "element", "two integers"),
    (0.5, (1, -2), "element", "two integers"),
    (0.5, (1, 2 ** 63), "element", "two integers"),
    (0.5, (1.5, 2), "element", "two integers"),
    (0.5, torch.zeros(2), "element", "int64"),
    (0.5, torch.zeros(3, dtype=torch.int64), "element", "int64"),
])
def test_dropout_arguments(p, rng, mode, match):
    with pytest.raises(ValueError, match=match):
        features._check_dropout(p, rng, mode, torch.zeros(2, 8), "dropout")


def test_dropout_arguments_accepted():
    x = torch.zeros(2, 8)
    assert features._check_dropout(0, None, "element", x, "dropout") == 0.0
    assert features._check_dropout(1, (0, 2 ** 63 - 1), "channel", x, "dropout") == 1.0
    assert features._check_dropout(0.5, torch.zeros(2, dtype=torch.int64), "element", x, "d") == 0.5


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from localcorr_b200.csrc import build

        build.build()
    return _lib.require_library()


def _dropout(lib, x=256, y=256, b=1, rows=4, c=8, dtype=_lib.F16, p=0.5, rng=None):
    return lib.launchLocalCorrB200Dropout(x, None, y, b, rows, c, dtype, p, False, 1, 2, rng, None,
                                          None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(c=0), "shape"), (dict(rows=-1), "shape"),
    (dict(b=-1), "shape"), (dict(b=2 ** 31 - 1, rows=2 ** 40), "too many"),
    (dict(p=1.5), "probability"), (dict(p=float("nan")), "probability"),
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(x=257), "aligned"),
    (dict(rng=260), "aligned"),
])
def test_c_dropout_refuses(lib, kw, match):
    assert not _dropout(lib, **kw)
    assert match in _lib.last_error(lib)


def _forward(lib, x=256, y=256, stats=256, weight=None, b=1, rows=4, c=8, g=2, dtype=_lib.F16,
             eps=1e-5, act=0, slope=0.0, p=0.0, ws=None, nws=0):
    return lib.launchLocalCorrB200GroupNormForward(
        x, weight, None, y, stats, b, rows, c, g, dtype, True, eps, act, slope, p, False, 0, 0,
        None, None, ws, nws, None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=-1), "dtype"), (dict(c=-8), "shape"), (dict(g=3), "divide"), (dict(g=0), "divide"),
    (dict(act=4), "activation"), (dict(slope=float("nan")), "slope"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(p=-0.5), "probability"), (dict(x=None), "null"),
    (dict(stats=None), "null"), (dict(stats=264), "aligned"), (dict(weight=258), "aligned"),
    (dict(x=255), "aligned"), (dict(ws=None), "workspace"), (dict(ws=256, nws=16), "workspace"),
    (dict(ws=260, nws=1 << 20), "workspace"),
])
def test_c_group_norm_refuses(lib, kw, match):
    assert not _forward(lib, **kw)
    assert match in _lib.last_error(lib)


def test_c_group_norm_backward_refuses(lib):
    def call(gy=256, x=256, stats=256, g=2, ws=None, nws=0):
        return lib.launchLocalCorrB200GroupNormBackward(
            gy, x, None, None, stats, 256, None, None, 1, 4, 8, g, _lib.F32, True, 0, 0.0, 0.0,
            False, 0, 0, None, ws, nws, None)

    for kw, match in ((dict(g=5), "divide"), (dict(gy=None), "null"), (dict(x=None), "null"),
                      (dict(stats=None), "null"), (dict(x=258), "aligned"),
                      (dict(), "workspace")):
        assert not call(**kw)
        assert match in _lib.last_error(lib)


def test_c_empty_problems_succeed(lib):
    assert _dropout(lib, x=None, y=None, rows=0)
    assert _dropout(lib, x=None, y=None, b=0)
    assert _forward(lib, x=None, y=None, stats=None, b=0)
    assert _forward(lib, x=None, y=None, stats=None, rows=0)


def test_c_workspace_sizes(lib):
    size = lib.localCorrB200GroupNormWorkspaceBytes
    assert size(0, 4, 8, 2, _lib.F16, False) == 0
    assert size(1, 4, 8, 3, _lib.F16, False) == 0
    assert size(1, 4, 8, 2, 7, False) == 0
    for b, rows, c, g in ((1, 1, 1, 1), (8, 32400, 256, 32), (3, 4000, 33, 11)):
        fwd, bwd = (size(b, rows, c, g, _lib.F16, back) for back in (False, True))
        # a pair of float64 per sample, slice and group; of float32 per channel
        assert fwd >= 4 * (b + 1) + 16 * b * g
        assert bwd >= 4 * (b + 1) + 8 * b * c + 16 * b * c + 16 * b * g
    assert ctypes.sizeof(ctypes.c_size_t) == 8
    # a million samples of one row: rows for the CTAs, not for the samples
    assert size(1 << 20, 1, 256, 32, _lib.F16, True) < 32 << 20
    assert size(64, 1 << 20, 64, 8, _lib.F16, True) < 1 << 30


@pytest.mark.parametrize("kw,match", [
    (dict(grad_y=torch.zeros(2, 5, 4)), "like x"),
    (dict(grad_y=torch.zeros(1, 5, 8)), "like x"),
    (dict(stats=torch.zeros(2, 4, 2)), "float64"),
    (dict(stats=torch.zeros(2, 2, 2, dtype=torch.float64)), "statistics"),
    (dict(stats=torch.zeros(1, 4, 2, dtype=torch.float64).expand(2, 4, 2)), "statistics"),
])
def test_norm_backward_arguments(kw, match):
    args = dict(grad_y=torch.zeros(2, 5, 8), x=torch.zeros(2, 5, 8),
                stats=torch.zeros(2, 4, 2, dtype=torch.float64), num_groups=4)
    features._check_norm_backward(**args)
    with pytest.raises(ValueError, match=match):
        features._check_norm_backward(**{**args, **kw})


@pytest.mark.parametrize("used,p,match", [
    (None, 0.5, "needs the stream"),
    (torch.zeros(0, dtype=torch.int64), 0.5, "needs the stream"),
    (torch.zeros(3, dtype=torch.int64), 0.5, "rng tensor"),
    (torch.zeros(2), 0.0, "rng tensor"),
    (torch.zeros(2, 2, dtype=torch.int64)[:, 0], 0.5, "contiguous"),
    (torch.zeros(2, dtype=torch.int64), 1.5, "probability"),
])
def test_used_stream_arguments(used, p, match):
    x = torch.zeros(2, 5, 8)
    features._check_used(None, 0.0, x, "backward")
    features._check_used(torch.zeros(2, dtype=torch.int64), 0.5, x, "backward")
    with pytest.raises(ValueError, match=match):
        features._check_used(used, p, x, "backward")


def test_only_the_map_of_a_registered_operator_is_differentiable():
    # the statistics have no gradient formula: a loss of them must not get a silent zero
    with FakeTensorMode():
        x = torch.empty(2, 5, 8, device="cuda", requires_grad=True)
        w = torch.empty(8, device="cuda", requires_grad=True)
        y, stats, used = torch.ops.localcorr.group_norm(x, w, None, 2, 1e-5, "relu", 0.0, 0.5,
                                                        False, None, 1, 2)
        assert y.requires_grad and not stats.requires_grad and not used.requires_grad
        y, used = torch.ops.localcorr.dropout(x, x, 0.5, True, None, 1, 2)
        assert y.requires_grad and not used.requires_grad


def test_tangents_are_refused():
    x = torch.ones(2, 8)
    features._check_tangents("dropout", x, None)
    with torch.autograd.forward_ad.dual_level():
        features._check_tangents("dropout", x, None)
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            features._check_tangents("dropout", x, dual)


def test_c_wait_limit(lib):
    before = lib.localCorrB200SetNormWaitLimit(-1)
    assert before == 2_000_000_000
    assert lib.localCorrB200SetNormWaitLimit(5) == before
    assert lib.localCorrB200SetNormWaitLimit(before) == 5
    assert lib.localCorrB200SetNormWaitLimit(-1) == before


def test_c_refuses_more_channels_than_the_kernels_count(lib):
    # their column loops add up to 256 to a 32-bit column before they compare it
    for c in (2 ** 30 + 1, 2 ** 31 - 1):
        assert not _dropout(lib, c=c) and "channels" in _lib.last_error(lib)
        assert not _forward(lib, c=c, g=1) and "channels" in _lib.last_error(lib)
        assert lib.localCorrB200GroupNormWorkspaceBytes(1, 1, c, 1, _lib.F16, False) == 0
    assert not _forward(lib, c=2 ** 30, g=1) and "workspace" in _lib.last_error(lib)


def test_c_wait_limit_is_bounded(lib):
    before = lib.localCorrB200SetNormWaitLimit(2 ** 62)
    assert lib.localCorrB200SetNormWaitLimit(before) == 10 ** 12
