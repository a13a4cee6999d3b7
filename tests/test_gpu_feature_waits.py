"""Waits inside the group norm's kernels that run out: the kernel ends by itself, the status
says so until it is reset, and the next call is right.

With a limit of 0 a wait gives up when its first looks find nothing.
"""

import pytest
import torch

import localcorr_b200 as lc
from localcorr_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    return _lib.require_library()


class _Limit:
    def __init__(self, lib, ns):
        self.lib, self.ns = lib, ns

    def __enter__(self):
        self.before = self.lib.localCorrB200SetNormWaitLimit(self.ns)

    def __exit__(self, *_):
        self.lib.localCorrB200SetNormWaitLimit(self.before)


def _leaves(shape, dtype):
    g = torch.Generator(DEV).manual_seed(sum(shape))
    x = torch.randn(shape, generator=g, device=DEV).to(dtype).requires_grad_(True)
    w = torch.rand(shape[-1], generator=g, device=DEV).requires_grad_(True)
    return x, w, torch.randn(shape, generator=g, device=DEV).to(dtype)


# divided and read element by element; wider than a CTA
PLAIN = [((2, 3000, 33), 3, torch.float16), ((1, 90, 4104), 8, torch.float32)]


def _run_out(lib, shape, groups, dtype):
    x, w, dy = _leaves(shape, dtype)

    def forward():
        return lc.group_norm(x, groups, w, activation="relu")

    want = forward()
    wants = torch.autograd.grad(want, (x, w), dy, retain_graph=True)
    assert lib.localCorrB200DeviceStatus(1) == 0
    side = torch.cuda.Stream()  # does not synchronise with the default stream
    for call in (forward, lambda: torch.autograd.grad(want, (x, w), dy, retain_graph=True)):
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(200):  # it may find all it looks for, if seldom
            with _Limit(lib, 0), torch.cuda.stream(side):
                call()
            if lib.localCorrB200DeviceStatus(0):
                break
        assert lib.localCorrB200DeviceStatus(1) == 1  # stays until it is reset
        assert lib.localCorrB200DeviceStatus(0) == 0
        torch.cuda.current_stream().wait_stream(side)
        y = forward()
        assert torch.equal(y, want)
        for a, b in zip(torch.autograd.grad(y, (x, w), dy), wants):
            assert torch.equal(a, b)
    assert lib.localCorrB200DeviceStatus(1) == 0


@pytest.mark.parametrize("shape,groups,dtype", PLAIN)
def test_plain_kernels(lib, shape, groups, dtype):
    _run_out(lib, shape, groups, dtype)


# streamed: groups of whole vectors and of single channels, one sample and several chunks
STREAMED = [((3, 4000, 64), 8, torch.float16), ((2, 2000, 64), 64, torch.float32),
            ((1, 40_000, 96), 12, torch.bfloat16), ((9, 40_000, 128), 16, torch.float16),
            ((33, 8192, 128), 128, torch.bfloat16)]


# the CTAs of small maps come to their sums within the microseconds that a first look takes:
# every wait may find what it looks for. Over a large map they drift apart.
@pytest.mark.parametrize("shape,groups,dtype", STREAMED[3:])
def test_streamed_kernels(lib, shape, groups, dtype):
    _run_out(lib, shape, groups, dtype)


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("shape,groups,dtype", STREAMED)
def test_limits_that_some_threads_reach(lib, shape, groups, dtype, act):
    # limits about as long as the waits: threads of one CTA give up at different times. A call
    # ends, and one that says it finished is right.
    x, w, dy = _leaves(shape, dtype)

    def call():
        y = lc.group_norm(x, groups, w, activation=act)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    want = call()
    for limit in (300, 1000, 2000, 4000, 8000, 16000, 32000, 64000):
        for _ in range(4):
            with _Limit(lib, limit):
                got = call()
            if lib.localCorrB200DeviceStatus(1) == 0:
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(call(), want))
