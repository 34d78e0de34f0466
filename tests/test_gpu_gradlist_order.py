"""Gradient lists on the GPU: order of work, memory and addresses.

The norm's tolerance counts roundings (u = 2^-24): the sum of squares is within
5u of the stored values', so the norm within 2.5u and its own rounding, 3.5u;
4u is checked.  Multiplying gradients by a power of two is exact.
"""
from __future__ import annotations

import math

import pytest

from slmopt import B200Adamw, GradientList, SlmError, StepOptions, TensorTable, _lib, synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BUSY = 40_000_000  # cycles: 20 ms and more, against microseconds of host work between two calls


@pytest.fixture(scope="module")
def torch():
    import torch as _torch

    if not _torch.cuda.is_available():
        pytest.fail("a gpu-marked test ran without a CUDA device")
    return _torch


def make(torch, sizes, kinds=("bfloat16", "float32"), seed=0, std=1e-2):
    gen = torch.Generator("cuda").manual_seed(seed)
    return [(std * torch.randn(n, generator=gen, device="cuda")).to(getattr(torch, kinds[i % len(kinds)]))
            for i, n in enumerate(sizes)]


def norm64(tensors):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in tensors))


def near(got, want, tol, what):
    assert abs(got - want) <= tol * abs(want), f"{what}: got {got!r}, want {want!r}"


# ---- results of calls on other streams ------------------------------------------------
READS = {"read": lambda r: r.read().norm, "norm": lambda r: float(r.norm),
         "values": lambda r: r.values.tolist()[0],
         "sum_squares": lambda r: math.sqrt(float(r.sum_squares))}


@pytest.mark.parametrize("how", ["another stream", "the default stream beside a side stream"])
@pytest.mark.parametrize("take", READS.values(), ids=READS.keys())
@pytest.mark.parametrize("sizes", [[3000, 33], [2_000_003, 70_001]], ids=["small", "large"])
def test_a_result_is_read_behind_its_call(torch, sizes, take, how):
    tensors = make(torch, sizes, seed=1)
    want = norm64(tensors)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with GradientList(tensors) as lst:
        on = side if how == "another stream" else torch.cuda.default_stream()
        reader = torch.cuda.default_stream() if how == "another stream" else side
        for k in range(1, 4):
            with torch.cuda.stream(on):
                torch.cuda._sleep(BUSY)
                for t in tensors:
                    t.mul_(2.0)
            with torch.cuda.stream(reader):
                r = lst.norm(stream=side if on is side else None)
                near(take(r), want * 2.0 ** k, 4 * U, "norm")


# ---- memory of calls on other streams -------------------------------------------------
@pytest.mark.parametrize("call", ["norm", "clip"])
@pytest.mark.parametrize("how", ["another stream", "the default stream beside a side stream"])
@pytest.mark.parametrize("sizes", [[3000, 33], [2_000_003, 70_001]], ids=["small", "large"])
def test_a_call_takes_no_memory_that_another_stream_still_uses(torch, sizes, how, call):
    """Blocks that were given back on the current stream, where kernels that use
    them are still queued, are not what a call on another stream writes to."""
    tensors = make(torch, sizes, seed=2)
    want = norm64(tensors)
    side = torch.cuda.Stream()
    with GradientList(tensors) as lst, \
            GradientList([torch.empty_like(t) for t in tensors]) as out:
        on = side if how == "another stream" else torch.cuda.default_stream()
        current = torch.cuda.default_stream() if how == "another stream" else side
        elements = [128, 256, 512, 1024, 4096, 16384]  # f32: blocks of results and workspaces
        with torch.cuda.stream(current):
            warm = [torch.empty(n, device="cuda") for n in elements for _ in range(8)]
            del warm
            torch.cuda.synchronize()
            for _ in range(3):
                blocks = [torch.full((n,), 3.0, device="cuda") for n in elements for _ in range(8)]
                kept = torch.empty(len(blocks), device="cuda")
                torch.cuda._sleep(BUSY)
                for k, b in enumerate(blocks):  # queued behind the sleep: reads, then writes
                    kept[k] = b.sum() / b.numel()
                    b.fill_(5.0)
                del blocks, b
                kw = dict(stream=side if on is side else None, per_tensor=True)
                r = lst.norm(**kw) if call == "norm" else lst.clip(want / 2, out=out, **kw)
                torch.cuda.synchronize()
                near(r.read().norm, want, 4 * U, "norm")
                near(float(r.tensor_max[0]), float(tensors[0].abs().max()), U, "largest")
                assert bool((kept == 3.0).all())
