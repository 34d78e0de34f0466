"""Gradient lists on the GPU: order of work, memory and addresses.

The norm's tolerance counts roundings (u = 2^-24): the sum of squares is within
5u of the stored values', so the norm within 2.5u and its own rounding, 3.5u;
4u is checked.  Multiplying gradients by a power of two is exact.
"""
from __future__ import annotations

import ctypes
import math

import pytest

from slmopt import B200Adamw, GradientList, SlmError, StepOptions, TensorTable, _lib, synth
from slmopt.trainer import canonical_learning_rate
from test_gpu_gradlist import check_state

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


# ---- clipped rows whose alignment changes ----------------------------------------------
def rows_of(torch, kind, first, columns=256, rows=3000, seed=0, width=328):
    """A column slice of a wider matrix; on vector boundaries when first % 8 == 0."""
    gen = torch.Generator("cuda").manual_seed(seed)
    wide = (1e-2 * torch.randn(rows, width, generator=gen, device="cuda")).to(getattr(torch, kind))
    return wide, wide[:, first:first + columns]


def half_step(torch, kind):
    return {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[kind]


def check_clipped(torch, got, before, factor):
    """round(x * (clip / scale)): clip 5u (sum to f32 6u, its root 3u + 1u, quotient 1u), over the
    scale 1u, product 1u: 7u, 7.5u are checked; and half a step of the output's type."""
    for y, x in zip(got, before):
        want = x.double() * factor
        off = (y.double() - want).abs()
        tol = (7.5 * U + half_step(torch, y.dtype)) * want.abs()
        if y.dtype == torch.float16:
            tol += 2.0 ** -25
        assert bool((off <= tol).all()), float((off - tol).max())


def outside_kept(torch, wide, keep, part):
    """Nothing but the slice has changed."""
    mask = torch.ones_like(wide, dtype=torch.bool)
    at = part.storage_offset() - wide.storage_offset()
    mask[:, at:at + part.shape[1]] = False
    return bool((wide[mask] == keep[mask]).all())


def captured(torch, call):
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        r = call(torch.cuda.current_stream())
    return g, r


@pytest.mark.parametrize("scale", [1.0, 8.0])
@pytest.mark.parametrize("kind", ["bfloat16", "float32", "float16"])
def test_a_captured_clip_in_place_follows_rows_off_the_boundaries(torch, kind, scale):
    wides, parts = zip(*[rows_of(torch, kind, first, seed=first) for first in (64, 61, 8, 3)])
    keeps = [w.clone() for w in wides]
    total = norm64(parts[:1]) / scale
    with GradientList([parts[0]]) as lst:
        g, r = captured(torch, lambda s: lst.clip(total / 2, loss_scale=scale, stream=s))
        for k in (1, 2, 3, 0):
            lst.bind([parts[k]])
            before = parts[k].clone()
            found = norm64([before]) / scale
            g.replay()
            torch.cuda.synchronize()
            near(r.read().norm, found, 4 * U, "norm")
            check_clipped(torch, [parts[k]], [before], total / 2 / found / scale)
            assert outside_kept(torch, wides[k], keeps[k], parts[k])


@pytest.mark.parametrize("out", ["bfloat16", "float32", "float16", "contiguous"])
@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_a_captured_clip_into_rows_follows_both_lists(torch, kind, out):
    ins = [rows_of(torch, kind, first, seed=first) for first in (64, 61)]
    outs = [rows_of(torch, "float32" if out == "contiguous" else out, first, seed=9)
            for first in (8, 5)]
    keeps = [w.clone() for w, _ in outs]
    targets = [p for _, p in outs]
    if out == "contiguous":
        room = torch.zeros(3000 * 256 + 8, device="cuda")
        targets = [room[a:a + 3000 * 256].view(3000, 256) for a in (0, 1)]
    with GradientList([ins[0][1]]) as lst, GradientList([targets[0]]) as to:
        g, _ = captured(torch, lambda s: lst.clip(0.25, loss_scale=8.0, out=to, stream=s))
        for i, o in ((1, 0), (0, 1), (1, 1), (0, 0)):
            lst.bind([ins[i][1]])
            to.bind([targets[o]])
            g.replay()
            torch.cuda.synchronize()
            found = norm64([ins[i][1]]) / 8.0
            check_clipped(torch, [targets[o]], [ins[i][1]], 0.25 / found / 8.0)
            if out != "contiguous":
                assert outside_kept(torch, outs[o][0], keeps[o], targets[o])


def test_calls_behind_a_replayed_bind_work_on_its_addresses(torch):
    wides, parts = zip(*[rows_of(torch, "bfloat16", first, seed=first) for first in (64, 61)])
    keeps = [w.clone() for w in wides]
    with GradientList([parts[0]]) as lst:
        g, _ = captured(torch, lambda s: lst.bind([parts[1]], stream=s))
        lst.bind([parts[0]])  # the host goes by this one
        g.replay()
        before = parts[1].clone()
        r = lst.clip(1.0, loss_scale=2.0)
        found = norm64([before]) / 2.0
        near(r.read().norm, found, 4 * U, "norm")
        check_clipped(torch, [parts[1]], [before], 1.0 / found / 2.0)
        assert torch.equal(wides[0], keeps[0])
        assert outside_kept(torch, wides[1], keeps[1], parts[1])


# ---- calls right behind a bind -----------------------------------------------------------
@pytest.mark.parametrize("sizes", [[3000, 33], [2_000_003, 70_001, 8192]], ids=["small", "large"])
def test_calls_right_behind_a_bind_read_the_new_addresses(torch, sizes):
    """No host synchronisation between binding and the calls, many times over."""
    sets = [make(torch, sizes, seed=20 + k, std=1e-2 * 2.0 ** k) for k in range(4)]
    wants = [norm64(s) for s in sets]
    flats = [torch.cat([t.float() for t in s]) for s in sets]
    n = sum(sizes)
    opts = StepOptions(one_based_update=3, max_grad_norm=1e6)
    with GradientList(sets[0]) as lst, B200Adamw(TensorTable.from_sizes(sizes)) as opt:
        room = -(-n // 4) * 4  # rows of the accumulators on 16-byte boundaries
        acc = [a[:n] for a in torch.empty(4, room, device="cuda")]
        for rep in range(20):
            norms = []
            for k in range(4):
                lst.bind(sets[k])
                norms.append(lst.norm())
                lst.bind(sets[(k + 1) % 4])
                lst.accumulate(acc[k], overwrite=True)
                lst.bind(sets[(k + 2) % 4])
                opt.norm_pass_accumulate(acc[k], lst, opts)
            for k in range(4):
                near(norms[k].read().norm, wants[k], 4 * U, "norm")
                assert torch.equal(acc[k], flats[(k + 1) % 4] + flats[(k + 2) % 4])


# ---- the update pass behind other work -----------------------------------------------------
def load(torch, opt, seed):
    st = synth.optimizer_state(opt.P, seed)
    opt.load_state(st["master"], st["moment"], st["variance"], st["bf16"])


def same_bits(torch, a, b):
    return all(torch.equal(a[k].view(torch.int16), b[k].view(torch.int16)) for k in a)


@pytest.mark.parametrize("form", ["list", "flat", "list accumulated", "flat accumulated"])
def test_an_update_pass_sees_what_ran_ahead_of_it(torch, form):
    """The norm pass, work on the state, then the update pass, without waiting in
    between, give what they give with a wait after each."""
    sizes = [2_000_003, 70_001, 8192]
    tensors = make(torch, sizes, ("float32",), seed=30)
    flat = torch.cat(tensors)
    opts = StepOptions(one_based_update=3, max_grad_norm=0.5)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        grads = lst if form.startswith("list") else flat
        start = torch.randn(opt.P, device="cuda")
        got = []
        for wait in (True, False, False, False):
            pause = torch.cuda.synchronize if wait else lambda: None
            load(torch, opt, 31)
            state, acc = opt.state_tensors(), start.clone()
            torch.cuda.synchronize()
            for k in range(8):
                if "accumulated" in form:
                    opt.norm_pass_accumulate(acc, grads, opts)
                else:
                    opt.norm_pass(grads, opts)
                pause()
                if k % 2:
                    state["moment"].mul_(0.5)
                    state["variance"].add_(1e-6)
                    pause()
                opt.update_pass(opts)
                pause()
            assert opt.read_result().skipped == 0
            got.append({k: v.clone() for k, v in state.items()})
        assert all(same_bits(torch, got[0], g) for g in got[1:])


@pytest.mark.parametrize("ahead", ["list", "flat", "list accumulated"])
@pytest.mark.parametrize("between", ["list step", "flat step", "uploaded step", "apply_update"])
def test_a_step_between_the_passes_ends_the_norm_pass(torch, ahead, between):
    """The decision of the norm pass is gone, so there is nothing to update by."""
    sizes = [70_001, 8192]
    tensors, other = (make(torch, sizes, ("float32",), seed=40 + k, std=1e-6) for k in (0, 1))
    opts = StepOptions(one_based_update=3)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst, \
            GradientList(other) as lst2:
        load(torch, opt, 41)
        if ahead == "list":
            opt.norm_pass(lst, opts)
        elif ahead == "flat":
            keep = opt.norm_pass(torch.cat(tensors), opts)
        else:
            opt.norm_pass_accumulate(torch.zeros(opt.P, device="cuda"), lst, opts)
        flat = torch.cat(other)
        if between == "list step":
            opt.step(lst2, opts)
        elif between == "flat step":
            opt.step(flat, opts)
        elif between == "uploaded step":
            opt.step_uploaded(opt.upload(flat.cpu().pin_memory()), opts)
        else:
            opt.apply_normalized_clipped_gradients(flat.cpu().numpy(), canonical_learning_rate(1), 1)
        with pytest.raises(SlmError) as e:
            opt.update_pass(opts)
        assert e.value.status == _lib.SLM_ERR_INVALID_ARGUMENT
        opt.norm_pass(lst, opts)  # and with one of its own it goes on
        opt.update_pass(opts)
        assert opt.read_result().skipped == 0


# ---- lists that end around captures --------------------------------------------------------
def test_a_list_collected_inside_a_capture_does_not_break_it(torch):
    tensors, other = make(torch, [70_001, 33], seed=50), make(torch, [5000], seed=51)
    with GradientList(tensors) as lst:
        spare = [GradientList(other), GradientList(other)]

        def call(s):
            r = lst.norm(stream=s)
            spare.pop()          # collected
            spare[0].close()
            lst.norm(stream=s)
            return r

        g, r = captured(torch, call)
        g.replay()
        torch.cuda.synchronize()
        near(r.read().norm, norm64(tensors), 4 * U, "norm")
        GradientList(other).close()
        near(lst.norm().read().norm, norm64(tensors), 4 * U, "norm")


def test_a_captured_update_pass_keeps_a_list_that_is_closed_ahead_of_it(torch):
    sizes = [70_001, 8192]
    tensors = make(torch, sizes, seed=52)
    opts = StepOptions(one_based_update=4, max_grad_norm=1e6)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        load(torch, opt, 53)
        opt.norm_pass(lst, opts)
        for _ in range(3):  # update passes by one decision, as the replays below
            opt.update_pass(opts)
            want = {k: v.clone() for k, v in opt.state_tensors().items()}
            opt.norm_pass(lst, opts)
        load(torch, opt, 53)
        gone = GradientList(tensors)
        opt.norm_pass(gone, opts)
        gone.close()
        g, _ = captured(torch, lambda s: opt.update_pass(opts, stream=s))
        for _ in range(3):
            g.replay()
        torch.cuda.synchronize()
        assert same_bits(torch, want, opt.state_tensors())
        opt.norm_pass(lst, opts)
        opt.update_pass(opts)
        assert opt.read_result().skipped == 0


# ---- the caller's context --------------------------------------------------------------------
@pytest.mark.parametrize("call", ["handle", "list"])
def test_calls_from_a_context_of_the_callers_own_run_in_the_primary_one(torch, call):
    """No kernel is launched here: copies of the loss scale, and the end of a list."""
    cuda = ctypes.CDLL("libcuda.so.1")

    def ok(status):
        assert status == 0, status

    with B200Adamw(TensorTable.from_sizes([100])) as opt, \
            GradientList([torch.ones(100, device="cuda")]) as lst:
        primary, own, now = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        torch.cuda.synchronize()
        ok(cuda.cuCtxGetCurrent(ctypes.byref(primary)))
        ok(cuda.cuCtxCreate_v2(ctypes.byref(own), 0, 0))
        try:
            ok(cuda.cuCtxGetCurrent(ctypes.byref(now)))
            assert now.value == own.value != primary.value
            if call == "handle":
                opt.set_loss_scale(512.0)
                assert opt.loss_scale() == (512.0, 0)
            else:
                handle, lst._h = lst._h, None
                assert lst.lib.slm_grad_list_destroy(handle) == _lib.SLM_OK
            ok(cuda.cuCtxGetCurrent(ctypes.byref(now)))
            assert now.value == primary.value
        finally:
            ok(cuda.cuCtxDestroy_v2(own))
            ok(cuda.cuCtxSetCurrent(primary))


# ---- gradients as large as the flat step takes them ------------------------------------------
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("accumulated", [False, True], ids=["step", "accumulated"])
@pytest.mark.parametrize("scale", [1.0, 1.5, 1024.0, 37888.0, 65536.0, 2.0 ** 20, 3e6])
def test_a_list_step_takes_large_gradients_as_the_flat_step(torch, scale, accumulated, kind):
    # the unscaled values' squares are f32 (up to 1e38), the stored ones' are not
    sizes = [4097, 33]
    scale = ctypes.c_float(scale).value
    tensors = make(torch, sizes, ("float32",), seed=60)
    for t in tensors:
        t.mul_(2.0 ** 20 * scale)
    tensors[0][5], tensors[1][32] = 3e18 * scale, -7e18 * scale
    tensors = [t.to(getattr(torch, kind)) for t in tensors]
    want = norm64(tensors) / scale
    opts = StepOptions(one_based_update=3, max_grad_norm=1.0, static_loss_scale=scale)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        load(torch, opt, 61)
        for grads in (torch.cat(tensors), lst):
            if accumulated:
                opt.norm_pass_accumulate(torch.empty(opt.P, device="cuda"), grads, opts,
                                         overwrite=True)
                opt.update_pass(opts)
                res = opt.read_result()
            else:
                res = opt.step(grads, opts)
            assert (res.skipped, res.nonfinite) == (0, 0)
            near(res.grad_norm, want, 4 * U, "norm")
        r = lst.norm(loss_scale=scale, per_tensor=True).values.tolist()
        near(r[0], want, 4 * U, "norm")
        assert r[3] == 0.0


@pytest.mark.parametrize("scale", [2.0 ** -149, 2.0 ** -127, 2.0 ** -126, 1.7 * 2.0 ** -126, 0.5,
                                   0.75, 1.0 - 2.0 ** -24, 1.0, 1.0 + 2.0 ** -23, 1.9, 2.0,
                                   1.5 * 2.0 ** 125, 2.0 ** 126, 1.5 * 2.0 ** 126, 2.0 ** 127,
                                   3.4e38])
def test_the_norm_at_any_loss_scale(torch, scale):
    """Unscaled values from 1 to 2, as far as the stored ones are normal numbers."""
    scale = ctypes.c_float(scale).value
    gen = torch.Generator("cuda").manual_seed(62)
    x = (torch.rand(20_001, generator=gen, device="cuda", dtype=torch.float64) + 1.0)
    x = (x * max(scale, 2.0 ** -126)).clamp(max=3.4e38).float()
    with GradientList([x]) as lst:
        r = lst.norm(loss_scale=scale, max_norm=3e38).values.tolist()
    near(r[0], norm64([x]) / scale, 4 * U, "norm")
    assert r[3] == 0.0


# ---- binds that fail -----------------------------------------------------------------------
def test_a_bind_that_fails_leaves_the_list_as_it_was(torch):
    """The launch is refused because a stream that the default stream waits for is
    being captured: an error from the runtime, nothing runs."""
    n = 4096
    old, new = torch.full((n,), 2.0, device="cuda"), torch.full((n,), 3.0, device="cuda")
    runtime = ctypes.CDLL("libcudart.so.12")
    blocking, graph = ctypes.c_void_p(), ctypes.c_void_p()
    with GradientList([old]) as lst:
        torch.cuda.synchronize()
        assert runtime.cudaStreamCreate(ctypes.byref(blocking)) == 0
        assert runtime.cudaStreamBeginCapture(blocking, 2) == 0  # relaxed
        with pytest.raises(SlmError) as e:
            lst.bind([new])
        assert e.value.status == _lib.SLM_ERR_CUDA
        runtime.cudaStreamEndCapture(blocking, ctypes.byref(graph))  # invalidated
        runtime.cudaGetLastError()
        assert runtime.cudaStreamDestroy(blocking) == 0
        assert lst.tensors == (old,)
        near(lst.norm().read().norm, 2.0 * math.sqrt(n), 4 * U, "norm")
        lst.accumulate(new)  # not one of the list's tensors
        torch.cuda.synchronize()
        assert bool((new == 5.0).all()) and bool((old == 2.0).all())
        lst.bind([new])
        near(lst.norm().read().norm, 5.0 * math.sqrt(n), 4 * U, "norm")


# ---- tensors between the rows of others ----------------------------------------------------
def test_tensors_between_the_rows_of_others_are_no_overlap(torch):
    w = torch.randn(64, 96, device="cuda")
    keep = w.clone()
    apart = [
        ([w[:, :40], w[5, 40:96]], None),                       # a run in one gap
        ([w[:, 32:64], w[0, :32], w[63, 64:]], None),           # ahead of, behind the rows
        ([w[::2, :40], w[:, 40:50], w[1::2, :40]], None),       # rows of two pitches
        ([w[:, :8], w[:4, 8:]], [w[:, :8], w[:4, 8:]]),
        ([w[:, :8]], [w[3, 40:40 + 8 * 5].new_empty(64, 8)]),
    ]
    for tensors, targets in apart:
        before = [t.clone() for t in tensors]
        found = norm64(before)
        with GradientList(tensors) as lst:
            to = GradientList(targets) if targets else None
            lst.clip(found / 2, out=to)
            check_clipped(torch, targets or tensors, before, 0.5)
            if to:
                to.close()
        inside = torch.zeros_like(w, dtype=torch.bool)
        for t in tensors:
            at = t.storage_offset()
            inside.view(-1).as_strided(t.shape, t.stride(), at).fill_(True)
        assert bool((w[~inside] == keep[~inside]).all())
        w.copy_(keep)
    with GradientList([w[:2, :4]]) as lst:  # an accumulator in the gap
        lst.accumulate(w[0, 8:16], overwrite=True)
        assert torch.equal(w[0, 8:16], w[:2, :4].reshape(-1))
    together = [[w[:, :40], w[5, 39:96]], [w[:, :40], w.view(-1)[5 * 96 + 50:6 * 96 + 1]],
                [w[::2, :40], w[:, 39:50]], [w[:, 32:64], w[0, :33]], [w[0], w[0, 5:6]],
                [w[:, :40], w[2:4].view(-1)]]
    for tensors in together:
        with GradientList(tensors) as lst, pytest.raises(SlmError):
            lst.clip(1.0)
    with GradientList([w[:2, :4]]) as lst, pytest.raises(SlmError):
        lst.accumulate(w.view(-1)[92:100])


# ---- tensors that a bind lets go -----------------------------------------------------------
@pytest.mark.parametrize("call", ["norm", "clip", "accumulate", "step"])
def test_tensors_let_go_by_a_bind_are_not_given_out_too_soon(torch, call):
    sizes = [2_000_003, 70_001]
    keep = make(torch, sizes, ("float32",), seed=70)
    new = make(torch, sizes, ("float32",), seed=71)
    want = norm64(keep)
    side = torch.cuda.Stream()
    acc = torch.zeros(sum(sizes), device="cuda")
    opts = StepOptions(one_based_update=3, max_grad_norm=1e6)
    out = [torch.empty_like(t) for t in keep]
    with GradientList(new) as lst, GradientList(out) as to, \
            B200Adamw(TensorTable.from_sizes(sizes)) as opt:
        load(torch, opt, 72)
        for _ in range(3):
            lst.bind([t.clone() for t in keep])
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                torch.cuda._sleep(BUSY)
            if call == "norm":
                r = lst.norm(stream=side)
            elif call == "clip":
                r = lst.clip(want / 2, out=to, stream=side)
            elif call == "accumulate":
                lst.accumulate(acc, overwrite=True, stream=side)
            else:
                opt.step(lst, opts, stream=side, wait=False)
            lst.bind(new, stream=side)
            junk = [torch.full((n,), 100.0, device="cuda") for n in sizes for _ in range(4)]
            torch.cuda.synchronize()
            del junk
            if call in ("norm", "clip"):
                near(r.read().norm, want, 4 * U, "norm")
            elif call == "accumulate":
                assert torch.equal(acc, torch.cat(keep))
            else:
                near(opt.read_result().grad_norm, want, 4 * U, "norm")


# ---- rows on the boundaries, and units beyond the smallest -----------------------------------
@pytest.mark.parametrize("rows", [3000, 40_000], ids=["0.8M", "10M"])
@pytest.mark.parametrize("scale", [1.0, 8.0])
@pytest.mark.parametrize("kind", ["bfloat16", "float32", "float16"])
def test_clip_of_rows_on_the_boundaries(torch, kind, scale, rows):
    """Beyond the lists that one cluster takes: in place, into rows of every type and
    into contiguous memory, with what lies beside the columns left as it was."""
    wide, part = rows_of(torch, kind, 64, rows=rows, seed=80)
    more = rows_of(torch, kind, 8, columns=64, rows=333, seed=81)[1]
    keep = wide.clone()
    before = [part.clone(), more.clone()]
    total = norm64(before) / scale
    for limit in (total / 3, total * 3):
        factor = min(1.0, limit / total)
        with GradientList([part, more]) as lst:
            for out in ("bfloat16", "float32", "float16"):
                room, target = rows_of(torch, out, 8, rows=rows, seed=82)
                room_keep = room.clone()
                flat = [torch.zeros(p.shape, device="cuda", dtype=room.dtype) for p in before]
                for targets in ([target, flat[1]], flat):
                    with GradientList(targets) as to:
                        r = lst.clip(limit, loss_scale=scale, out=to, per_tensor=rows > 3000)
                        near(r.read().norm, total, 4 * U, "norm")
                    check_clipped(torch, targets, before, factor / scale)
                assert outside_kept(torch, room, room_keep, target)
            r = lst.clip(limit, loss_scale=scale)
            near(r.read().norm, total, 4 * U, "norm")
            check_clipped(torch, [part, more], before, factor / scale)
            assert outside_kept(torch, wide, keep, part)
            if scale == 1.0 and limit > total:
                assert torch.equal(part, before[0])
        part.copy_(before[0]), more.copy_(before[1])


def test_units_beyond_the_smallest_over_mixed_layouts(torch):
    """141M elements (units of 16,384) in contiguous memory off the boundaries, rows with
    an odd pitch and rows on the boundaries: norm, clip, accumulate and the step."""
    gen = torch.Generator("cuda").manual_seed(90)

    def values(*shape, kind):
        return (1e-3 * torch.randn(shape, generator=gen, device="cuda")).to(kind)

    odd = values(30_000, 1003, kind=torch.float32)
    even = values(50_000, 1032, kind=torch.bfloat16)
    tensors = [values(60_000_002, kind=torch.bfloat16)[1:], odd[:, 1:1002], even[:, 8:],
               values(777, kind=torch.float16)]
    sizes = [t.numel() for t in tensors]
    n = sum(sizes)
    assert n // 8192 > 16384
    keeps = [odd.clone(), even.clone()]
    before = [t.clone() for t in tensors]
    flat = torch.cat([t.reshape(-1).float() for t in tensors])
    total = norm64(before)
    limit = ctypes.c_float(total / 2).value
    opts = StepOptions(learning_rate=3e-4, one_based_update=10, max_grad_norm=limit)
    decay = [True, False, True, False]
    with GradientList(tensors) as lst, B200Adamw(TensorTable.from_sizes(sizes, decay)) as opt:
        r = lst.norm(per_tensor=True)
        near(r.read().norm, total, 4 * U, "norm")
        for k, t in enumerate(before):
            near(float(r.tensor_norms[k]), norm64([t]), 4 * U, f"norm of tensor {k}")
            assert float(r.tensor_max[k]) == float(t.abs().max())
        acc = torch.randn(n, generator=gen, device="cuda")
        old = acc.clone()
        lst.accumulate(acc)
        assert torch.equal(acc, old + flat)
        lst.accumulate(acc, overwrite=True)
        assert torch.equal(acc, flat)
        opt.norm_pass_accumulate(acc, lst, opts)
        assert torch.equal(acc, flat + flat)
        near(opt.read_result().grad_norm, 2.0 * total, 4 * U, "accumulated norm")
        del acc, old
        state = opt.state_tensors()
        state["master"].copy_(0.02 * torch.randn(n, generator=gen, device="cuda"))
        state["moment"].copy_(1e-4 * torch.randn(n, generator=gen, device="cuda"))
        state["variance"].copy_((1e-3 * torch.randn(n, generator=gen, device="cuda")).square())
        state["bf16"].copy_(state["master"].bfloat16())
        start = {k: v.clone() for k, v in state.items()}
        res = opt.step(lst, opts)
        near(res.grad_norm, total, 4 * U, "norm of the step")
        check_state(torch, state, start, before, decay, opts, 1.0, 0.5)
        del start
        wide = torch.zeros(30_000, 1008, device="cuda")
        targets = [torch.empty(sizes[0], device="cuda", dtype=torch.float16), wide[:, 3:1004],
                   torch.empty(50_000, 1024, device="cuda"), torch.empty(777, device="cuda")]
        with GradientList(targets) as to:
            lst.clip(limit, out=to)
            check_clipped(torch, targets, before, 0.5)
        assert not bool(wide[:, :3].any()) and not bool(wide[:, 1004:].any())
        lst.clip(limit)
        check_clipped(torch, tensors, before, 0.5)
        assert outside_kept(torch, odd, keeps[0], tensors[1])
        assert outside_kept(torch, even, keeps[1], tensors[2])


def test_streams_of_the_callers_own_may_end_before_results_are_read(torch):
    tensors, new = make(torch, [70_001, 33], seed=100), make(torch, [70_001, 33], seed=101)
    want = norm64(tensors)
    acc = torch.zeros(70_034, device="cuda")
    runtime = ctypes.CDLL("libcudart.so.12")
    with GradientList(tensors) as lst:
        torch.cuda.synchronize()
        for k in range(3):
            own = ctypes.c_void_p()
            assert runtime.cudaStreamCreateWithFlags(ctypes.byref(own), 1) == 0  # non-blocking
            r = lst.norm(stream=own.value)
            lst.accumulate(acc, overwrite=True, stream=own.value)
            assert runtime.cudaStreamSynchronize(own) == 0
            assert runtime.cudaStreamDestroy(own) == 0
            near(r.read().norm, want, 4 * U, "norm")
            del r
            lst.bind(new)
            lst.bind(tensors)


@pytest.mark.parametrize("mode", [0, 1, 2], ids=["global", "thread", "relaxed"])
def test_a_list_destroyed_through_the_abi_inside_a_capture_lives_on(torch, mode):
    """The runtime refuses the wait (and ends the capture): an error, nothing runs."""
    tensors = make(torch, [70_001, 33], seed=110)
    runtime = ctypes.CDLL("libcudart.so.12")
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    with GradientList(tensors) as lst:
        torch.cuda.synchronize()
        assert runtime.cudaStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
        assert runtime.cudaStreamBeginCapture(stream, mode) == 0
        got = lst.lib.slm_grad_list_destroy(lst.handle)
        runtime.cudaStreamEndCapture(stream, ctypes.byref(graph))
        runtime.cudaGetLastError()
        assert runtime.cudaStreamDestroy(stream) == 0
        assert got == _lib.SLM_ERR_CUDA
        near(lst.norm().read().norm, norm64(tensors), 4 * U, "norm")
