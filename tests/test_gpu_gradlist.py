"""Gradient lists on the GPU: norm, clip, accumulate and step against plain
implementations in 64 bits, at the sizes, layouts, types and values where they
can go wrong.

Tolerances count roundings (u = 2^-24, half a step of f32):

* sum of squares: of the stored values, 4 fused multiply-adds
  and one add in f32 -> 5u; the f64 adds are negligible.  norm: half of that, and
  its own rounding -> 3.5u (checked with 4u; the flat norm rounds u = g / s too).
* clip scale: the sum rounded to f32 -> 6u, root 3u + 1u, quotient 1u -> 5u (5.5u).
* clipped value: clip 5, over the scale 1, product 1 -> 7u (7.5u), and the output type's
  half step (f32: that product's; bf16 2^-8 at most, f16 2^-11, and 2^-25
  absolute among f16's subnormals).
* moments: see check_state.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from slmopt import (B200Adamw, GqaDimensions, GradientList, SlmError, StepOptions, TensorTable,
                    _lib, synth)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def torch():
    import torch as _torch

    if not _torch.cuda.is_available():
        pytest.fail("a gpu-marked test ran without a CUDA device")
    return _torch


def kind_of(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


SIZES = {
    "one": [1],
    "below a vector": [7],
    "a vector": [8],
    "vector and one": [9],
    "nothing, little, nothing": [0, 5, 0],
    "half a unit": [4096],
    "half a unit and one": [4097],
    "a unit": [8192],
    "a unit and one": [8193],
    "units": [2048 * 256, 8191, 12288, 3],
    "odd": [70001, 33, 1, 1, 65537, 777],
    "many tiny": [1 + (7 * i) % 40 for i in range(500)],
    "larger units": [40_000_003, 11],
}


def make(torch, sizes, types, place, seed=0, std=1e-2):
    """Tensors of the sizes with the types cycled; place: separate, packed (back
    to back behind one odd element), columns (slices of wider matrices)."""
    gen = torch.Generator("cuda").manual_seed(1000 + seed)
    kinds = [kind_of(torch, types[i % len(types)]) for i in range(len(sizes))]

    def values(shape, k):
        return (std * torch.randn(shape, generator=gen, device="cuda")).to(k)

    if place == "separate":
        return [values((n,), k) for n, k in zip(sizes, kinds)]
    if place == "packed":
        out = []
        room = {k: values((1 + sum(n for n, q in zip(sizes, kinds) if q == k),), k)
                for k in set(kinds)}
        at = {k: 1 for k in room}
        for n, k in zip(sizes, kinds):
            out.append(room[k][at[k]:at[k] + n])
            at[k] += n
        return out
    out = []
    for i, (n, k) in enumerate(zip(sizes, kinds)):
        # the largest row count that divides n, at most 64
        rows = max(r for r in range(1, 65) if n % r == 0) if n else 1
        cols = n // rows
        wide = values((rows, cols + (8 if i % 2 else 5)), k)
        out.append(wide[:, :cols] if i % 3 else wide[:, 3:3 + cols])
    return out


def same(a, b):
    return a == b or (math.isnan(a) and math.isnan(b))


def near(got, want, tol, what):
    if not (same(got, want) or abs(got - want) <= tol * abs(want)):
        raise AssertionError(f"{what}: got {got!r} want {want!r}, off {abs(got - want):.3g}, "
                             f"allowed {tol * abs(want):.3g}")


def norms64(torch, tensors, scale, kind):
    each, tops = [], []
    for t in tensors:
        x = t.detach().double().reshape(-1) / float(np.float32(scale))
        if x.numel() == 0:
            each.append(0.0), tops.append(0.0)
            continue
        tops.append(float(x.abs().max()))
        each.append(tops[-1] if kind == "max" else float(x.square().sum().sqrt()))
    if any(math.isnan(v) for v in each + tops):
        total = top = math.nan
    else:
        top = max(tops)
        total = top if kind == "max" else math.sqrt(math.fsum(v * v for v in each))
    return total, top, each, tops


def check_norm(torch, got, tensors, scale, limit, kind="l2"):
    total, top, each, tops = norms64(torch, tensors, scale, kind)
    v = got.values.tolist()
    fine = math.isfinite(total) and math.isfinite(top)
    near(v[0], total, 4 * U, "norm")
    near(v[2], top, U, "largest")
    assert v[3] == (0.0 if fine else 1.0)
    clip = 0.0 if not fine else 1.0 if total <= limit else limit / total
    near(v[1], clip, 5.5 * U, "clip scale")
    assert v[1] <= 1.0
    if len(v) > 4:
        n = len(tensors)
        for k in range(n):
            near(v[4 + k], each[k], 4 * U, f"norm of tensor {k}")
            near(v[4 + n + k], tops[k], U, f"largest of tensor {k}")
    if kind == "l2" and fine:
        near(float(got.sum_squares), total * total, 7 * U, "sum of squares")
    return v


# ---- norm ------------------------------------------------------------------------
@pytest.mark.parametrize("place", ["separate", "packed", "columns"])
@pytest.mark.parametrize("types", [["f32"], ["bf16"], ["f16"], TYPES], ids="-".join)
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_norm(torch, sizes, types, place):
    tensors = make(torch, sizes, types, place)
    with GradientList(tensors) as lst:
        assert len(lst) == len(sizes) and lst.elements == sum(sizes)
        check_norm(torch, lst.norm(max_norm=0.3, per_tensor=True), tensors, 1.0, 0.3)
        check_norm(torch, lst.norm(loss_scale=1000.0), tensors, 1000.0, 1.0)
        check_norm(torch, lst.norm(loss_scale=0.25, max_norm=1e-3, kind="max", per_tensor=True),
                   tensors, 0.25, 1e-3, "max")


def tree_sum(pieces, unit):
    """The documented tree, restated: per unit 256 lanes of 8-element vectors (two
    runs of 4 fused multiply-adds in f32, whose f64 product is exact, added in f32),
    f64 lane sums, halving folds; then 1,024 lanes over units."""
    parts = []
    for x in pieces:
        for a in range(0, x.size, unit):
            part = x[a:a + unit].astype(np.float32)
            rows = -(-part.size // 2048)
            q = np.zeros(rows * 2048)
            q[:part.size] = part.astype(np.float64) ** 2
            q = q.reshape(rows, 256, 2, 4)
            s = q[..., 0].astype(np.float32)
            for j in (1, 2, 3):
                s = (s + q[..., j]).astype(np.float32)
            p = s[..., 0] + s[..., 1]
            lanes = np.zeros(256)
            for r in range(rows):
                lanes = lanes + p[r].astype(np.float64)
            parts.append(fold(lanes))
    lanes = np.zeros(1024)
    for a in range(0, len(parts), 1024):
        row = np.zeros(1024)
        row[:len(parts[a:a + 1024])] = parts[a:a + 1024]
        lanes = lanes + row
    return fold(lanes)


def fold(lanes):
    w = lanes.reshape(-1, 32)
    for off in (16, 8, 4, 2, 1):
        w = w.copy()
        w[:, :off] = w[:, :off] + w[:, off:2 * off]
    s = w[:, 0].copy()
    off = s.size // 2
    while off:
        s[:off] = s[:off] + s[off:2 * off]
        off //= 2
    return s[0]


@pytest.mark.parametrize("place", ["separate", "packed", "columns"])
@pytest.mark.parametrize("sizes", [SIZES["odd"], SIZES["units"], SIZES["many tiny"]],
                         ids=["odd", "units", "many tiny"])
def test_norm_is_the_documented_tree_whatever_the_layout(torch, sizes, place):
    tensors = make(torch, sizes, ["bf16", "f32"], place)
    want = tree_sum([t.float().reshape(-1).cpu().numpy() for t in tensors], 8192)
    with GradientList(tensors) as lst:
        first = lst.norm()
        assert float(first.sum_squares) == want
        for _ in range(3):  # and the same bits run to run
            assert float(lst.norm().sum_squares) == want


@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("place", ["separate", "packed"])
def test_norm_flags_what_is_not_finite(torch, name, value, kind, place):
    tensors = make(torch, [70001, 33, 8192], [name], place)
    for k, i in ((0, 0), (0, 70000), (1, 32), (2, 4096)):
        keep = tensors[k][i].clone()
        with GradientList(tensors) as lst:
            check_norm(torch, lst.norm(kind=kind, per_tensor=True), tensors, 1.0, 1.0, kind)
            tensors[k][i] = value
            v = lst.norm(kind=kind, per_tensor=True).values.tolist()
            assert v[1] == 0.0 and v[3] == 1.0 and not math.isfinite(v[0])
            for j in range(3):  # only the tensor that holds it
                assert math.isfinite(v[4 + j]) == (j != k)
                assert math.isfinite(v[4 + 3 + j]) == (j != k)
        tensors[k][i] = keep


def test_norm_of_zeros_and_of_nothing(torch):
    zeros = [torch.zeros(5000, device="cuda"), torch.zeros(0, device="cuda")]
    for tensors in (zeros, zeros[1:]):
        with GradientList(tensors) as lst:
            assert lst.norm(per_tensor=True).values.tolist() == \
                [0.0, 1.0, 0.0, 0.0] + [0.0] * (2 * len(tensors))
            lst.clip()


def test_accumulate_of_nothing(torch):
    with GradientList([torch.zeros(0, device="cuda"), torch.zeros(0, 4, device="cuda")]) as lst:
        lst.accumulate(torch.zeros(0, device="cuda"))
        lst.accumulate(torch.zeros(0, device="cuda"), overwrite=True)
        with pytest.raises(ValueError):
            lst.accumulate(torch.zeros(1, device="cuda"))
    with GradientList([torch.zeros(3, device="cuda")]) as lst:
        with pytest.raises(SlmError):  # elements, but no accumulator
            _lib.check(lst.lib.slm_grad_list_accumulate(lst.handle, None, 3, 0, None))
    torch.cuda.synchronize()


def test_squares_that_overflow_count_as_non_finite(torch):
    with GradientList([torch.full((100,), 1e20, device="cuda")]) as lst:
        v = lst.norm().values.tolist()
        assert v[1] == 0.0 and v[3] == 1.0
        v = lst.norm(kind="max").values.tolist()  # no square is formed for this one
        near(v[0], float(np.float32(1e20)), 0, "max norm")
        assert v[3] == 0.0
    # unscaling can overflow by itself
    with GradientList([torch.full((100,), 1e38, device="cuda")]) as lst:
        assert lst.norm(kind="max", loss_scale=2.0 ** -10).values.tolist()[3] == 1.0


def test_subnormal_gradients_and_scales(torch):
    x = (torch.arange(1, 4001, device="cuda") * 2.0 ** -140).float()
    with GradientList([x]) as lst:
        v = lst.norm(kind="max", loss_scale=2.0 ** -100).values.tolist()
        near(v[0], 4000 * 2.0 ** -40, U, "max norm")
        v = lst.norm(loss_scale=2.0 ** -100).values.tolist()
        near(v[0], math.sqrt(sum(k * k for k in range(1, 4001))) * 2.0 ** -40, 4 * U, "norm")
    h = torch.full((4097,), 2.0 ** -24, device="cuda", dtype=torch.float16)
    with GradientList([h]) as lst:
        near(lst.norm().read().norm, math.sqrt(4097) * 2.0 ** -24, 4 * U, "f16 subnormals")


# ---- clip ------------------------------------------------------------------------
def half_step(torch, kind):
    return {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[kind]


def check_clipped(torch, got, before, scale, clip):
    for k, (y, x) in enumerate(zip(got, before)):
        y = y.reshape(-1)
        want = x.double().reshape(-1) / float(np.float32(scale)) * clip
        tol = (7.5 * U + half_step(torch, y.dtype)) * want.abs()
        if y.dtype == torch.float16:
            tol += 2.0 ** -25
            assert float(want.abs().max() if want.numel() else 0) < 65504
        off = (y.double() - want).abs()
        assert bool((off <= tol).all()), f"tensor {k}: {float((off - tol).max())} too far"


@pytest.mark.parametrize("place", ["separate", "packed", "columns"])
@pytest.mark.parametrize("out", TYPES + ["itself"])
@pytest.mark.parametrize("types", [["f32"], ["bf16"], ["f16"], TYPES], ids="-".join)
@pytest.mark.parametrize("sizes", [SIZES[k] for k in ("one", "vector and one",
                                                      "nothing, little, nothing", "odd", "units",
                                                      "many tiny", "larger units")],
                         ids=["one", "vector and one", "nothing", "odd", "units", "many tiny",
                              "larger"])
def test_clip(torch, sizes, types, out, place):
    tensors = make(torch, sizes, types, place, seed=3)
    before = [t.clone() for t in tensors]
    total = norms64(torch, before, 8.0, "l2")[0]
    for limit in (total / 3, total * 3):  # clipped, and below the limit
        for t, b in zip(tensors, before):
            t.copy_(b)
        with GradientList(tensors) as lst:
            if out == "itself":
                r = lst.clip(limit, loss_scale=8.0, per_tensor=True)
                got = tensors
            else:
                targets = make(torch, sizes, [out], "columns" if place == "packed" else "separate",
                               seed=4)
                with GradientList(targets) as to:
                    r = lst.clip(limit, loss_scale=8.0, out=to, per_tensor=True)
                    r.read()
                for t, b in zip(tensors, before):
                    assert bool((t == b).all())
                got = targets
            v = check_norm(torch, r, before, 8.0, limit)
            check_clipped(torch, got, before, 8.0, 1.0 if limit > total else limit / total)
            assert (v[1] == 1.0) == (limit > total)


@pytest.mark.parametrize("scale", [1.0, 37888.0, 1000.0, 2.0 ** -3, 3e-3])
def test_clip_with_other_scales_and_the_max_norm(torch, scale):
    tensors = make(torch, [70001, 4096], ["f32", "bf16"], "separate", seed=5)
    before = [t.clone() for t in tensors]
    top = norms64(torch, before, scale, "max")[0]
    limit = float(np.float32(top / 2))
    targets = [torch.empty_like(t, dtype=torch.float32) for t in tensors]
    with GradientList(tensors) as lst, GradientList(targets) as to:
        r = lst.clip(limit, loss_scale=scale, kind="max", out=to)
        check_norm(torch, r, before, scale, limit, "max")
        check_clipped(torch, targets, before, scale, limit / top)


@pytest.mark.parametrize("scale, std", [(1e-38, 1e-37), (2.0 ** -140, 2.0 ** -138), (1e38, 1e36),
                                        (2.0 ** 127, 2.0 ** 120), (2.0 ** 20, 1e4),
                                        (1.5 * 2.0 ** 20, 1e4), (0.99, 1e-2), (3e38, 1e37)])
def test_extreme_loss_scales(torch, scale, std):
    # the stored values, their quotients and the clipped values are all normal f32
    gen = torch.Generator("cuda").manual_seed(9)
    x = torch.rand(50_001, generator=gen, device="cuda", dtype=torch.float64) + 0.5
    x = (x * (torch.arange(50_001, device="cuda") % 2 * 2 - 1) * std).float()
    total = norms64(torch, [x], scale, "l2")[0]
    top = norms64(torch, [x], scale, "max")[0]
    # the quantised values of a subnormal scale: it is the f32 that counts
    for kind, found in (("l2", total), ("max", top)):
        for part in (0.5, 2.0):
            limit = float(np.float32(found * part))
            y = torch.empty_like(x)
            with GradientList([x]) as lst, GradientList([y]) as to:
                r = lst.clip(limit, loss_scale=scale, kind=kind, out=to)
                check_norm(torch, r, [x], scale, limit, kind)
                check_clipped(torch, [y], [x], scale, min(1.0, limit / found))


LIMITS = [n * 8192 + d for n in (40, 80, 192, 1024) for d in (-1, 0, 1)]


@pytest.mark.parametrize("n", LIMITS)
def test_around_the_sizes_where_the_form_changes(torch, n):
    sizes = [n - 3 * 8192, 8192, 8192, 8192] if n % 8192 else [n]
    tensors = make(torch, sizes, ["bf16", "f32"], "separate", seed=14)
    before = [t.clone() for t in tensors]
    want = tree_sum([t.float().cpu().numpy() for t in tensors], 8192)
    total = norms64(torch, tensors, 1.0, "l2")[0]
    targets = [torch.empty_like(t, dtype=torch.float16) for t in tensors]
    with GradientList(tensors) as lst, GradientList(targets) as to, \
            B200Adamw(TensorTable.from_sizes(sizes)) as opt:
        assert float(lst.norm().sum_squares) == want
        check_norm(torch, lst.norm(per_tensor=True), before, 1.0, 1.0)
        for per_tensor in (True, False):
            r = lst.clip(total / 2, out=to, per_tensor=per_tensor)
            assert float(r.sum_squares) == want
            check_norm(torch, r, before, 1.0, total / 2)
            check_clipped(torch, targets, before, 1.0, 0.5)
        start = load(torch, opt, 15)
        opts = StepOptions(one_based_update=10, max_grad_norm=float(np.float32(total / 2)))
        assert opt.step(lst, opts).sum_squares == want
        check_state(torch, opt.state_tensors(), start, before, [True] * len(sizes), opts, 1.0, 0.5)
        r = lst.clip(total / 2)
        assert float(r.sum_squares) == want
        check_clipped(torch, tensors, before, 1.0, 0.5)


def test_values_around_a_clipped_tensor_stay(torch):
    wide = torch.randn(64, 100, device="cuda")
    bucket = torch.randn(5001, device="cuda", dtype=torch.bfloat16)
    keep, keep_bucket = wide.clone(), bucket.clone()
    with GradientList([wide[:, 30:61], bucket[7:4990]]) as lst:
        lst.clip(0.5)
        torch.cuda.synchronize()
    inside = torch.zeros_like(wide, dtype=torch.bool)
    inside[:, 30:61] = True
    assert bool((wide[~inside] == keep[~inside]).all()) and bool((wide != keep)[inside].any())
    assert bool((bucket[:7] == keep_bucket[:7]).all())
    assert bool((bucket[4990:] == keep_bucket[4990:]).all())


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_clip_writes_nothing_when_a_gradient_is_not_finite(torch, value):
    tensors = make(torch, [9000, 77], ["bf16", "f32"], "separate", seed=6)
    tensors[1][76] = value
    before = [t.clone() for t in tensors]
    targets = [torch.full_like(t, 3.0) for t in tensors]
    with GradientList(tensors) as lst, GradientList(targets) as to:
        assert lst.clip(1e-3, out=to).read().nonfinite == 1.0
        assert all(bool((t == 3.0).all()) for t in targets)
        assert lst.clip(1e-3).read().clip_scale == 0.0
        for t, b in zip(tensors, before):
            assert torch.equal(t.view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32),
                               b.view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32))


def test_clip_below_the_limit_in_place_changes_no_bit(torch):
    # -0.0 and subnormals survive
    x = torch.tensor([-0.0, 0.0, 1e-40, -1e-3], device="cuda").repeat(3000)
    keep = x.clone()
    with GradientList([x]) as lst:
        assert lst.clip(1e3).read().clip_scale == 1.0
    assert torch.equal(x.view(torch.int32), keep.view(torch.int32))


def test_clip_refuses_outputs_that_share_elements(torch):
    a = torch.ones(1000, device="cuda")
    w = torch.ones(10, 64, device="cuda")
    refused = [
        ([a, a], None),                       # the same tensor twice
        ([a[:600], a[500:]], None),           # overlapping pieces
        ([w[:, :40], w[:, 30:]], None),       # overlapping columns
        ([a[:500]], [a[100:600]]),            # onto other gradients
        ([a[:500], a[500:]], [a[500:], a[:500]]),
        ([a], [torch.ones(999, device="cuda")]),
        ([a], [a[:500], a[500:]]),
        ([w[:6, :4]], [w[:4, :6]]),           # as many elements from the same one on, other rows
        ([w[:, :30]], [w[:, 1:31]]),
    ]
    for tensors, targets in refused:
        with GradientList(tensors) as lst:
            lst.norm()  # reading them is fine
            to = GradientList(targets) if targets else None
            with pytest.raises(SlmError) as e:
                lst.clip(1.0, out=to)
            assert e.value.status == _lib.SLM_ERR_INVALID_ARGUMENT
            if to:
                to.close()
    torch.cuda.synchronize()
    assert bool((a == 1).all()) and bool((w == 1).all())
    # neighbours are no overlap, nor is a list as its own output
    with GradientList([w[:, :40], w[:, 40:], a[:500], a[500:]]) as lst:
        lst.clip(1.0)
        with GradientList([w[:, :40], w[:, 40:], a[:500], a[500:]]) as again:
            lst.clip(0.5, out=again)
    total = math.sqrt(640 + 1000)
    near(float(a[3]), 0.5 / total, 24 * U, "clipped twice")


# ---- accumulate ------------------------------------------------------------------
@pytest.mark.parametrize("place", ["separate", "packed", "columns"])
@pytest.mark.parametrize("types", [["f32"], ["bf16"], ["f16"], TYPES], ids="-".join)
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_accumulate(torch, sizes, types, place):
    tensors = make(torch, sizes, types, place, seed=7)
    n = sum(sizes)
    flat = torch.cat([t.reshape(-1).float() for t in tensors])
    room = torch.full((n + 64,), 7.0, device="cuda")
    acc = room[:n]
    with GradientList(tensors) as lst:
        lst.accumulate(acc, overwrite=True)
        assert torch.equal(acc, flat)
        other = torch.randn(n, device="cuda")
        acc.copy_(other)
        lst.accumulate(acc)
        assert torch.equal(acc, other + flat)
    assert bool((room[n:] == 7.0).all())


def test_accumulate_refusals(torch):
    g = torch.ones(100, device="cuda")
    with GradientList([g]) as lst:
        for bad in (torch.zeros(99, device="cuda"), torch.zeros(100, device="cuda").bfloat16(),
                    torch.zeros(100), torch.zeros(200, device="cuda")[::2]):
            with pytest.raises(ValueError):
                lst.accumulate(bad)
        for bad in (torch.zeros(101, device="cuda")[1:], g):  # misaligned, the gradient itself
            with pytest.raises(SlmError):
                lst.accumulate(bad)


# ---- the step ----------------------------------------------------------------------
def load(torch, opt, seed):
    st = synth.optimizer_state(opt.P, seed)
    opt.load_state(st["master"], st["moment"], st["variance"], st["bf16"])
    return {k: v.clone() for k, v in opt.state_tensors().items()}


def check_state(torch, got, before, grads, decay, opts, scale, clip):
    """The state against 64 bits.  Gradient g' = fl(fl(g/s) * clip): 7.5u.  m': the
    products 1u each (g' carried: 8.5u), the sum 1u.  v': (1-b2) g' g' 2u + 15u,
    the sum 1u.  master is checked from the stored m', v': quotients 1u each,
    root half of its argument's and 1u, eps added 1u, quotient 1u: 5u on the
    step, decay product 1u, their sum 1u, lr product 1u, the difference 1u."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    b1, b2, lr, eps = f(opts.beta1), f(opts.beta2), f(opts.learning_rate), f(opts.epsilon)
    t = opts.one_based_update

    def power(b):  # f32 square-and-multiply, as the library
        r, x, k = np.float32(1), np.float32(b), t
        while k:
            if k & 1:
                r = np.float32(r * x)
            x, k = np.float32(x * x), k >> 1
        return float(r)

    c1, c2 = f(1 - np.float32(power(b1))), f(1 - np.float32(power(b2)))
    g = torch.cat([x.double().reshape(-1) for x in grads]) / f(scale) * clip
    m0, v0, w0 = (before[k].double() for k in ("moment", "variance", "master"))
    m1, v1, w1 = (got[k].double() for k in ("moment", "variance", "master"))
    # 2^-149: the step of f32's subnormals, which products of tiny values round to
    off = (m1 - (b1 * m0 + (1 - b1) * g)).abs()
    assert bool((off <= U * (2 * (b1 * m0).abs() + 9.5 * ((1 - b1) * g).abs()) + 2.0 ** -148).all())
    off = (v1 - (b2 * v0 + (1 - b2) * g * g)).abs()
    assert bool((off <= U * (2 * b2 * v0 + 18 * (1 - b2) * g * g) + 2.0 ** -148).all())
    wd = torch.cat([torch.full((x.numel(),), f(opts.decay_weight) if d else f(opts.no_decay_weight),
                               device="cuda", dtype=torch.float64) for x, d in zip(grads, decay)])
    move = m1 / c1 / ((v1 / c2).sqrt() + eps)
    want = w0 - lr * (move + wd * w0)
    allowed = U * (want.abs() + lr * (7 * move.abs() + 3 * (wd * w0).abs())) + 2.0 ** -148
    assert bool(((w1 - want).abs() <= allowed).all())
    assert torch.equal(got["bf16"].view(torch.int16), got["master"].bfloat16().view(torch.int16))


STEP_SIZES = {k: SIZES[k] for k in SIZES if 0 not in SIZES[k]}
STEP_SIZES["tiles"] = [2048 * 9, 2048 * 3 + 1024, 768, 4096 * 2, 2047]
STEP_SIZES["thousands of one"] = [1] * 3000 + [5000]


@pytest.mark.parametrize("place", ["separate", "packed", "columns"])
@pytest.mark.parametrize("types", [["f32"], ["bf16"], ["f16"], TYPES], ids="-".join)
@pytest.mark.parametrize("sizes", STEP_SIZES.values(), ids=STEP_SIZES.keys())
def test_step(torch, sizes, types, place):
    if sum(sizes) > 10_000_000 and place != "separate":
        sizes = [n // 8 for n in sizes if n > 8]
    tensors = make(torch, sizes, types, place, seed=8)
    decay = [i % 3 != 1 for i in range(len(sizes))]
    total = norms64(torch, tensors, 16.0, "l2")[0]
    with B200Adamw(TensorTable.from_sizes(sizes, decay)) as opt, GradientList(tensors) as lst:
        for limit, scale in ((float(np.float32(total / 3)), 16.0), (1e4, 1000.0)):
            before = load(torch, opt, 9)
            opts = StepOptions(learning_rate=3e-4, one_based_update=10, max_grad_norm=limit,
                               static_loss_scale=scale)
            res = opt.step(lst, opts)
            assert res.skipped == 0 and res.nonfinite == 0
            want = norms64(torch, tensors, scale, "l2")[0]
            near(res.grad_norm, want, 4 * U, "norm")
            clip = min(1.0, limit / want)
            near(res.clip_scale, clip, 5.5 * U, "clip")
            check_state(torch, opt.state_tensors(), before, tensors, decay, opts, scale, clip)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", STEP_SIZES.values(), ids=STEP_SIZES.keys())
def test_step_below_the_limit_is_the_flat_step_bit_for_bit(torch, sizes, dtype):
    tensors = make(torch, sizes, [dtype], "separate", seed=10)
    flat = torch.cat(tensors)
    opts = StepOptions(one_based_update=3, max_grad_norm=1e6, static_loss_scale=1000.0)
    got = []
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        for grads in (flat, lst):
            load(torch, opt, 11)
            assert opt.step(grads, opts).clip_scale == 1.0
            got.append({k: v.clone() for k, v in opt.state_tensors().items()})
        assert int(opt.read_result().status) == 0
    for k in got[0]:
        assert torch.equal(got[0][k].view(torch.int16), got[1][k].view(torch.int16)), k


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("place", ["separate", "columns"])
def test_step_skips_and_halves_the_scale(torch, value, place):
    sizes = [70001, 33, 8192]
    tensors = make(torch, sizes, ["bf16", "f16"], place, seed=12)
    opts = StepOptions(loss_scale_mode=_lib.SCALE_DYNAMIC, growth_interval=2)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        before = load(torch, opt, 13)
        opt.set_loss_scale(1024.0)
        where = tensors[0].view(-1) if tensors[0].is_contiguous() else tensors[0][-1]
        keep = where[-1].clone()
        where[-1] = value
        res = opt.step(lst, opts)
        assert res.skipped == 1 and res.nonfinite == 1 and res.clip_scale == 0.0
        assert opt.loss_scale() == (512.0, 0)
        for k, v in opt.state_tensors().items():
            assert torch.equal(v.view(torch.int16), before[k].view(torch.int16)), k
        with pytest.raises(SlmError) as e:
            opt.step(lst, StepOptions(nonfinite_policy=_lib.NONFINITE_ERROR))
        assert e.value.status == _lib.SLM_ERR_MODEL_GRADIENT_NONFINITE
        where[-1] = keep
        for want in ((512.0, 1), (1024.0, 0)):
            res = opt.step(lst, opts)
            assert res.skipped == 0 and res.loss_scale_used == 512.0
            assert opt.loss_scale() == want


def test_step_refusals(torch):
    a, b = torch.zeros(100, device="cuda"), torch.zeros(20, device="cuda")
    with B200Adamw(TensorTable.from_sizes([100, 20])) as opt:
        for tensors in ([b, a], [a], [a, b, b], [torch.zeros(120, device="cuda")]):
            with GradientList(tensors) as lst:
                for call in (lambda: opt.step(lst), lambda: opt.norm_pass(lst),
                             lambda: opt.norm_pass_accumulate(torch.zeros(120, device="cuda"), lst)):
                    with pytest.raises(SlmError) as e:
                        call()
                    assert e.value.code == "E1_PARAMETER_LAYOUT_MISMATCH"
        with pytest.raises(SlmError):
            opt.update_pass()
        with GradientList([a, b]) as lst:
            with pytest.raises(SlmError) as e:
                opt.step(lst, StepOptions(one_based_update=0))
            assert e.value.code == "MODEL_OPTIMIZER_INPUT_INVALID"
            opt.norm_pass(lst)
        lst2 = GradientList([a, b])
        lst2.close()
        with pytest.raises(ValueError):
            opt.step(lst2)


def test_list_refusals(torch):
    a = torch.zeros(100, device="cuda")
    with pytest.raises(TypeError):
        GradientList([a, a.double()])
    with pytest.raises(ValueError):
        GradientList([a, torch.zeros(3)])
    with pytest.raises(ValueError):
        GradientList([a, torch.zeros(6, 10, device="cuda").t()])
    with GradientList([a]) as lst:
        with pytest.raises(ValueError):
            lst.norm(kind="l1")
        for kw in (dict(loss_scale=0.0), dict(loss_scale=math.inf), dict(max_norm=0.0),
                   dict(max_norm=math.nan), dict(max_norm=-1.0)):
            with pytest.raises(SlmError):
                lst.norm(**kw)
            with pytest.raises(SlmError):
                lst.clip(**kw)
        with pytest.raises(ValueError):
            lst.bind([torch.zeros(99, device="cuda")])
        with pytest.raises(ValueError):
            lst.norm().tensor_norms
    # an address that is no device memory, through the C ABI
    import ctypes

    host = np.zeros(64, np.float32)
    pinned = torch.zeros(64).pin_memory()
    for address in (host.ctypes.data, pinned.data_ptr(), None, a.data_ptr() + 2):
        v = (_lib.GradView * 1)()
        v[0].data, v[0].rows, v[0].columns, v[0].row_stride = address, 1, 16, 16
        h = ctypes.c_void_p()
        got = _lib.load().slm_grad_list_create(v, 1, 0, ctypes.byref(h))
        assert got == _lib.SLM_ERR_INVALID_ARGUMENT and not h.value
    # a workspace that is too small or misaligned
    with GradientList([a]) as lst:
        lib, out = _lib.load(), torch.zeros(64, device="cuda")
        need = lib.slm_grad_list_workspace_bytes(lst.handle)
        ws = torch.zeros(need + 64, dtype=torch.uint8, device="cuda")
        for ptr, size in ((ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
            got = lib.slm_grad_list_norm(lst.handle, 1.0, 1.0, 0, out.data_ptr(), None, None, None,
                                         ptr, size, None)
            assert got == _lib.SLM_ERR_INVALID_ARGUMENT


# ---- a run of them together --------------------------------------------------------
@pytest.mark.parametrize("form", ["step", "passes", "accumulated"])
def test_an_update_as_it_is_used(torch, form):
    """Micro-batches of a small model's tensors, accumulated or stepped on, give
    the flat path's state, update after update."""
    table = TensorTable.from_dimensions(GqaDimensions.from_model_json(
        {"vocab_size": 257, "d_model": 64, "d_ff": 160, "n_layers": 2, "n_heads": 4,
         "n_kv_heads": 2, "tie_embeddings": False}))
    P = table.parameter_count
    with B200Adamw(table) as one, B200Adamw(table) as two:
        for opt in (one, two):
            load(torch, opt, 20)
        acc1, acc2 = (torch.empty(P, device="cuda") for _ in range(2))
        lst = None
        for t in (1, 2, 3):
            micro = [[x.view(s) for x, s in zip(make(torch, table.elements, ["bf16"], "separate",
                                                     seed=100 * t + i), table.shapes)]
                     for i in range(3)]
            opts = StepOptions(one_based_update=t, max_grad_norm=1e6, static_loss_scale=37888.0)
            if form == "accumulated":
                for i, tensors in enumerate(micro):
                    flat = torch.cat([x.reshape(-1) for x in tensors])
                    if lst is None:
                        lst = GradientList(tensors)
                    else:
                        lst.bind(tensors)
                    if i < 2:
                        one.accumulate(acc1, flat, overwrite=i == 0)
                        two.accumulate(acc2, lst, overwrite=i == 0)
                    else:
                        one.norm_pass_accumulate(acc1, flat, opts)
                        two.norm_pass_accumulate(acc2, lst, opts)
                        assert torch.equal(acc1, acc2)
                        one.update_pass(opts)
                        two.update_pass(opts)
            else:
                flat = torch.cat([x.reshape(-1) for x in micro[0]])
                one.step(flat, opts)
                if lst is None:
                    lst = GradientList(micro[0])
                else:
                    lst.bind(micro[0])
                if form == "step":
                    two.step(lst, opts, wait=False)
                else:
                    two.norm_pass(lst, opts)
                    two.update_pass(opts)
            a, b = one.read_result(), two.read_result()
            # The list's sum is within 5u, its norm within 2.5u; the flat norm also
            # rounds each quotient (2u of a square): 4 + 2u on the sum, 3u.
            near(b.grad_norm, a.grad_norm, 5.5 * U, "norm of the two trees")
            assert a.clip_scale == b.clip_scale == 1.0
        assert one.state_sha256() == two.state_sha256()


def test_accumulated_and_clipped_update(torch):
    sizes = [70001, 33, 8192, 5]
    decay = [True, False, True, False]
    micro = [make(torch, sizes, TYPES, place, seed=30 + i)
             for i, place in enumerate(("separate", "packed", "columns"))]
    lists = [GradientList(m) for m in micro]
    total = sum(torch.cat([x.double().reshape(-1) for x in m]) for m in micro)
    limit = float(np.float32(float(total.square().sum().sqrt()) / 5.0 / 16.0))
    opts = StepOptions(one_based_update=2, max_grad_norm=limit, static_loss_scale=16.0)
    with B200Adamw(TensorTable.from_sizes(sizes, decay)) as opt:
        before = load(torch, opt, 31)
        acc = torch.empty(opt.P, device="cuda")
        opt.accumulate(acc, lists[0], overwrite=True)
        opt.accumulate(acc, lists[1])
        opt.norm_pass_accumulate(acc, lists[2], opts)
        opt.update_pass(opts)
        res = opt.read_result()
        # from the f32 sums that the passes left: the rest is rounding of this pass alone
        sums = acc.double()
        assert bool(((sums - total).abs() <= 3 * U * sum(
            torch.cat([x.double().reshape(-1) for x in m]).abs() for m in micro)).all())
        norm = float((sums / 16.0).square().sum().sqrt())
        near(res.grad_norm, norm, 4 * U, "norm")
        near(res.clip_scale, limit / norm, 5.5 * U, "clip")
        check_state(torch, opt.state_tensors(), before, list(acc.split(sizes)), decay, opts, 16.0,
                    limit / norm)
    for lst in lists:
        lst.close()


def test_the_trainer_takes_lists(torch):
    from slmopt import trainer as tr

    table = TensorTable.from_sizes([40000, 77, 128 * 65], [True, False, True])
    with B200Adamw(table) as one, B200Adamw(table) as two:
        shas = []
        for opt, as_list in ((one, False), (two, True)):
            load(torch, opt, 40)
            run = tr.B200Trainer(opt)
            cursor = 0
            for t in range(2):
                for i in range(4):
                    tensors = make(torch, table.elements, ["f32"], "separate", seed=50 + 4 * t + i)
                    if as_list:
                        with GradientList(tensors) as lst:
                            ev = run.process_batch(cursor, 16_384, 1.0, lst)
                    else:
                        ev = run.process_batch(cursor, 16_384, 1.0, torch.cat(tensors))
                    cursor += 16_384
            shas.append(ev.update_state_sha256)
        assert shas[0] == shas[1]


# ---- rows with a pitch -----------------------------------------------------------
# (rows, columns, row stride, first column): odd and even pitches, rows shorter and
# longer than a vector, a block's 2,048 elements and a unit
ROWS = [(37, 25, 31, 3), (100, 24, 25, 0), (5, 4096, 5000, 8), (3, 1, 7, 2), (1000, 7, 9, 1),
        (2, 3001, 3008, 5), (513, 8, 16, 0), (64, 1000, 1024, 8), (9, 2048, 2056, 8),
        (700, 40, 41, 1), (2, 20_000, 20_001, 1), (4097, 1, 2, 1), (300, 16, 24, 8)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows, columns, stride, first", ROWS)
def test_rows(torch, rows, columns, stride, first, name):
    k = kind_of(torch, name)
    gen = torch.Generator("cuda").manual_seed(rows)

    def slab(kind):
        room = (1e-2 * torch.randn(rows * stride + first, generator=gen, device="cuda")).to(kind)
        return room, room[first:first + rows * stride].view(rows, stride)[:, :columns]

    room, x = slab(k)
    keep = room.clone()
    other = (1e-2 * torch.randn(333, generator=gen, device="cuda")).to(k)
    tensors = [x, other]
    before = [t.clone() for t in tensors]
    n = rows * columns + 333
    limit = norms64(torch, tensors, 2.0, "l2")[0] / 2
    with GradientList(tensors) as lst:
        check_norm(torch, lst.norm(per_tensor=True, loss_scale=3.0), tensors, 3.0, 1.0)
        want = tree_sum([t.float().reshape(-1).cpu().numpy() for t in before], 8192)
        assert float(lst.norm().sum_squares) == want
        flat = torch.cat([t.reshape(-1).float() for t in tensors])
        for start in (0, 1):  # an accumulator on and off the 32-byte boundaries
            acc = torch.randn(n + 8, generator=gen, device="cuda")[4 * start:4 * start + n]
            old = acc.clone()
            lst.accumulate(acc)
            assert torch.equal(acc, old + flat)
            lst.accumulate(acc, overwrite=True)
            assert torch.equal(acc, flat)
        for out in TYPES:  # rows into rows of another pitch, and into contiguous memory
            for pitched in (True, False):
                to, y = slab(kind_of(torch, out))
                to_keep = to.clone()
                if not pitched:
                    y = torch.empty(rows, columns, dtype=kind_of(torch, out), device="cuda")
                targets = [y, torch.empty_like(other, dtype=kind_of(torch, out))]
                with GradientList(targets) as o:
                    r = lst.clip(limit, loss_scale=2.0, out=o)
                    check_norm(torch, r, before, 2.0, limit)
                    check_clipped(torch, targets, before, 2.0, 0.5)
                if pitched:  # nothing beside the columns
                    y.copy_(to_keep[first:first + rows * stride].view(rows, stride)[:, :columns])
                    assert torch.equal(to, to_keep)
        lst.clip(limit, loss_scale=2.0)
        check_clipped(torch, tensors, before, 2.0, 0.5)
        x.copy_(before[0])
        assert torch.equal(room, keep)
    with B200Adamw(TensorTable.from_sizes([rows * columns, 333])) as opt:
        tensors[1].copy_(before[1])
        opts = StepOptions(one_based_update=10, max_grad_norm=limit, static_loss_scale=2.0)
        with GradientList(tensors) as lst:
            st = load(torch, opt, 9)
            opt.step(lst, opts)
            check_state(torch, opt.state_tensors(), st, before, [True, True], opts, 2.0, 0.5)
            # the last micro-batch, added to what is there
            acc = torch.randn(n, generator=gen, device="cuda")
            old = acc.clone()
            opt.norm_pass_accumulate(acc, lst, opts)
            assert torch.equal(acc, old + flat)
            res = opt.read_result()
            near(res.grad_norm, float((acc.double() / 2.0).square().sum().sqrt()), 4 * U, "norm")


# ---- streams, graphs, addresses ----------------------------------------------------
def test_bind_follows_new_addresses(torch):
    sizes = [1 + (37 * i) % 5000 for i in range(700)]  # more than two bind batches
    sets = [make(torch, sizes, ["bf16", "f32"], place, seed=60 + i, std=1e-2 * (i + 1))
            for i, place in enumerate(["separate", "packed", "separate"])]
    with GradientList(sets[0]) as lst:
        for tensors in sets + sets[:1]:
            lst.bind(tensors)
            check_norm(torch, lst.norm(per_tensor=True), tensors, 1.0, 1.0)


def test_two_streams_at_once(torch):
    big = make(torch, [3_000_001, 500_000], ["bf16"], "separate", seed=70)
    targets = [[torch.empty_like(t) for t in big] for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    with GradientList(big) as lst:
        outs = [GradientList(t) for t in targets]
        limits = [0.1, 0.2, 0.4, 0.8]
        want = float(lst.norm().sum_squares)
        for _ in range(20):
            got = []
            for s, o, limit in zip(streams, outs, limits):
                with torch.cuda.stream(s):
                    got.append(lst.clip(limit, out=o, stream=s))
            torch.cuda.synchronize()
            for r, limit, t in zip(got, limits, targets):
                assert float(r.sum_squares) == want
                check_norm(torch, r, big, 1.0, limit)
                check_clipped(torch, t, big, 1.0, limit / math.sqrt(want))
        for o in outs:
            o.close()


def test_a_stream_that_is_not_the_current_one(torch):
    tensors = make(torch, [100_001], ["f16"], "separate", seed=71)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with GradientList(tensors) as lst:
        for _ in range(50):
            r = lst.norm(stream=s)          # results allocated on the default stream
            junk = torch.full((100_000,), 5.0, device="cuda")
            del junk
            s.synchronize()
            check_norm(torch, r, tensors, 1.0, 1.0)
        with torch.cuda.stream(s):
            r = lst.norm()                  # None: the legacy default stream
            torch.cuda.synchronize()
            check_norm(torch, r, tensors, 1.0, 1.0)


def test_two_captured_graphs_of_one_list(torch):
    tensors = make(torch, [2_000_003, 4096, 65], ["bf16", "f32"], "separate", seed=72)
    targets = [[torch.empty_like(t) for t in tensors] for _ in range(2)]
    with GradientList(tensors) as lst:
        outs = [GradientList(t) for t in targets]
        graphs, results = [], []
        for o, limit in zip(outs, (0.25, 0.5)):
            g = torch.cuda.CUDAGraph()
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(g, stream=s):
                results.append(lst.clip(limit, out=o, per_tensor=True,
                                        stream=torch.cuda.current_stream()))
            graphs.append(g)
        side = [torch.cuda.Stream() for _ in graphs]
        for rep in range(10):
            for t in tensors:
                t.mul_(1.01)
            torch.cuda.synchronize()
            for g, s in zip(graphs, side):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for r, limit, t in zip(results, (0.25, 0.5), targets):
                check_norm(torch, r, tensors, 1.0, limit)
                check_clipped(torch, t, tensors, 1.0,
                              limit / norms64(torch, tensors, 1.0, "l2")[0])
        for o in outs:
            o.close()


def test_a_captured_step(torch):
    sizes = [70001, 33, 8192]
    tensors = make(torch, sizes, ["bf16"], "separate", seed=73)
    opts = StepOptions(one_based_update=4, max_grad_norm=1e6)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        load(torch, opt, 74)
        for _ in range(3):
            opt.step(lst, opts)
        want = {k: v.clone() for k, v in opt.state_tensors().items()}
        load(torch, opt, 74)
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            opt.step(lst, opts, stream=torch.cuda.current_stream(), wait=False)
        for _ in range(3):
            g.replay()
        torch.cuda.synchronize()
        for k, v in opt.state_tensors().items():
            assert torch.equal(v.view(torch.int16), want[k].view(torch.int16)), k


def test_rebinding_inside_a_captured_graph(torch):
    sets = [make(torch, [9000, 33], ["bf16"], "separate", seed=80 + i, std=1e-2 * (1 + i))
            for i in range(2)]
    with GradientList(sets[0]) as lst:
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            cur = torch.cuda.current_stream()
            a = lst.norm(stream=cur)
            lst.bind(sets[1], stream=cur)
            b = lst.norm(stream=cur)
            lst.bind(sets[0], stream=cur)
        for _ in range(3):
            g.replay()
            torch.cuda.synchronize()
            check_norm(torch, a, sets[0], 1.0, 1.0)
            check_norm(torch, b, sets[1], 1.0, 1.0)


def test_a_captured_clip_in_place(torch):
    # small and larger lists, below the limit and above it, as the gradients change
    for sizes in ([5000, 33], [900_000, 70_001]):
        tensors = make(torch, sizes, ["bf16", "f32"], "separate", seed=75)
        keep = [t.clone() for t in tensors]
        total = norms64(torch, keep, 1.0, "l2")[0]
        with GradientList(tensors) as lst:
            g = torch.cuda.CUDAGraph()
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(g, stream=s):
                r = lst.clip(total, stream=torch.cuda.current_stream())
            for factor in (0.5, 2.0, 0.25, 4.0):
                for t, k in zip(tensors, keep):
                    t.copy_(k * factor)
                now = [t.clone() for t in tensors]
                g.replay()
                torch.cuda.synchronize()
                check_norm(torch, r, now, 1.0, total)
                found = norms64(torch, now, 1.0, "l2")[0]
                check_clipped(torch, tensors, now, 1.0, min(1.0, total / found))


def test_a_list_closed_between_the_passes(torch):
    sizes = [70001, 8192]
    tensors = make(torch, sizes, ["bf16"], "separate", seed=76)
    opts = StepOptions(one_based_update=4, max_grad_norm=1e6)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt:
        got = []
        for close in (False, True):
            load(torch, opt, 77)
            lst = GradientList(tensors)
            opt.norm_pass(lst, opts)
            if close:
                lst.close()
            opt.update_pass(opts)
            assert opt.read_result().skipped == 0
            got.append({k: v.clone() for k, v in opt.state_tensors().items()})
            lst.close()
        for k in got[0]:
            assert torch.equal(got[0][k].view(torch.int16), got[1][k].view(torch.int16))
        lst = GradientList(tensors)
        opt.norm_pass(lst, opts)
        lst.close()  # the handle lets go of it when it is closed itself


def test_threads_share_a_list(torch):
    import threading

    tensors = make(torch, [3_000_001, 77], ["f16"], "separate", seed=78)
    with GradientList(tensors) as lst:
        want = lst.norm(per_tensor=True).values.tolist()
        wrong = []

        def work():
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(100):
                    r = lst.norm(per_tensor=True, stream=s)
                    if r.values.tolist() != want:
                        wrong.append(1)

        torch.cuda.synchronize()
        pool = [threading.Thread(target=work) for _ in range(4)]
        for t in pool:
            t.start()
        for t in pool:
            t.join()
        assert not wrong


# ---- sizes beyond 32 bits -----------------------------------------------------------
def test_a_tensor_of_more_than_2_to_the_31_elements(torch):
    n = 2 ** 31 + 4099
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[::1_000_003] = 0.5
    x[-1] = 3.0
    count = -(-n // 1_000_003)
    want = math.sqrt(0.25 * (count - ((n - 1) % 1_000_003 == 0)) + 9.0)
    with GradientList([x[1:], x[:1]]) as lst, GradientList([x]) as whole:
        for r in (lst.norm(per_tensor=True), whole.norm()):
            near(r.read().norm, want, 4 * U, "norm")
            assert r.read().max_abs == 3.0
        whole.clip(want / 4)
        near(float(x[-1]), 0.75, 2.0 ** -8, "last element")
        near(float(x[1_000_003 * 2000]), 0.125, 2.0 ** -8, "element 2,000,006,000")
    del x


def test_column_offsets_beyond_32_bits(torch):
    rows, width = 70_000, 70_016
    wide = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")  # 9.8 GB, unwritten
    aligned, odd = wide[:, 64:128], wide[:, 201:264]
    for t in (aligned, odd):
        t.copy_(1e-2 * torch.randn(t.shape, device="cuda"))
    with GradientList([aligned, odd]) as lst:
        check_norm(torch, lst.norm(per_tensor=True), [aligned, odd], 1.0, 1.0)
        acc = torch.empty(lst.elements, device="cuda")
        lst.accumulate(acc, overwrite=True)
        assert torch.equal(acc, torch.cat([aligned.reshape(-1), odd.reshape(-1)]).float())
    del wide


def test_bind_takes_only_what_the_list_was_made_of(torch):
    a = [torch.ones(100, device="cuda"), torch.ones(6, 20, device="cuda").bfloat16()[:, :10]]
    same = [torch.full((100,), 2.0, device="cuda"),
            torch.full((6, 20), 2.0, device="cuda").bfloat16()[:, 5:15]]
    other = [
        [same[0]], [same[0], same[1], same[0]],
        [same[0].bfloat16(), same[1]],               # another type
        [same[0][:99], same[1]],                      # another size
        [same[0], same[1].contiguous()],              # another layout
        [same[0], torch.ones(6, 30, device="cuda").bfloat16()[:, :10]],
        [torch.ones(200, device="cuda")[::2], same[1]],
    ]
    with GradientList(a) as lst:
        before = lst.norm().read().norm
        for tensors in other:
            with pytest.raises(ValueError):
                lst.bind(tensors)
        with pytest.raises(ValueError):
            lst.bind([same[0].cpu(), same[1]])
        assert lst.norm().read().norm == before and lst.tensors == tuple(a)
        # the same elements in another shape are the same run in memory
        lst.bind([same[0].view(10, 10), same[1]])
        near(lst.norm().read().norm, 2.0 * math.sqrt(160), 4 * U, "norm")


def test_closed_lists_are_refused_and_a_list_is_its_own_output(torch):
    x, y = torch.full((9000,), 2.0, device="cuda"), torch.empty(9000, device="cuda")
    closed, lst = GradientList([y]), GradientList([x])
    closed.close()
    closed.close()
    for call in (closed.norm, closed.clip, lambda: closed.accumulate(y),
                 lambda: closed.bind([y]), lambda: lst.clip(out=closed)):
        with pytest.raises(ValueError):
            call()
    lst.clip(1.0, out=lst)
    near(float(x[77]), 1.0 / math.sqrt(9000), 8 * U, "clipped")
    lst.close()


def test_phase_times_of_a_step_on_a_list(torch):
    sizes = [70001, 8192]
    tensors = make(torch, sizes, ["bf16"], "separate", seed=90)
    with B200Adamw(TensorTable.from_sizes(sizes)) as opt, GradientList(tensors) as lst:
        load(torch, opt, 91)
        opt.phase_timing(True)
        for t in (1, 2, 3):
            opt.step(lst, StepOptions(one_based_update=t))
        times, steps = opt.phase_times()
        assert len(times) == 2 and steps == 3 and all(v > 0.0 for v in times.values())
