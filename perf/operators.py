"""Cases of the gradient-list operators: what is measured, in plain torch and with the kernels.

A backward pass leaves its gradients in many tensors of several types.  Four operators take them
as they lie:

  norm        global L2 (or largest-magnitude) norm over all tensors of the gradients divided by
              the loss scale, the clip scale min(max_norm / norm, 1), a non-finite flag, and each
              tensor's own norm and largest magnitude
  clip        unscaled and clipped gradients, into tensors of another type or in place;
              nothing is written when a gradient is inf or NaN
  accumulate  a micro-batch's tensors added to (or starting) one flat f32 accumulator
  step        norm + clip + AdamW over f32 master weights and moments, and the bf16 weight copy;
              no state is written when a gradient is inf or NaN

A case says how the tensors are laid out:

  kind "model"   the tensor list of a grouped-query transformer (embedding, per block: norm, q, k,
                 v, o, norm, gate, up, down; final norm, untied head unless "tied")
  kind "pieces"  "tensors" tensors of "elements" values in all, spread by "shape_seed"; "odd" leaves
                 sizes as they fall, else they are multiples of 8
  place          "separate" allocations, "packed" one after another in a bucket of their type
                 (an odd size misaligns all that follow), "columns" of pairwise fused matrices
  dtype          "bf16", "f16", "f32", or "mixed": the 1-D tensors f32, the matrices bf16
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
BETA1, BETA2, EPS, DECAY, LR, UPDATE = 0.9, 0.95, 1e-8, 0.1, 3e-4, 10

SMOKE = {"kind": "model", "vocabulary": 32000, "width": 128, "ffn": 384, "layers": 2, "kv_width": 64, "tied": True}
CANONICAL = {"kind": "model", "vocabulary": 32000, "width": 768, "ffn": 2432, "layers": 12, "kv_width": 256, "tied": False}


def listed():
    return [
        # the gradients of a handful of small tensors (adapters, a probe's head): latency is all there is
        {"name": "norm, 9 small tensors", "op": "norm", "kind": "pieces", "tensors": 9, "elements": 98304, "shape_seed": 3, "odd": False,
         "place": "separate", "dtype": "bf16", "scale": 1.0, "max_norm": 1.0, "measure": "l2", "spread": 1e-3, "bad": ""},
        # the canonical model's backward pass: one norm per update, with the per-tensor norms that training logs
        {"name": "norm, 135M bf16", "op": "norm", **CANONICAL, "place": "separate", "dtype": "bf16", "scale": 65536.0, "max_norm": 1.0, "measure": "l2", "spread": 1e-3, "bad": ""},
        # buckets filled back to back with odd sizes, norm scales in f32 among bf16 matrices; a loss scale that is no power of two
        {"name": "norm, 257 ragged, packed", "op": "norm", "kind": "pieces", "tensors": 257, "elements": 30000001, "shape_seed": 11, "odd": True,
         "place": "packed", "dtype": "mixed", "scale": 37888.0, "max_norm": 0.5, "measure": "l2", "spread": 1e-3, "bad": ""},
        # f16 gradients of a small model unscaled and clipped into f32 for another optimizer
        {"name": "clip, smoke f16 to f32", "op": "clip", **SMOKE, "place": "separate", "dtype": "f16", "out": "f32", "scale": 1024.0, "max_norm": 1.0, "measure": "l2", "spread": 1e-3, "bad": ""},
        # the canonical model, clipped by its norm, type kept
        {"name": "clip, 135M bf16", "op": "clip", **CANONICAL, "place": "separate", "dtype": "bf16", "out": "bf16", "scale": 1.0, "max_norm": 1.0, "measure": "l2", "spread": 1e-3, "bad": ""},
        # column slices of fused projections' gradients, f32
        {"name": "clip, 48 column slices f32", "op": "clip", "kind": "pieces", "tensors": 48, "elements": 24000000, "shape_seed": 5, "odd": False,
         "place": "columns", "dtype": "f32", "out": "f32", "scale": 8.0, "max_norm": 1.0, "measure": "l2", "spread": 1e-2, "bad": ""},
        # late training: the norm is below the limit, the gradients stay as they are
        {"name": "clip in place, 135M below the limit", "op": "clip", **CANONICAL, "place": "packed", "dtype": "bf16", "out": "", "scale": 1.0, "max_norm": 1000.0, "measure": "l2", "spread": 1e-3, "bad": ""},
        # first micro-batch of a small model's update
        {"name": "accumulate, smoke, first", "op": "accumulate", **SMOKE, "place": "separate", "dtype": "bf16", "overwrite": True, "spread": 1e-3, "bad": ""},
        # a later micro-batch of the canonical model's update
        {"name": "accumulate, 135M bf16", "op": "accumulate", **CANONICAL, "place": "separate", "dtype": "bf16", "overwrite": False, "spread": 1e-3, "bad": ""},
        # the whole update, small model
        {"name": "step, smoke bf16", "op": "step", **SMOKE, "place": "separate", "dtype": "bf16", "scale": 65536.0, "max_norm": 1.0, "spread": 1e-3, "bad": ""},
        # the whole update, canonical model
        {"name": "step, 135M bf16", "op": "step", **CANONICAL, "place": "separate", "dtype": "bf16", "scale": 65536.0, "max_norm": 1.0, "spread": 1e-3, "bad": ""},
        # odd sizes: neither the state's tensors nor the gradients start on vector boundaries
        {"name": "step, 61 ragged, mixed types", "op": "step", "kind": "pieces", "tensors": 61, "elements": 9000011, "shape_seed": 23, "odd": True,
         "place": "packed", "dtype": "mixed", "scale": 1024.0, "max_norm": 1.0, "spread": 1e-3, "bad": ""},
    ]


def draw(rng):
    op = rng.choice(["norm", "clip", "accumulate", "step"])
    most = {"norm": 135e6, "clip": 135e6, "accumulate": 135e6, "step": 100e6}[op]
    elements = int(math.exp(rng.uniform(math.log(2000), math.log(most))))
    tensors = min(int(math.exp(rng.uniform(0, math.log(400)))), max(1, elements // 64))
    c = {"op": op, "kind": "pieces", "tensors": tensors, "elements": elements, "shape_seed": rng.randrange(1 << 30), "odd": rng.random() < 0.6,
         "place": rng.choice(["separate", "separate", "packed", "columns"]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32", "mixed"]),
         "spread": rng.choice([1e-4, 1e-3, 1e-2]), "bad": rng.choice(["", "", "", "", "", "", "inf", "nan"])}
    if op == "accumulate":
        return {**c, "bad": "", "overwrite": rng.random() < 0.4}
    c.update(scale=rng.choice([1.0, 1.0, 1024.0, 65536.0 if c["dtype"] != "f16" else 512.0, 1000.0, 37888.0 if c["dtype"] != "f16" else 96.0]),
             max_norm=rng.choice([0.25, 1.0, 1.0, 1000.0]))
    if op != "step":
        c["measure"] = rng.choice(["l2", "l2", "l2", "max"])
    if op == "clip":
        c["out"] = rng.choice(["f32", "bf16", "f16", c["dtype"] if c["dtype"] != "mixed" else "f32"])
        if rng.random() < 0.2:  # in place: the gradients come back in their buckets, and below the limit so that every pass sees the same
            c.update(out="", place="packed", scale=1.0, max_norm=1e6)
    return c


def shapes_of(case):
    """The tensors' shapes; a 1-D tensor is a norm scale or a bias."""
    if case["kind"] == "model":
        w, f, kv = case["width"], case["ffn"], case["kv_width"]
        block = [(w,), (w, w), (kv, w), (kv, w), (w, w), (w,), (f, w), (f, w), (w, f)]
        head = [] if case["tied"] else [(case["vocabulary"], w)]
        return [(case["vocabulary"], w)] + block * case["layers"] + [(w,)] + head
    r = random.Random(case["shape_seed"])
    weights = [math.exp(r.gauss(0, 1.5)) for _ in range(case["tensors"])]
    sizes = [max(1, int(case["elements"] * x / sum(weights))) for x in weights]
    if case["place"] == "columns":
        # pairs of slices [rows, c] of one matrix of c0 + c1 columns
        rows = [max(1, min(4096, int(math.sqrt(n)))) for n in sizes[0::2] for _ in (0, 1)]
        cols = [max(1, n // k) for n, k in zip(sizes, rows)]
        return [(k, c if case["odd"] else max(8, c // 8 * 8)) for k, c in zip(rows, cols)]
    sizes = [n if case["odd"] else max(8, n // 8 * 8) for n in sizes]
    return [(n,) if i % 3 == 0 else (1, n) for i, n in enumerate(sizes)]


def types_of(case, shapes):
    return [TYPES[("f32" if len(s) == 1 else "bf16") if case["dtype"] == "mixed" else case["dtype"]] for s in shapes]


def numbers_of(case):
    return [math.prod(s) for s in shapes_of(case)]


def gradients(case, gen):
    """The tensors, and the buckets that hold them where they are packed.  Each tensor has a size of
    its own (log-normal), its values are normal with a heavy tail, times the loss scale."""
    shapes = shapes_of(case)
    types = types_of(case, shapes)
    if case["place"] == "packed":
        kinds = list(dict.fromkeys(types))
        buckets = [torch.empty(sum(math.prod(s) for s, t in zip(shapes, types) if t == k), dtype=k, device="cuda") for k in kinds]
        pieces = {k: iter(b.split([math.prod(s) for s, t in zip(shapes, types) if t == k])) for k, b in zip(kinds, buckets)}
        tensors = [next(pieces[t]).view(s) for s, t in zip(shapes, types)]
    elif case["place"] == "columns":
        buckets, tensors = [], []
        for i in range(0, len(shapes), 2):
            wide = torch.empty(shapes[i][0], sum(s[1] for s in shapes[i:i + 2]), dtype=types[i], device="cuda")
            buckets.append(wide)
            tensors += wide.split([s[1] for s in shapes[i:i + 2]], 1)
    else:
        tensors = [torch.empty(s, dtype=t, device="cuda") for s, t in zip(shapes, types)]
        buckets = tensors
    sizes = torch.exp(0.5 * torch.randn(len(tensors), generator=gen, device="cuda"))
    for k, t in enumerate(tensors):
        x = torch.randn(t.shape, generator=gen, device="cuda")
        t.copy_(x * (1 + 0.25 * x * x) * (sizes[k] * case["spread"] * case.get("scale", 1.0)))
    if case["bad"]:
        k = random.Random(case["shape_seed"] + 1).randrange(len(tensors))
        tensors[k].select(0, tensors[k].shape[0] // 2)[..., -1:].fill_(float(case["bad"]))
    return tensors, buckets


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    tensors, buckets = gradients(case, gen)
    numbers = [t.numel() for t in tensors]
    s = {"case": case, "tensors": tensors, "buckets": buckets, "numbers": numbers}
    if case["op"] == "clip" and case["out"]:
        # the clipped gradients' tensors, each on a 64-byte boundary of one buffer
        room = [(n + 31) // 32 * 32 for n in numbers]
        s["flat"] = torch.zeros(sum(room), dtype=TYPES[case["out"]], device="cuda")
        s["outs"] = [p[:n].view(t.shape) for p, n, t in zip(s["flat"].split(room), numbers, tensors)]
    if case["op"] == "accumulate":
        s["acc"] = case["spread"] * torch.randn(sum(numbers), generator=gen, device="cuda")
    if case["op"] == "step":
        total = sum(numbers)
        master = 0.02 * torch.randn(total, generator=gen, device="cuda")
        moment = 1e-4 * torch.randn(total, generator=gen, device="cuda")
        variance = (1e-3 * torch.randn(total, generator=gen, device="cuda")).square()
        s["decay"] = [len(t.shape) > 1 for t in tensors]
        s["state"] = {"master": master, "moment": moment, "variance": variance, "bf16": master.bfloat16()}
    if own:
        import sys
        if "python-slm_b200" not in sys.path:
            sys.path.insert(0, "python-slm_b200")
        import slmopt
        s["list"] = slmopt.GradientList(tensors)
        if case["op"] == "clip":
            s["out_list"] = slmopt.GradientList(s["outs"]) if case["out"] else None
        if case["op"] == "step":
            s["opt"] = slmopt.B200Adamw(slmopt.TensorTable.from_sizes(numbers, s["decay"]))
            mine = s["opt"].state_tensors()
            for name, start in s["state"].items():
                mine[name].copy_(start)
            s["state"] = mine
            s["options"] = slmopt.StepOptions(learning_rate=LR, one_based_update=UPDATE, beta1=BETA1, beta2=BETA2, epsilon=EPS, decay_weight=DECAY,
                                              max_grad_norm=case["max_norm"], static_loss_scale=case["scale"])
    elif case["op"] == "step":
        s["decay_weight"] = torch.cat([torch.full((n,), DECAY if d else 0.0, device="cuda") for n, d in zip(numbers, s["decay"])])
    return s


def values(tensors, scale, max_norm, measure):
    """norm, clip scale, largest magnitude and non-finite flag over all tensors, then each tensor's norm
    and largest magnitude, as one f32 tensor; and the unscaled gradients in f32."""
    g = [t.float() / scale for t in tensors]
    squares = torch.stack([x.square().sum(dtype=torch.float64) for x in g])
    largest = torch.stack([x.abs().max() for x in g])
    top = largest.max()
    norm = top if measure == "max" else squares.sum().sqrt().float()
    bad = ~torch.isfinite(norm) | ~torch.isfinite(top)
    clip = torch.where(bad, 0.0, torch.where(norm > 0, max_norm / norm, 1.0).clamp(max=1.0))
    each = largest if measure == "max" else squares.sqrt().float()
    return torch.cat([torch.stack([norm, clip, top, bad.float()]), each, largest]), g


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "norm":
            return s["list"].norm(loss_scale=case["scale"], max_norm=case["max_norm"], kind=case["measure"], per_tensor=True).values
        if op == "clip":
            r = s["list"].clip(case["max_norm"], loss_scale=case["scale"], kind=case["measure"], out=s["out_list"])
            return r.values, s["flat"] if case["out"] else s["buckets"]
        if op == "accumulate":
            s["list"].accumulate(s["acc"], overwrite=case["overwrite"])
            return s["acc"]
        s["opt"].step(s["list"], s["options"], wait=False)
        return s["state"]
    if op == "accumulate":
        micro = torch.cat([t.reshape(-1).float() for t in s["tensors"]])
        s["acc"] = micro if case["overwrite"] else s["acc"].add_(micro)
        return s["acc"]
    found, g = values(s["tensors"], case["scale"], case["max_norm"], case.get("measure", "l2"))
    if op == "norm":
        return found
    clip, bad = found[1], found[3] > 0
    if op == "clip":
        outs = s["outs"] if case["out"] else s["tensors"]
        [o.copy_(torch.where(bad, o.float(), x * clip)) for o, x in zip(outs, g)]
        return found[:4], s["flat"] if case["out"] else s["buckets"]
    x = torch.cat([t.reshape(-1) for t in g]) * clip
    master, m, v = (s["state"][k] for k in ("master", "moment", "variance"))
    m1 = BETA1 * m + (1 - BETA1) * x
    v1 = BETA2 * v + (1 - BETA2) * x * x
    root = (v1 / (1 - BETA2 ** UPDATE)).sqrt() + EPS
    w1 = master - LR * (m1 / (1 - BETA1 ** UPDATE) / root + s["decay_weight"] * master)
    [old.copy_(torch.where(bad, old, new)) for old, new in ((master, w1), (m, m1), (v, v1))]
    s["state"]["bf16"].copy_(master)
    return s["state"]


def exact(case, seed):
    """The same from the definitions, in 64 bits; what is stored in fewer bits is left unrounded."""
    s = prepare(case, seed)
    if case["op"] == "accumulate":
        total = torch.zeros_like(s["acc"], dtype=torch.float64) if case["overwrite"] else s["acc"].double()
        at = 0
        for t in s["tensors"]:
            total[at:at + t.numel()] += t.double().flatten()
            at += t.numel()
        return total
    measure, scale, limit = case.get("measure", "l2"), case["scale"], case["max_norm"]
    norms, tops = [], []
    for t in s["tensors"]:
        x = t.double().flatten() / scale
        tops.append(x.abs().amax())
        norms.append(torch.linalg.vector_norm(x) if measure == "l2" else tops[-1])
    norms, tops = torch.stack(norms), torch.stack(tops)
    norm = torch.linalg.vector_norm(norms) if measure == "l2" else tops.amax()
    fine = bool(torch.isfinite(norm)) and bool(torch.isfinite(tops).all())
    factor = 0.0 if not fine else 1.0 if float(norm) <= limit else limit / float(norm)
    head = torch.tensor([float(norm), factor, float(tops.amax()), 0.0 if fine else 1.0], dtype=torch.float64, device="cuda")
    if case["op"] == "norm":
        return torch.cat([head, norms, tops])
    if case["op"] == "clip":
        if fine:
            if not case["out"]:
                for b in s["buckets"]:
                    s["wide"] = s.get("wide", []) + [b.double() / scale * factor]
                return head, s["wide"]
            wide = torch.zeros(s["flat"].numel(), dtype=torch.float64, device="cuda")
            at = 0
            for t in s["tensors"]:
                wide[at:at + t.numel()] = t.double().flatten() / scale * factor
                at += -(-t.numel() // 32) * 32
            return head, wide
        return head, s["flat"].double() if case["out"] else [b.double() for b in s["buckets"]]
    w, m, v = (s["state"][k].double() for k in ("master", "moment", "variance"))
    if fine:
        at = 0
        for t, decayed in zip(s["tensors"], s["decay"]):
            here = slice(at, at + t.numel())
            x = t.double().flatten() / scale * factor
            m[here] += (1 - BETA1) * (x - m[here])
            v[here] += (1 - BETA2) * (x ** 2 - v[here])
            move = m[here] / (1 - BETA1 ** UPDATE) / ((v[here] / (1 - BETA2 ** UPDATE)) ** 0.5 + EPS)
            w[here] -= LR * (move + (DECAY * w[here] if decayed else 0.0))
            at += t.numel()
    return {"master": w, "moment": m, "variance": v, "bf16": w}


def work(case):
    """Each gradient read once, each output written once; the state of a step read and written once."""
    shapes = shapes_of(case)
    numbers = [math.prod(x) for x in shapes]
    total = sum(numbers)
    read = sum(n * (4 if t == torch.float32 else 2) for n, t in zip(numbers, types_of(case, shapes)))
    if case["op"] == "norm":
        return {"bytes": read + 4 * (4 + 2 * len(numbers)), "flops": 4 * total}
    if case["op"] == "clip":
        kept = not case["out"]  # in place and below the limit nothing has to be written
        return {"bytes": read + (0 if kept else total * SIZE[case["out"]]), "flops": 4 * total if kept else 6 * total}
    if case["op"] == "accumulate":
        return {"bytes": read + total * (4 if case["overwrite"] else 8), "flops": 0 if case["overwrite"] else total}
    return {"bytes": read + 26 * total, "flops": 20 * total}
