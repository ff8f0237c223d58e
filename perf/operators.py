"""The layer norm, gradient clipping and clipped SGD step of vince_amd as measurable calls: cases, inputs, plain forms, exact values.

Three operators of a training step:

  layer_norm_fwd   y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, with the ReLU of a projection head in its epilogue
  layer_norm_bwd   its input gradient and the gradients of weight and bias (sums over all rows); `act` is the ReLU's output
  grad_clip        the 2-norm over many gradient tensors, and the gradients scaled in place to a largest norm
  clipped_step     the same norm, then SGD with momentum and weight decay over flat ranges with the clipping coefficient folded in

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls a user makes of the library.
"""
import torch

own = False

EPS = 1e-5           # layer norm
CLIP_EPS = 1e-6      # coefficient = min(1, max_norm / (norm + CLIP_EPS))
LR, MOMENTUM, WEIGHT_DECAY = 0.03, 0.9, 1e-4
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one frame through ResNet-18's projection head at inference: latency
        dict(name="fwd one row", op="layer_norm_fwd", rows=1, cols=512, dtype="float32", relu=True),
        # ResNet-50's projection head, the benchmark's batch
        dict(name="fwd head", op="layer_norm_fwd", rows=256, cols=2048, dtype="float32", relu=True),
        # odd in both sizes: most rows start off a 4-byte boundary
        dict(name="fwd odd", op="layer_norm_fwd", rows=4099, cols=1023, dtype="bfloat16", relu=False),
        # a long batch of wide bfloat16 activations
        dict(name="fwd large", op="layer_norm_fwd", rows=65536, cols=2048, dtype="bfloat16", relu=False),
        # the backward pass of "fwd head"
        dict(name="bwd head", op="layer_norm_bwd", rows=256, cols=2048, dtype="float32", relu=True),
        # many ragged rows: the sums for weight and bias are long, the rows short
        dict(name="bwd ragged", op="layer_norm_bwd", rows=10007, cols=515, dtype="bfloat16", relu=False),
        # the largest: 805 MB through one pass
        dict(name="bwd large", op="layer_norm_bwd", rows=32768, cols=4096, dtype="bfloat16", relu=False),
        # the gradients of ResNet-18's projection head with its norm, clipped
        dict(name="clip head", op="grad_clip", tensors=6, elements=296512, dtype="float32", align=64, clipped=True),
        # all trainable tensors of ResNet-50 with its heads, every gradient scaled
        dict(name="clip trunk", op="grad_clip", tensors=167, elements=27970688, dtype="float32", align=64, clipped=True),
        # a large model's bfloat16 and float32 gradients, packed without alignment, whose norm stays below the limit (most steps)
        dict(name="clip large mixed", op="grad_clip", tensors=301, elements=160000001, dtype="mixed", align=1, clipped=False),
        # the flat range of ResNet-18's head
        dict(name="step head", op="clipped_step", elements=296512, first=64, clipped=True),
        # ResNet-50's flat buffer: trunk and head ranges
        dict(name="step trunk", op="clipped_step", elements=27970688, first=23454912, clipped=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["layer_norm_fwd", "layer_norm_bwd", "grad_clip", "clipped_step"])
    if op.startswith("layer_norm"):
        cols = _log(rng, 16, 16384)
        rows = _log(rng, 1, min(131072, 130000000 // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["float32", "bfloat16"]) if rows * cols < 60000000 else "bfloat16",
                    relu=rng.random() < 0.5 and rows * cols < 60000000)
    if op == "grad_clip":
        dtype = rng.choice(["float32", "bfloat16", "mixed"])
        elements = _log(rng, 2000, 40000000)
        return dict(op=op, tensors=max(2, min(_log(rng, 2, 600), elements // 8)), elements=elements, dtype=dtype, align=rng.choice([1, 64]),
                    clipped=rng.random() < 0.5)
    elements = _log(rng, 2000, 27000000)
    # (a flat range starts on a boundary of 64 elements, as in the model's flat buffer)
    return dict(op=op, elements=elements, first=rng.randrange(1, elements // 64 + 1) * 64, clipped=rng.random() < 0.5)


def work(case):
    if case["op"].startswith("layer_norm"):
        rows, cols = case["rows"], case["cols"]
        size = 4 if case["dtype"] == "float32" else 2
        n = rows * cols
        if case["op"] == "layer_norm_fwd":      # x in, y out, weight and bias in, mean and rstd out
            return {"bytes": 2 * n * size + 8 * cols + 8 * rows, "flops": 8 * n}
        return {"bytes": (4 if case["relu"] else 3) * n * size + 12 * cols + 8 * rows, "flops": 14 * n}
    if case["op"] == "grad_clip":
        n, sizes = case["elements"], _sizes(case["tensors"], case["elements"])
        nbytes = {"float32": 4 * n, "bfloat16": 2 * n, "mixed": 4 * sum(sizes[::2]) + 2 * sum(sizes[1::2])}[case["dtype"]]
        return {"bytes": nbytes * (2 if case["clipped"] else 1) + 8, "flops": n * (3 if case["clipped"] else 2)}
    # gradient, parameter and momentum in, parameter and momentum out
    return {"bytes": 20 * case["elements"] + 8, "flops": 9 * case["elements"]}


# ------------------------------------------------------------------------------------------------ inputs
def _sizes(count, total):
    """`count` sizes from 1 element to a large part of `total`, which is their sum: most tensors of a network are small, a few are large."""
    weights = [((i * 7919 + 13) % 997 + 1) ** 3 for i in range(count)]
    spare, whole = total - count, sum(weights)
    sizes = [1 + spare * w // whole for w in weights]
    sizes[-1] += total - sum(sizes)
    return sizes


def _starts(sizes, align):
    places, at = [], 0
    for n in sizes:
        places.append(at)
        at += -(-n // align) * align
    return places, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    state = dict(case)
    if case["op"].startswith("layer_norm"):
        rows, cols, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]
        # rows of different mean and spread, as a Linear layer leaves them
        x = normal(rows, cols).mul_(normal(rows, 1).abs_().add_(0.3)).add_(normal(rows, 1).mul_(0.5)).to(dtype)
        state.update(x=x, weight=normal(cols).mul_(0.2).add_(1.0), bias=normal(cols).mul_(0.3))
        if case["op"] == "layer_norm_bwd":
            wide = x.float()
            mean = wide.mean(1)
            rstd = (wide.sub_(mean[:, None]).square_().mean(1) + EPS).rsqrt()
            state.update(mean=mean, rstd=rstd, dout=normal(rows, cols).mul_(0.01).to(dtype),
                         act=normal(rows, cols).clamp_(min=0.0).to(dtype) if case["relu"] else None)
        return state
    target = 3.0 if case["clipped"] else 0.7          # against a largest norm of 1
    n = case["elements"]
    if case["op"] == "grad_clip":
        sizes = _sizes(case["tensors"], n)
        halves = {"float32": ["float32"], "bfloat16": ["bfloat16"], "mixed": ["float32", "bfloat16"]}[case["dtype"]]
        state.update(fresh=[], flat=[], grads=[])
        for k, dtype in enumerate(halves):
            mine = sizes[k::len(halves)]
            places, whole = _starts(mine, case["align"])
            fresh = torch.zeros(whole, device="cuda", dtype=DTYPES[dtype])
            parts = [fresh[at:at + m] for at, m in zip(places, mine)]
            for part in parts:
                part.copy_(normal(part.numel()).mul_(target / n ** 0.5))
            flat = fresh.clone()
            state["fresh"].append(fresh)
            state["flat"].append(flat)
            state["grads"] += [flat[at:at + m] for at, m in zip(places, mine)]
        if own:
            from vince_amd import ops
            state["table"] = ops.GradTable(state["grads"])
        return state
    # gradients summed over two ranks, halved by the step
    grad, param, buf = normal(n).mul_(2 * target / n ** 0.5), normal(n).mul_(0.05), normal(n).mul_(target / n ** 0.5)
    a = min(case["first"], n)
    ranges = [(0, a), (a, n)] if a < n else [(0, n)]
    state.update(grad=grad, param=param, buf=buf, ranges=ranges)
    if own:
        from vince_amd import ops
        state["table"] = ops.GradTable([grad[i:j] for i, j in ranges], scales=[0.5] * len(ranges))
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from vince_amd import ops
    if s["op"] == "layer_norm_fwd":
        return ops.layer_norm_fwd(s["x"], s["weight"], s["bias"], eps=EPS, relu=s["relu"])
    if s["op"] == "layer_norm_bwd":
        return ops.layer_norm_bwd(s["x"], s["weight"], s["mean"], s["rstd"], s["dout"], act=s["act"])
    if s["op"] == "grad_clip":
        _new_gradients(s)
        clip = ops.grad_clip(s["table"], 1.0)
        return [clip] + s["flat"]
    clip = ops.grad_norm(s["table"], 1.0)
    [ops.sgd_flat(s["param"][i:j], s["grad"][i:j], s["buf"][i:j], LR, MOMENTUM, WEIGHT_DECAY, grad_scale=0.5, clip=clip) for i, j in s["ranges"]]
    return [clip, s["param"], s["buf"]]


def _new_gradients(s):
    """Where clipping rewrites the gradients, a step's backward pass has written new ones before: the copy stands for it."""
    if s["clipped"]:
        [flat.copy_(fresh) for flat, fresh in zip(s["flat"], s["fresh"])]


def _clip_of(norm):
    return torch.stack([norm, (1.0 / (norm + CLIP_EPS)).clamp(max=1.0)])


def _run_plain(s):
    if s["op"] == "layer_norm_fwd":
        x = s["x"].float()
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((centred * centred).mean(1) + EPS)
        y = centred * rstd[:, None] * s["weight"] + s["bias"]
        y = torch.where(y < 0, torch.zeros_like(y), y) if s["relu"] else y
        return y.to(s["x"].dtype), mean, rstd
    if s["op"] == "layer_norm_bwd":
        d = s["dout"].float()
        d = d * (s["act"] > 0) if s["relu"] else d
        xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        g = d * s["weight"]
        dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        return dx.to(s["x"].dtype), (d * xhat).sum(0), d.sum(0)
    if s["op"] == "grad_clip":
        _new_gradients(s)
        wide = [g.float() for g in s["grads"]]
        clip = _clip_of(torch.stack([(g * g).sum() for g in wide]).sum().sqrt())
        [g.copy_(w * clip[1]) for g, w in zip(s["grads"], wide)]
        return [clip] + s["flat"]
    parts = [s["grad"][i:j] * 0.5 for i, j in s["ranges"]]
    clip = _clip_of(torch.stack([(g * g).sum() for g in parts]).sum().sqrt())
    for g, (i, j) in zip(parts, s["ranges"]):
        p, b = s["param"][i:j], s["buf"][i:j]
        d = g * clip[1] + WEIGHT_DECAY * p
        b.copy_(b * MOMENTUM + d)
        p.copy_(p - LR * b)
    return [clip, s["param"], s["buf"]]


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + EPS).pow(-0.5)
        y = torch.addcmul(s["bias"].double(), x.sub_(mean.unsqueeze(1)).mul_(rstd.unsqueeze(1)), s["weight"].double())
        return (y.clamp_(min=0.0) if case["relu"] else y), mean, rstd
    if case["op"] == "layer_norm_bwd":
        cols = case["cols"]
        mean, rstd, w = s["mean"].double().unsqueeze(1), s["rstd"].double().unsqueeze(1), s["weight"].double()
        xhat = s["x"].double().sub_(mean).mul_(rstd)
        d = s["dout"].double()
        if case["relu"]:
            d[s["act"] <= 0] = 0.0
        along = (xhat * d) @ w.unsqueeze(1)          # sum over a row of g * xhat
        level = d @ w.unsqueeze(1)                   # sum over a row of g
        dw, db = (xhat * d).sum(0), d.sum(0)
        return d.mul_(w).mul_(cols).sub_(level).sub_(xhat.mul_(along)).mul_(rstd / cols), dw, db
    if case["op"] == "grad_clip":
        flats = [f.double() for f in s["fresh"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(f) for f in flats]))
        coefficient = torch.minimum(torch.ones_like(norm), 1.0 / (norm + CLIP_EPS))
        return [torch.stack([norm, coefficient])] + [f.mul_(coefficient) for f in flats]
    grad = s["grad"].double().mul_(0.5)
    norm = torch.linalg.vector_norm(grad)
    coefficient = torch.minimum(torch.ones_like(norm), 1.0 / (norm + CLIP_EPS))
    param = s["param"].double()
    buf = s["buf"].double().mul_(MOMENTUM).add_(grad.mul_(coefficient)).add_(param, alpha=WEIGHT_DECAY)
    return [torch.stack([norm, coefficient]), param.sub_(buf, alpha=LR), buf]
