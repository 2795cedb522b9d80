"""The trainable block's operators: cases, plain forms and the framework's calls.

Three operators that a training or serving program uses together: layer normalisation (forward, and backward with the weights'
gradients), the matrix product with bias, activation and residual in its epilogue (forward, and backward to all operands), and the
global gradient norm with clipping.  `own` selects between elementary torch operations in 32 bits and the framework's operators.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the encoder's normalisation of one 34-frame inference window (width 768): a launch, where latency counts
        {"name": "norm_window_fp32", "op": "norm", "rows": 34, "width": 768, "dtype": "fp32", "backward": False, "pad": 0},
        # the same layer in a training step of 128 clips of 34 frames, 16-bit activations
        {"name": "norm_train_bf16", "op": "norm", "rows": 4352, "width": 768, "dtype": "bf16", "backward": True, "pad": 0},
        # an odd width in rows that lie apart (a slice of a wider tensor): no row is aligned
        {"name": "norm_odd_fp16", "op": "norm", "rows": 2171, "width": 1001, "dtype": "fp16", "backward": True, "pad": 19},
        # the widest: long sequences of a wide model, fp32 activations
        {"name": "norm_wide_fp32", "op": "norm", "rows": 8192, "width": 4096, "dtype": "fp32", "backward": True, "pad": 0},
        # one token through the fused Q|K|V projection (768 -> 2304): the weight's bytes are all there is
        {"name": "linear_token_bf16", "op": "linear", "m": 1, "k": 768, "n": 2304, "dtype": "bf16", "act": "none", "bias": True, "residual": False,
         "backward": False},
        # one inference window through the attention output projection with its residual
        {"name": "linear_window_bf16", "op": "linear", "m": 34, "k": 768, "n": 768, "dtype": "bf16", "act": "none", "bias": True, "residual": True,
         "backward": False},
        # a training step's MLP-in product with its activation, 128 clips of 34 frames, to all gradients
        {"name": "linear_train_bf16", "op": "linear", "m": 4352, "k": 768, "n": 2304, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False,
         "backward": True},
        # odd sizes, where neither rows nor columns are aligned (an adapter between feature widths)
        {"name": "linear_odd_fp16", "op": "linear", "m": 2171, "k": 1021, "n": 427, "dtype": "fp16", "act": "silu", "bias": True, "residual": True,
         "backward": True},
        # the largest: 16k tokens of a wide model, activation and residual in one
        {"name": "linear_wide_bf16", "op": "linear", "m": 16384, "k": 4096, "n": 4096, "dtype": "bf16", "act": "gelu", "bias": True, "residual": True,
         "backward": True},
        # a small network's gradients, under the limit (most steps of a run): nothing is scaled
        {"name": "clip_small_fp32", "op": "clip", "tensors": 40, "total": 1100000, "dtype": "fp32", "into": False},
        # the generator's gradients (172 tensors, 65.8 M values), under the limit, in place
        {"name": "clip_generator_fp32", "op": "clip", "tensors": 172, "total": 65800000, "dtype": "fp32", "into": False},
        # 16-bit gradients of a larger model, clipped into the fp32 tensors that the optimizer reads
        {"name": "clip_into_bf16", "op": "clip", "tensors": 148, "total": 160000000, "dtype": "bf16", "into": True},
    ]


def _size(rng, lo, hi, step=1):
    """An integer spread over the logarithm of lo..hi; half of them multiples of `step`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if step > 1 and rng.random() < 0.5:
        v = v // step * step
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm", "linear", "clip"])
    if op == "norm":
        width = _size(rng, 32, 8192, 8)
        return {"op": op, "rows": _size(rng, 1, min(65536, 8192 * 4096 // width)), "width": width, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "backward": rng.random() < 0.7, "pad": rng.choice([0, 0, 0, 8, 19])}
    if op == "linear":
        k, n = _size(rng, 64, 4096, 8), _size(rng, 32, 4096, 8)
        return {"op": op, "m": _size(rng, 1, 16384), "k": k, "n": n, "dtype": rng.choice(["bf16", "fp16"]),
                "act": rng.choice(["none", "relu", "gelu", "silu"]), "bias": rng.random() < 0.8, "residual": rng.random() < 0.5,
                "backward": rng.random() < 0.6}
    total = _size(rng, 10000, 160000000)
    return {"op": op, "tensors": _size(rng, 1, min(400, total // 100)), "total": total, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
            "into": rng.random() < 0.5}


# --------------------------------------------------------------------------------------------------------------- inputs
def _clip_sizes(case):
    """Sizes of a model's parameter tensors: a few large, many small, odd ones among them, `total` values in all."""
    n, total = case["tensors"], case["total"]
    weights = [1.0 / (1 + i % 37) ** 2 for i in range(n)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    sizes[0] = max(1, sizes[0] + total - sum(sizes))
    return sizes


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=dev) * scale + mean

    s = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # a residual stream: rows of different magnitude, an offset, a few channels far larger than the others
        big = 1 + 12 * (torch.rand(width, generator=g, device=dev) < 0.01).float()
        x = (normal(rows, width) * big + 0.3) * torch.exp(normal(rows, 1, scale=0.3))
        buf = torch.zeros(rows, width + case["pad"], device=dev, dtype=t)
        buf[:, :width] = x
        s["x"] = buf[:, :width]
        s["weight"] = normal(width, scale=0.1, mean=1.0).to(t)
        s["bias"] = normal(width, scale=0.1).to(t)
        if case["backward"]:
            s["dy"] = normal(rows, width).to(t)
            s["leaves"] = [s[n].detach().requires_grad_() for n in ("x", "weight", "bias")]
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k).to(t)
        s["w"] = normal(n, k, scale=k ** -0.5).to(t)
        s["bias"] = normal(n, scale=0.5).to(t) if case["bias"] else None
        s["res"] = normal(m, n).to(t) if case["residual"] else None
        if case["backward"]:
            s["dy"] = normal(m, n).to(t)
            s["leaves"] = [s[i].detach().requires_grad_() if s[i] is not None else None for i in ("x", "w", "bias", "res")]
    else:
        sizes = _clip_sizes(case)
        # each tensor on a 16-byte boundary at least, as an allocator gives them; the gaps between them hold zeros
        starts = [0]
        for z in sizes:
            starts.append(starts[-1] + (z + 7) // 8 * 8)
        s["flat"] = torch.zeros(starts[-1], device=dev, dtype=t)
        values = normal(starts[-1], scale=1e-3)
        s["grads"] = [s["flat"][a:a + z] for a, z in zip(starts, sizes)]
        for a, gr in zip(starts, s["grads"]):
            gr.copy_(values[a:a + gr.numel()])
        s["limit"] = 1.0 if case["into"] else 1e3
        s["out_flat"] = torch.zeros(starts[-1], device=dev) if case["into"] else None
        s["outs"] = [s["out_flat"][a:a + z] for a, z in zip(starts, sizes)] if case["into"] else None
        if own:
            # a training program keeps its plan over the gradient tensors, as it keeps its optimizer's
            import hopmi
            s["plan"] = hopmi.ops.GradClip(s["grads"], out=s["outs"])
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    t = s["x"].dtype
    x, weight, bias = s["x"].float(), s["weight"].float(), s["bias"].float()
    c = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    xhat = c * rstd
    y = xhat * weight + bias
    if "dy" not in s:
        return [y.to(t)]
    dy = s["dy"].float()
    gdy = dy * weight
    dx = rstd * (gdy - gdy.mean(-1, keepdim=True) - xhat * (gdy * xhat).mean(-1, keepdim=True))
    return [y.to(t), dx.to(t), (dy * xhat).sum(0).to(t), dy.sum(0).to(t)]


def _plain_linear(s):
    t, act = s["x"].dtype, s["case"]["act"]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        a = z * cdf
    elif act == "silu":
        cdf = 1.0 / (1.0 + torch.exp(-z))
        a = z * cdf
    else:
        a = torch.where(z > 0, z, torch.zeros_like(z)) if act == "relu" else z
    y = (a if s["res"] is None else a + s["res"].float()).to(t)
    if "dy" not in s:
        return [y]
    dy = s["dy"].float()
    if act == "gelu":
        dz = dy * (cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    elif act == "silu":
        dz = dy * cdf * (1.0 + z * (1.0 - cdf))
    else:
        dz = torch.where(z > 0, dy, torch.zeros_like(dy)) if act == "relu" else dy
    out = [y, (dz @ w).to(t), (dz.t() @ x).to(t)]
    if s["bias"] is not None:
        out.append(dz.sum(0).to(t))
    if s["res"] is not None:
        out.append(s["dy"])
    return out


def _plain_clip(s):
    # all gradients as one stretch of memory (the gaps between them are zeros, which change neither the norm nor themselves)
    flat = s["flat"].float()
    norm = torch.sqrt((flat * flat).sum())
    scaled = flat * torch.clamp(s["limit"] / (norm + 1e-6), max=1.0)
    return [norm, scaled if s["case"]["into"] else scaled.to(s["flat"].dtype)]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "clip": _plain_clip}[op](s)
    import hopmi
    if op == "norm":
        if "dy" not in s:
            return [hopmi.ops.layer_norm(s["x"], s["weight"], s["bias"], 1e-5)]
        y = hopmi.ops.layer_norm(*s["leaves"], 1e-5)
        return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]
    if op == "linear":
        if "dy" not in s:
            return [hopmi.ops.linear_act(s["x"], s["w"], s["bias"], s["res"], s["case"]["act"])]
        y = hopmi.ops.linear_act(*s["leaves"], s["case"]["act"])
        return [y.detach(), *torch.autograd.grad(y, [v for v in s["leaves"] if v is not None], s["dy"])]
    norm = s["plan"].clip_(s["limit"])
    return [norm, s["out_flat"] if s["case"]["into"] else s["flat"]]


# ----------------------------------------------------------------------------------------------------- what it has to cost
def work(case):
    e = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "norm":
        n, d = case["rows"] * case["width"], case["width"]
        # forward: x in, y out; backward: dy in, dx out (x is counted once), the weights in and their gradients out
        return {"bytes": e * (4 * n + 4 * d if case["backward"] else 2 * n + 2 * d), "flops": (22 if case["backward"] else 8) * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        b, r = case["bias"] * n, case["residual"] * m * n
        once = m * k + n * k + b + r + m * n                       # x, W, bias, residual in, y out
        if not case["backward"]:
            return {"bytes": e * once, "flops": 2 * m * n * k}
        return {"bytes": e * (once + m * n + m * k + n * k + b), "flops": 6 * m * n * k}      # dy in; dx, dW, db out (dres is dy)
    n = case["total"]
    # the norm reads every value before the first can be scaled: read once; written where they go into other tensors
    return {"bytes": n * e + (4 * n if case["into"] else 0), "flops": 3 * n}


# ------------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.nn.functional
    if case["op"] == "norm":
        x, w, b = (s[i].double().requires_grad_(case["backward"]) for i in ("x", "weight", "bias"))
        y = f.layer_norm(x, (case["width"],), w, b, 1e-5)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], s["dy"].double())] if case["backward"] else [y]
    if case["op"] == "linear":
        v = {i: s[i].double().requires_grad_(case["backward"]) for i in ("x", "w", "bias", "res") if s[i] is not None}
        y = f.linear(v["x"], v["w"], v.get("bias"))
        y = {"none": lambda z: z, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}[case["act"]](y)
        y = y + v["res"] if "res" in v else y
        return [y.detach(), *torch.autograd.grad(y, list(v.values()), s["dy"].double())] if case["backward"] else [y]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in s["grads"]]))
    return [norm, s["flat"].double() * min(1.0, s["limit"] / (norm.item() + 1e-6))]
