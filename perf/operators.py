"""The training operators' cases: what is timed, in plain form and through ``commux_b200.ops``.

Four kinds of call, each a part of one training step of a decoder-only
transformer (``commux_b200.models.gpt``) or, for the norm, of serving a token:

``norm``    layer norm of a residual stream, forward alone or with its
            backward pass, with or without the residual sum in the same call
            and with the normalised input kept in 8 bits or not.
``gelu8``   GELU whose input is kept in 8 bits for the backward pass.
``wgrad8``  a linear layer's input kept in 8 bits, and the weight and bias
            gradients formed from it.
``xent``    softmax cross entropy over the vocabulary with its gradient.

The 8-bit form: groups of 32 neighbours of a row share a scale, the smallest
power of two s >= 2^-126 with 127 s >= the group's largest magnitude; a value x
is held as rint(x / s).
"""

import math

import torch

own = False

GROUP = 32
EPS = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100


def listed():
    return [
        # one token of a served request at the GPT's width: launch latency
        {"name": "norm 1 token", "op": "norm", "rows": 1, "cols": 768, "x": "bf16", "out": "bf16", "weight": "bf16",
         "residual": True, "pack": False, "train": False},
        # one norm of the GPT's step (micro-batch 8 x 1024 tokens) under bf16 autocast: fp32 stream and weights
        {"name": "norm gpt step", "op": "norm", "rows": 8192, "cols": 768, "x": "fp32", "out": "bf16", "weight": "fp32",
         "residual": True, "pack": False, "train": True},
        # a wide model trained in bf16 throughout, its normalised input kept in 8 bits
        {"name": "norm wide packed", "op": "norm", "rows": 32768, "cols": 4096, "x": "bf16", "out": "bf16",
         "weight": "bf16", "residual": False, "pack": True, "train": True},
        # the last, short batch of an epoch: latency
        {"name": "gelu8 short", "op": "gelu8", "rows": 16, "cols": 3072, "x": "bf16", "form": "tanh", "pack": False},
        # the GPT's feed-forward activation, its output handed on in 8 bits as well
        {"name": "gelu8 gpt step", "op": "gelu8", "rows": 8192, "cols": 3072, "x": "bf16", "form": "tanh", "pack": True},
        # training without autocast, the exact GELU, rows of odd length
        {"name": "gelu8 fp32 odd", "op": "gelu8", "rows": 4099, "cols": 10001, "x": "fp32", "form": "none",
         "pack": False},
        # a small head on a few tokens, nothing a multiple of anything
        {"name": "wgrad8 small odd", "op": "wgrad8", "rows": 37, "cols": 100, "outs": 61, "x": "fp32", "dw": "fp32",
         "bias": True},
        # the GPT's first feed-forward product: fp32 gradients for fp32 master weights
        {"name": "wgrad8 gpt fc", "op": "wgrad8", "rows": 8192, "cols": 768, "outs": 3072, "x": "bf16", "dw": "fp32",
         "bias": True},
        # a square projection of a wide model over a long batch
        {"name": "wgrad8 wide", "op": "wgrad8", "rows": 16384, "cols": 4096, "outs": 4096, "x": "bf16", "dw": "bf16",
         "bias": False},
        # fine-tuning on a single sequence's answer tokens
        {"name": "xent 8 rows", "op": "xent", "rows": 8, "cols": 32000, "x": "fp32", "masked": 0},
        # the GPT's loss: every position of the micro-batch over its vocabulary
        {"name": "xent gpt step", "op": "xent", "rows": 8192, "cols": 32000, "x": "bf16", "masked": 0},
        # a large vocabulary of odd size, its unused tail masked
        {"name": "xent long odd", "op": "xent", "rows": 1021, "cols": 128257, "x": "bf16", "masked": 257},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gelu8", "wgrad8", "xent"])
    x = rng.choice(["fp32", "bf16", "fp16"])
    if op == "norm":
        cols = _between(rng, 64, 8192)
        rows = _between(rng, 1, min(32768, 2 ** 27 // cols // (2 if x == "fp32" else 1)))
        half = x != "fp32"
        return {"op": op, "rows": rows, "cols": cols, "x": x, "out": x if half else rng.choice(["fp32", "bf16"]),
                "weight": x if half else "fp32", "residual": rng.random() < 0.5, "pack": half and rng.random() < 0.5,
                "train": rng.random() < 0.8}
    if op == "gelu8":
        cols = _between(rng, 64, 16384)
        rows = _between(rng, 1, min(16384, 40_000_000 // cols))
        return {"op": op, "rows": rows, "cols": cols, "x": x, "form": rng.choice(["tanh", "none"]),
                "pack": x != "fp32" and rng.random() < 0.5}
    if op == "wgrad8":
        cols, outs = _between(rng, 32, 4096), _between(rng, 32, 4096)
        rows = _between(rng, 1, 16384)
        if x != "bf16":  # three times the products of bf16
            rows = min(rows, 4096)
        return {"op": op, "rows": rows, "cols": cols, "outs": outs, "x": x, "dw": rng.choice(["fp32", x]),
                "bias": rng.random() < 0.5}
    cols = _between(rng, 100, 131072)
    rows = _between(rng, 1, min(8192, 2 ** 28 // cols // (2 if x == "fp32" else 1)))
    return {"op": op, "rows": rows, "cols": cols, "x": x, "masked": rng.choice([0, cols // 16])}


def _size(kind):
    return 4 if kind == "fp32" else 2


def work(case):
    n, op = case["rows"] * case["cols"], case["op"]
    b = _size(case["x"])
    if op == "norm":
        out, w = _size(case["out"]), _size(case["weight"])
        r = out if case["residual"] else 0
        s = b if case["residual"] else 0
        total = n * (b + r + out + s) + 2 * case["cols"] * w  # x, residual -> y, sum
        if case["train"]:
            total += n * (out + s + b + r) + 2 * case["cols"] * w  # dy, dsum -> dx, dresidual; dweight, dbias
        return {"bytes": total, "flops": n * (22 if case["train"] else 8)}
    if op == "gelu8":  # x, dy -> y, dx (, y's checkpoint as values)
        return {"bytes": n * b * (5 if case["pack"] else 4), "flops": n * 40}
    if op == "wgrad8":
        m, k = case["outs"], case["cols"]
        return {"bytes": case["rows"] * (k + m) * b + m * k * _size(case["dw"]) + (m * 4 if case["bias"] else 0),
                "flops": 2 * case["rows"] * k * m}
    return {"bytes": 2 * n * b + 8 * case["rows"], "flops": n * 8}


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, d, op = case["rows"], case["cols"], case["op"]
    t = TYPES[case["x"]]
    s = {"case": case}
    if op == "norm":
        # a residual stream: columns of unlike scale and offset, rows that grow with depth
        col = torch.exp(0.5 * _normal(g, d))
        s["x"] = (_normal(g, n, d) * col + 0.3 * _normal(g, d)).to(t)
        s["weight"] = (1 + 0.2 * _normal(g, d)).to(TYPES[case["weight"]])
        s["bias"] = (0.1 * _normal(g, d)).to(TYPES[case["weight"]])
        s["residual"] = (0.3 * _normal(g, n, d)).to(TYPES[case["out"]]) if case["residual"] else None
        if case["train"]:
            s["dy"] = _normal(g, n, d).to(TYPES[case["out"]])
            s["ds"] = _normal(g, n, d).to(t) if case["residual"] else None
            for k in ("x", "weight", "bias", "residual"):
                if s[k] is not None:
                    s[k].requires_grad_()
    elif op == "gelu8":
        # pre-activations: most columns ordinary, a few large ones
        col = torch.where(torch.rand(d, generator=g, device="cuda") < 0.01, 6.0, 1.0)
        s["x"] = (_normal(g, n, d) * col).to(t).requires_grad_()
        s["dy"] = _normal(g, n, d).to(t)
    elif op == "wgrad8":
        # a layer's input and the gradient of its output; the latter spans the sizes of a loss averaged over tokens
        s["x"] = (_normal(g, n, d) * torch.exp(0.5 * _normal(g, d))).to(t)
        s["dy"] = (_normal(g, n, case["outs"]) * torch.exp(_normal(g, n, 1))).to(t)
    else:
        s["x"] = 2.0 * _normal(g, n, d)
        target = torch.randint(0, d - case["masked"], (n,), generator=g, device="cuda")
        # a model that has learnt something favours the target; a twentieth of the positions is padding
        s["x"].scatter_add_(1, target[:, None], 8.0 * torch.rand(n, 1, generator=g, device="cuda"))
        if case["masked"]:
            s["x"][:, d - case["masked"]:] = -math.inf
        pad = torch.rand(n, generator=g, device="cuda") < 0.05
        pad[0] = False
        s["target"] = torch.where(pad, IGNORE, target)
        s["x"] = s["x"].to(t).requires_grad_()
    return s


def run(state):
    case = state["case"]
    return (_RUN_OWN if own else _RUN_PLAIN)[case["op"]](case, state)


# --- through the framework ---------------------------------------------------

def _own_norm(case, s):
    from commux_b200 import ops

    kw = {"residual": s["residual"], "out_dtype": TYPES[case["out"]], "pack": case["pack"]}
    got = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS, **kw)
    got = got if isinstance(got, tuple) else (got,)
    y, total = got[0], got[1] if case["residual"] else None
    out = {"y": y.detach(), "sum": total.detach() if total is not None else None}
    if case["train"]:
        names = [k for k in ("x", "residual", "weight", "bias") if s[k] is not None]
        outs, grads = ([y, total], [s["dy"], s["ds"]]) if case["residual"] else ([y], [s["dy"]])
        out.update(("d" + k, v) for k, v in zip(names, torch.autograd.grad(outs, [s[k] for k in names], grads)))
    return out


def _own_gelu8(case, s):
    from commux_b200 import ops

    got = ops.gelu8(s["x"], approximate=case["form"], pack=case["pack"])
    y, kept = got if case["pack"] else (got, None)
    (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y.detach(), "dx": dx, "kept": kept.unpack() if kept is not None else None}


def _own_wgrad8(case, s):
    from commux_b200 import ops

    kept = ops.pack8(s["x"])
    got = ops.weight_grad8(s["dy"], kept, bias=case["bias"], out_dtype=TYPES[case["dw"]])
    return {"dw": got[0], "db": got[1]} if case["bias"] else {"dw": got}


def _own_xent(case, s):
    from commux_b200 import ops

    loss = ops.cross_entropy(s["x"], s["target"], ignore_index=IGNORE)
    (dx,) = torch.autograd.grad(loss, s["x"])
    return {"loss": loss.detach(), "dx": dx}


_RUN_OWN = {"norm": _own_norm, "gelu8": _own_gelu8, "wgrad8": _own_wgrad8, "xent": _own_xent}


# --- plain form: elementary operations in 32 bits, rounded once at the end ---

def _held(x):
    """The values that the 8-bit form of the rows of x (32 bits) stands for."""
    n, d = x.shape
    pad = -d % GROUP
    v = torch.nn.functional.pad(x, (0, pad)).view(n, -1, GROUP)
    big = v.abs().amax(2, keepdim=True)
    part, power = torch.frexp(big)  # big = part * 2^power, part in [0.5, 1)
    power = torch.where(part > 127 / 128, power - 6, power - 7).clamp(min=-126)
    power = torch.where(big == 0, -126, power)
    step = torch.ldexp(torch.ones_like(big), power)
    return (torch.round(v / step) * step).view(n, d + pad)[:, :d]


@torch.no_grad()
def _plain_norm(case, s):
    x, t, out_t = s["x"].float(), s["x"].dtype, TYPES[case["out"]]
    out = {"sum": None}
    if case["residual"]:  # the stream is what is handed on and normalised
        out["sum"] = (x + s["residual"].float()).to(t)
        x = out["sum"].float()
    w, b = s["weight"].float(), s["bias"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    hat = c * rstd
    out["y"] = (hat * w + b).to(out_t)
    if case["train"]:
        if case["pack"]:
            hat = _held(hat)
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + s["ds"].float()
            out["dresidual"] = dx.to(out_t)
        out["dx"] = dx.to(t)
        out["dweight"], out["dbias"] = (dy * hat).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["weight"].dtype)
    return out


@torch.no_grad()
def _plain_gelu8(case, s):
    t = s["x"].dtype
    x = s["x"].float()
    h = _held(x)
    if case["form"] == "tanh":
        a, c = math.sqrt(2 / math.pi), 0.044715
        y = 0.5 * x * (1 + torch.tanh(a * (x + c * x * x * x)))
        th = torch.tanh(a * (h + c * h * h * h))
        slope = 0.5 * (1 + th) + 0.5 * h * (1 - th * th) * a * (1 + 3 * c * h * h)
    else:
        y = 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
        slope = 0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    return {"y": y.to(t), "dx": (s["dy"].float() * slope).to(t), "kept": _held(y).to(t) if case["pack"] else None}


@torch.no_grad()
def _plain_wgrad8(case, s):
    dy = s["dy"].float()
    out = {"dw": (dy.t() @ _held(s["x"].float())).to(TYPES[case["dw"]])}
    if case["bias"]:
        out["db"] = dy.sum(0).to(TYPES[case["dw"]])
    return out


@torch.no_grad()
def _plain_xent(case, s):
    x, target = s["x"].float(), s["target"]
    valid = target != IGNORE
    at = torch.where(valid, target, 0)[:, None]
    count = valid.sum()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    rows = (top + torch.log(total) - x.gather(1, at))[:, 0]
    loss = torch.where(valid, rows, 0).sum() / count
    p = e / total
    p.scatter_add_(1, at, torch.full_like(total, -1.0))
    return {"loss": loss, "dx": (p * (valid / count)[:, None]).to(s["x"].dtype)}


_RUN_PLAIN = {"norm": _plain_norm, "gelu8": _plain_gelu8, "wgrad8": _plain_wgrad8, "xent": _plain_xent}


# --- 64 bits, from the definitions -------------------------------------------

def _exact_held(x):
    """What the 8-bit form stands for, in 64 bits: the step comes from log2, mended where that rounded."""
    out = torch.zeros_like(x)
    d = x.shape[1]
    for first in range(0, d, GROUP):
        v = x[:, first:first + GROUP]
        big = v.abs().amax(1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2(big / 127)).clamp(min=-126.0))
        step = torch.where(127 * step < big, 2 * step, step)
        half = step / 2
        step = torch.where((127 * half >= big) & (half >= 2.0 ** -126), half, step)
        out[:, first:first + GROUP] = torch.round(v / step) * step
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op, x = case["op"], s["x"].detach().double()
    if op == "norm":
        out = {"sum": None}
        if case["residual"]:
            out["sum"] = x + s["residual"].double()
            x = out["sum"].to(s["x"].dtype).double()
        w, b, d = s["weight"].double(), s["bias"].double(), case["cols"]
        mean = x.sum(1, keepdim=True) / d
        var = ((x - mean) ** 2).sum(1, keepdim=True) / d
        sd = torch.sqrt(var + EPS)
        hat = (x - mean) / sd
        out["y"] = hat * w + b
        if case["train"]:
            if case["pack"]:
                hat = _exact_held(hat)
            dy = s["dy"].double()
            dhat = dy * w
            dx = (d * dhat - dhat.sum(1, keepdim=True) - hat * (dhat * hat).sum(1, keepdim=True)) / (d * sd)
            if case["residual"]:
                dx = dx + s["ds"].double()
                out["dresidual"] = dx
            out["dx"], out["dweight"], out["dbias"] = dx, (dy * hat).sum(0), dy.sum(0)
        return out
    if op == "gelu8":
        h = _exact_held(x)
        if case["form"] == "tanh":
            # x (1 + tanh u) / 2 = x / (1 + exp(-2u))
            k = 2 * math.sqrt(2 / math.pi)
            y = x / (1 + torch.exp(-k * (x + 0.044715 * x ** 3)))
            sig = 1 / (1 + torch.exp(-k * (h + 0.044715 * h ** 3)))
            slope = sig + h * sig * (1 - sig) * k * (1 + 0.134145 * h ** 2)
        else:
            y = x * 0.5 * torch.erfc(-x / math.sqrt(2))
            slope = 0.5 * torch.erfc(-h / math.sqrt(2)) + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
        return {"y": y, "dx": s["dy"].double() * slope, "kept": _exact_held(y) if case["pack"] else None}
    if op == "wgrad8":
        dy = s["dy"].double()
        out = {"dw": torch.einsum("to,ti->oi", dy, _exact_held(x))}
        if case["bias"]:
            out["db"] = dy.sum(0)
        return out
    valid = (s["target"] != IGNORE).nonzero()[:, 0]
    at = s["target"][valid]
    logp = torch.log_softmax(x[valid], 1)
    loss = -logp[torch.arange(len(valid), device=x.device), at].sum() / len(valid)
    grad = torch.zeros_like(x)
    p = torch.exp(logp)
    p[torch.arange(len(valid), device=x.device), at] -= 1
    grad[valid] = p / len(valid)
    return {"loss": loss, "dx": grad}
