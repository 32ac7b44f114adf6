"""Measured cases of the operators that stand behind a reduction: what a training or serving
program does with a sum over ranks (or micro-batches) next.

* ``norm``: the partial sums of a row-parallel product are added, the residual is added, and the
  root-mean-square norm of the result goes out in the input's type or in e4m3 with scales.
* ``norm_backward``: its gradient with respect to the input and the weight.
* ``adamw``: one AdamW step over many tensors, states in 32 or in 8 bits.
* ``grad_norm``: the norm of all gradients and the coefficient that clips them.

``run`` has two forms of each: elementary torch operations (``own`` false) and this package's
operators (``own`` true).
"""
import functools
import math
import operator
import random

import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # least scale of a block or group, so that its reciprocal is finite
BLOCK = 256         # elements that share one scale in the 8-bit states
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "": 0}
BETA1, BETA2, EPS, LR, T, SEED = 0.9, 0.95, 1e-8, 1e-4, 1000, 20
NORM_EPS = 1e-6
MAX_NORM = 1.0


def listed():
    return [
        # One new token of a served model: latency is all that counts.
        dict(name="norm decode 1x8192", op="norm", rows=1, hidden=8192, type="bf16", weight="bf16",
             parts=1, residual=True, fp8=False, group=0),
        # A prompt, or a training micro-batch, through one norm.
        dict(name="norm prefill 8192x4096", op="norm", rows=8192, hidden=4096, type="bf16",
             weight="bf16", parts=1, residual=True, fp8=False, group=0),
        # The same where an 8-bit product follows that wants one scale per 128 columns.
        dict(name="norm fp8 16384x5120 g128", op="norm", rows=16384, hidden=5120, type="bf16",
             weight="fp32", parts=1, residual=True, fp8=True, group=128),
        # Partial sums of four ranks, a ragged batch, a hidden size that no vector divides, one
        # scale per token.
        dict(name="norm 4 parts 1013x5001 fp8", op="norm", rows=1013, hidden=5001, type="fp16",
             weight="fp16", parts=4, residual=True, fp8=True, group=0),
        # The gradient of the prefill's norm, with the gradient of the residual stream added.
        dict(name="backward 16384x4096", op="norm_backward", rows=16384, hidden=4096, type="bf16",
             weight="fp32", heads=0, stream=True),
        # The norm over each head of the queries, read out of a packed projection.
        dict(name="backward heads 8192x32x128", op="norm_backward", rows=8192, hidden=128,
             type="bf16", weight="bf16", heads=32, stream=False),
        # Small and odd in 32 bits.
        dict(name="backward 999x1001 fp32", op="norm_backward", rows=999, hidden=1001, type="fp32",
             weight="fp32", heads=0, stream=True),
        # The tensors of one transformer layer: 32-bit weights and states, 16-bit gradients, and the
        # 16-bit copy of the weights that the next step computes with.
        dict(name="adamw layer 4096", op="adamw", layer=4096, tensors=0, largest=0, layout=0,
             align=64, type="fp32", copy="bf16", grad="bf16", parts=1, bits=32),
        # A wider layer with states in 8 bits, and the gradients of two micro-batches.
        dict(name="adamw 8-bit layer 4608", op="adamw", layer=4608, tensors=0, largest=0, layout=0,
             align=BLOCK, type="fp32", copy="bf16", grad="bf16", parts=2, bits=8),
        # Many small tensors of odd sizes, packed without gaps (biases, norms, adapters).
        dict(name="adamw 64 small tensors", op="adamw", layer=0, tensors=64, largest=20000, layout=1,
             align=1, type="fp32", copy="", grad="fp32", parts=1, bits=32),
        # The norm of a layer's gradients before the step.
        dict(name="grad norm layer 4096", op="grad_norm", layer=4096, tensors=0, largest=0, layout=0,
             align=64, grad="bf16", parts=1),
        # The same for many small ones, summed over three micro-batches.
        dict(name="grad norm 200 small tensors", op="grad_norm", layer=0, tensors=200, largest=50000,
             layout=2, align=1, grad="fp32", parts=3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "adamw", "grad_norm"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op in ("norm", "norm_backward"):
        heads = rng.choice([0, 0, rng.randint(1, 40)]) if op == "norm_backward" else 0
        hidden = _log_int(rng, 32, 512) if heads else _log_int(rng, 16, 16384)
        rows = _log_int(rng, 1, max(1, min(32768, (24 << 20) // (hidden * max(1, heads)))))
        weight = rng.choice([kind, "fp32"])
        if op == "norm_backward":
            return dict(op=op, rows=rows, hidden=hidden, type=kind, weight=weight, heads=heads,
                        stream=rng.random() < 0.5)
        fp8 = rng.random() < 0.5
        return dict(op=op, rows=rows, hidden=hidden, type=kind, weight=weight,
                    parts=rng.choice([1, 1, 2, 3, 4, 8]), residual=rng.random() < 0.75, fp8=fp8,
                    group=rng.choice([0, 32, 64, 128]) if fp8 else 0)
    tensors = _log_int(rng, 1, 300)
    case = dict(op=op, layer=0, tensors=tensors, largest=_log_int(rng, 16, (48 << 20) // tensors),
                layout=rng.randrange(1 << 20), align=rng.choice([1, 8, 64]), grad=kind,
                parts=rng.choice([1, 1, 2, 4, 8]))
    if op == "adamw":
        case["bits"] = rng.choice([8, 32])
        case["type"] = rng.choice(["fp32", "fp32", "bf16", "fp16"])
        case["copy"] = rng.choice(["", "bf16", "fp16"]) if case["type"] == "fp32" else ""
        if case["bits"] == 8:
            case["align"] = BLOCK
    return case


# ---------------------------------------------------------------- inputs

def _sizes(case):
    if case["layer"]:
        h = case["layer"]
        return [3 * h * h, 3 * h, h * h, h, 4 * h * h, 4 * h, 4 * h * h, h, h, h]
    rng = random.Random(case["layout"])
    return [_log_int(rng, 1, case["largest"]) for _ in range(case["tensors"])]


def _starts(case):
    """Each tensor's first element in the flat buffers, and the buffers' length."""
    at, starts = 0, []
    for n in _sizes(case):
        starts.append(at)
        at += -(-n // case["align"]) * case["align"]
    return starts, at


def _views(flat, case, unit=1):
    starts, _ = _starts(case)
    return [flat[s // unit:s // unit + -(-n // unit)] for s, n in zip(starts, _sizes(case))]


def _mask(case, dev):
    """1 where a tensor is, 0 in the gaps between them."""
    starts, total = _starts(case)
    keep = torch.zeros(total, dtype=torch.float32, device=dev)
    for v in _views(keep, case):
        v.fill_(1.0)
    return keep


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if case["op"] in ("norm", "norm_backward"):
        kind, wkind = DTYPES[case["type"]], DTYPES[case["weight"]]
        rows, hidden = case["rows"], case["hidden"]
        state = {"case": case, "weight": (1 + 0.1 * randn(hidden)).to(wkind)}
        # Activations have a few columns that are much larger than the others.
        spread = torch.exp(0.5 * randn(hidden))
        if case["op"] == "norm":
            state["x"] = [(randn(rows, hidden) * spread).to(kind) for _ in range(case["parts"])]
            state["residual"] = (2 * randn(rows, hidden)).to(kind) if case["residual"] else None
            return state
        if case["heads"]:  # a third of a packed projection
            shape = (rows, case["heads"], hidden)
            h = (randn(rows, 3 * case["heads"], hidden) * spread).to(kind)[:, :case["heads"]]
        else:
            shape = (rows, hidden)
            h = (randn(*shape) * spread).to(kind)
        state["h"] = h
        state["rstd"] = (h.double().square().mean(-1) + NORM_EPS).rsqrt().float()
        state["dy"] = randn(*shape).to(kind)
        state["dh"] = randn(*shape).to(kind) if case["stream"] else None
        return state

    kind = DTYPES[case["grad"]]
    _, total = _starts(case)
    mask = _mask(case, dev)
    # Gradients differ by orders of magnitude between weights, and some weights get none.
    size = torch.exp(randn(total) - 7) * (torch.rand(total, device=dev, generator=gen) > 0.02) * mask
    flats = [(randn(total) * size).to(kind) for _ in range(case["parts"])]
    state = {"case": case, "flat_grads": flats,
             "grads": [list(g) for g in zip(*[_views(f, case) for f in flats])]}
    if case["op"] == "grad_norm":
        if own:
            from scc26_nccl_shim_b200.ops import optim
            state["norm"] = optim.GradNorm(state["grads"])
        return state

    state["p"] = (0.02 * randn(total) * mask).to(DTYPES[case["type"]])
    state["params"] = _views(state["p"], case)
    state["copy"] = state["p"].to(DTYPES[case["copy"]]) if case["copy"] else None
    state["copies"] = _views(state["copy"], case) if case["copy"] else None
    # Matrices decay, vectors do not.
    state["decay"] = [0.1 if n >= 4096 else 0.0 for n in _sizes(case)]
    m = 0.3 * size * randn(total)
    v = size * size * torch.exp(0.3 * randn(total))
    if case["bits"] == 32:
        state["m"], state["v"] = m, v
        state["states"] = (_views(m, case), _views(v, case))
    else:
        starts, _ = _starts(case)
        state["m"], state["ms"] = _nearest(m)
        state["v"], state["vs"] = _nearest(v.sqrt())
        state["states"] = (list(zip(_views(state["m"], case), _views(state["ms"], case, BLOCK))),
                           list(zip(_views(state["v"], case), _views(state["vs"], case, BLOCK))))
        # Which tensor each block of the flat buffers belongs to, and its number there.
        tensor = torch.zeros(total // BLOCK, dtype=torch.int32, device=dev)
        block = torch.zeros_like(tensor)
        for i, (t, b) in enumerate(zip(_views(tensor, case, BLOCK), _views(block, case, BLOCK))):
            t.fill_(i)
            b.copy_(torch.arange(b.numel(), device=dev))
        state["tensor_of"], state["block_of"] = tensor, block
    if own:
        from scc26_nccl_shim_b200.ops import optim
        state["optimizer"] = optim.AdamW(
            state["params"], state["grads"], betas=(BETA1, BETA2), eps=EPS,
            weight_decay=state["decay"], state="float32" if case["bits"] == 32 else "8bit",
            states=state["states"], copies=state["copies"], seed=SEED)
    return state


def _nearest(x):
    """Blocks of 256 in e4m3 and their scales, rounded to nearest (what a checkpoint holds)."""
    x = x.view(-1, BLOCK)
    scale = (x.abs().amax(1) / E4M3_MAX).clamp(min=TINY)
    return (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).view(-1), scale


# ---------------------------------------------------------------- the operators

def run(state):
    op = state["case"]["op"]
    if op == "norm":
        return _norm(state)
    if op == "norm_backward":
        return _norm_backward(state)
    if op == "adamw":
        return _adamw(state)
    return _grad_norm(state)


def _fold(parts):
    return functools.reduce(operator.add, [p.float() for p in parts])


def _norm(state):
    case = state["case"]
    if own:
        from scc26_nccl_shim_b200.ops import norm
        out = norm.add_rms_norm(state["x"], state["weight"], state["residual"], eps=NORM_EPS,
                                out_dtype=E4M3 if case["fp8"] else None, group=case["group"])
        return {"y": out.y, "scale": out.scale, "h": out.h, "rstd": out.rstd}
    kind = state["x"][0].dtype
    h = _fold(state["x"])
    if state["residual"] is not None:
        h = h + state["residual"].float()
    rstd = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + NORM_EPS)
    y = h * rstd * state["weight"].float()
    scale = None
    if case["fp8"]:
        hidden = y.shape[1]
        group = case["group"] or hidden
        width = -(-hidden // group) * group
        blocks = torch.nn.functional.pad(y, (0, width - hidden)).view(y.shape[0], -1, group)
        scale = (blocks.abs().amax(-1) / E4M3_MAX).clamp(min=TINY)
        q = (blocks * (1 / scale)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        y = q.view(y.shape[0], width)[:, :hidden]
    else:
        y = y.to(kind)
    return {"y": y, "scale": scale, "h": h.to(kind), "rstd": rstd[:, 0]}


def _norm_backward(state):
    if own:
        from scc26_nccl_shim_b200.ops import norm
        dx, dw = norm.add_rms_norm_backward(state["dy"], state["h"], state["weight"], state["rstd"],
                                            dh=state["dh"])
        return {"dx": dx, "dweight": dw}
    h, dy = state["h"].float(), state["dy"].float()
    rstd = state["rstd"][..., None]
    n = h * rstd
    g = dy * state["weight"].float()
    dx = rstd * (g - n * (g * n).mean(-1, keepdim=True))
    if state["dh"] is not None:
        dx = dx + state["dh"].float()
    dw = (dy * n).view(-1, h.shape[-1]).sum(0)
    return {"dx": dx.to(state["h"].dtype), "dweight": dw.to(state["weight"].dtype)}


def _grad_norm(state):
    if own:
        return state["norm"](MAX_NORM, scale=0.5)
    g = _fold(state["flat_grads"])
    total = 0.5 * torch.sqrt(g.square().sum(dtype=torch.float64))
    coefficient = 0.5 * (MAX_NORM / (total + 1e-6)).clamp(max=1.0)
    coefficient = torch.where(torch.isfinite(total), coefficient, torch.nan)  # no step is taken
    return torch.stack([total, coefficient]).float()


def _hash(tensor_of, block_of):
    """32 pseudo-random bits for each element of each block: a function of the seed, the step, the
    tensor's number and the element's number."""
    key = tensor_of * 0x3C6EF35F + _int32(SEED * 0x27D4EB2F + T * 0x165667B1)
    x = (block_of * BLOCK)[:, None] + torch.arange(BLOCK, dtype=torch.int32, device=block_of.device)
    x = x * _int32(0x9E3779B9) + key[:, None]
    x = x ^ ((x >> 16) & 0xFFFF)
    x = x * _int32(0xA5CB9243)
    x = x ^ ((x >> 15) & 0x1FFFF)
    x = x * _int32(0x5D8A37E5)
    return x ^ ((x >> 16) & 0xFFFF)


def _int32(x):
    return (x + (1 << 31)) % (1 << 32) - (1 << 31)


def _to_codes(x, u):
    """e4m3 by blocks of 256: the next value below x/scale + u steps, 0 <= u < 1."""
    scale = (x.abs().amax(1, keepdim=True) / E4M3_MAX).clamp(min=TINY)
    z = (x.abs() * (1 / scale)).clamp(max=E4M3_MAX)
    step = torch.exp2((torch.frexp(z)[1] - 4).clamp(min=-9).float())
    return (torch.floor(z / step + u) * step).copysign(x), scale


def _adamw(state):
    case = state["case"]
    if own:
        state["optimizer"].step(T, LR, scale=0.5)
    else:
        p = state["p"]
        g = _fold(state["flat_grads"]) * 0.5
        c1, c2 = 1 - BETA1 ** T, 1 - BETA2 ** T
        if case["bits"] == 32:
            m = state["m"].mul_(BETA1).add_(g * (1 - BETA1))
            v = state["v"].mul_(BETA2).add_(g * g * (1 - BETA2))
        else:
            g = g.view(-1, BLOCK)
            m = state["m"].view(-1, BLOCK).float() * state["ms"][:, None]
            r = state["v"].view(-1, BLOCK).float() * state["vs"][:, None]
            m = m * BETA1 + g * (1 - BETA1)
            v = r * r * BETA2 + g * g * (1 - BETA2)
            bits = _hash(state["tensor_of"], state["block_of"])
            q, scale = _to_codes(m, ((bits >> 16) & 0xFFFF).float() * 2.0 ** -16)
            state["m"].copy_(q.view(-1))
            state["ms"].copy_(scale[:, 0])
            q, scale = _to_codes(torch.sqrt(v), (bits & 0xFFFF).float() * 2.0 ** -16)
            q = torch.where(v > 0, q.clamp(min=2.0 ** -9), q)
            state["v"].copy_(q.view(-1))
            state["vs"].copy_(scale[:, 0])
            m, v = m.view(-1), v.view(-1)
        update = m * (LR / c1) / (torch.sqrt(v) * (1 / math.sqrt(c2)) + EPS)
        if p.dtype == torch.float32:
            torch._foreach_mul_(state["params"], [1 - LR * d for d in state["decay"]])
            p.sub_(update)
        else:
            wide = p.float()
            torch._foreach_mul_(_views(wide, case), [1 - LR * d for d in state["decay"]])
            p.copy_(wide.sub_(update))
        if state["copy"] is not None:
            state["copy"].copy_(p)
    names = ["p", "m", "v", "copy"] + (["ms", "vs"] if case["bits"] == 8 else [])
    return {k: state[k] for k in names}


# ---------------------------------------------------------------- costs and the definition

def work(case):
    if case["op"] in ("norm", "norm_backward"):
        rows = case["rows"] * max(1, case.get("heads", 0))
        n, e, w = rows * case["hidden"], BYTES[case["type"]], BYTES[case["weight"]] * case["hidden"]
        if case["op"] == "norm_backward":
            return {"bytes": n * e * (3 + case["stream"]) + 4 * rows + 2 * w, "flops": 10 * n}
        sums = case["parts"] + case["residual"] > 1
        out = 1 if case["fp8"] else e
        scales = rows * -(-case["hidden"] // (case["group"] or case["hidden"])) if case["fp8"] else 0
        return {"bytes": n * (e * (case["parts"] + case["residual"] + sums) + out) + 4 * (rows + scales) + w,
                "flops": (5 + case["parts"]) * n}
    n, e = sum(_sizes(case)), BYTES[case["grad"]]
    if case["op"] == "grad_norm":
        return {"bytes": n * e * case["parts"] + 8, "flops": (1 + case["parts"]) * n}
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": int(n * (2 * BYTES[case["type"]] + BYTES[case["copy"]] + e * case["parts"] + states)),
            "flops": (15 + case["parts"]) * n}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["op"] == "norm_backward":
        h, dy, w, r = s["h"].double(), s["dy"].double(), s["weight"].double(), s["rstd"].double()
        inner = torch.einsum("...i,...i,i->...", dy, h, w) * r.pow(3) / h.shape[-1]
        dx = dy * w * r.unsqueeze(-1) - h * inner.unsqueeze(-1)
        dx = dx if s["dh"] is None else dx + s["dh"].double()
        return {"dx": dx, "dweight": (dy * h * r.unsqueeze(-1)).reshape(-1, h.shape[-1]).sum(0)}
    if case["op"] == "grad_norm":
        total = 0.5 * torch.linalg.vector_norm(sum(f.double() for f in s["flat_grads"]))
        clipped = 0.5 * MAX_NORM / (total + 1e-6)
        return torch.stack([total, torch.minimum(clipped, torch.full_like(clipped, 0.5))])
    return _exact_adamw(case, s)


def _exact_norm(case, s):
    h = torch.zeros_like(s["x"][0], dtype=torch.float64)
    for part in s["x"] + ([s["residual"]] if case["residual"] else []):
        h += part.double()
    rstd = (h.pow(2).sum(1) / case["hidden"] + NORM_EPS).pow(-0.5)
    y = h * rstd[:, None] * s["weight"].double()
    if not case["fp8"]:
        return {"y": y, "scale": None, "h": h, "rstd": rstd}
    parts = [c.abs().max(1).values for c in y.split(case["group"] or case["hidden"], 1)]
    scale = (torch.stack(parts, 1) / E4M3_MAX).clamp(min=TINY)
    wide = scale.repeat_interleave(case["group"] or case["hidden"], 1)[:, :case["hidden"]]
    q = (y / wide).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).double()
    return {"y": q, "scale": scale, "h": h, "rstd": rstd}


def _exact_codes(x, u):
    x = x.view(-1, BLOCK)
    scale = (x.abs().max(1).values / E4M3_MAX).clamp(min=TINY)
    z = (x.abs() / scale[:, None]).clamp(max=E4M3_MAX)
    exponent = torch.floor(torch.log2(z.clamp(min=2.0 ** -9)))
    step = torch.pow(2.0, exponent.clamp(min=-6) - 3)
    return (z / step + u).floor() * step * torch.sign(x), scale


def _exact_adamw(case, s):
    sizes, (starts, total) = _sizes(case), _starts(case)
    g = sum(f.double() for f in s["flat_grads"]) * 0.5
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = s["m"].double() * s["ms"].double().repeat_interleave(BLOCK)
        v = (s["v"].double() * s["vs"].double().repeat_interleave(BLOCK)) ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = s["p"].double()
    for start, n, decay in zip(starts, sizes, s["decay"]):
        p[start:start + n] *= 1 - LR * decay
    p -= LR * (m / (1 - BETA1 ** T)) / ((v / (1 - BETA2 ** T)).sqrt() + EPS)
    out = {"p": p, "m": m, "v": v, "copy": p if case["copy"] else None}
    if case["bits"] == 8:
        bits = torch.zeros(total, dtype=torch.int64, device=p.device)
        low = 0xFFFFFFFF
        for i, (start, n) in enumerate(zip(starts, sizes)):
            n = -(-n // BLOCK) * BLOCK
            x = torch.arange(n, dtype=torch.int64, device=p.device)
            x = (x * 0x9E3779B9 + i * 0x3C6EF35F + SEED * 0x27D4EB2F + T * 0x165667B1) & low
            x = ((x ^ (x >> 16)) * 0xA5CB9243) & low
            x = ((x ^ (x >> 15)) * 0x5D8A37E5) & low
            bits[start:start + n] = x ^ (x >> 16)
        bits = bits.view(-1, BLOCK)
        q, out["ms"] = _exact_codes(m, (bits >> 16).double() / 65536)
        out["m"] = q.view(-1)
        root = v.sqrt()
        q, out["vs"] = _exact_codes(root, (bits & 0xFFFF).double() / 65536)
        out["v"] = torch.where(root > 0, q.view(-1).clamp(min=2.0 ** -9), q.view(-1))
    return out
