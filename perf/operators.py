"""Workloads of the gradient-norm and 4-bit weight operators.

Four operators, in two pairs:

  norm    the global norm of a list of gradient tensors (L1, L2 or the largest
          magnitude), one float32
  clip    the same norm, then every gradient scaled so that the global norm is
          at most max_norm, in place or into other tensors
  quant   a weight matrix to 4-bit codes with one scale (and, where asked, one
          zero point) per group of columns, and back to the values they stand for
  matvec  a few rows of activations times a 4-bit weight matrix

`run` computes them in elementary torch operations while `own` is false and
through quickruncuda_b200 while it is true.  `exact` gives the same answers
from the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ORDERS = {"1": 1.0, "2": 2.0, "inf": math.inf}


# -- cases --------------------------------------------------------------------
# Gradient lists are written as "count*dims:type" items, e.g. "24*16x2048:bf16".

def listed():
    return [
        # the gains of the normalisations alone, tuned on their own: the smallest call
        {"name": "norm_gains_f32", "op": "norm", "grads": "33*2048:f32", "ord": "2"},
        # one flat gradient bucket of a sharded optimizer, 1e9 floats
        {"name": "norm_flat_1e9_f32", "op": "norm", "grads": "1*1000000000:f32", "ord": "2"},
        # largest gradient of a model with odd sizes, watched for fp16 overflow
        {"name": "norm_odd_inf_f16", "op": "norm",
         "grads": "7*1023x5001:f16 7*5001x1023:f16 14*5001:f16 1*333x77:f16", "ord": "inf"},
        # low-rank adapters of 24 blocks, gradients clipped where they lie
        {"name": "clip_adapters_bf16", "op": "clip", "grads": "24*16x2048:bf16 24*2048x16:bf16", "ord": "2",
         "to": "place"},
        # a whole 12-block model of width 2048 with its embedding: bf16 gradients, clipped
        # into the float32 gradients that the optimizer reads
        {"name": "clip_blocks_bf16_to_f32", "op": "clip",
         "grads": "1*32000x2048:bf16 12*6144x2048:bf16 12*2048x2048:bf16 12*11264x2048:bf16 12*2048x5632:bf16"
                  " 1*25x2048:f32", "ord": "2", "to": "f32"},
        # float32 gradients of a small model with odd sizes, about the size of the L2
        {"name": "clip_odd_f32", "op": "clip", "grads": "9*777x1301:f32 9*1301x777:f32 5*1301:f32 1*1:f32",
         "ord": "2", "to": "same"},
        # the weight matrix of the FP8 quantize workload, to 4 bits
        {"name": "quant_16384x8192_bf16", "op": "quant", "n": 16384, "k": 8192, "type": "bf16", "group": 128,
         "symmetric": True},
        # odd sizes, the smallest group, with zero points
        {"name": "quant_odd_f16", "op": "quant", "n": 1021, "k": 2999, "type": "f16", "group": 32,
         "symmetric": False},
        # one token through a square projection: latency
        {"name": "matvec_4096x4096_bf16", "op": "matvec", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "group": 128,
         "symmetric": True, "bias": False, "out": "same"},
        # one token through the output layer, larger than the L2, logits in float32
        {"name": "matvec_65536x8192_bf16", "op": "matvec", "m": 1, "n": 65536, "k": 8192, "type": "bf16",
         "group": 128, "symmetric": True, "bias": False, "out": "f32"},
        # five streams, odd sizes, zero points and a bias
        {"name": "matvec_odd_f16", "op": "matvec", "m": 5, "n": 5003, "k": 11007, "type": "f16", "group": 32,
         "symmetric": False, "bias": True, "out": "same"},
        # a decode batch of 32 streams
        {"name": "matvec_batch_bf16", "op": "matvec", "m": 32, "n": 16384, "k": 8192, "type": "bf16", "group": 64,
         "symmetric": False, "bias": False, "out": "same"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "quant", "matvec"])
    if op in ("norm", "clip"):
        left, items = _spread(rng, 1000, 400_000_000), []
        for _ in range(rng.randint(1, 5)):
            count = _spread(rng, 1, 64 if op == "norm" else 12)
            each = max(1, left // (5 * count))
            cols = _spread(rng, 1, max(1, min(each, 9000)))
            rows = max(1, each // cols)
            dims = "%dx%d" % (rows, cols) if rng.random() < 0.8 else "%d" % (rows * cols)
            items.append("%d*%s:%s" % (count, dims, rng.choice(list(TYPES))))
        case = {"op": op, "grads": " ".join(items), "ord": rng.choice(["2", "2", "1", "inf"])}
        if op == "clip":
            case["to"] = rng.choice(["place", "same", "f32"])
        return case
    kind = {"op": op, "type": rng.choice(["bf16", "f16"]), "group": rng.choice([32, 64, 128, 256]),
            "symmetric": rng.random() < 0.5}
    if op == "quant":
        n = _spread(rng, 1, 16384)
        return dict(kind, n=n, k=_spread(rng, 1, min(16384, (1 << 27) // n)))
    n = _spread(rng, 16, 65536)
    k = _spread(rng, 33, min(32768, (1 << 28) // n))
    m = _spread(rng, 1, min(32, (1 << 32) // (n * k)))
    return dict(kind, m=m, n=n, k=k, bias=rng.random() < 0.5, out=rng.choice(["same", "f32"]))


def _shapes(case):
    """[(shape, torch type)] of a gradient list."""
    found = []
    for item in case["grads"].split():
        count, rest = item.split("*")
        dims, kind = rest.split(":")
        found += [(tuple(int(d) for d in dims.split("x")), TYPES[kind])] * int(count)
    return found


def _groups(case):
    return -(-case["k"] // case["group"])


# -- inputs -------------------------------------------------------------------

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    made = {}
    if case["op"] in ("norm", "clip"):
        # magnitudes differ from tensor to tensor, as gradients' do
        made["grads"] = []
        for i, (shape, kind) in enumerate(_shapes(case)):
            grad = torch.randn(shape, generator=gen, device="cuda").mul_(2.0 ** -(4 + i % 7))
            made["grads"].append(grad.to(kind))
        # a step that has to be clipped: the norm is well above the limit
        count = sum(g.numel() for g in made["grads"])
        made["max_norm"] = {"1": 0.0006 * count, "2": 0.003 * math.sqrt(count), "inf": 0.002}[case["ord"]]
    elif case["op"] == "quant":
        w = torch.randn(case["n"], case["k"], generator=gen, device="cuda").mul_(0.02)
        made["w"] = w.to(TYPES[case["type"]])
    else:
        # codes, scales and zero points as a checkpoint of 4-bit weights holds them
        n, k, g, kind = case["n"], case["k"], _groups(case), TYPES[case["type"]]
        made["codes"] = torch.randint(0, 16, (n, k), generator=gen, device="cuda", dtype=torch.uint8)
        made["scales"] = (torch.rand(g, n, generator=gen, device="cuda") * 0.008 + 0.002).to(kind)
        made["zeros"] = None
        if not case["symmetric"]:
            made["zeros"] = torch.randint(5, 11, (g, n), generator=gen, device="cuda", dtype=torch.uint8)
        made["x"] = torch.randn(case["m"], k, generator=gen, device="cuda").to(kind)
        made["bias"] = torch.randn(n, generator=gen, device="cuda").to(kind) if case["bias"] else None
    return made


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["op"] == "clip" and case["to"] == "place":
        state["fresh"] = state["grads"]
        state["grads"] = [torch.empty_like(g) for g in state["fresh"]]
    if not own:
        return state
    import quickruncuda_b200 as q
    if case["op"] in ("norm", "clip"):
        if case["op"] == "clip" and case["to"] != "place":
            state["out"] = [torch.empty_like(g, dtype=torch.float32 if case["to"] == "f32" else g.dtype)
                            for g in state["grads"]]
        state["list"] = q.TensorList(state["grads"], out=state.get("out"))
    elif case["op"] == "matvec":
        state["w4"] = q.Weight4.from_codes(state.pop("codes"), state.pop("scales"), state.pop("zeros"),
                                           group=case["group"])
    return state


# -- one pass -----------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case = state["case"]
    op = case["op"]
    if op == "norm":
        return state["list"].norm(ORDERS[case["ord"]])
    if op == "clip":
        if "fresh" in state:
            torch._foreach_copy_(state["grads"], state["fresh"])    # the backward pass writes the gradients
        norm = state["list"].clip_norm(state["max_norm"], ORDERS[case["ord"]])
        return norm, state.get("out", state["grads"])
    if op == "quant":
        import quickruncuda_b200 as q
        w4 = q.quant_w4(state["w"], group=case["group"], symmetric=case["symmetric"])
        return w4.dequant(), w4.scales, w4.zeros
    return state["w4"].matvec(state["x"], bias=state["bias"],
                              out_dtype=torch.float32 if case["out"] == "f32" else None)


def _plain_norm(grads, order):
    """The norm in 64 bits: sums of up to 1e9 terms."""
    parts = []
    for g in grads:
        for piece in g.reshape(-1).split(1 << 27):
            a = piece.float().abs()
            if order == "inf":
                parts.append(a.max().double())
            else:
                parts.append((a if order == "1" else a * a).sum(dtype=torch.float64))
    parts = torch.stack(parts)
    if order == "inf":
        return parts.max()
    return parts.sum() if order == "1" else parts.sum().sqrt()


def _plain_scale(value, kind):
    """value (64 bits) rounded once to kind: its border cases decide codes."""
    bits, low = (8, -125) if kind == torch.bfloat16 else (11, -13)
    _, e = torch.frexp(value)
    step = torch.ldexp(torch.ones_like(value), e.clamp(min=low) - bits)
    return (torch.round(value / step) * step).float()


def _plain_quant(w, group, symmetric):
    n, k = w.shape
    g = -(-k // group)
    x = torch.zeros(n, g * group, device=w.device)
    x[:, :k] = w.float()
    x = x.view(n, g, group)
    if symmetric:
        scale = _plain_scale(x.abs().amax(2).double() / 7.0, w.dtype)
        zero = torch.full_like(scale, 8.0)
        low, high = 1.0, 15.0
    else:
        least, most = x.amin(2).clamp(max=0.0), x.amax(2).clamp(min=0.0)
        scale = _plain_scale((most.double() - least.double()) / 15.0, w.dtype)
        low, high = 0.0, 15.0
    inverse_ok = scale > 0
    safe = torch.where(inverse_ok, scale, torch.ones_like(scale))
    if not symmetric:
        zero = torch.where(inverse_ok, torch.round(-least / safe), torch.zeros_like(scale)).clamp(0.0, 15.0)
    # 32-bit quotients of 16-bit numbers keep their side of every border k + 1/2
    code = torch.where(inverse_ok[..., None], torch.round(x / safe[..., None]), torch.zeros_like(x)) + zero[..., None]
    values = (code.clamp(low, high) - zero[..., None]) * scale[..., None]
    values = values.view(n, g * group)[:, :k].to(w.dtype).contiguous()
    scales = scale.t().contiguous().to(w.dtype)
    return values, scales, None if symmetric else zero.t().contiguous().to(torch.uint8)


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "norm":
        return _plain_norm(state["grads"], case["ord"]).float()
    if op == "clip":
        grads = state["grads"]
        if "fresh" in state:
            torch._foreach_copy_(grads, state["fresh"])
        norm = _plain_norm(grads, case["ord"])
        coef = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
        if "fresh" in state:
            for g in grads:
                g.copy_(g.float() * coef)
            return norm.float(), grads
        return norm.float(), [(g.float() * coef).to(torch.float32 if case["to"] == "f32" else g.dtype) for g in grads]
    if op == "quant":
        return _plain_quant(state["w"], case["group"], case["symmetric"])
    codes, group, k = state["codes"], case["group"], case["k"]
    zero = 8.0 if state["zeros"] is None else state["zeros"].float().t().repeat_interleave(group, 1)[:, :k]
    w = (codes.float() - zero) * state["scales"].float().t().repeat_interleave(group, 1)[:, :k]
    y = state["x"].float() @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y if case["out"] == "f32" else y.to(state["x"].dtype)


# -- what one pass cannot do without -------------------------------------------

def work(case):
    op = case["op"]
    if op in ("norm", "clip"):
        shapes = [(math.prod(s), t.itemsize) for s, t in _shapes(case)]
        count = sum(c for c, _ in shapes)
        read = sum(c * b for c, b in shapes)
        if op == "norm":
            return {"bytes": read + 4, "flops": 2 * count}
        wrote = 4 * count if case["to"] == "f32" else read
        return {"bytes": read + wrote + 4, "flops": 3 * count}
    n, k, g = case["n"], case["k"], _groups(case)
    side = g * n * (2 if case["symmetric"] else 3)
    if op == "quant":
        return {"bytes": 2 * n * k * 2 + side, "flops": 4 * n * k}
    m = case["m"]
    size = 4 if case["out"] == "f32" else 2
    return {"bytes": n * k // 2 + side + 2 * m * k + size * m * n + (2 * n if case["bias"] else 0),
            "flops": 2 * m * n * k}


# -- the definitions in 64 bits -------------------------------------------------

def exact(case, seed):
    state, op = _inputs(case, seed), case["op"]
    if op in ("norm", "clip"):
        grads = state["grads"]
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for g in grads:
            flat = g.flatten()
            for at in range(0, flat.numel(), 1 << 26):
                d = flat[at:at + (1 << 26)].to(torch.float64)
                if case["ord"] == "inf":
                    total = torch.maximum(total, torch.maximum(d.max(), -d.min()))
                elif case["ord"] == "1":
                    total = total + torch.where(d < 0, -d, d).sum()
                else:
                    total = total + torch.dot(d, d)
        norm = torch.sqrt(total) if case["ord"] == "2" else total
        if op == "norm":
            return norm
        coef = torch.minimum(torch.ones_like(norm), state["max_norm"] / (norm + 1e-6))
        return norm, [g.double() * coef for g in grads]
    if op == "quant":
        return _exact_quant(state["w"].double(), case)
    codes, scales, zeros = state["codes"], state["scales"], state["zeros"]
    x, group = state["x"].double(), case["group"]
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    for j in range(_groups(case)):
        cols = slice(j * group, min(case["k"], (j + 1) * group))
        zero = 8.0 if zeros is None else zeros[j].double()[:, None]
        y += (x[:, cols] @ (codes[:, cols].double() - zero).t()) * scales[j].double()
    return y if state["bias"] is None else y + state["bias"].double()


def _exact_quant(w, case):
    """The codes follow from the scale as it is kept, in 16 bits, so its
    rounding is part of the definition."""
    group, digits, least_exponent = (case["group"],) + ((8, -126) if case["type"] == "bf16" else (11, -14))
    values = torch.empty_like(w)
    scales, zeros = [], []
    for j in range(_groups(case)):
        part = w[:, j * group:(j + 1) * group]
        top, bottom = part.max(1).values.clamp(min=0), part.min(1).values.clamp(max=0)
        s = torch.maximum(top, -bottom) / 7 if case["symmetric"] else (top - bottom) / 15
        exponent = torch.floor(torch.log2(s.clamp(min=1e-300)))
        exponent = torch.where(torch.exp2(exponent) > s, exponent - 1, exponent)
        exponent = torch.where(torch.exp2(exponent + 1) <= s, exponent + 1, exponent).clamp(min=least_exponent)
        unit = torch.exp2(exponent - (digits - 1))
        s = torch.round(s / unit) * unit
        whole = s > 0
        d = torch.where(whole, s, torch.ones_like(s))
        if case["symmetric"]:
            code = torch.round(part / d[:, None]).clamp(-7, 7)
        else:
            z = torch.where(whole, torch.round(-bottom / d), torch.zeros_like(s)).clamp(0, 15)
            code = (torch.round(part / d[:, None]) + z[:, None]).clamp(0, 15) - z[:, None]
            zeros.append(z)
        values[:, j * group:(j + 1) * group] = torch.where(whole[:, None], code * s[:, None], torch.zeros_like(part))
        scales.append(s)
    return values, torch.stack(scales), None if case["symmetric"] else torch.stack(zeros)
