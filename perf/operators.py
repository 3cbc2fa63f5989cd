"""The 4-bit and mixture-of-experts operators, case by case: their inputs, their plain forms and the
calls a user makes.

Five operators of one serving and training path, the experts' feed-forward network in 4 bits:

* ``quantise``: bf16 / fp16 / fp32 to MXFP4 (blocks of 32 values of 4 bits, E2M1, that share a
  power-of-two scale, E8M0), along the rows or along the columns, behind the group-256 rotation or
  not, and read back;
* ``linear``: activations quantised and multiplied with an MXFP4 weight (serving);
* ``train``: the same with both operands quantised each step, and both gradients;
* ``route``: tokens sorted by expert, gathered, and combined again with their weights, and the
  gradients of both;
* ``experts``: tokens quantised in sorted order and multiplied with their expert's weight, and the
  gradients.

The MXFP4 arithmetic is exact up to the sums: a block's scale is 2^(floor(log2 amax) - 2) (at least
2^-127), the values are divided by it, which is exact, and rounded to the nearest of 0, 0.5, 1, 1.5,
2, 3, 4, 6 (ties to the even code, values above 6 to 6).
"""

import math

import torch

own = False

BLOCK = 32      # values that share a scale
GROUP = 256     # the rotation's group
TILE = 128      # rows of a scale tile, and contraction values of one
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoded token's activation, the smallest call there is: latency
        {"name": "quantise_token", "op": "quantise", "rows": 1, "cols": 4096, "dtype": "bf16",
         "rotate": True, "columns": False},
        # a prefill's activations: bandwidth
        {"name": "quantise_batch", "op": "quantise", "rows": 16384, "cols": 4096, "dtype": "bf16",
         "rotate": True, "columns": False},
        # a gradient quantised along the tokens for the weight gradient, an odd number of them
        {"name": "quantise_columns", "op": "quantise", "rows": 4097, "cols": 5120, "dtype": "f32",
         "rotate": False, "columns": True},
        # one decoded token through an up-projection: the weight is read once, latency counts
        {"name": "linear_token", "op": "linear", "rows": 1, "inner": 4096, "outer": 14336,
         "dtype": "bf16", "rotate": True, "bias": False},
        # a short prompt, a number of rows that fills no tile, fp16 and a bias
        {"name": "linear_prompt", "op": "linear", "rows": 77, "inner": 1280, "outer": 10240,
         "dtype": "f16", "rotate": False, "bias": True},
        # a prefill through the same up-projection: the tensor cores
        {"name": "linear_batch", "op": "linear", "rows": 8192, "inner": 4096, "outer": 14336,
         "dtype": "bf16", "rotate": True, "bias": True},
        # a training step of one layer: output, input gradient, weight gradient
        {"name": "train_step", "op": "train", "rows": 4096, "inner": 1280, "outer": 5120,
         "dtype": "bf16", "rotate": True},
        # a smaller one in fp32 over a ragged batch
        {"name": "train_ragged", "op": "train", "rows": 1000, "inner": 1024, "outer": 1024,
         "dtype": "f32", "rotate": False},
        # one token's routing while decoding: eight rows out and back
        {"name": "route_token", "op": "route", "tokens": 1, "width": 4096, "experts": 64, "top": 8,
         "dtype": "bf16", "train": False, "dropped": False},
        # a training step's routing with its gradients, padding tokens among them (no expert)
        {"name": "route_train", "op": "route", "tokens": 16384, "width": 2048, "experts": 128,
         "top": 8, "dtype": "bf16", "train": True, "dropped": True},
        # a decoding batch: few rows an expert, the weights' bytes count
        {"name": "experts_decode", "op": "experts", "tokens": 16, "inner": 2048, "outer": 2816,
         "experts": 64, "top": 4, "dtype": "bf16", "rotate": True, "train": False},
        # a training step of the experts' product: both gradients
        {"name": "experts_train", "op": "experts", "tokens": 8192, "inner": 2048, "outer": 5632,
         "experts": 8, "top": 2, "dtype": "bf16", "rotate": True, "train": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["quantise", "linear", "linear", "train", "route", "experts", "experts"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        rotate = dtype != "f32" and rng.random() < 0.6

        def width(low, high):
            w = _spread(rng, low, high)  # even half of the time, odd ones among the others
            return max(GROUP, w // GROUP * GROUP) if rotate else w // 32 * 32 if rng.random() < 0.5 else w

        if op == "quantise":
            columns = not rotate and rng.random() < 0.5
            case = {"op": op, "rows": _spread(rng, 1, 16384), "cols": width(64, 16384),
                    "dtype": dtype, "rotate": rotate, "columns": columns}
            if columns:
                case["cols"] = _spread(rng, 1, 8192)
        elif op == "linear":
            case = {"op": op, "rows": _spread(rng, 1, 8192), "inner": width(256, 14336),
                    "outer": _spread(rng, 16, 14336), "dtype": dtype, "rotate": rotate,
                    "bias": rng.random() < 0.5}
        elif op == "train":
            case = {"op": op, "rows": _spread(rng, 1, 8192), "inner": width(256, 5120),
                    "outer": _spread(rng, 64, 8192), "dtype": dtype, "rotate": rotate}
        elif op == "route":
            experts = _spread(rng, 2, 256)
            case = {"op": op, "tokens": _spread(rng, 1, 16384), "width": _spread(rng, 64, 8192),
                    "experts": experts, "top": min(experts, rng.randint(1, 8)), "dtype": dtype,
                    "train": rng.random() < 0.5, "dropped": rng.random() < 0.5}
        else:
            experts = _spread(rng, 4, 64)
            case = {"op": op, "tokens": _spread(rng, 1, 8192), "inner": width(256, 4096),
                    "outer": _spread(rng, 64, 8192), "experts": experts,
                    "top": min(experts, rng.randint(1, 4)), "dtype": dtype, "rotate": rotate,
                    "train": rng.random() < 0.4}
            if case["experts"] * case["inner"] * case["outer"] > 400_000_000:
                continue
        if _cost(case) <= most and 3 * 1024 not in case.values():
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _size(case):
    return {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]


def work(case):
    s, q = _size(case), 0.5 + 1 / BLOCK
    op = case["op"]
    if op == "quantise":  # read, 4 bits and a scale written, both read back, the values written
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * s + 2 * q), "flops": n * (30 if case["rotate"] else 4)}
    if op == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"bytes": m * k * s + n * k * q + m * n * s + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "train":  # x, w, dy in; y, dx, dw out
        m, k, n = case["rows"], case["inner"], case["outer"]
        return {"bytes": 2 * s * (m * k + n * k + m * n), "flops": 6 * m * n * k}
    if op == "route":
        t, h, p = case["tokens"], case["width"], case["tokens"] * case["top"]
        forward = s * (t * h + p * h) + s * (p * h + t * h) + 4 * p * 4
        backward = s * (p * h + t * h) + s * (t * h + p * h + p * h) + 4 * p * 2
        return {"bytes": forward + (backward if case["train"] else 0),
                "flops": p * h * (2 + (5 if case["train"] else 0))}
    t, k, n, e = (case[i] for i in ("tokens", "inner", "outer", "experts"))
    p = t * case["top"]
    used = min(e, p)
    if not case["train"]:
        return {"bytes": t * k * s + used * n * k * q + p * n * s + 4 * p, "flops": 2 * p * n * k}
    return {"bytes": s * (2 * t * k + 2 * e * n * k + 2 * p * n) + 4 * p, "flops": 6 * p * n * k}


# ------------------------------------------------------------------------------------------ inputs

def _normal(g, shape, dtype, scale=1.0, outliers=False):
    x = torch.randn(shape, generator=g, device="cuda") * scale
    if outliers:  # a few channels far above the others, as activations have them
        count = max(1, shape[-1] // 128)
        at = torch.randint(0, shape[-1], (count,), generator=g, device="cuda")
        x[..., at] *= 20
    return x.to(dtype)


def _routing(g, case):
    """Expert ids [tokens, top], some experts asked for more than others; -1: no expert."""
    t, e = case["tokens"], case["experts"]
    scores = torch.randn(t, e, generator=g, device="cuda")
    scores += 0.7 * torch.randn(e, generator=g, device="cuda")
    best = scores.topk(case["top"], dim=1)
    ids = best.indices.to(torch.int32)
    if case.get("dropped"):
        ids[torch.rand(t, generator=g, device="cuda") < 0.05] = -1
    return ids, torch.softmax(best.values, dim=1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]
    state = dict(case)
    if op == "quantise":
        state["x"] = _normal(g, (case["rows"], case["cols"]), dtype, outliers=True)
    elif op == "linear":
        state["x"] = _normal(g, (case["rows"], case["inner"]), dtype, outliers=True)
        w = _normal(g, (case["outer"], case["inner"]), dtype, 0.02)
        state["codes"], state["scales"] = _stored(_turned(w.float(), dtype) if case["rotate"] else w)
        state["bias"] = 0.01 * torch.randn(case["outer"], generator=g, device="cuda") if case["bias"] else None
    elif op == "train":
        state["x"] = _normal(g, (case["rows"], case["inner"]), dtype, outliers=True).requires_grad_()
        state["w"] = _normal(g, (case["outer"], case["inner"]), dtype, 0.02).requires_grad_()
        state["dy"] = _normal(g, (case["rows"], case["outer"]), dtype, 1e-3)
    elif op == "route":
        rows, h = case["tokens"] * case["top"], case["width"]
        state["ids"], state["weights"] = _routing(g, case)
        state["x"] = _normal(g, (case["tokens"], h), dtype)
        state["y"] = _normal(g, (rows, h), dtype)        # the experts' outputs, sorted
        if case["train"]:
            state["dx"] = _normal(g, (rows, h), dtype, 1e-2)  # of the gathered rows
            state["dy"] = _normal(g, (case["tokens"], h), dtype, 1e-2)
            for name in ("x", "y", "weights"):
                state[name].requires_grad_()
    else:
        state["ids"], _ = _routing(g, case)
        state["x"] = _normal(g, (case["tokens"], case["inner"]), dtype, outliers=True)
        w = _normal(g, (case["experts"], case["outer"], case["inner"]), dtype, 0.02)
        if case["train"]:
            state["x"].requires_grad_()
            state["w"] = w.requires_grad_()
            state["dy"] = _normal(g, (case["tokens"] * case["top"], case["outer"]), dtype, 1e-3)
        else:
            state["codes"], state["scales"] = _stored(_turned(w.float(), dtype) if case["rotate"] else w)
    return state


# -------------------------------------------------------------------------------------- plain forms

def _turned(x, dtype):
    """The rotation along the last axis: in each group of 256, four radix-4 steps (one a base-4 digit
    of the index, the lowest first) of [[1,1,1,-1],[1,1,-1,1],[1,-1,1,1],[-1,1,1,1]] / 2, in 32 bits;
    the result rounded to `dtype`."""
    t = x.reshape(*x.shape[:-1], -1, 4, 4, 4, 4)

    def chain(t, axis):
        a, b, c, d = t.unbind(axis)
        p, m = a + b, a - b
        return torch.stack([(p + c) - d, (p - c) + d, (m + c) + d, (c - m) + d], axis)

    def pairs(t, axis):
        a, b, c, d = t.unbind(axis)
        p, m, q, n = a + b, a - b, c + d, c - d
        return torch.stack([p + n, p - n, m + q, q - m], axis)

    t = pairs(pairs(chain(chain(t, -1), -2), -3), -4) * 0.0625
    return t.reshape(x.shape).to(dtype)


def _blocks(x):
    """(code magnitudes and signs, scale exponents) of x's rows in 32 bits: [.., B, 32], [.., B]."""
    x = x.float()
    pad = -x.shape[-1] % BLOCK
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))
    x = x.reshape(*x.shape[:-1], -1, BLOCK)
    amax = x.abs().amax(-1)
    e = (((amax.view(torch.int32) >> 23) & 255) - 2).clamp_min(0)     # the scale 2^(e - 127)
    a = x.abs() * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5))
    return code + 8 * (x < 0).to(torch.uint8), e.to(torch.uint8)


def _values(code, e):
    """The values that codes [.., B, 32] and exponents [.., B] stand for, in 32 bits: [.., K]."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    two = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e.to(torch.int32) - 127)
    return (grid[code.long()] * two.unsqueeze(-1)).flatten(-2)


def _rounded(x):
    """x's rows as MXFP4 holds them, in 32 bits."""
    return _values(*_blocks(x))[..., :x.shape[-1]]


def _stored(x):
    """x's rows as they are kept: codes [.., R, B * 16], two to a byte, the first in the low half, and
    scales [.., tiles of 128 rows, tiles of 4 blocks, 32, 16]: row 32 j + l of a tile and its block b
    at [l, 4 j + b]."""
    code, e = _blocks(x)
    packed = (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2)
    rows, blocks = e.shape[-2:]
    e = torch.nn.functional.pad(e, (0, -blocks % 4, 0, -rows % TILE))
    n = e.dim() - 2
    e = e.reshape(*e.shape[:-2], -1, 4, 32, -(-blocks // 4), 4)
    e = e.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    return packed.contiguous(), e.flatten(-2).contiguous()


def _read(codes, scales, k):
    """The values of stored rows, in 32 bits: [.., R, k]."""
    rows, blocks = codes.shape[-2], codes.shape[-1] // 16
    n = scales.dim() - 4
    e = scales.reshape(*scales.shape[:-1], 4, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    e = e.reshape(*scales.shape[:-4], -1, scales.shape[-3] * 4)[..., :rows, :blocks]
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], blocks, BLOCK)
    return _values(code, e)[..., :k]


def _order(ids, experts):
    """(order, offsets, positions): the slots (token, choice) sorted by expert, equal ones in their
    order and those of no expert last; where each expert's rows begin and end; each slot's row."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(key, stable=True)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device=order.device)
    return order, offsets, positions.reshape(ids.shape)


def _plain_route(s):
    dtype, top = DTYPES[s["dtype"]], s["top"]
    x, y, weights = (s[i].detach() for i in ("x", "y", "weights"))
    order, offsets, positions = _order(s["ids"], s["experts"])
    taken = torch.arange(order.numel(), device=order.device) < offsets[-1]
    gathered = torch.where(taken[:, None], x[order // top], torch.zeros((), dtype=dtype, device=x.device))
    slot = (positions < offsets[-1]).unsqueeze(-1)
    rows = torch.where(slot, y[positions].float(), 0.0)
    out = {"order": order.int(), "offsets": offsets.int(), "positions": positions.int(),
           "gathered": gathered, "combined": (rows * weights.unsqueeze(-1)).sum(1).to(dtype)}
    if s["train"]:
        dy = s["dy"].float()
        out["grad_x"] = torch.where(slot, s["dx"][positions].float(), 0.0).sum(1).to(dtype)
        out["grad_weights"] = (rows * dy.unsqueeze(1)).sum(-1)
        grad = weights.reshape(-1)[order].unsqueeze(-1) * dy[order // top]
        out["grad_y"] = torch.where(taken[:, None], grad, 0.0).to(dtype)
    return out


def _plain_experts(s):
    dtype, top, k = DTYPES[s["dtype"]], s["top"], s["inner"]
    x = s["x"].detach()
    x = _turned(x.float(), dtype) if s["rotate"] else x
    order, offsets, _ = _order(s["ids"], s["experts"])
    row = torch.arange(order.numel(), device=x.device)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    at = row - offsets[expert]
    most = int((offsets[1:] - offsets[:-1]).max())            # every expert's rows, to one length

    def spread(rows):
        wide = torch.zeros(s["experts"], most, rows.shape[1], device=x.device)
        wide[expert, at] = rows.float()
        return wide

    if not s["train"]:
        wide = spread(_rounded(x)[order // top])
        return {"y": (wide @ _read(s["codes"], s["scales"], k).mT)[expert, at].to(dtype)}
    w = s["w"].detach()
    w = _turned(w.float(), dtype) if s["rotate"] else w
    dy = s["dy"]
    y = (spread(_rounded(x)[order // top]) @ _rounded(w).mT)[expert, at]
    dx = (spread(_rounded(dy)) @ _rounded(w.mT).mT)[expert, at]
    dx = torch.zeros(x.shape, device=x.device).index_add_(0, order // top, dx)
    dw = _rounded(spread(dy).mT) @ _rounded(spread(x[order // top]).mT).mT
    if s["rotate"]:
        dx, dw = _turned(dx, torch.float32), _turned(dw, torch.float32)
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}


def _plain(s):
    op, dtype = s["op"], DTYPES[s["dtype"]]
    if op == "quantise":
        x = s["x"].mT if s["columns"] else s["x"]
        x = _turned(x.float(), dtype) if s["rotate"] else x
        return {"values": _rounded(x).to(dtype)}
    if op == "linear":
        x = _turned(s["x"].float(), dtype) if s["rotate"] else s["x"]
        y = _rounded(x) @ _read(s["codes"], s["scales"], s["inner"]).mT
        return {"y": (y if s["bias"] is None else y + s["bias"]).to(dtype)}
    if op == "train":
        x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
        if s["rotate"]:
            x, w = _turned(x.float(), dtype), _turned(w.float(), dtype)
        y = _rounded(x) @ _rounded(w).mT
        dx = _rounded(dy) @ _rounded(w.mT).mT
        dw = _rounded(dy.mT) @ _rounded(x.mT).mT
        if s["rotate"]:
            dx, dw = _turned(dx, torch.float32), _turned(dw, torch.float32)
        return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}
    return _plain_route(s) if op == "route" else _plain_experts(s)


# ------------------------------------------------------------------------------------- the framework

def _package():
    import importlib
    import os
    import sys
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oko-xpu-kernels_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    return importlib.import_module("xpu_kernels")


def _framework(s):
    xk, op, rotate = _package(), s["op"], s.get("rotate", False)
    if op == "quantise":
        q = xk.quantize_mxfp4(s["x"], rotate=rotate, transpose=s["columns"])
        return {"values": xk.dequantize_mxfp4(q, dtype=s["x"].dtype)}
    if op == "linear":
        w = xk.MXFP4(s["codes"], s["scales"], (s["outer"], s["inner"]))
        return {"y": xk.linear_mxfp4(s["x"], w, s["bias"], rotate=rotate)}
    if op == "train":
        y = xk.mxfp4_linear(s["x"], s["w"], rotate=rotate)
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    plan = xk.expert_sort(s["ids"], s["experts"])
    if op == "route":
        gathered = xk.expert_gather(s["x"], plan)
        combined = xk.expert_combine(s["y"], s["weights"], plan)
        out = {"order": plan.order, "offsets": plan.offsets, "positions": plan.positions,
               "gathered": gathered, "combined": combined}
        if s["train"]:
            out["grad_x"], out["grad_y"], out["grad_weights"] = torch.autograd.grad(
                (gathered, combined), (s["x"], s["y"], s["weights"]), (s["dx"], s["dy"]))
        return out
    if not s["train"]:
        w = xk.MXFP4(s["codes"], s["scales"], (s["experts"], s["outer"], s["inner"]))
        return {"y": xk.expert_linear_mxfp4(s["x"], w, plan, rotate=rotate)}
    y = xk.mxfp4_expert_linear(s["x"], s["w"], plan, rotate=rotate)
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def run(state):
    if own:
        return _framework(state)
    with torch.no_grad():
        return _plain(state)


# -------------------------------------------------------------------------------------- in 64 bits

def _h256(device):
    h = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]],
                     dtype=torch.float64, device=device) / 2
    h = torch.kron(h, h)
    return torch.kron(h, h)


def _turned64(x):
    return (x.double().reshape(-1, GROUP) @ _h256(x.device)).reshape(x.shape)


def _round64(x):
    """x's rows (64 bits) as MXFP4 holds them."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(amax)[1] - 1 - 2).clamp(-127, 127)  # frexp: amax = m 2^e, m in [1/2, 1)
    exponent = torch.where(amax == 0, -127, exponent)
    scale = torch.ldexp(torch.ones_like(amax), exponent)
    v = x / scale
    step = 0.5 + 0.5 * (v.abs() >= 2) + 1.0 * (v.abs() >= 4)
    v = (torch.round(v / step) * step).clamp(-6, 6) * scale       # round: ties to even
    return v.flatten(-2)[..., :k]


def exact(case, seed):
    s = prepare(case, seed)
    op, dtype, rotate = case["op"], DTYPES[case["dtype"]], case.get("rotate", False)
    with torch.no_grad():
        if op == "quantise":
            x = s["x"].double()
            x = _turned64(x).to(dtype).double() if rotate else x
            return {"values": _round64(x.mT if case["columns"] else x)}
        if op == "route":
            return _exact_route(s)
        x = _turned64(s["x"]).to(dtype).double() if rotate else s["x"].double()
        if "w" in s:
            w = _turned64(s["w"]).to(dtype).double() if rotate else s["w"].double()
            wq = _round64(w)
        else:
            wq = _read64(s["codes"], s["scales"], case["inner"])
        back = _turned64 if rotate else (lambda v: v)
        if op == "linear":
            y = _round64(x) @ wq.mT
            return {"y": y if s["bias"] is None else y + s["bias"].double()}
        dy = s["dy"].double() if "dy" in s else None
        if op == "train":
            return {"y": _round64(x) @ wq.mT, "dx": back(_round64(dy) @ _round64(w.mT).mT),
                    "dw": back(_round64(dy.mT) @ _round64(x.mT).mT)}
        top = case["top"]
        rows = s["ids"].numel()
        y = torch.zeros(rows, case["outer"], dtype=torch.float64, device=x.device)
        train = case["train"]
        if train:
            dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        xq, begin = _round64(x), 0
        for e in range(case["experts"]):
            token = torch.nonzero((s["ids"] == e).any(1)).flatten()    # a token's experts differ
            if not token.numel():
                continue
            end = begin + token.numel()
            y[begin:end] = xq[token] @ wq[e].T
            if train:
                d = dy[begin:end]
                dx[token] += _round64(d) @ _round64(w[e].T.contiguous()).T
                dw[e] = _round64(d.T.contiguous()) @ _round64(x[token].T.contiguous()).T
            begin = end
        return {"y": y, "dx": back(dx), "dw": back(dw)} if train else {"y": y}


def _read64(codes, scales, k):
    rows, blocks = codes.shape[-2], codes.shape[-1] // 16
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange(blocks, device=codes.device)[None, :]
    e = scales[..., r // 128, b // 4, r % 32, (r % 128) // 32 * 4 + b % 4]
    low, high = codes & 15, codes >> 4
    c = torch.stack([low, high], -1).flatten(-2).int()
    m = c & 7
    v = torch.where(m < 2, m * 0.5, torch.ldexp(1 + (m & 1) * 0.5, (m >> 1) - 1)).double()
    v = torch.where(c >= 8, -v, v)
    scale = torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.int() - 127)
    return (v.unflatten(-1, (blocks, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)[..., :k]


def _exact_route(s):
    experts, top = s["experts"], s["top"]
    device = s["x"].device
    x, y, w = s["x"].double(), s["y"].double(), s["weights"].double().reshape(-1)
    flat = s["ids"].reshape(-1)
    lists = [torch.nonzero(flat == e).flatten() for e in range(experts)]
    none = torch.nonzero((flat < 0) | (flat >= experts)).flatten()
    order = torch.cat(lists + [none])
    ends, total = [0], 0
    for at in lists:
        total += at.numel()
        ends.append(total)
    kept = order[:total]
    position = torch.empty(flat.numel(), dtype=torch.int64, device=device)
    position.scatter_(0, order, torch.arange(flat.numel(), device=device))
    gathered = torch.zeros(flat.numel(), x.shape[1], dtype=torch.float64, device=device)
    gathered[:total] = x[kept // top]
    combined = torch.zeros_like(x).index_add_(0, kept // top, y[:total] * w[kept, None])
    out = {"order": order.int(), "offsets": torch.tensor(ends, dtype=torch.int32, device=device),
           "positions": position.reshape(s["ids"].shape).int(), "gathered": gathered,
           "combined": combined}
    if s["train"]:
        dy = s["dy"].double()
        out["grad_x"] = torch.zeros_like(x).index_add_(0, kept // top, s["dx"].double()[:total])
        grad_y = torch.zeros_like(y)
        grad_y[:total] = w[kept, None] * dy[kept // top]
        out["grad_y"] = grad_y
        dot = torch.zeros(flat.numel(), dtype=torch.float64, device=device)
        dot[kept] = (y[:total] * dy[kept // top]).sum(1)
        out["grad_weights"] = dot.reshape(s["ids"].shape)
    return out
