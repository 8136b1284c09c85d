"""Cases of the expert and projection operators, their plain forms, and the calls a user makes of them.

dispatch   ``expert_sort`` + ``expert_gather``: a router's selection, sorted by expert, and the tokens' rows in that order
combine    ``expert_combine``: the experts' outputs back in token order, weighted and summed, onto a residual
backward   ``expert_combine_grad`` + ``expert_gather_grad``: the gradients of both directions
linear     ``linear``: residual + mul * activation(x @ W.T + bias) from the packed weights of one projection
experts    ``expert_linear``: the same product for rows sorted by expert, each segment with its own expert's weights
"""
import math
import os
import sys

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
ACTIVATIONS = ("none", "relu", "relu2", "gelu", "gelu_tanh", "silu", "sigmoid")

# Projection shapes (n, k) of this repository's configurations: fused QKV+gate, output, pooler, unpooler, and the
# smaller set it is compared with.
SHAPES = ((14336, 6144), (6144, 6144), (1536, 6144), (6144, 1536), (2304, 8192), (8192, 1024), (4096, 8192))


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "muse-bf16-proj_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mbp
    return mbp


def listed():
    return [
        # one decoded token's eight experts of 256: pure latency
        {"name": "dispatch 1x8/256", "op": "dispatch", "m": 1, "k": 8, "experts": 256, "d": 6144, "f32": False, "dropped": 0.0},
        # a small ragged batch with padding tokens and assignments over capacity
        {"name": "dispatch 333x6/60 dropped", "op": "dispatch", "m": 333, "k": 6, "experts": 60, "d": 1536, "f32": False, "dropped": 0.1},
        # a prompt
        {"name": "dispatch 4096x8/256", "op": "dispatch", "m": 4096, "k": 8, "experts": 256, "d": 6144, "f32": False, "dropped": 0.0},
        # a decode batch back in token order, onto the residual stream
        {"name": "combine 16x8/256 residual", "op": "combine", "m": 16, "k": 8, "experts": 256, "d": 6144, "f32": False, "residual": True, "dropped": 0.0},
        # a prompt, an uneven token count
        {"name": "combine 4001x8/256", "op": "combine", "m": 4001, "k": 8, "experts": 256, "d": 6144, "f32": False, "residual": False, "dropped": 0.02},
        # a training step's gradients through both directions
        {"name": "backward 2048x8/64", "op": "backward", "m": 2048, "k": 8, "experts": 64, "d": 6144, "f32": False, "dropped": 0.0},
        # the output projection of one decoded token, onto the residual stream
        {"name": "linear 1 o residual", "op": "linear", "m": 1, "n": 6144, "kk": 6144, "act": "none", "bias": True, "mul": False, "residual": True},
        # a decode batch through the fused projection with a bias
        {"name": "linear 24 qkv_gate gelu", "op": "linear", "m": 24, "n": 14336, "kk": 6144, "act": "gelu", "bias": True, "mul": False, "residual": False},
        # a verify batch of an uneven size: gated and added
        {"name": "linear 200 unpooler silu", "op": "linear", "m": 200, "n": 6144, "kk": 1536, "act": "silu", "bias": False, "mul": True, "residual": True},
        # one decoded token through its eight experts
        {"name": "experts 1x8/64 silu", "op": "experts", "m": 1, "k": 8, "experts": 64, "n": 1536, "kk": 6144, "act": "silu", "bias": False, "mul": False},
        # a decode batch through the experts' second product
        {"name": "experts 30x8/64 down", "op": "experts", "m": 30, "k": 8, "experts": 64, "n": 6144, "kk": 1536, "act": "none", "bias": True, "mul": False},
        # a prompt chunk: gated activation, about 128 rows an expert
        {"name": "experts 1024x8/64 silu mul", "op": "experts", "m": 1024, "k": 8, "experts": 64, "n": 1536, "kk": 6144, "act": "silu", "bias": False, "mul": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("dispatch", "combine", "backward", "linear", "experts"))
    if op == "linear":
        if rng.random() < 0.5:
            n, kk = rng.choice(SHAPES)
        else:
            n, kk = 16 * _log(rng, 16, 800), 64 * _log(rng, 4, 128)
        return {"op": op, "m": _log(rng, 1, 256), "n": n, "kk": kk, "act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.5,
                "mul": rng.random() < 0.4, "residual": rng.random() < 0.5}
    experts = _log(rng, 4, 64 if op == "experts" else 256)
    k = rng.randint(1, min(8, experts))
    if op == "experts":
        if rng.random() < 0.5:
            n, kk = rng.choice(((1536, 6144), (6144, 1536)))
        else:
            n, kk = 16 * _log(rng, 16, 96), 64 * _log(rng, 4, 96)
        return {"op": op, "m": _log(rng, 1, 1024), "k": k, "experts": experts, "n": n, "kk": kk, "act": rng.choice(ACTIVATIONS),
                "bias": rng.random() < 0.5, "mul": rng.random() < 0.4}
    d = rng.choice((1024, 1536, 6144)) if rng.random() < 0.5 else _log(rng, 64, 6144)
    case = {"op": op, "m": _log(rng, 1, 2048 if op == "backward" else 4000), "k": k, "experts": experts, "d": d,
            "f32": rng.random() < 0.25 and d <= 2048, "dropped": rng.choice((0.0, 0.0, 0.05, 0.3))}
    if op == "combine":
        case["residual"] = rng.random() < 0.5
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------


def _selection(g, m, k, experts, dropped):
    """A router's top-k (some experts more popular than others), with padding (-1) where an assignment is dropped."""
    logits = torch.randn((m, experts), generator=g, device="cuda") + 0.5 * torch.randn((1, experts), generator=g, device="cuda")
    top, ids = logits.topk(k, dim=1)
    w = torch.softmax(top, dim=1)
    if dropped:
        out = torch.rand((m, k), generator=g, device="cuda") < dropped
        out[m - m // 16:] = True  # padding tokens at the end of the batch
        ids = ids.masked_fill(out, -1)
        w = w.masked_fill(out, 0.0)
    return ids.to(torch.int32), w


def _plan(ids, experts):
    """Row of each assignment, assignment of each row, and segment borders, as the forward pass left them."""
    m, k = ids.shape
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.argsort(key, stable=True)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)
    rows = torch.arange(m * k, device=ids.device)
    used = rows < offsets[-1]
    src = torch.where(used, order, -1)
    pos = torch.empty_like(order).scatter_(0, order, torch.where(used, rows, -1))
    return pos.view(m, k).to(torch.int32), src.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rn = lambda *s, dtype=BF16: torch.randn(s, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    s = {"case": case}
    op, m = case["op"], case["m"]
    if op in ("dispatch", "combine", "backward"):
        dtype, k, d = F32 if case["f32"] else BF16, case["k"], case["d"]
        s["ids"], s["weights"] = _selection(g, m, k, case["experts"], case["dropped"])
        if op == "dispatch":
            s["x"] = rn(m, d, dtype=dtype)
            return s
        s["pos"], s["src"], s["offsets"] = _plan(s["ids"], case["experts"])
        s["ys"] = rn(m * k, d, dtype=dtype)
        if op == "combine":
            s["residual"] = rn(m, d, dtype=dtype) if case["residual"] else None
        else:
            s["dout"], s["dxs"] = rn(m, d, dtype=dtype), rn(m * k, d, dtype=dtype)
        return s
    n, kk = case["n"], case["kk"]
    if op == "linear":
        w = rn(n, kk) * 0.02
        s["x"] = rn(m, kk)
        s["bias"] = rn(n, dtype=F32) if case["bias"] else None
        rows = m
    else:
        ids, _ = _selection(g, m, case["k"], case["experts"], 0.0)
        s["pos"], s["src"], s["offsets"] = _plan(ids, case["experts"])
        w = rn(case["experts"], n, kk) * 0.02
        rows = m * case["k"]
        s["x"] = rn(rows, kk)
        s["bias"] = rn(case["experts"], n, dtype=F32) if case["bias"] else None
    s["mul"] = rn(rows, n) if case["mul"] else None
    s["residual"] = rn(rows, n) if case.get("residual") else None
    if own:  # a program that serves from packed weights packs them once, when it loads them
        mbp = _package()
        s["packed"] = mbp.pack_c12(w) if op == "linear" else mbp.pack_experts(w)
    else:
        s["w"] = w
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------


def _activate(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "relu2":
        return torch.clamp(z, min=0) ** 2
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _finish(z, s, bias):
    if bias is not None:
        z = z + bias.float()
    z = _activate(z, s["case"]["act"])
    if s["mul"] is not None:
        z = z * s["mul"].float()
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(BF16)


def _rows(ys, pos):
    """The rows of ys at pos (zeros for -1) in 32 bits."""
    return torch.where((pos >= 0).unsqueeze(-1), ys[pos.clamp(min=0).long()].float(), 0.0)


def _plain(s):
    case = s["case"]
    op, m = case["op"], case["m"]
    if op == "dispatch":
        pos, src, offsets = _plan(s["ids"], case["experts"])
        used = (src >= 0).unsqueeze(-1)
        xs = torch.where(used, s["x"][(src.clamp(min=0) // case["k"]).long()], 0)
        return {"pos": pos, "src": src, "offsets": offsets, "xs": xs.to(s["x"].dtype)}
    if op == "combine":
        out = (_rows(s["ys"], s["pos"]) * s["weights"].unsqueeze(-1)).sum(1)
        if s["residual"] is not None:
            out = out + s["residual"].float()
        return {"out": out.to(s["ys"].dtype)}
    if op == "backward":
        dtype, used = s["ys"].dtype, (s["src"] >= 0).unsqueeze(-1)
        src = s["src"].clamp(min=0).long()
        dys = torch.where(used, s["weights"].reshape(-1)[src].unsqueeze(-1) * s["dout"][src // case["k"]].float(), 0.0)
        dw = (_rows(s["ys"], s["pos"]) * s["dout"].float().unsqueeze(1)).sum(-1)
        dx = _rows(s["dxs"], s["pos"]).sum(1)
        return {"dys": dys.to(dtype), "dweights": dw, "dx": dx.to(dtype)}
    if op == "linear":
        return {"out": _finish(s["x"].float() @ s["w"].float().T, s, s["bias"])}
    # each used expert's rows, padded to the longest segment, as one batched product
    offsets = s["offsets"].long()
    counts = offsets.diff()
    used = counts.nonzero().squeeze(1)
    rows = torch.arange(s["x"].shape[0], device="cuda")
    expert = torch.searchsorted(offsets[1:], rows, right=True)
    slot = torch.searchsorted(used, expert)
    inside = rows - offsets[expert]
    xp = torch.zeros((used.numel(), int(counts.max()), case["kk"]), device="cuda")
    xp[slot, inside] = s["x"].float()
    z = torch.bmm(xp, s["w"][used].float().transpose(1, 2))[slot, inside]
    return {"out": _finish(z, s, None if s["bias"] is None else s["bias"][expert])}


def run(s):
    if not own:
        return _plain(s)
    mbp = _package()
    case = s["case"]
    op, m = case["op"], case["m"]
    if op == "dispatch":
        plan = mbp.expert_sort(s["ids"], case["experts"])
        return {"pos": plan.pos, "src": plan.src, "offsets": plan.offsets, "xs": mbp.expert_gather(s["x"], plan)}
    if op == "linear":
        return {"out": mbp.linear(s["packed"], s["x"], bias=s["bias"], activation=case["act"], mul=s["mul"], residual=s["residual"])}
    plan = mbp.ExpertPlan(s["pos"], s["src"], s["offsets"])
    if op == "combine":
        return {"out": mbp.expert_combine(s["ys"], s["weights"], plan, residual=s["residual"])}
    if op == "backward":
        dys, dw = mbp.expert_combine_grad(s["dout"], s["ys"], s["weights"], plan)
        return {"dys": dys, "dweights": dw, "dx": mbp.expert_gather_grad(s["dxs"], plan)}
    return {"out": mbp.expert_linear(s["packed"], s["x"], plan, bias=s["bias"], activation=case["act"], mul=s["mul"],
                                     residual=s["residual"])}


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    op, m = case["op"], case["m"]
    if op in ("dispatch", "combine", "backward"):
        a, es = m * case["k"], 4 if case["f32"] else 2
        kept = a * (1 - case["dropped"]) * (15 / 16 if case["dropped"] and m >= 16 else 1)
        row = case["d"] * es
        if op == "dispatch":  # ids; the tokens once; every row of xs and the plan
            return {"bytes": 4 * a + m * row + a * row + 8 * a + 4 * case["experts"] + 4, "flops": 0}
        if op == "combine":
            return {"bytes": 8 * a + kept * row + m * row * (2 if case["residual"] else 1), "flops": 2 * kept * case["d"]}
        # dout once; ys and dxs read, dys written; dx written; weights, positions and dweights
        return {"bytes": 2 * m * row + 2 * kept * row + a * row + 12 * a, "flops": 4 * kept * case["d"]}
    n, kk = case["n"], case["kk"]
    rows, used = m, 1.0
    if op == "experts":
        e = case["experts"]
        rows, used = m * case["k"], e * (1 - (1 - case["k"] / e) ** m)
    side = 1 + bool(case["mul"]) + bool(case.get("residual"))
    byt = 1.5 * used * n * kk + 2 * rows * (kk + side * n) + (4 * used * n if case["bias"] else 0)
    return {"bytes": byt, "flops": 2.0 * rows * n * kk}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def _act64(z, act):
    if act == "none":
        return z
    if act in ("relu", "relu2"):
        r = torch.where(z > 0, z, torch.zeros_like(z))
        return r if act == "relu" else r * r
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    if act == "gelu_tanh":
        return z * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z) if act == "silu" else torch.sigmoid(z)


def exact(case, seed):
    s = prepare(case, seed)
    op, m = case["op"], case["m"]
    if op in ("linear", "experts"):
        x, rows = s["x"].double(), s["x"].shape[0]
        z = torch.empty((rows, case["n"]), dtype=torch.float64, device="cuda")
        at = [0, rows] if op == "linear" else s["offsets"].tolist()
        for e in range(len(at) - 1):
            if at[e] < at[e + 1]:
                w = s["w"] if op == "linear" else s["w"][e]
                y = x[at[e]:at[e + 1]] @ w.double().T
                if s["bias"] is not None:
                    y += (s["bias"] if op == "linear" else s["bias"][e]).double()
                z[at[e]:at[e + 1]] = y
        z = _act64(z, case["act"])
        if s["mul"] is not None:
            z *= s["mul"].double()
        if s["residual"] is not None:
            z += s["residual"].double()
        return {"out": z}
    k, experts, d = case["k"], case["experts"], case["d"]
    # the position of assignment i: all kept ones of lower experts, then the earlier ones of its own
    ids = s["ids"].reshape(-1).tolist()
    count = [0] * experts
    for e in ids:
        if e >= 0:
            count[e] += 1
    start, total = [], 0
    for c in count:
        start.append(total)
        total += c
    pos = []
    for e in ids:
        pos.append(start[e] if e >= 0 else -1)
        if e >= 0:
            start[e] += 1
    pos = torch.tensor(pos, device="cuda").view(m, k)
    if op == "dispatch":
        xs = torch.zeros((m * k, d), dtype=torch.float64, device="cuda")
        for j in range(k):
            keep = pos[:, j] >= 0
            xs[pos[keep, j]] = s["x"][keep].double()
        return {"pos": None, "src": None, "offsets": None, "xs": xs}
    if op == "combine":
        out = torch.zeros((m, d), dtype=torch.float64, device="cuda") if s["residual"] is None else s["residual"].double()
        for j in range(k):
            keep = pos[:, j] >= 0
            out[keep] += s["weights"][keep, j].double().unsqueeze(1) * s["ys"][pos[keep, j]].double()
        return {"out": out}
    dys = torch.zeros((m * k, d), dtype=torch.float64, device="cuda")
    dw = torch.zeros((m, k), dtype=torch.float64, device="cuda")
    dx = torch.zeros((m, d), dtype=torch.float64, device="cuda")
    for j in range(k):
        keep = pos[:, j] >= 0
        dout = s["dout"][keep].double()
        dys[pos[keep, j]] = s["weights"][keep, j].double().unsqueeze(1) * dout
        dw[keep, j] = (dout * s["ys"][pos[keep, j]].double()).sum(1)
        dx[keep] += s["dxs"][pos[keep, j]].double()
    return {"dys": dys, "dweights": dw, "dx": dx}
