"""Cases of the operators of a mixture of 1-bit experts: the router's choice,
the experts' linears over ragged groups of rows, and the weighted sum of what
the experts give.

A case is a dict of plain values; `kind` names the call:

  route    bonsai_b1.route: router logits -> each token's experts and weights,
           and the rows of every expert, one expert after another
  linear   bonsai_b1.linear_experts: packed fp16 activations -> the B1_0
           linear of each row's expert
  combine  bonsai_b1.combine_experts: each token's rows, weighted and added
           to the residual stream

A token has `top_k` routes.  Route rows are in the experts' order, within an
expert in the tokens' order.  `rows` says which activations a route row reads:
its token's ("tokens", the up projections) or its own ("routes", the down
projections).  `out` is "packed" (the packed fp16 activations of the next
linear, through `act`; returned as fp16 values in their stored order) or
"rows" (fp32).  `out_dim` counts weight rows: SwiGLU's [gate | value] are two
of them a column.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request's decoding step: a single row of logits, bound by latency
        {"name": "route_one", "kind": "route", "tokens": 1, "experts": 128, "top_k": 8, "type": "fp32",
         "score": "softmax", "bias": False, "renormalize": True, "scale": 1.0, "off": 0},
        # a batch of prompts
        {"name": "route_prompts", "kind": "route", "tokens": 8192, "experts": 128, "top_k": 8, "type": "bf16",
         "score": "softmax", "bias": False, "renormalize": True, "scale": 1.0, "off": 0},
        # many experts, chosen by balanced scores, some of them off
        {"name": "route_balanced", "kind": "route", "tokens": 4099, "experts": 256, "top_k": 6, "type": "fp32",
         "score": "sigmoid", "bias": True, "renormalize": True, "scale": 2.5, "off": 5},
        # one request's decoding step: eight experts of one row each
        {"name": "up_one", "kind": "linear", "tokens": 1, "experts": 128, "top_k": 8, "in_dim": 2048, "out_dim": 1536,
         "rows": "tokens", "act": "swiglu", "out": "packed"},
        # a decoding step of 64 requests: about four rows an expert, bound by the weights
        {"name": "up_step", "kind": "linear", "tokens": 64, "experts": 128, "top_k": 8, "in_dim": 2048,
         "out_dim": 1536, "rows": "tokens", "act": "swiglu", "out": "packed"},
        # its down projections
        {"name": "down_step", "kind": "linear", "tokens": 64, "experts": 128, "top_k": 8, "in_dim": 768,
         "out_dim": 2048, "rows": "routes", "act": "none", "out": "rows"},
        # a chunk of a prompt through few experts of odd widths
        {"name": "up_odd", "kind": "linear", "tokens": 509, "experts": 20, "top_k": 3, "in_dim": 1344, "out_dim": 1408,
         "rows": "tokens", "act": "gelu_tanh", "out": "packed"},
        # prompts through few wide experts
        {"name": "down_wide", "kind": "linear", "tokens": 1777, "experts": 8, "top_k": 2, "in_dim": 7168,
         "out_dim": 4096, "rows": "routes", "act": "none", "out": "rows"},
        # a batch of prompts, up and down: bound by the matrix cores
        {"name": "up_prompts", "kind": "linear", "tokens": 8192, "experts": 128, "top_k": 8, "in_dim": 2048,
         "out_dim": 1536, "rows": "tokens", "act": "swiglu", "out": "packed"},
        {"name": "down_prompts", "kind": "linear", "tokens": 8192, "experts": 128, "top_k": 8, "in_dim": 768,
         "out_dim": 2048, "rows": "routes", "act": "none", "out": "rows"},
        # the sums of that decoding step and of those prompts
        {"name": "combine_step", "kind": "combine", "tokens": 64, "experts": 128, "top_k": 8, "h": 2048},
        {"name": "combine_prompts", "kind": "combine", "tokens": 8192, "experts": 128, "top_k": 8, "h": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# a drawn case costs no more than the largest listed one, and its plain form's
# decoded weights and padded rows fit what the listed ones' do
MOST = {"flops": 4.2e11, "bytes": 8.0e8}
MOST_WEIGHTS, MOST_PADDED = 5.0e8, 1.2e9


def draw(rng):
    """A case of the listed ones' ranges: 1 to 8192 tokens, odd counts among
    them, 2 to 256 experts, 1 to 8 routes a token, widths of 64 to 8192."""
    while True:
        experts = rng.choice([2, 5, 8, 16, 20, 32, 64, 96, 128, 160, 256])
        case = {"kind": rng.choice(["route", "linear", "linear", "linear", "combine"]), "tokens": _log(rng, 1, 8192),
                "experts": experts, "top_k": rng.randint(1, min(8, experts))}
        if case["kind"] == "route":
            off = rng.randint(1, experts - case["top_k"]) if case["top_k"] < experts and rng.random() < 0.3 else 0
            return case | {"type": rng.choice(["fp32", "fp32", "fp16", "bf16"]),
                           "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.4,
                           "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 1.0, 2.5]), "off": off}
        if case["kind"] == "combine":
            case |= {"h": 4 * _log(rng, 16, 2048)}
        else:
            out = rng.choice(["packed", "rows"])
            act = rng.choice(["swiglu", "swiglu", "gelu_tanh", "none"]) if out == "packed" else "none"
            step = {"swiglu": 64, "gelu_tanh": 32, "none": 32 if out == "packed" else 1}[act]
            case |= {"in_dim": 64 * _log(rng, 1, 128), "out_dim": step * _log(rng, -(-64 // step), 8192 // step),
                     "rows": rng.choice(["tokens", "routes"]), "act": act, "out": out}
            rows = case["tokens"] * case["top_k"]
            most = min(case["tokens"], 8 * -(-rows // experts) + 64)
            if experts * case["in_dim"] * case["out_dim"] > MOST_WEIGHTS or \
                    experts * most * (case["in_dim"] + case["out_dim"]) > MOST_PADDED:
                continue
        w = work(case)
        if w["flops"] <= MOST["flops"] and w["bytes"] <= MOST["bytes"]:
            return case


def work(case):
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    routes = tokens * k
    if case["kind"] == "route":
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": size * tokens * experts + 16 * routes + 4 * (experts + 1),
                "flops": 6 * tokens * experts}
    if case["kind"] == "combine":
        return {"bytes": 4 * case["h"] * (routes + 2 * tokens) + 8 * routes, "flops": 2 * case["h"] * routes}
    # experts that some token goes to (as many as with even chances)
    used = experts * (1.0 - (1.0 - k / experts) ** tokens)
    cols = case["out_dim"] // (2 if case["act"] == "swiglu" else 1)
    read = 2 * case["in_dim"] * (tokens if case["rows"] == "tokens" else routes)
    return {"bytes": int(used * case["out_dim"] * (case["in_dim"] // 32) * 6) + read
            + (2 if case["out"] == "packed" else 4) * cols * routes + 4 * (routes + experts + 1),
            "flops": 2 * case["in_dim"] * case["out_dim"] * routes}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, spread=1.0):
        return torch.randn(shape, generator=g, device="cuda") * spread

    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    s = {"case": case}
    # tokens differ in what they want, and some experts are wanted more
    logits = normal(tokens, experts, spread=1.5) + normal(experts, spread=0.6)
    if case["kind"] == "route":
        if case["off"]:
            logits[:, torch.randperm(experts, generator=g, device="cuda")[:case["off"]]] = -math.inf
        s["logits"] = logits.to(TYPES[case["type"]])
        s["bias"] = normal(experts, spread=0.1) if case["bias"] else None
        return s
    chosen = torch.topk(logits, k, 1)
    s["expert"], s["weight"] = chosen.indices.int(), torch.softmax(chosen.values, 1)
    flat = chosen.indices.flatten()
    at = torch.argsort(flat, stable=True)
    s["order"] = at.int()
    s["place"] = torch.empty_like(s["order"])
    s["place"][at] = torch.arange(len(at), dtype=torch.int32, device="cuda")
    s["place"] = s["place"].view(tokens, k)
    count = torch.bincount(flat, minlength=experts)
    s["start"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).int()
    if case["kind"] == "combine":
        s["y"], s["x"] = normal(tokens * k, case["h"]), normal(tokens, case["h"], spread=3.0)
        return s
    s["most"] = int(count.max())  # rows of the largest group
    rows = tokens if case["rows"] == "tokens" else tokens * k
    # what a norm or an activation leaves, already in the packed order
    s["act"] = normal(rows, case["in_dim"]).to(torch.float16)
    blocks = experts * case["out_dim"] * (case["in_dim"] // 32)
    s["w"] = torch.randint(0, 256, (blocks, 6), generator=g, device="cuda", dtype=torch.uint8)
    scale = (0.5 + torch.rand(blocks, generator=g, device="cuda")) * case["in_dim"] ** -0.5
    s["w"][:, :2] = scale.to(torch.float16)[:, None].view(torch.uint8)
    s["w"] = s["w"].flatten()
    return s


# ---- the plain forms -------------------------------------------------------


def _packed(y):
    """fp32 rows -> the packed fp16 activations: within 32 columns, j beside j + 16."""
    rows, cols = y.shape
    return y.to(torch.float16).view(rows, cols // 32, 2, 16).transpose(2, 3).reshape(rows, cols)


def _unpacked(a):
    """Packed fp16 activations -> fp32 rows."""
    rows, cols = a.shape
    return a.view(rows, cols // 32, 16, 2).transpose(2, 3).reshape(rows, cols).float()


def _plain_route(s):
    case, k = s["case"], s["case"]["top_k"]
    x = s["logits"].float()
    # chosen in 64 bits where a score is what is compared; ties to the lowest index
    choice = x
    if s["bias"] is not None:
        z = x.double()
        if case["score"] == "sigmoid":
            z = 1.0 / (1.0 + torch.exp(-z))
        else:
            z = torch.exp(z - z.amax(1, keepdim=True))
            z = z / z.sum(1, keepdim=True)
        choice = torch.where(x == -math.inf, x.double(), z + s["bias"].double())
    expert = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k]
    if case["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    weight = score.gather(1, expert)
    if case["renormalize"]:
        weight = weight / weight.sum(1, keepdim=True)
    flat = expert.flatten()
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device="cuda")
    each = (flat[:, None] == torch.arange(case["experts"], device="cuda")).sum(0)
    start = torch.cat([each.new_zeros(1), each.cumsum(0)])
    return {"expert": expert.int(), "weight": weight * case["scale"], "start": start.int(), "order": order.int(),
            "place": place.view(-1, k).int()}


def _plain_linear(s):
    case = s["case"]
    k, n, routes = case["in_dim"], case["out_dim"], len(s["order"])
    start = s["start"].long()
    # the experts with the most rows, as many as can have any
    mine = torch.sort(start.diff(), descending=True).indices[:routes]
    block = s["w"].view(case["experts"], -1, 6)[mine]
    scale = block[:, :, :2].contiguous().view(torch.float16).float()
    bits = (block[:, :, 2:, None] >> torch.arange(8, dtype=torch.uint8, device="cuda")) & 1
    w = torch.where(bits.flatten(2).view(-1, 32) == 1, scale.view(-1, 1), -scale.view(-1, 1))
    w = w.view(len(mine), n, k).transpose(1, 2).contiguous()
    # each expert's rows, as many as the largest group has
    at = start[mine, None] + torch.arange(s["most"], device="cuda")
    there = at < start[mine + 1, None]
    source = torch.where(there, at, 0)
    if case["rows"] == "tokens":
        source = s["order"].long()[source] // case["top_k"]
    y = torch.empty(routes, n, device="cuda")
    y[at[there]] = (_unpacked(s["act"])[source] @ w)[there]
    if case["act"] == "swiglu":
        gate, value = y[:, :n // 2], y[:, n // 2:]
        y = gate / (1.0 + torch.exp(-gate)) * value
    elif case["act"] == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return _packed(y) if case["out"] == "packed" else y


def _plain_combine(s):
    return s["x"] + (s["weight"][:, :, None] * s["y"][s["place"].long()]).sum(1)


# ---- the framework's calls -------------------------------------------------


_b1 = None


def _framework():
    global _b1
    if _b1 is None:
        import sys
        from pathlib import Path
        sys.path.insert(0, str(Path.cwd() / "bonsai.cpp_amd"))
        import bonsai_b1
        _b1 = bonsai_b1
    return _b1


def _own(s):
    b1, case = _framework(), s["case"]
    if case["kind"] == "route":
        r = b1.route(s["logits"], case["top_k"], score=case["score"], bias=s["bias"],
                     renormalize=case["renormalize"], scale=case["scale"])
        return {"expert": r.expert, "weight": r.weight, "start": r.start, "order": r.order, "place": r.place}
    routes = b1.Routes(s["expert"], s["weight"], s["start"], s["order"], s["place"])
    if case["kind"] == "combine":
        return b1.combine_experts(s["y"], routes, residual=s["x"])
    out = b1.linear_experts(s["act"], s["w"], routes, case["in_dim"], case["out_dim"], act=case["act"],
                            rows=case["rows"], packed=case["out"] == "packed" or None)
    if case["out"] == "packed":
        out = out.view(torch.float16).view(case["tokens"] * case["top_k"], -1)
    return out


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    return _plain_route(state) if kind == "route" else _plain_linear(state) if kind == "linear" else \
        _plain_combine(state)


# ---- the definitions in 64 bits --------------------------------------------


def _exact_route(case, s):
    x = s["logits"].double()
    score = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, 1)
    by = x if s["bias"] is None else (score + s["bias"].double()).masked_fill(x == -math.inf, -math.inf)
    # one expert at a time: the first of the highest that are left
    left, chosen = by.clone(), []
    for _ in range(case["top_k"]):
        top = left.max(1, keepdim=True).values
        chosen.append((left == top).int().argmax(1, keepdim=True))
        left.scatter_(1, chosen[-1], -math.inf)
    expert = torch.cat(chosen, 1)
    weight = torch.take_along_dim(score, expert, 1)
    if case["renormalize"]:
        weight = weight / weight.sum(1, keepdim=True)
    rows = [(expert == e).flatten().nonzero().flatten() for e in range(case["experts"])]
    order = torch.cat(rows)
    place = torch.argsort(order).view(expert.shape)
    ends = [0]
    for r in rows:
        ends.append(ends[-1] + len(r))
    return {"expert": expert.int(), "weight": weight * case["scale"],
            "start": torch.tensor(ends, dtype=torch.int32, device="cuda"), "order": order.int(),
            "place": place.int()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, s)
    if case["kind"] == "combine":
        out = s["x"].double()
        for j in range(case["top_k"]):
            out += s["weight"][:, j, None].double() * s["y"].double()[s["place"][:, j].long()]
        return out
    k, n, routes = case["in_dim"], case["out_dim"], case["tokens"] * case["top_k"]
    # column 32 b + j + 16 e of a packed row is stored at 32 b + 2 j + e
    def stored(cols):
        c = torch.arange(cols, device="cuda")
        return c // 32 * 32 + 2 * (c % 16) + c % 32 // 16

    a = s["act"][:, stored(k)].double()
    w = s["w"].view(case["experts"], n, k // 32, 6)
    shift = torch.arange(32, device="cuda")
    starts = s["start"].tolist()
    y = torch.zeros(routes, n, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        lo, hi = starts[e], starts[e + 1]
        if lo == hi:
            continue
        word = w[e, :, :, 2:].contiguous().view(torch.int32).long()
        scale = w[e, :, :, :2].contiguous().view(torch.float16).double()
        mine = (scale * (2.0 * (word >> shift & 1) - 1.0)).view(n, k)
        rows = torch.arange(lo, hi, device="cuda")
        if case["rows"] == "tokens":
            rows = torch.div(s["order"][lo:hi].long(), case["top_k"], rounding_mode="floor")
        y[lo:hi] = a[rows] @ mine.t()
    if case["act"] == "swiglu":
        y = torch.nn.functional.silu(y[:, :n // 2]) * y[:, n // 2:]
    elif case["act"] == "gelu_tanh":
        y = torch.nn.functional.gelu(y, approximate="tanh")
    if case["out"] == "rows":
        return y
    out = torch.empty_like(y)
    out[:, stored(y.shape[1])] = y
    return out
