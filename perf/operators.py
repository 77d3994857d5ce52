"""Cases of the operators around the 1-bit linears of a transformer block: the
RMS norm in front of them, the q/k/v columns' norm and rotation, and attention
over whole prompts and over a paged cache.

A case is a dict of plain values; `kind` names the call:

  norm    bonsai_b1.rms_norm: x + add -> the new residual stream (fp32) and
          its RMS norm as packed fp16 activations
  qkv     bonsai_b1.qkv_rope: fp32 q/k/v rows -> head norm, rotary, 16 bit
  append  bonsai_b1.qkv_rope_paged: the same, k and v into a paged cache
  attn    bonsai_b1.attention over packed sequences
  paged   bonsai_b1.attention_paged: new tokens over a paged cache

Sequence lengths are texts, "q" new tokens and "kv" keys (new ones included)
of each sequence.  `out` is "rows" (the inputs' type) or "packed" (the packed
fp16 activations of the next linear, returned as fp16 values in their stored
order).
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the pre-norm of a decoding step: a few tokens, bound by latency
        {"name": "norm_step", "kind": "norm", "rows": 8, "h": 2560},
        # the pre-norm of a batch of prompts
        {"name": "norm_prompts", "kind": "norm", "rows": 8192, "h": 4096},
        # one decoding step of 64 requests: a token each, into the cache
        {"name": "append_step", "kind": "append", "q": ",".join(["1"] * 64),
         "kv": ",".join(str(40 + 37 * i) for i in range(64)), "heads": 32, "kv_heads": 8, "d": 128, "type": "bf16",
         "rope": "half", "page": 64, "order": "head"},
        # prompts of odd lengths into the cache, pages ending inside them
        {"name": "append_prompts", "kind": "append", "q": "1500,17,333,998,1", "kv": "1500,17,461,3000,78",
         "heads": 32, "kv_heads": 8, "d": 128, "type": "fp16", "rope": "half", "page": 16, "order": "token"},
        # q/k/v of a diffuser's block: 64 x 64 latents and 512 text tokens
        {"name": "qkv_image", "kind": "qkv", "rows": 4608, "heads": 24, "kv_heads": 24, "d": 128, "type": "fp16",
         "rope": "pairs"},
        # that block's attention: every token sees every other, into the output projection's packed input
        {"name": "attn_image", "kind": "attn", "q": "4608", "kv": "4608", "heads": 24, "kv_heads": 24, "d": 128,
         "type": "fp16", "causal": False, "window": 0, "out": "packed"},
        # short prompts of a text encoder in one call, where latency counts
        {"name": "attn_short", "kind": "attn", "q": "77,5,31,1,64,19,40,12", "kv": "77,5,31,1,64,19,40,12",
         "heads": 32, "kv_heads": 8, "d": 128, "type": "fp16", "causal": True, "window": 0, "out": "packed"},
        # a batch of prompts of a decoder with grouped heads
        {"name": "attn_prompts", "kind": "attn", "q": "2048,1,333,1024,17,1777,3000", "kv": "2048,1,333,1024,17,1777,3000",
         "heads": 32, "kv_heads": 8, "d": 128, "type": "bf16", "causal": True, "window": 0, "out": "rows"},
        # a long document through narrow heads
        {"name": "attn_long", "kind": "attn", "q": "8191", "kv": "8191", "heads": 16, "kv_heads": 4, "d": 64,
         "type": "fp16", "causal": True, "window": 0, "out": "packed"},
        # one request's decoding step over a long cache
        {"name": "paged_one", "kind": "paged", "q": "1", "kv": "32700", "heads": 32, "kv_heads": 8, "d": 128,
         "type": "fp16", "causal": True, "window": 0, "out": "packed", "page": 64, "order": "head"},
        # a decoding step of 64 requests of every age
        {"name": "paged_batch", "kind": "paged", "q": ",".join(["1"] * 64),
         "kv": ",".join(str(60 + (i * 1297) % 8100) for i in range(64)), "heads": 32, "kv_heads": 8, "d": 128,
         "type": "bf16", "causal": True, "window": 0, "out": "packed", "page": 16, "order": "token"},
        # chunks of new prompt tokens over what earlier chunks left in the cache
        {"name": "paged_chunk", "kind": "paged", "q": "512,300,512,45", "kv": "9000,4111,512,13045", "heads": 32,
         "kv_heads": 8, "d": 128, "type": "fp16", "causal": True, "window": 0, "out": "packed", "page": 64,
         "order": "head"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


# a drawn case costs no more than the largest listed one, and its plain form's
# padded scores fit what the listed ones' do
MOST = {"flops": 2.6e11, "bytes": 1.0e9}
MOST_SCORES = 2.0e9


def draw(rng):
    """A case of the listed ones' ranges: 1 to 8192 tokens, odd counts among
    them, 1 to 64 sequences, 1 to 8 query heads a key head, pages of 1 to 256
    tokens, caches of up to 32768 keys."""
    while True:
        kind = rng.choice(["norm", "qkv", "append", "attn", "attn", "attn", "paged", "paged", "paged"])
        if kind == "norm":
            case = {"kind": kind, "rows": _log(rng, 1, 8192), "h": 32 * _log(rng, 8, 256)}
            if work(case)["bytes"] <= MOST["bytes"]:
                return case
            continue
        d = rng.choice([64, 128, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
        group = rng.choice([1, 1, 2, 3, 4, 6, 8])
        case = {"kind": kind, "heads": kv_heads * group, "kv_heads": kv_heads, "d": d,
                "type": rng.choice(["fp16", "bf16"])}
        if kind == "qkv":
            case |= {"rows": _log(rng, 1, 8192), "rope": rng.choice(["half", "pairs"])}
        else:
            n = _log(rng, 1, 64)
            if kind == "attn":
                n = min(n, 16)
                q = [_log(rng, 1, 4096) for _ in range(n)]
                kv = q if rng.random() < 0.7 else [_log(rng, 1, 4096) for _ in range(n)]
            else:
                single = rng.random() < (0.6 if kind == "paged" else 0.4)
                q = [1] * n if single else [_log(rng, 1, 512 if kind == "paged" else 2048) for _ in range(n)]
                kv = [v + _log(rng, 1, 32768 if kind == "paged" else 2048) - 1 for v in q]
                case |= {"page": 1 << rng.randint(0, 8), "order": rng.choice(["head", "token"])}
            case |= {"q": _text(q), "kv": _text(kv)}
            if kind == "append":
                case |= {"rope": rng.choice(["half", "pairs"])}
            else:
                causal = kind == "paged" or rng.random() < 0.7
                case |= {"causal": causal, "window": _log(rng, 1, 4096) if causal and rng.random() < 0.2 else 0,
                         "out": rng.choice(["rows", "packed"])}
                if len(q) * case["heads"] * max(q) * max(kv) > MOST_SCORES:
                    continue
        w = work(case)
        if w["flops"] <= MOST["flops"] and w["bytes"] <= MOST["bytes"]:
            return case


def _lens(case):
    return [int(v) for v in case["q"].split(",")], [int(v) for v in case["kv"].split(",")]


def _visible(case):
    """The visible (query, key) pairs of each sequence, and the keys that any of its queries sees."""
    pairs, keys = [], []
    for nq, nk in zip(*_lens(case)):
        if not case["causal"]:
            pairs.append(nq * nk)
            keys.append(nk if nq else 0)
            continue
        first = nk - nq
        w = case["window"] or nk + nq + 1
        pairs.append(sum(max(0, min(p + 1, w)) for p in range(first, nk)))
        keys.append(min(nk, nk - max(0, first) + w - 1) if nq else 0)
    return pairs, keys


def work(case):
    if case["kind"] == "norm":
        values = case["rows"] * case["h"]
        return {"bytes": 14 * values + 4 * case["h"], "flops": 5 * values}
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    if case["kind"] in ("qkv", "append"):
        rows = case["rows"] if case["kind"] == "qkv" else sum(_lens(case)[0])
        values = rows * (heads + 2 * kv_heads) * d
        return {"bytes": 6 * values + 4 * rows * d, "flops": 8 * values}
    pairs, keys = _visible(case)
    q = sum(_lens(case)[0])
    return {"bytes": 4 * q * heads * d + 4 * sum(keys) * kv_heads * d, "flops": 4 * d * heads * sum(pairs)}


def _pages(kv, page, g):
    """A page table of shuffled pages, -1 behind each sequence's last, and the number of pages."""
    need = [-(-v // page) for v in kv]
    total = sum(need) + 3
    table = torch.full((len(kv), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(total, generator=g, device="cuda").int()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _starts(lens):
    total, starts = 0, [0]
    for v in lens:
        total += v
        starts.append(total)
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def _rope_table(rows, d):
    """cos and sin of each position's angles, in 64 bits and rounded once."""
    angle = torch.arange(rows, device="cuda").double()[:, None] * \
        10000.0 ** (-torch.arange(d // 2, device="cuda").double() / (d // 2))
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, spread=1.0):
        return torch.randn(shape, generator=g, device="cuda") * spread

    s = {"case": case}
    if case["kind"] == "norm":
        s["x"] = normal(case["rows"], case["h"], spread=3.0)
        s["add"] = normal(case["rows"], case["h"])
        s["w"] = 1.0 + normal(case["h"], spread=0.2)
        return s
    heads, kv_heads, d, dtype = case["heads"], case["kv_heads"], case["d"], TYPES[case["type"]]
    if case["kind"] != "qkv":
        q, kv = _lens(case)
        s |= {"q_start": _starts(q), "most_q": max(q), "most_kv": max(kv), "rows": sum(q)}
        if case["kind"] == "attn":
            s["kv_start"] = s["q_start"] if q == kv else _starts(kv)
        else:
            s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
            s["pages"], total = _pages(kv, case["page"], g)
            shape = (total, kv_heads, case["page"], d)
            if case["order"] == "token":
                shape = (total, case["page"], kv_heads, d)
            s["k_cache"], s["v_cache"] = normal(*shape, spread=1.5).to(dtype), normal(*shape).to(dtype)
            if case["order"] == "token":
                s["k_cache"], s["v_cache"] = s["k_cache"].transpose(1, 2), s["v_cache"].transpose(1, 2)
    rows = case["rows"] if case["kind"] == "qkv" else s["rows"]
    if case["kind"] in ("qkv", "append"):
        qkv = normal(rows, (heads + 2 * kv_heads) * d)  # one linear's output columns
        s["q"], s["k"], s["v"] = qkv.split([heads * d, kv_heads * d, kv_heads * d], 1)
        s["q_weight"], s["k_weight"] = 1.0 + normal(d, spread=0.2), 1.0 + normal(d, spread=0.2)
        s["rope"] = _rope_table(rows if case["kind"] == "qkv" else s["most_kv"], d)
        return s
    s["q"] = normal(rows, heads, d, spread=1.5).to(dtype)
    if case["kind"] == "attn":
        keys = sum(_lens(case)[1])
        s["k"], s["v"] = normal(keys, kv_heads, d, spread=1.5).to(dtype), normal(keys, kv_heads, d).to(dtype)
    return s


# ---- the plain forms -------------------------------------------------------


def _packed(y):
    """fp32 rows -> the packed fp16 activations: within 32 columns, j beside j + 16."""
    rows, cols = y.shape
    return y.to(torch.float16).view(rows, cols // 32, 2, 16).transpose(2, 3).reshape(rows, cols)


def _plain_norm(s):
    h = s["x"] + s["add"]
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["w"]
    return {"residual": h, "packed": _packed(y)}


def _rotate(x, rope, form):
    half = x.shape[-1] // 2
    c, sn = rope[:, None, :half], rope[:, None, half:]
    if form == "half":
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * sn, b * c + a * sn], -1)
    a, b = x[..., ::2], x[..., 1::2]
    return torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)


def _plain_qkv(s, positions):
    case = s["case"]
    d, dtype, rows = case["d"], TYPES[case["type"]], s["q"].shape[0]
    q, k, v = (s[n].reshape(rows, -1, d) for n in ("q", "k", "v"))
    rope = s["rope"] if positions is None else s["rope"][positions]
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_weight"]
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_weight"]
    return _rotate(q, rope, case["rope"]).to(dtype), _rotate(k, rope, case["rope"]).to(dtype), v.to(dtype)


def _token_places(s):
    """Each new token's sequence and its position among that sequence's keys."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), row.int(), right=True)
    return seq, s["kv_len"][seq].long() - s["q_start"][seq + 1].long() + row


def _plain_append(s):
    seq, pos = _token_places(s)
    q, k, v = _plain_qkv(s, pos)
    page = s["case"]["page"]
    where = s["pages"][seq, pos // page].long()
    s["k_cache"][where, :, pos % page] = k
    s["v_cache"][where, :, pos % page] = v
    return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}


def _padded(x, start, most):
    """Packed rows -> [sequences, most, ...] and which of them are there."""
    at = start[:-1, None].long() + torch.arange(most, device="cuda")
    there = at < start[1:, None]
    return x[torch.where(there, at, 0)], there


def _plain_attention(s):
    case = s["case"]
    group, d = case["heads"] // case["kv_heads"], case["d"]
    q, q_there = _padded(s["q"], s["q_start"], s["most_q"])
    if case["kind"] == "attn":
        k, _ = _padded(s["k"], s["kv_start"], s["most_kv"])
        v, _ = _padded(s["v"], s["kv_start"], s["most_kv"])
        nk = s["kv_start"].diff()
    else:
        at = torch.arange(s["most_kv"], device="cuda")
        where = s["pages"][:, at // case["page"]].long().clamp(min=0)
        k, v = s["k_cache"][where, :, at % case["page"]], s["v_cache"][where, :, at % case["page"]]
        nk = s["kv_len"]
    nq = s["q_start"].diff()
    n, lq, lk = len(nq), s["most_q"], s["most_kv"]
    q = q.float().view(n, lq, case["kv_heads"], group, d).permute(0, 2, 3, 1, 4).reshape(n, -1, group * lq, d)
    k, v = k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
    score = (q @ k.transpose(2, 3).contiguous()).mul_(d ** -0.5).view(n, -1, group, lq, lk)
    key = torch.arange(lk, device="cuda")
    seen = (key < nk[:, None])[:, None, :]
    if case["causal"]:
        last = (nk - nq)[:, None] + torch.arange(lq, device="cuda")
        seen = seen & (key <= last[:, :, None])
        if case["window"]:
            seen = seen & (key > last[:, :, None] - case["window"])
    seen = seen[:, None, None].expand(n, 1, 1, lq, lk)
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, -1, group * lq, lk) @ v).view(n, -1, group, lq, d) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, lq, -1)[q_there]
    return _packed(o) if case["out"] == "packed" else o.to(TYPES[case["type"]]).view(-1, case["heads"], d)


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
    if case["kind"] == "norm":
        h, packed = b1.rms_norm(s["x"], s["w"], EPS, add=s["add"], packed=True)
        return {"residual": h, "packed": packed.view(torch.float16).view(s["x"].shape)}
    if case["kind"] in ("qkv", "append"):
        options = {"q_weight": s["q_weight"], "k_weight": s["k_weight"], "eps": EPS, "rope": s["rope"],
                   "interleaved": case["rope"] == "pairs"}
        if case["kind"] == "qkv":
            return dict(zip("qkv", b1.qkv_rope(s["q"], s["k"], s["v"], case["d"], dtype=TYPES[case["type"]],
                                               **options)))
        q = b1.qkv_rope_paged(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["q_start"], s["kv_len"],
                              s["pages"], **options)
        return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}
    options = {"causal": case["causal"], "window": case["window"], "packed": case["out"] == "packed" or None}
    if case["kind"] == "attn":
        out = b1.attention(s["q"], s["k"], s["v"], s["q_start"], s["kv_start"], **options)
    else:
        out = b1.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["q_start"], s["kv_len"], s["pages"], **options)
    if case["out"] == "packed":
        out = out.view(torch.float16).view(s["rows"], -1)
    return out


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "qkv":
        return dict(zip("qkv", _plain_qkv(state, None)))
    if kind == "append":
        return _plain_append(state)
    return _plain_attention(state)


# ---- the definitions in 64 bits --------------------------------------------


def _exact_packed(y):
    """Column 32 b + j + 16 e of a row is stored at 32 b + 2 j + e."""
    col = torch.arange(y.shape[1], device=y.device)
    at = col // 32 * 32 + 2 * (col % 16) + col % 32 // 16
    out = torch.empty_like(y)
    out[:, at] = y
    return out


def _exact_head(x, weight, rope, form):
    """One row's heads [heads, d] normalised and turned by complex factors."""
    x = x * weight / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    half = x.shape[-1] // 2
    turn = torch.complex(rope[..., :half], rope[..., half:])[:, None]
    if form == "half":
        z = torch.complex(x[..., :half], x[..., half:]) * turn
        return torch.cat([z.real, z.imag], -1)
    return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) * turn).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = s["x"].double() + s["add"].double()
        norm = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        return {"residual": h, "packed": _exact_packed(h * s["w"].double() / (norm * norm / case["h"] + EPS).sqrt())}
    d = case["d"]
    if case["kind"] in ("qkv", "append"):
        rows = s["q"].shape[0]
        q, k, v = (s[n].double().view(rows, -1, d) for n in ("q", "k", "v"))
        if case["kind"] == "append":
            at = [nk - nq + i for nq, nk in zip(*_lens(case)) for i in range(nq)]
            rope = s["rope"].double()[torch.tensor(at, device="cuda")]
        else:
            rope = s["rope"].double()
        q = _exact_head(q, s["q_weight"].double(), rope, case["rope"])
        k = _exact_head(k, s["k_weight"].double(), rope, case["rope"])
        if case["kind"] == "qkv":
            return {"q": q, "k": k, "v": v}
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        row, page = 0, case["page"]
        pages = s["pages"].tolist()
        for b, (nq, nk) in enumerate(zip(*_lens(case))):
            pos = list(range(nk - nq, nk))
            where = torch.tensor([pages[b][p // page] for p in pos], device="cuda")
            slot = torch.tensor([p % page for p in pos], device="cuda")
            kc[where, :, slot], vc[where, :, slot] = k[row:row + nq], v[row:row + nq]
            row += nq
        return {"q": q, "k": kc, "v": vc}
    out = torch.zeros(s["rows"], case["heads"], d, dtype=torch.float64, device="cuda")
    group, row, keys = case["heads"] // case["kv_heads"], 0, 0
    for b, (nq, nk) in enumerate(zip(*_lens(case))):
        if case["kind"] == "attn":
            k, v = s["k"][keys:keys + nk].double(), s["v"][keys:keys + nk].double()
        else:
            used = s["pages"][b, :-(-nk // case["page"])].long()
            k, v = (s[n][used].double().transpose(1, 2).reshape(-1, case["kv_heads"], d)[:nk]
                    for n in ("k_cache", "v_cache"))
        apart = torch.arange(nk, device="cuda")[None] - torch.arange(nk - nq, nk, device="cuda")[:, None]
        hidden = apart > (0 if case["causal"] else nk + nq)
        if case["window"]:
            hidden |= apart <= -case["window"]
        there = ~hidden.all(1)
        for h in range(case["heads"] if bool(there.any()) else 0):
            z = s["q"][row:row + nq, h].double()[there] @ k[:, h // group].t() / math.sqrt(d)
            z = torch.softmax(z.masked_fill(hidden[there], -math.inf), 1)
            mine = out[row:row + nq, h]
            mine[there] = z @ v[:, h // group]
        row += nq
        keys += nk
    return _exact_packed(out.view(s["rows"], -1)) if case["out"] == "packed" else out
