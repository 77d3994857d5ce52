"""Plain routing, grouped linears and weighted sums in float64 on the CPU, and
how far a kernel's rounded steps may take them: what the GPU tests of the
mixture-of-experts operators compare with."""
import math

import torch

from tests.attention_ref import U32

# tokens, experts, top_k, in_dim, out_dim -> the kernel that runs it: rows of a
# tile, or 0 and the few-rows kernel's waves and 256s of K a wave
KERNELS = {
    (40, 3, 2, 192, 256): (0, 3, 1), (33, 7, 2, 704, 320): (0, 3, 1), (20, 5, 2, 1024, 128): (0, 4, 1),
    (9, 6, 3, 1344, 192): (0, 3, 2), (21, 4, 2, 2048, 192): (0, 4, 2), (13, 3, 1, 4096, 128): (0, 8, 2),
    (30, 3, 2, 8192, 128): (0, 8, 4),
    (20, 20, 2, 192, 2496): (32, 0, 0), (100, 20, 3, 1088, 2304): (32, 0, 0), (200, 33, 6, 128, 576): (32, 0, 0),
    (7, 3, 2, 8256, 64): (32, 0, 0), (6, 2, 1, 16384, 320): (32, 0, 0),
    (2721, 5, 3, 192, 128): (64, 0, 0), (512, 20, 1, 1088, 2368): (64, 0, 0), (4000, 2, 1, 128, 2048): (64, 0, 0),
    (2829, 3, 3, 320, 320): (128, 0, 0), (2774, 20, 3, 832, 320): (128, 0, 0), (6000, 2, 1, 64, 2112): (128, 0, 0)}


def layout(expert, experts):
    """start, order and place of expert ids [tokens, top_k] (-1: no route)."""
    flat = expert.flatten().tolist()
    rows = [s for e in range(experts) for s, x in enumerate(flat) if x == e]
    start = [0]
    for e in range(experts):
        start.append(start[-1] + sum(x == e for x in flat))
    place = [-1] * len(flat)
    for r, s in enumerate(rows):
        place[s] = r
    i32 = torch.int32
    return (torch.tensor(start, dtype=i32), torch.tensor(rows + [-1] * (len(flat) - len(rows)), dtype=i32),
            torch.tensor(place, dtype=i32).view(expert.shape))


def route(logits, top_k, score="softmax", bias=None, renormalize=True, scale=1.0):
    """expert, weight and the weights' bound.  logits [tokens, experts].

    Softmax: the difference to the peak is rounded (half a step of at most 110
    counts: weights beyond e^-103 are 0), an exponential is off by at most 2
    steps, a sum of n positive terms by n/64 + 8 half steps, two divisions and
    the scale by half a step each; numerator and denominator both.  Sigmoid:
    64 bits but for the last rounding."""
    x = logits.double().cpu()
    tokens, experts = x.shape
    expert = torch.full((tokens, top_k), -1, dtype=torch.int32)
    weight = torch.zeros(tokens, top_k, dtype=torch.float64)
    off = torch.zeros(tokens, top_k, dtype=torch.float64)
    for t in range(tokens):
        row = x[t]
        if score == "softmax":
            peak = row[~row.isnan()].max() if bool((~row.isnan()).any()) else torch.tensor(math.nan)
            s = torch.exp(row - peak)
            s = s / s.nansum()
        else:
            s = torch.sigmoid(row)
        key = row if bias is None or bool((row == math.inf).any() and score == "softmax") else s + bias.double().cpu()
        live = [e for e in range(experts) if not row[e] == -math.inf and not key[e] == -math.inf]
        chosen = sorted(live, key=lambda e: (math.isnan(key[e]), -float(key[e].nan_to_num(0.0, math.inf, -math.inf)), e))
        chosen = chosen[:top_k]
        n = len(chosen)
        expert[t, :n] = torch.tensor(chosen, dtype=torch.int32)
        if not n:
            continue
        w = s[chosen]
        if renormalize:
            total = w.sum()
            w = w / total if not total == 0 else torch.zeros(n, dtype=torch.float64)
        nan = bool(row.isnan().any()) or (score == "softmax" and bool((row == math.inf).any()))
        if bias is not None:
            nan = nan or bool((key.isnan() & ~(row == -math.inf)).any())
        weight[t, :n] = math.nan if nan else w * scale
        if score == "softmax" and not nan:
            spread = min(110.0, float((peak - row[row > -math.inf]).max()))
            off[t, :n] = (w * scale).abs() * (2 * spread + 8 + experts / 64 + 16) * U32 + abs(scale) * 2.0 ** -126
        elif not nan:
            off[t, :n] = (w * scale).abs() * 2.0 ** -45
    return expert, weight, off


def linear(a, w):
    """a [rows, k] fp16 values, w [n, k] float64: float64 and its bound, k
    exact products summed in fp32 in any order, each addition off by a step at
    most (a matrix unit may cut where it does not round)."""
    a = a.double()
    return a @ w.T, a.abs() @ w.abs().T * (2 * (a.shape[1] + 16) * U32)


def activation(y, off, act):
    """act(y) and its bound for y off by `off`: silu' stays below 1.1, the
    tanh form of gelu's slope below 1.13.  silu(g) by 2^(-g log2 e): the
    exponent |g| log2 e is off by half a step for its product and a quarter for
    its factor, times ln 2 in the power, 0.75 |g| steps = 1.5 |g| U32; power and reciprocal
    by a step each, the sum, the product and the one with the value by half a
    step each, and the constant 1 more: 1.5 |g| + 8 half steps.  gelu's are
    within 3e-7 max(1, |y|)."""
    if act == "swiglu":
        h = y.shape[1] // 2
        g, v, og, ov = y[:, :h], y[:, h:], off[:, :h], off[:, h:]
        silu = g * torch.sigmoid(g)
        out = silu * v
        return out, 1.1 * og * v.abs() + silu.abs() * ov + 1.1 * og * ov + (1.5 * g.abs() + 8) * U32 * out.abs() + 2.0 ** -126
    if act == "gelu_tanh":
        out = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
        return out, 1.13 * off + 3e-7 * y.abs().clamp(min=1.0)
    return y, off


def experts(acts, weights, start, order, top_k, by_token, act="none"):
    """acts [rows, k] fp16 (unpacked), weights [experts, n, k] float64 -> (out,
    bound) of the rows start[0] .. start[-1]."""
    outs, offs = [], []
    for e in range(len(start) - 1):
        rows = torch.arange(int(start[e]), int(start[e + 1]))
        src = order[rows].long() // top_k if by_token else rows
        y, off = linear(acts[src], weights[e])
        y, off = activation(y, off, act)
        outs.append(y)
        offs.append(off)
    return torch.cat(outs), torch.cat(offs)


def combine(y, weight, place, residual):
    """out and its bound: top_k fused multiply-adds, each off by half a step of
    a partial sum."""
    t, k = place.shape
    out = residual.double().cpu().clone() if residual is not None else torch.zeros(t, y.shape[1], dtype=torch.float64)
    mags = out.abs()
    for j in range(k):
        there = place[:, j] >= 0
        part = weight[there, j, None].double() * y[place[there, j].long()].double()
        out[there] += part
        mags[there] += part.abs()
    return out, mags * (k + 2) * U32
