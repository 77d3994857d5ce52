"""Plain attention, norms and rotation in float64 on the CPU, and how far a
kernel's rounded steps may take it: what the GPU tests compare with."""
import math

import torch

U32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def seen(nq, nk, causal, window):
    """[nq, nk]: which keys each token sees."""
    i = torch.arange(nq)[:, None] + (nk - nq)
    j = torch.arange(nk)[None]
    m = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        m &= j <= i
        if window:
            m &= j > i - window
    return m


def attention(q, k, v, scale, causal=False, window=0):
    """One sequence: q [nq, heads, d], k, v [nk, kv_heads, d] (16 bit).
    Returns (out, bound before the output's own rounding), float64.

    The bound, per element, with A = sum_j p_j |v_j| / sum_j p_j and the
    largest weight 1: each weight is rounded to the inputs' type, for the
    product with v and for the sum it is divided by (half a step of it times
    A in the product, and in the sum half a step times |out| <= A; where that
    type is fp16 half its smallest step, 2^-25, in place of half a step for
    weights below 2^-14, in both); a score's fp32
    sum of d products is off by at most e = (d + 2) U32 scale sum_d |q_d k_d|,
    which changes a weight by a factor 1 + e and the maximum it is relative to
    cancels, so numerator and denominator are off by e each; the sums over nk
    keys and the exponentials add (nk + 16) U32 each."""
    nq, heads, d = q.shape
    nk = k.shape[0]
    dtype = q.dtype
    group = heads // k.shape[1]
    out = torch.zeros(nq, heads, d, dtype=torch.float64)
    off = torch.zeros_like(out)
    mask = seen(nq, nk, causal, window)
    some = mask.any(1)
    if nk == 0 or not bool(some.any()):
        return out, off
    for h in range(heads):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        s = (q[:, h].double() @ kh.T * scale).masked_fill(~mask, -math.inf)
        mags = (q[:, h].double().abs() @ kh.abs().T * scale).masked_fill(~mask, 0.0)
        top = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(some[:, None], top, 0.0))
        total = torch.where(some, p.sum(1), 1.0)[:, None]
        vis = torch.where(mask.any(0)[:, None], vh, 0.0)
        # a masked key's value does not reach the row
        o = torch.zeros(nq, d, dtype=torch.float64)
        big = torch.zeros(nq, d, dtype=torch.float64)
        flat = torch.zeros(nq, d, dtype=torch.float64)
        if bool(torch.isfinite(vis).all()):
            o, big, flat = p @ vis, p @ vis.abs(), mask.double() @ vis.abs()
        else:
            for i in range(nq):
                vi = vh[mask[i]]
                o[i], big[i], flat[i] = p[i][mask[i]] @ vi, p[i][mask[i]] @ vi.abs(), vi.abs().sum(0)
        e = (d + 2) * U32 * mags.amax(1, keepdim=True)
        rel = 2 * half_step(dtype) + 2 * e + 2 * (nk + 16) * U32
        tiny = 2.0 ** -25 * (flat + nk * big / total) if dtype == torch.float16 else 0.0
        out[:, h] = torch.where(some[:, None], o / total, 0.0)
        off[:, h] = torch.where(some[:, None], (rel * big + tiny) / total, 0.0)
    return out, off


def packed_order(cols):
    """Stored position -> column of packed fp16 activations."""
    at = torch.arange(cols)
    return at // 32 * 32 + at % 32 // 2 + 16 * (at % 2)


def unpack(packed, rows, cols, ldp=None, first=0):
    """fp16 [rows, cols] of the packed activations in a uint8 buffer."""
    ldp = cols if ldp is None else ldp
    flat = packed.cpu().view(torch.float16)
    m = torch.stack([flat[first + r * ldp:first + r * ldp + cols] for r in range(rows)]) if rows else \
        torch.zeros(0, cols, dtype=torch.float16)
    out = torch.empty_like(m)
    out[:, packed_order(cols)] = m
    return out


def check(got, want, off, dtype, what):
    """got within off of want, after one rounding to dtype (half its smallest
    step, for results near zero, included); NaN where want is NaN."""
    got = got.double().cpu()
    u, least = half_step(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bound = off * (1 + u) + u * want.abs() + least
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(got)), f"{what}: NaN in other places"
    bad = ~nan & ~((got - want).abs() <= bound)
    if bool(bad.any()):
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: got {got[at]:.6g}, "
                             f"want {want[at]:.6g}, bound {bound[at]:.3g}")
