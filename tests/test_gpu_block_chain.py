"""GPU check of a decoder block's attention half in chunks and single tokens
through a paged cache: every operator of every step, element by element,
against float64 on the operands that it read."""
import math

import pytest

from tests import attention_ref as ref
from tests.test_gpu_block_ops import b1, head_ref, i32, norm_ref, normal, say, table, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def linear_ref(a, w):
    """a [rows, k] fp16 values, w [n, k] float64: float64 and its bound, k
    exact products summed in fp32 in any order, each addition off by a step at
    most (a matrix unit may cut where it does not round)."""
    a, w = a.double(), w.cpu()
    return a @ w.T, a.abs() @ w.abs().T * (2 * (a.shape[1] + 16) * ref.U32)


@pytest.mark.parametrize("t,window", [("fp16", 0), ("bf16", 60)])
def test_each_step_of_chunks_through_a_cache(torch, b1, unpack, t, window):
    from bonsai_b1 import synth
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[t]
    lens, hidden, heads, kv_heads, d, page = [70, 133, 5], 768, 6, 2, 128, 16
    total, nq, nk = sum(lens), heads * d, kv_heads * d
    width = nq + 2 * nk
    x = normal(torch, 60, total, hidden)
    w_norm = 1.0 + normal(torch, 61, hidden, spread=0.2)
    wqkv, wo = synth.device_packed_weights(width, hidden, 62), synth.device_packed_weights(hidden, nq, 63)
    wqkv64, wo64 = unpack(wqkv, width, hidden), unpack(wo, hidden, nq)
    qw, kw = 1.0 + normal(torch, 64, d, spread=0.2), 1.0 + normal(torch, 65, d, spread=0.2)
    rope = table(torch, 256, d)
    at = ref.starts(lens)
    pages = torch.randperm(3 * 9, generator=torch.Generator().manual_seed(3)).int().view(3, 9).cuda()
    kc, vc = (torch.full((27, kv_heads, page, d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    done = [0, 0, 0]
    for turn, step in enumerate([[50, 100, 1], [17, 30, 0], [1, 1, 1], [2, 1, 3], [0, 1, 0]]):
        say(f"step {turn} {step}")
        rows = torch.cat([torch.arange(at[b] + done[b], at[b] + done[b] + c) for b, c in enumerate(step)]).cuda()
        xs, n = x[rows].contiguous(), len(rows)
        pos = torch.cat([torch.arange(a, a + c) for a, c in zip(done, step)])
        done = [a + c for a, c in zip(done, step)]
        st, kl = i32(torch, ref.starts(step)), i32(torch, done)

        packed = b1.rms_norm(xs, w_norm, packed=True)
        want, off = norm_ref(torch, xs, w_norm, 1e-6)
        a16 = ref.unpack(packed, n, hidden)
        ref.check(a16, want, off, torch.float16, "norm")

        qkv = b1.linear_packed_f16(packed, wqkv, hidden, width, n)
        want, off = linear_ref(a16, wqkv64)
        ref.check(qkv, want, off, torch.float32, "q/k/v linear")

        before = kc.clone(), vc.clone()
        q, k, v = qkv.split([nq, nk, nk], 1)
        q16 = b1.qkv_rope_paged(q, k, v, kc, vc, st, kl, pages, qw, kw, rope=rope, bad=bad)
        want, off = head_ref(torch, q.reshape(n, heads, d), qw, rope[pos.cuda()], False, 1e-6)
        ref.check(q16, want, off, dtype, "q")
        seq = torch.repeat_interleave(torch.arange(3), torch.tensor(step))
        place = pages[seq.cuda(), (pos // page).cuda()].long(), (pos % page).cuda()
        for name, cache, old, src, w, r in (("k", kc, before[0], k, kw, rope[pos.cuda()]),
                                            ("v", vc, before[1], v, None, None)):
            want, off = head_ref(torch, src.reshape(n, kv_heads, d), w, r, False, 1e-6)
            ref.check(cache[place[0], :, place[1]], want, off, dtype, name)
            same = torch.ones(27, page, dtype=torch.bool, device="cuda")
            same[place] = False
            assert torch.equal(cache.transpose(1, 2)[same].nan_to_num(7.0), old.transpose(1, 2)[same].nan_to_num(7.0))

        out = b1.attention_paged(q16, kc, vc, st, kl, pages, window=window, packed=True, bad=bad)
        wants, offs = [], []
        for b, c in enumerate(step):
            if c == 0:
                continue
            used = pages[b, :-(-done[b] // page)].long()
            ks, vs = (m[used].transpose(1, 2).reshape(-1, kv_heads, d)[:done[b]].cpu() for m in (kc, vc))
            first = ref.starts(step)[b]
            o, e = ref.attention(q16[first:first + c].cpu(), ks, vs, d ** -0.5, True, window)
            wants.append(o)
            offs.append(e)
        o16 = ref.unpack(out, n, nq)
        ref.check(o16.view(n, heads, d), torch.cat(wants), torch.cat(offs), torch.float16, "attention")

        y = b1.linear_packed_f16(out, wo, nq, hidden, n)
        want, off = linear_ref(o16, wo64)
        ref.check(y, want, off, torch.float32, "output linear")
        assert int(bad) == 0
    assert done == lens
