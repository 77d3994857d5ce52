"""GPU checks of attention from bf16 inputs into packed fp16 activations: the
softmax weights are as fine as the output, in tiles and few rows alike."""
import pytest

from tests import attention_ref as ref
from tests.test_gpu_attention import b1, i32, make, paged, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def expect(torch, q, k, v, ql, kl, scale, causal, window):
    """ref.attention with the bound of weights of two bf16 parts: of the half
    steps of one part, 2 * 2^-8 of the sum of weights times |v|, only 2^-8 of
    2^-8 is left, for the product and for the sum each.  (That sum over the
    sum of weights is the attention of |v|.)"""
    outs, offs = [], []
    for a, b, n, m in zip(ref.starts(ql), ref.starts(kl), ql, kl):
        args = q[a:a + n].cpu(), k[b:b + m].cpu()
        o, e = ref.attention(*args, v[b:b + m].cpu(), scale, causal, window)
        size, _ = ref.attention(*args, v[b:b + m].cpu().abs(), scale, causal, window)
        outs.append(o)
        offs.append(e - 2 * (2.0 ** -8 - 2.0 ** -16) * size)
    return torch.cat(outs), torch.cat(offs)


CASES = [
    # (query lengths, key lengths, heads, key heads, head dim, causal, window, page)
    ([200], [200], 4, 2, 128, True, 0, 16), ([129, 40], [129, 300], 2, 1, 64, True, 0, 64),
    ([70, 33], [200, 33], 4, 4, 256, True, 0, 16), ([300], [300], 5, 1, 128, False, 0, None),
    ([100, 9, 260], [1500, 2900, 260], 4, 2, 128, True, 0, 16),  # split
    ([130, 257], [3000, 5000], 4, 2, 64, True, 1536, 4), ([65], [4000], 4, 4, 256, True, 1023, 256),
    ([1, 3], [3000, 70], 8, 2, 128, True, 0, 16),  # few rows
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}")
def test_packed_output_of_bf16_inputs(torch, b1, case):
    ql, kl, heads, kv_heads, d, causal, window, page = case
    say(f"packed bf16 {case}")
    q, k, v = make(torch, 71, ql, kl, heads, kv_heads, d, torch.bfloat16)
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, causal, window)
    assert bool((off >= 0).all())
    starts, n = i32(torch, ref.starts(ql)), sum(ql)
    out = b1.attention(q, k, v, starts, i32(torch, ref.starts(kl)), causal=causal, window=window, packed=True)
    ref.check(ref.unpack(out, n, heads * d).view(n, heads, d), want, off, torch.float16, "contiguous")
    if page:
        kc, vc, table = paged(torch, 9, k, v, kl, page, "token")
        out = b1.attention_paged(q, kc, vc, starts, i32(torch, kl), table, window=window, packed=True)
        ref.check(ref.unpack(out, n, heads * d).view(n, heads, d), want, off, torch.float16, "paged")
