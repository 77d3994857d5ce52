"""GPU checks of windowed causal attention whose tiles' keys are split, with
contiguous and paged keys, against float64."""
import pytest

from tests import attention_ref as ref
from tests.test_gpu_attention import b1, dtype_of, i32, make, paged, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def expect(torch, q, k, v, ql, kl, scale, window, block=512):
    """ref.attention of every sequence, a block of tokens with the keys that
    any of them sees at a time."""
    outs, offs = [], []
    for a, b, n, m in zip(ref.starts(ql), ref.starts(kl), ql, kl):
        for i in range(0, n, block):
            end = min(i + block, n)
            lo, hi = max(0, m - n + i - window + 1), max(0, m - n + end)
            o, e = ref.attention(q[a + i:a + end].cpu(), k[b + lo:b + hi].cpu(), v[b + lo:b + hi].cpu(), scale, True,
                                 window)
            outs.append(o)
            offs.append(e)
    return torch.cat(outs), torch.cat(offs)


# (query lengths, key lengths, heads, key heads, head dim, type, window, page):
# the last tile of a sequence has fewer rows, and so fewer keys, than the others
SPLIT = [
    ([129, 129], [4096, 4096], 8, 8, 128, "fp16", 2048, 64),
    ([4097, 4097], [4097, 4097], 1, 1, 128, "bf16", 1024, 16),
    ([19713], [30000], 1, 1, 128, "fp16", 4096, 64),
    ([130, 70, 257], [3000, 2000, 5000], 4, 2, 64, "fp16", 1536, 16),
    ([65, 200], [4000, 4100], 8, 4, 256, "bf16", 1023, 256),
]


@pytest.mark.parametrize("case", SPLIT, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}")
def test_split_windows(torch, b1, case):
    ql, kl, heads, kv_heads, d, t, window, page = case
    say(f"split windows {case}")
    dtype = dtype_of(torch, t)
    q, k, v = make(torch, 51, ql, kl, heads, kv_heads, d, dtype)
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, window)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = i32(torch, ref.starts(ql))
    out = torch.full_like(q, float("nan"))  # rows that no work-group writes
    b1.attention(q, k, v, starts, i32(torch, ref.starts(kl)), causal=True, window=window, out=out, bad=bad)
    ref.check(out, want, off, dtype, "contiguous")
    kc, vc, table = paged(torch, 7, k, v, kl, page, "head")
    out.fill_(float("nan"))
    b1.attention_paged(q, kc, vc, starts, i32(torch, kl), table, window=window, out=out, bad=bad)
    ref.check(out, want, off, dtype, "paged")
    assert int(bad) == 0
