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


@pytest.mark.parametrize("ql,kl,heads,kv_heads,d,window,page", [
    ([130, 40], [400, 150], 4, 2, 128, 50, 16), ([200], [333], 2, 2, 64, 33, 4), ([90, 70], [300, 90], 4, 1, 64, 77, 1),
    ([150], [2100], 2, 1, 256, 300, 2), ([129, 60], [5000, 4000], 8, 8, 128, 2000, 16), ([3, 1], [500, 90], 8, 2, 128, 45, 16),
    ([1], [3000], 4, 4, 64, 1030, 1)])
def test_pages_that_a_window_left(torch, b1, ql, kl, heads, kv_heads, d, window, page):
    """Pages before the first key that any of a call's tokens sees may be gone:
    their table entries are anything, what they held too."""
    say(f"pages left {ql} {kl} {d} {window} {page}")
    q, k, v = make(torch, 52, ql, kl, heads, kv_heads, d, torch.float16)
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, window)
    kc, vc, table = paged(torch, 8, k, v, kl, page, "head")
    gone = 0
    for b, (n, m) in enumerate(zip(ql, kl)):
        for j in range(max(0, m - n - window + 1) // page):  # all keys before the first token's window
            kc[table[b, j]], vc[table[b, j]] = float("nan"), float("nan")
            table[b, j] = (-1, 1 << 30)[j % 2]
            gone += 1
    assert gone > 0
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = b1.attention_paged(q, kc, vc, i32(torch, ref.starts(ql)), i32(torch, kl), table, window=window, bad=bad)
    ref.check(out, want, off, torch.float16, "rows")
    assert int(bad) == 0


@pytest.mark.parametrize("ql,kl", [([40], [40]), ([90, 33], [3000, 2000]), ([2, 1], [30, 3000])])
def test_scores_past_fp32(torch, b1, ql, kl):
    """A score that only its scale takes past fp32's range gives NaN, never
    the zeros of a row that sees nothing; rows that do not see it are right."""
    say(f"scores past fp32 {ql} {kl}")
    heads, d = 2, 64
    q, k, v = make(torch, 53, ql, kl, heads, heads, d, torch.bfloat16)
    q[..., 1:] *= 2.0 ** -6
    q[..., 0], k[..., 0] = 2.0 ** 60, 0.0
    last = ref.starts(kl)[1] - 1
    k[last, 0, 0] = 2.0 ** 66  # seen by the first sequence's last token: 2^126, times 16 log2(e)
    out = b1.attention(q, k, v, i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl)), causal=True, scale=16.0)
    row = ql[0] - 1
    assert bool(out[row, 0].isnan().all())
    rest = torch.ones(out.shape[:2], dtype=torch.bool)
    rest[row, 0] = False
    assert bool(out.cpu()[rest].isfinite().all())
    k[last, 0, 0] = 0.0
    want, off = [], []
    for a, b, n, m in zip(ref.starts(ql), ref.starts(kl), ql, kl):
        o, e = ref.attention(q[a:a + n].cpu(), k[b:b + m].cpu(), v[b:b + m].cpu(), 16.0, True)
        want.append(o)
        off.append(e)
    want, off = torch.cat(want), torch.cat(off)
    ref.check(out.cpu()[rest], want[rest], off[rest], torch.bfloat16, "rows that do not see it")
