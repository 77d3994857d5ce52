"""GPU checks of bonsai_b1_attention: packed sequences with contiguous and
paged keys, against float64 (tests/attention_ref.py derives the bounds)."""
import math
import sys

import pytest

from tests import attention_ref as ref

pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need the MI355X"
    return t


@pytest.fixture(scope="module")
def b1(torch):
    import bonsai_b1
    bonsai_b1.load()
    return bonsai_b1


def dtype_of(torch, name):
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[name]


def i32(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(torch, seed, q, kv, heads, kv_heads, d, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(n, h, spread):
        return (torch.randn((n, h, d), generator=g, device="cuda") * spread).to(dtype)

    return normal(sum(q), heads, 1.5), normal(sum(kv), kv_heads, 1.5), normal(sum(kv), kv_heads, 1.0)


def expect(torch, q, k, v, ql, kl, scale, causal, window):
    """Reference and bound of all sequences' rows (k, v packed per sequence)."""
    outs, offs = [], []
    for a, b, n, m in zip(ref.starts(ql), ref.starts(kl), ql, kl):
        o, e = ref.attention(q[a:a + n].cpu(), k[b:b + m].cpu(), v[b:b + m].cpu(), scale, causal, window)
        outs.append(o)
        offs.append(e)
    return torch.cat(outs), torch.cat(offs)


# (query lengths, key lengths, heads, key heads, head dim, type, causal, window, packed)
CASES = [
    ([1], [1], 1, 1, 64, "fp16", False, 0, False),
    ([1], [300], 8, 1, 128, "fp16", True, 0, True),
    ([128], [64], 1, 1, 128, "fp16", False, 0, False),
    ([129], [65], 2, 2, 128, "bf16", False, 0, True),
    ([63, 64, 65], [63, 64, 65], 4, 2, 64, "fp16", True, 0, False),
    ([127, 1, 200], [127, 1, 200], 3, 3, 128, "bf16", True, 0, False),
    ([5, 77, 31, 1], [5, 77, 31, 1], 8, 2, 128, "fp16", True, 0, True),
    ([300], [300], 5, 1, 128, "fp16", True, 0, False),
    ([260], [260], 6, 2, 256, "fp16", True, 0, True),
    ([70, 33], [200, 33], 4, 4, 256, "bf16", True, 0, False),
    ([40, 90], [700, 90], 8, 4, 64, "bf16", True, 0, True),
    # tokens that see no key (more tokens than keys), no keys at all, no tokens
    ([150, 10, 0, 7], [20, 0, 9, 3], 4, 2, 128, "fp16", True, 0, False),
    ([9, 0, 5], [0, 0, 40], 2, 1, 64, "fp16", False, 0, True),
    # windows, wider and narrower than a tile, and of one key
    ([333], [333], 4, 2, 128, "fp16", True, 100, False),
    ([200], [500], 2, 2, 64, "bf16", True, 1, False),
    ([1, 1, 1], [500, 70, 3], 8, 2, 128, "fp16", True, 65, True),
    # few rows over many keys: split
    ([1], [5000], 4, 2, 128, "fp16", True, 0, False),
    ([2, 1], [3001, 1200], 8, 8, 64, "bf16", True, 0, True),
    ([3], [2500], 4, 1, 256, "bf16", False, 0, False),
    ([100], [4000], 2, 1, 128, "fp16", True, 0, True),
    ([40, 130], [3000, 1500], 8, 2, 128, "bf16", False, 0, False),
    ([1] * 70, [3 * i + 1 for i in range(70)], 4, 2, 128, "fp16", True, 0, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}-{c[7]}")
def test_attention(torch, b1, case):
    ql, kl, heads, kv_heads, d, t, causal, window, packed = case
    say(f"attention {case}")
    dtype = dtype_of(torch, t)
    q, k, v = make(torch, 11, ql, kl, heads, kv_heads, d, dtype)
    qs, ks = i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl))
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, causal, window)
    out = b1.attention(q, k, v, qs, ks, causal=causal, window=window, packed=packed, bad=bad)
    if packed:
        got = ref.unpack(out, sum(ql), heads * d).view(-1, heads, d)
        ref.check(got, want, off, torch.float16, "packed")
    else:
        ref.check(out, want, off, dtype, "rows")
    assert int(bad) == 0
    if len(ql) == 1:  # the same without starts
        again = b1.attention(q, k, v, causal=causal, window=window, packed=packed)
        assert torch.equal(out, again)


# Tiles: many sequences (past the 64 a wave holds at once), split and not;
# sequences of unlike lengths split by the call's work
MANY = [
    # few rows: as many whole sequences as fill the device several times, some
    # of them without tokens; whole by their equal lengths
    ([i % 5 // 2 for i in range(300)], [30 + 7 * i for i in range(300)], 16, 8, 64, "fp16", True, 0, True),
    ([1] * 80, [1200] * 80, 16, 8, 64, "bf16", True, 0, False),
    ([20 + i % 31 for i in range(70)], None, 4, 1, 64, "fp16", True, 0, False),
    ([17 + i % 40 for i in range(130)], None, 2, 1, 128, "bf16", False, 0, True),
    ([20 + i % 9 for i in range(66)], [700 + 7 * i for i in range(66)], 2, 1, 64, "fp16", True, 0, True),
    ([100, 9, 260], [1500, 2900, 260], 4, 2, 128, "fp16", True, 0, False),
    ([60, 500, 33], [3000, 600, 40], 8, 4, 64, "bf16", True, 300, True),
    ([129, 40], [2000, 1100], 2, 2, 256, "fp16", False, 0, False),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{len(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}-{c[7]}")
def test_many_and_unlike_sequences(torch, b1, case):
    ql, kl, heads, kv_heads, d, t, causal, window, packed = case
    say(f"many {case}")
    dtype = dtype_of(torch, t)
    kl = ql if kl is None else kl
    q, k, v = make(torch, 41, ql, kl, heads, kv_heads, d, dtype)
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, causal, window)
    out = b1.attention(q, k, v, i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl)), causal=causal, window=window,
                       packed=packed)
    if packed:
        ref.check(ref.unpack(out, sum(ql), heads * d).view(-1, heads, d), want, off, torch.float16, "packed")
    else:
        ref.check(out, want, off, dtype, "rows")


@pytest.mark.parametrize("ql,kl", [([150, 40], [20, 30]), ([6, 9], [2, 700])])
def test_window_of_any_size(torch, b1, ql, kl):
    """A window that no sequence fills is none, with tokens before the first key too."""
    say(f"window {ql} {kl}")
    q, k, v = make(torch, 43, ql, kl, 4, 2, 128, torch.float16)
    want, off = expect(torch, q, k, v, ql, kl, 128 ** -0.5, True, 0)
    for window in (2 ** 31 - 1, 2 ** 30 + 1, 1000, 2 ** 32 + 1, 2 ** 40):
        out = b1.attention(q, k, v, i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl)), causal=True, window=window)
        ref.check(out, want, off, torch.float16, f"window {window}")
    with pytest.raises(ValueError):
        b1.attention(q, k, v, i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl)), causal=True, window=-2 ** 32)


@pytest.mark.parametrize("n,heads,d", [(2100, 48, 64), (1300, 72, 128)])
def test_last_round_of_equal_tiles(torch, b1, n, heads, d):
    """More equal tiles than the device holds at once, by a part of a round:
    the last ones are split (on 256 CUs: 816 and 792 tiles of 768 places)."""
    say(f"last round {n} {heads} {d}")
    q, k, v = make(torch, 42, [n], [n], heads, heads, d, torch.float16)
    out = b1.attention(q, k, v)
    for h in (0, heads // 2, heads - 1):
        want, off = ref.attention(q[:, h:h + 1].cpu(), k[:, h:h + 1].cpu(), v[:, h:h + 1].cpu(), d ** -0.5)
        ref.check(out[:, h:h + 1], want, off, torch.float16, f"head {h}")
    whole = b1.attention(q, k, v, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    # both within the bound of the exact value and a rounding of it: 2^-9 of
    # the largest value bounds twice either with room
    assert float((out.double() - whole.double()).abs().max()) <= 2.0 ** -9 * float(v.abs().max())


@pytest.mark.parametrize("m", [0, 1, 700])
@pytest.mark.parametrize("paged", [True, False])
def test_last_round_of_equal_tiles_over_few_keys(torch, b1, m, paged):
    """The same where the cache could hold more keys than the sequence has, or has none."""
    say(f"last round {m} {paged}")
    n, heads, d, page = 12800, 8, 64, 64
    q, k, v = make(torch, 44, [n], [2048], heads, heads, d, torch.float16)
    if paged:
        kc, vc = (x.view(2048 // page, page, heads, d).transpose(1, 2) for x in (k, v))
        pages = torch.arange(2048 // page, dtype=torch.int32, device="cuda")[None]
        out = b1.attention_paged(q, kc, vc, None, i32(torch, [m]), pages, causal=False)
    else:
        out = b1.attention(q, k, v, i32(torch, [0, n]), i32(torch, [0, m]))
    if m == 0:
        assert bool((out == 0).all())
        return
    rows = torch.cat([torch.arange(0, 300), torch.arange(n - 300, n)]).cuda()
    want, off = ref.attention(q[rows].cpu(), k[:m].cpu(), v[:m].cpu(), d ** -0.5)
    ref.check(out[rows], want, off, torch.float16, "first and last rows")


PAGED = [
    # (query lengths, key lengths, heads, key heads, head dim, type, page size, order, window, packed)
    ([1], [1], 2, 1, 64, "fp16", 16, "head", 0, False),
    ([1, 1, 1, 1], [17, 1, 300, 64], 8, 2, 128, "bf16", 16, "token", 0, True),
    ([1, 1], [33, 200], 4, 4, 128, "fp16", 1, "head", 0, False),
    ([1, 1, 2], [90, 31, 7], 4, 1, 256, "fp16", 2, "token", 0, False),
    ([1, 0, 3, 1], [40, 12, 260, 9], 6, 2, 64, "bf16", 32, "head", 0, True),
    ([130, 1, 40], [500, 77, 40], 4, 2, 128, "fp16", 16, "head", 0, True),
    ([70, 150], [333, 150], 8, 1, 128, "bf16", 4, "token", 0, False),
    ([65], [190], 2, 2, 256, "fp16", 64, "token", 0, False),
    ([200], [201], 4, 4, 64, "fp16", 8, "head", 50, False),
    ([1, 1], [4000, 2500], 8, 2, 128, "fp16", 64, "head", 0, True),
    ([1, 1], [3000, 90], 8, 2, 64, "bf16", 256, "token", 700, False),
    ([60], [5000], 4, 1, 128, "fp16", 128, "head", 0, False),
    ([12], [5], 4, 2, 128, "fp16", 16, "head", 0, False),  # tokens before the first key
    # tiles over pages of fewer keys than one copy of a wave takes
    ([150], [170], 2, 2, 64, "fp16", 1, "head", 0, False),
    ([40, 90], [140, 333], 4, 2, 64, "bf16", 2, "token", 0, True),
    ([130], [261], 2, 1, 64, "fp16", 4, "head", 70, False),
    ([33, 70], [45, 301], 4, 2, 128, "fp16", 1, "token", 0, False),
    ([129], [2000], 2, 1, 128, "bf16", 2, "head", 0, True),
    ([40, 5], [170, 77], 4, 1, 256, "fp16", 1, "head", 0, False),
    # many sequences as tiles
    ([20 + i % 9 for i in range(70)], [30 + 5 * i for i in range(70)], 2, 1, 128, "fp16", 16, "token", 0, True),
]


@pytest.mark.parametrize("d,page", [(64, 1), (64, 16), (128, 2), (256, 1), (256, 64)])
def test_bad_page_in_tiles(torch, b1, d, page):
    """A page out of range in a sequence of tiles: NaN from the first token that sees it on."""
    say(f"bad page {d} {page}")
    heads, kv_heads, ql, kl = 4, 2, [100, 90], [100, 200]
    q, k, v = make(torch, 45, ql, kl, heads, kv_heads, d, torch.float16)
    kc, vc, table = paged(torch, 6, k, v, kl, page, "head")
    table[1, 3] = 1 << 20
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = b1.attention_paged(q, kc, vc, i32(torch, ref.starts(ql)), i32(torch, kl), table, bad=bad)
    assert int(bad) > 0
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, True, 0)
    ref.check(out[:100], want[:100], off[:100], torch.float16, "the other sequence")
    if 4 * page <= 110:  # every token sees places 0 .. 110
        assert bool(out[100:].isnan().all())
    else:  # page 3 of 64 keys: places 192 on, the last 8 tokens'
        assert bool(out[182:].isnan().all())


def paged(torch, seed, k, v, kl, page, order, spare=2):
    """Caches of shuffled pages holding k and v; every place that no key has is NaN."""
    kv_heads, d = k.shape[1:]
    need = [-(-n // page) for n in kl]
    total = sum(need) + spare
    shape = (total, kv_heads, page, d) if order == "head" else (total, page, kv_heads, d)
    kc, vc = (torch.full(shape, math.nan, dtype=k.dtype, device="cuda") for _ in range(2))
    if order == "token":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    g = torch.Generator()
    g.manual_seed(seed)
    order_of = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(kl), max(need + [1]) + 1), -1, dtype=torch.int32)
    at, row = 0, 0
    for b, n in enumerate(kl):
        for j in range(need[b]):
            page_id = order_of[at]
            at += 1
            table[b, j] = page_id
            m = min(page, n - j * page)
            kc[page_id, :, :m] = k[row:row + m].transpose(0, 1)
            vc[page_id, :, :m] = v[row:row + m].transpose(0, 1)
            row += m
    return kc, vc, table.cuda()


@pytest.mark.parametrize("case", PAGED, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}{c[7]}")
def test_attention_paged(torch, b1, case):
    ql, kl, heads, kv_heads, d, t, page, order, window, packed = case
    say(f"paged {case}")
    dtype = dtype_of(torch, t)
    q, k, v = make(torch, 12, ql, kl, heads, kv_heads, d, dtype)
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, True, window)
    kc, vc, table = paged(torch, 3, k, v, kl, page, order)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = b1.attention_paged(q, kc, vc, i32(torch, ref.starts(ql)), i32(torch, kl), table, window=window,
                             packed=packed, bad=bad)
    if packed:
        ref.check(ref.unpack(out, sum(ql), heads * d).view(-1, heads, d), want, off, torch.float16, "packed")
    else:
        ref.check(out, want, off, dtype, "rows")
    assert int(bad) == 0


@pytest.mark.parametrize("ql,kl,heads,kv_heads,d", [([200], [200], 4, 2, 128), ([140], [333], 2, 2, 64),
                                                    ([3, 1], [90, 40], 8, 2, 128), ([70], [70], 1, 1, 256)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_masked_keys_may_hold_anything(torch, b1, ql, kl, heads, kv_heads, d, value):
    """NaN and infinities in keys and values that a row does not see leave it
    alone; rows that see a NaN value are NaN in that column."""
    say(f"masked {value} {ql} {kl} {heads} {d}")
    q, k, v = make(torch, 13, ql, kl, heads, kv_heads, d, torch.float16)
    # the last key of each sequence: seen by its last token alone
    for end in ref.starts(kl)[1:]:
        k[end - 1, :, 5] = value
        v[end - 1, :, 3] = value
    qs, ks = i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl))
    out = b1.attention(q, k, v, qs, ks, causal=True).cpu()
    row = 0
    for n, m, b in zip(ql, kl, ref.starts(kl)):
        want, off = ref.attention(q[row:row + n - 1].cpu(), k[b:b + m - 1].cpu(), v[b:b + m - 1].cpu(), d ** -0.5,
                                  True)
        ref.check(out[row:row + n - 1], want, off, torch.float16, "rows that do not see it")
        row += n
    # a NaN among the seen values
    k[:, :, 5] = 0.25
    v[:, :, 3] = 0.5
    last = ref.starts(kl)[1] - 1
    v[last, :, 3] = value
    out = b1.attention(q, k, v, qs, ks, causal=True).cpu()
    assert not bool(out[ql[0] - 1, :, 3].isfinite().any())
    assert bool(out[ql[0] - 1, :, 4:].isfinite().all())


def test_overflowing_partial_sums(torch, b1):
    """bf16 values near the type's largest: the weighted mean is finite."""
    ql, heads, d = [3, 100], 2, 128
    q, k, v = make(torch, 14, ql, ql, heads, heads, d, torch.bfloat16)
    v = (v.float().sign() * 2.5e38).to(torch.bfloat16)
    qs = i32(torch, ref.starts(ql))
    want, off = expect(torch, q, k, v, ql, ql, d ** -0.5, True, 0)
    out = b1.attention(q, k, v, qs, causal=True)
    assert bool(out.isfinite().all())
    ref.check(out, want, off, torch.bfloat16, "rows")


@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_flat_and_sharp_scores(torch, b1, spread):
    """Scores all equal, and scores so far apart that one key takes all."""
    ql = [1, 90, 257]
    q, k, v = make(torch, 15, ql, ql, 4, 2, 128, torch.float16)
    q = q * spread
    qs = i32(torch, ref.starts(ql))
    want, off = expect(torch, q, k, v, ql, ql, 128 ** -0.5, True, 0)
    ref.check(b1.attention(q, k, v, qs, causal=True), want, off, torch.float16, "rows")


def test_scale(torch, b1):
    ql = [130, 2]
    q, k, v = make(torch, 16, ql, ql, 2, 2, 64, torch.float16)
    qs = i32(torch, ref.starts(ql))
    for scale in (1.0, 0.01, 7.5):
        want, off = expect(torch, q, k, v, ql, ql, scale, True, 0)
        ref.check(b1.attention(q, k, v, qs, causal=True, scale=scale), want, off, torch.float16, "rows")


@pytest.mark.parametrize("ql,kl", [([40, 3], [40, 30]), ([1, 2], [90, 31]), ([1, 1], [3000, 1200])])
def test_strides_and_rows_of_no_sequence(torch, b1, ql, kl):
    """q, k, v as slices of wider tensors, out and packed as column ranges,
    rows before the first sequence and behind the last left as they were."""
    say(f"strides {ql} {kl}")
    heads, kv_heads, d, before, behind = 4, 2, 128, 2, 3
    n = sum(ql) + before + behind
    g = torch.Generator(device="cuda")
    g.manual_seed(17)
    wide_q = torch.randn((n, heads + 3, d + 8), generator=g, device="cuda").half()
    wide_kv = torch.randn((sum(kl), 2, kv_heads + 1, d), generator=g, device="cuda").half()
    q = wide_q[:, 1:heads + 1, :d]
    k, v = wide_kv[:, 0, :kv_heads], wide_kv[:, 1, 1:]
    qs = i32(torch, [before + x for x in ref.starts(ql)])
    ks = i32(torch, ref.starts(kl))
    want, off = expect(torch, q[before:], k, v, ql, kl, d ** -0.5, True, 0)
    wide = torch.full((n, heads * d + 64), 7.0, dtype=torch.float16, device="cuda")
    out = wide[:, 32:32 + heads * d].view(n, heads, d)
    b1.attention(q, k, v, qs, ks, causal=True, out=out)
    ref.check(out[before:before + sum(ql)], want, off, torch.float16, "rows")
    assert bool((wide[:before] == 7).all()) and bool((wide[before + sum(ql):] == 7).all())
    assert bool((wide[:, :32] == 7).all()) and bool((wide[:, 32 + heads * d:] == 7).all())
    ldp = heads * d + 96
    buf = torch.full((n * ldp * 2,), 0x3A, dtype=torch.uint8, device="cuda")
    b1.attention(q, k, v, qs, ks, causal=True, packed=buf[64 * 2:(64 + (n - 1) * ldp + heads * d) * 2], ldp=ldp)
    got = ref.unpack(buf, n, heads * d, ldp, 64).view(n, heads, d)
    ref.check(got[before:before + sum(ql)], want, off, torch.float16, "packed")
    rows = buf.view(n, ldp * 2)
    assert bool((rows[:before] == 0x3A).all()) and bool((rows[before + sum(ql):] == 0x3A).all())
    assert bool((rows[:, :128] == 0x3A).all()) and bool((rows[:, (64 + heads * d) * 2:] == 0x3A).all())


@pytest.mark.parametrize("ql,kl", [([1, 1], [5000, 900]), ([60], [4000])])
def test_with_and_without_a_workspace(torch, b1, ql, kl):
    """The caller's workspace gives the library's bits; one too small runs the
    keys unsplit, within the same bounds."""
    heads, kv_heads, d = 8, 2, 128
    q, k, v = make(torch, 18, ql, kl, heads, kv_heads, d, torch.float16)
    qs, ks = i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl))
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, True, 0)
    own = b1.attention(q, k, v, qs, ks, causal=True)
    big = b1.attention(q, k, v, qs, ks, causal=True, workspace=torch.empty(256 << 20, dtype=torch.uint8,
                                                                           device="cuda"))
    none = b1.attention(q, k, v, qs, ks, causal=True, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert torch.equal(own, big)
    ref.check(own, want, off, torch.float16, "split")
    ref.check(none, want, off, torch.float16, "unsplit")


def test_offsets_past_32_bits(torch, b1):
    """A cache of more than 2^32 bytes, keys on its last pages; and a sequence
    of contiguous keys that begins past 2^31 elements."""
    heads, kv_heads, d, page, n = 4, 2, 128, 64, 300
    pages = (1 << 32) // (kv_heads * page * d * 2) + 40
    kc, vc = (torch.zeros((pages, kv_heads, page, d), dtype=torch.float16, device="cuda") for _ in range(2))
    q, k, v = make(torch, 19, [1, 70], [n, n], heads, kv_heads, d, torch.float16)
    table = torch.tensor([[pages - 1 - i for i in range(5)], [pages - 10 - 3 * i for i in range(5)]],
                         dtype=torch.int32)
    for b in range(2):
        for j in range(5):
            m = min(page, n - j * page)
            at = b * n + j * page
            kc[table[b, j], :, :m] = k[at:at + m].transpose(0, 1)
            vc[table[b, j], :, :m] = v[at:at + m].transpose(0, 1)
    want, off = expect(torch, q, k, v, [1, 70], [n, n], d ** -0.5, True, 0)
    for ql, part in (([1, 70], slice(0, 71)), ([1, 0], slice(0, 1))):
        out = b1.attention_paged(q[:sum(ql)].contiguous(), kc, vc, i32(torch, ref.starts(ql)), i32(torch, [n, n]),
                                 table.cuda())
        ref.check(out, want[part], off[part], torch.float16, f"paged {ql}")
    rows = kc.view(-1, kv_heads, d), vc.view(-1, kv_heads, d)
    first = rows[0].shape[0] - 2 * n
    assert first * kv_heads * d > 1 << 31
    for full, part in zip(rows, (k, v)):
        full[first:] = part
    out = b1.attention(q, rows[0], rows[1], i32(torch, [0, 1, 71]), i32(torch, [first, first + n, first + 2 * n]),
                       causal=True)
    ref.check(out, want, off, torch.float16, "contiguous")


def test_other_streams_and_two_at_once(torch, b1):
    """Calls on two streams, each with its own workspace, while the default
    stream works."""
    heads, kv_heads, d = 8, 2, 128
    ql, kl = [1, 1], [4000, 2100]
    sets = [make(torch, 20 + i, ql, kl, heads, kv_heads, d, torch.float16) for i in range(2)]
    qs, ks = i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl))
    want = [b1.attention(*s, qs, ks, causal=True) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = [b1.attention(*s, qs, ks, causal=True, stream=st) for s, st in zip(sets, streams)]
        torch.randn(1000, device="cuda").sum()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_captured_and_replayed(torch, b1):
    """Two graphs of split calls on one stream, replayed in turn with eager
    calls between: every replay gives the eager bits."""
    heads, kv_heads, d = 8, 2, 128
    shapes = [([1, 1], [4000, 2100]), ([40], [3000])]
    stream = torch.cuda.Stream()
    calls = []
    with torch.cuda.stream(stream):
        for i, (ql, kl) in enumerate(shapes):
            q, k, v = make(torch, 30 + i, ql, kl, heads, kv_heads, d, torch.float16)
            qs, ks = i32(torch, ref.starts(ql)), i32(torch, ref.starts(kl))
            out = torch.zeros_like(q)
            calls.append((q, k, v, qs, ks, out))

        def run(c):
            b1.attention(*c[:5], causal=True, out=c[5])

        want = []
        for c in calls:
            run(c)
            want.append(c[5].clone())
        stream.synchronize()
        graphs = []
        for c in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                run(c)
            graphs.append(g)
        for turn in range(4):
            for c, g, w in zip(calls, graphs, want):
                c[5].zero_()
                g.replay()
                stream.synchronize()
                assert torch.equal(c[5], w), f"replay {turn}"
            for c in calls:
                run(c)
            stream.synchronize()
    del graphs


def test_no_tokens_no_sequences(torch, b1):
    q = torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda")
    k = torch.zeros((5, 2, 64), dtype=torch.float16, device="cuda")
    assert b1.attention(q, k, k).shape == (0, 4, 64)
    q = torch.ones((3, 4, 64), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 3.0)
    b1.attention(q, q[:, :2], q[:, :2], i32(torch, [0]), out=out)  # rows of no sequence
    assert bool((out == 3).all())
    out = b1.attention(q, k[:0], k[:0])
    assert bool((out == 0).all())


def test_bits_do_not_depend_on_other_sequences_order(torch, b1):
    """Unsplit, a sequence's rows have the bits it has alone."""
    ql = [200, 33, 129]
    q, k, v = make(torch, 23, ql, ql, 4, 2, 128, torch.float16)
    ws = torch.empty(16, dtype=torch.uint8, device="cuda")
    whole = b1.attention(q, k, v, i32(torch, ref.starts(ql)), causal=True, workspace=ws)
    for a, n in zip(ref.starts(ql), ql):
        s = slice(a, a + n)
        assert torch.equal(whole[s], b1.attention(q[s], k[s], v[s], causal=True, workspace=ws))


BAD = [
    # (starts, key lengths, table entries to change, rows NaN, rows right)
    ("page below 0", {"table": (0, 1, -7)}),
    ("page past the last", {"table": (0, 0, 1 << 30)}),
    ("length below 0", {"kv": (0, -3)}),
    ("length past the table", {"kv": (0, 1 << 29)}),
]


@pytest.mark.parametrize("what,change", BAD, ids=[b[0] for b in BAD])
@pytest.mark.parametrize("ql", [[1, 1], [90, 20]])
def test_bad_pages_and_lengths(torch, b1, what, change, ql):
    """Rows that depend on an index out of range are NaN and counted; the
    other sequence is right."""
    say(f"bad index: {what} {ql}")
    heads, kv_heads, d, page, kl = 4, 2, 128, 16, [100, 64]
    q, k, v = make(torch, 24, ql, kl, heads, kv_heads, d, torch.float16)
    kc, vc, table = paged(torch, 5, k, v, kl, page, "head")
    lens = i32(torch, kl)
    if "table" in change:
        b, j, p = change["table"]
        table[b, j] = p
    else:
        lens[change["kv"][0]] = change["kv"][1]
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = b1.attention_paged(q, kc, vc, i32(torch, ref.starts(ql)), lens, table, bad=bad)
    assert int(bad) > 0
    assert bool(out[:ql[0]].isnan().all())
    want, off = expect(torch, q, k, v, ql, kl, d ** -0.5, True, 0)
    ref.check(out[ql[0]:], want[ql[0]:], off[ql[0]:], torch.float16, "the other sequence")


@pytest.mark.parametrize("kind", ["past the end", "below 0", "descending", "huge"])
@pytest.mark.parametrize("tokens", [4, 40])
def test_bad_starts(torch, b1, kind, tokens):
    """Starts out of range or out of order: counted, and nothing outside the
    tensors is touched."""
    heads, kv_heads, d = 4, 1, 64
    starts = {"past the end": [0, 300, tokens], "below 0": [-5, tokens // 2, tokens],
              "descending": [tokens - 1, 1, tokens], "huge": [0, tokens // 2, 1 << 30]}[kind]
    q, k, v = make(torch, 25, [tokens], [40], heads, kv_heads, d, torch.float16)
    buf = torch.full((tokens + 20, heads, d), 5.0, dtype=torch.float16, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    b1.attention(q, k, v, i32(torch, starts), i32(torch, [0, 20, 40]), causal=True, out=buf[10:10 + tokens], bad=bad)
    assert int(bad) > 0
    assert bool((buf[:10] == 5).all()) and bool((buf[10 + tokens:] == 5).all())
