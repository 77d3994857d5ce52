"""GPU checks of the operators around a block's linears: rms_norm, qkv_rope
(rows and paged cache), and a block's chain of them with the linears and
attention, against float64."""
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


def normal(torch, seed, *shape, spread=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * spread


def i32(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def norm_ref(torch, h, w, eps):
    """RMS norm in float64 and its bound: the sum of squares is off by at most
    96 half steps of fp32 relative (at most 64 terms a thread, an 8-step tree
    and the squares; wider rows as many more terms), the root halves that;
    root, division and two products add 4."""
    h = h.double().cpu()
    y = h / (h.square().mean(1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double().cpu()
    terms = max(96, h.shape[1] / 256 + 32)
    return y, y.abs() * (terms / 2 + 4) * ref.U32


@pytest.mark.parametrize("rows,h", [(1, 32), (5, 96), (3, 2048), (2, 2080), (7, 2560), (4, 4096), (3, 4128),
                                    (300, 1024), (2, 16384), (3, 16416), (2, 20000), (9, 512), (5, 544), (3, 8192), (2, 8224),
                                    (2, 32768), (3, 32800), (2, 70016)])
@pytest.mark.parametrize("with_add", [True, False])
def test_rms_norm(torch, b1, rows, h, with_add):
    say(f"rms_norm {rows} {h} {with_add}")
    x, add = normal(torch, 1, rows, h, spread=3.0), normal(torch, 2, rows, h)
    w = 1.0 + normal(torch, 3, h, spread=0.2)
    eps = 1e-5
    total = x + add if with_add else x  # one fp32 addition a value
    want, off = norm_ref(torch, total, w, eps)
    if with_add:
        res, y = b1.rms_norm(x, w, eps, add=add)
        assert torch.equal(res, total)
        _, p = b1.rms_norm(x, w, eps, add=add, packed=True)
    else:
        y, p = b1.rms_norm(x, w, eps), b1.rms_norm(x, w, eps, packed=True)
    ref.check(y, want, off, torch.float32, "fp32")
    ref.check(ref.unpack(p, rows, h), want, off, torch.float16, "packed")
    # the packing is the one of the fp32 rows
    assert torch.equal(p[:rows * h * 2], b1.pack_act_f16(y)[:rows * h * 2])
    bare = b1.rms_norm(total, None, eps)
    want, off = norm_ref(torch, total, None, eps)
    ref.check(bare, want, off, torch.float32, "no weight")


@pytest.mark.parametrize("h", [64, 2560, 20000, 40000])
@pytest.mark.parametrize("into", ["x", "add"])
def test_rms_norm_in_place_and_strided(torch, b1, h, into):
    rows = 37
    wide = normal(torch, 4, 3, rows, h + 32)
    x, add = wide[0][:, :h], wide[1][:, 16:16 + h]
    w = 1.0 + normal(torch, 5, h, spread=0.2)
    total = x + add
    want, off = norm_ref(torch, total, w, 1e-6)
    out = wide[2][:, 4:4 + h]
    edge = wide[2].clone()
    res, y = b1.rms_norm(x, w, add=add, residual=x if into == "x" else add, out=out)
    assert y is out and torch.equal(res, total)
    ref.check(y, want, off, torch.float32, "strided")
    assert torch.equal(wide[2][:, :4], edge[:, :4]) and torch.equal(wide[2][:, 4 + h:], edge[:, 4 + h:])


def test_rms_norm_of_zeros_and_odd_values(torch, b1):
    x = normal(torch, 6, 4, 256)
    x[0] = 0.0
    x[1, 7] = math.nan
    x[2, 9] = math.inf
    y = b1.rms_norm(x, None, 1e-6).cpu()
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all())
    assert bool((y[2, :9] == 0).all()) and bool(y[2, 9].isnan())
    want, off = norm_ref(torch, x[3:], None, 1e-6)
    ref.check(y[3:], want, off, torch.float32, "the row beside them")
    assert b1.rms_norm(x[:0]).shape == (0, 256)


def test_rms_norm_of_more_rows_than_a_launch(torch, b1):
    rows, h = (1 << 26) + 5, 32
    x = torch.empty((rows, h), dtype=torch.float32, device="cuda")
    some = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, (1 << 24) + 1, rows - 2, rows - 1], device="cuda")
    x.fill_(1.0)
    x[some] = normal(torch, 9, len(some), h)
    packed = b1.rms_norm(x, None, 1e-6, packed=True)
    want, off = norm_ref(torch, x[some], None, 1e-6)
    got = packed.view(torch.float16).view(rows, h)[some].contiguous().view(torch.uint8).flatten()
    ref.check(ref.unpack(got, len(some), h), want, off, torch.float16, "rows")


def table(torch, rows, dim):
    angle = torch.arange(rows).double()[:, None] * 100.0 ** (-torch.arange(dim // 2).double() / max(1, dim // 2))
    return torch.cat([angle.cos(), angle.sin()], 1).float().cuda().contiguous()


def head_ref(torch, x, w, rope, interleaved, eps):
    """x [tokens, heads, d] fp32 -> float64 and bound: the norm's (d squares
    over d / 4 lanes) and the rotation's few fp32 roundings, on the larger of
    the pair's terms."""
    x = x.double().cpu()
    d = x.shape[-1]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
    mags = x.abs()
    if rope is not None:
        r = rope.double().cpu()
        dim = r.shape[1]
        c, s = r[:, None, :dim // 2], r[:, None, dim // 2:]
        rot = x[..., :dim]
        a, b = (rot[..., ::2], rot[..., 1::2]) if interleaved else (rot[..., :dim // 2], rot[..., dim // 2:])
        ra, rb = a * c - b * s, b * c + a * s
        ma, mb = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()

        def join(p, q):
            return torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)

        x = torch.cat([join(ra, rb), x[..., dim:]], -1)
        mags = torch.cat([join(ma, mb), mags[..., dim:]], -1)
    return x, mags * 16 * ref.U32 + 0 * d


@pytest.mark.parametrize("tokens,heads,kv_heads,d", [(1, 1, 1, 64), (5, 8, 2, 128), (3, 5, 5, 256), (70, 3, 1, 64),
                                                     (33, 24, 24, 128), (1100, 6, 2, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t", ["fp16", "bf16"])
def test_qkv_rope(torch, b1, tokens, heads, kv_heads, d, interleaved, t):
    say(f"qkv_rope {tokens} {heads} {kv_heads} {d} {interleaved} {t}")
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[t]
    x = normal(torch, 7, tokens, (heads + 2 * kv_heads) * d + 8)
    q, k, v = x[:, :heads * d], x[:, heads * d:(heads + kv_heads) * d], x[:, (heads + kv_heads) * d:-8]
    qw, kw = 1.0 + normal(torch, 8, d, spread=0.3), 1.0 + normal(torch, 9, d, spread=0.3)
    pos = torch.randperm(tokens + 9, generator=torch.Generator().manual_seed(1))[:tokens]
    for dim, weights, at in ((d, True, pos), (d // 2, False, None), (None, True, None), (8, True, pos)):
        rope = table(torch, tokens + 9, dim) if dim else None
        used = None if rope is None else rope[at.cuda()] if at is not None else rope[:tokens]
        got = b1.qkv_rope(q, k, v, d, q_weight=qw if weights else None, k_weight=kw if weights else None, eps=1e-6,
                          rope=rope, positions=at.int().cuda() if at is not None else None, interleaved=interleaved,
                          dtype=dtype)
        for name, g, src, w, r, n in (("q", got[0], q, qw, used, heads), ("k", got[1], k, kw, used, kv_heads),
                                      ("v", got[2], v, None, None, kv_heads)):
            want, off = head_ref(torch, src.reshape(tokens, n, d), w if weights else None, r, interleaved, 1e-6)
            ref.check(g, want, off, dtype, f"{name}, rope_dim {dim}")


@pytest.mark.parametrize("page,order", [(1, "head"), (16, "token"), (64, "head")])
def test_qkv_rope_paged(torch, b1, page, order):
    """Keys and values at their places, everything else in the cache and rows
    of no sequence as they were."""
    ql, kl, heads, kv_heads, d = [1, 20, 0, 3], [50, 20, 7, 90], 4, 2, 128
    n = sum(ql)
    x = normal(torch, 10, n + 2, (heads + 2 * kv_heads) * d)
    q, k, v = x.split([heads * d, kv_heads * d, kv_heads * d], 1)
    kw = 1.0 + normal(torch, 11, d, spread=0.3)
    rope = table(torch, 100, d)
    need = [-(-m // page) for m in kl]
    total = sum(need) + 2
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(2)).tolist()
    pages = torch.full((4, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        pages[b, :m] = torch.tensor(ids[at:at + m])
        at += m
    shape = (total, kv_heads, page, d) if order == "head" else (total, page, kv_heads, d)
    kc, vc = (torch.full(shape, 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    if order == "token":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    qo = torch.full((n + 2, heads, d), 9.0, dtype=torch.float16, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = b1.qkv_rope_paged(q, k, v, kc, vc, i32(torch, ref.starts(ql)), i32(torch, kl), pages.cuda(), k_weight=kw,
                            rope=rope, q_out=qo, bad=bad)
    assert got is qo and int(bad) == 0
    pos = torch.tensor([m - c + i for c, m in zip(ql, kl) for i in range(c)])
    seq = [b for b, c in enumerate(ql) for _ in range(c)]
    used = rope[pos.cuda()]
    want, off = head_ref(torch, q[:n].reshape(n, heads, d), None, used, False, 1e-6)
    ref.check(qo[:n], want, off, torch.float16, "q")
    assert bool((qo[n:] == 9).all())
    untouched = torch.ones(total, page, dtype=torch.bool)
    for name, cache, src, w, r in (("k", kc, k, kw, used), ("v", vc, v, None, None)):
        want, off = head_ref(torch, src[:n].reshape(n, kv_heads, d), w, r, False, 1e-6)
        for i in range(n):
            p, slot = int(pages[seq[i], pos[i] // page]), int(pos[i]) % page
            untouched[p, slot] = False
            ref.check(cache[p, :, slot], want[i], off[i], torch.float16, f"{name} of token {i}")
    for cache in (kc, vc):
        assert bool((cache.transpose(1, 2)[untouched.cuda()] == 9).all())


def test_qkv_rope_bad_indexes(torch, b1):
    """Positions outside the table, pages outside the cache, more tokens than
    places: NaN queries, nothing stored, counted."""
    heads, d, page = 2, 64, 16
    x = normal(torch, 12, 6, 3 * heads * d)
    q, k, v = x.split([heads * d] * 3, 1)
    rope = table(torch, 8, d)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo, ko, vo = b1.qkv_rope(q, k, v, d, rope=rope, positions=i32(torch, [0, -1, 8, 1 << 30, 7, 3]), bad=bad)
    assert int(bad) == 3
    for t in (qo, ko, vo):
        assert bool(t[1:4].isnan().all()) and bool(t[[0, 4, 5]].isfinite().all())
    for pages, kl in (([[0, 5]], [20]), ([[0, -1]], [20]), ([[0, 1]], [4]), ([[0, 1]], [1000]), ([[0, 1]], [-1])):
        kc, vc = (torch.full((2, heads, page, d), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
        bad.zero_()
        qo = b1.qkv_rope_paged(q, k, v, kc, vc, i32(torch, [0, 6]), i32(torch, kl), i32(torch, pages), bad=bad)
        assert int(bad) > 0 and bool(qo.isnan().any())
        wrong = qo.isnan().all(2).all(1)
        assert int((kc != 9).any(3).any(1).sum()) == int((~wrong).sum())


def test_qkv_rope_starts_that_do_not_ascend(torch, b1):
    """Tokens that such starts put behind their sequence's end are stored
    nowhere: places past a table's row are not looked up."""
    heads, d, page, n = 2, 64, 16, 24
    x = normal(torch, 13, n, 3 * heads * d)
    q, k, v = x.split([heads * d] * 3, 1)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    for at, kl in (([0, 20, 5, 6], [20, 5, 16]), ([0, 24, 2, 3, 3], [24, 7, 1, 32]), ([7, 2, 1, 24], [3, 3, 30])):
        kc, vc = (torch.full((9, heads, page, d), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
        pages = torch.arange(2 * len(kl), dtype=torch.int32, device="cuda").view(len(kl), 2)
        bad.zero_()
        qo = b1.qkv_rope_paged(q, k, v, kc, vc, i32(torch, at), i32(torch, kl), pages, bad=bad)
        assert int(bad) > 0
        if at[1] == 20:  # tokens 6 .. 19: of sequence 2 by the ends, behind its one row
            assert bool(qo[6:20].isnan().all()) and bool((kc[2:] == 9).all()) and bool((vc[2:] == 9).all())
        assert bool((kc[8] == 9).all()) and bool((vc[8] == 9).all())


def test_block_chain_whole_and_in_chunks(torch, b1):
    """A decoder block's attention half over prompts at once (contiguous keys)
    and in chunks and single tokens through a paged cache, both against
    float64 on the rounded operands of each step: the norm's packing, the
    1-bit q/k/v linear, qkv_rope, attention into the packed input of the
    output linear, and that linear added to the residual."""
    from bonsai_b1 import synth
    lens, hidden, heads, kv_heads, d, page = [70, 133], 768, 6, 2, 128, 16
    total, width = sum(lens), (heads + 2 * kv_heads) * d
    x = normal(torch, 20, total, hidden)
    w_norm = 1.0 + normal(torch, 21, hidden, spread=0.2)
    wqkv, wo = synth.device_packed_weights(width, hidden, 22), synth.device_packed_weights(hidden, heads * d, 23)
    qw, kw = 1.0 + normal(torch, 24, d, spread=0.2), 1.0 + normal(torch, 25, d, spread=0.2)
    rope = table(torch, 256, d)
    split = [heads * d, kv_heads * d, kv_heads * d]

    def front(rows):
        n = rows.shape[0]
        packed = b1.rms_norm(rows, w_norm, packed=True)
        return b1.linear_packed_f16(packed, wqkv, hidden, width, n).split(split, 1)

    def back(packed, rows):
        return rows + b1.linear_packed_f16(packed, wo, heads * d, hidden, rows.shape[0])

    # whole prompts
    at = ref.starts(lens)
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    q, k, v = front(x)
    q16, k16, v16 = b1.qkv_rope(q, k, v, d, qw, kw, rope=rope, positions=pos)
    starts = i32(torch, at)
    whole = b1.attention(q16, k16, v16, starts, causal=True, packed=True)
    y = back(whole, x)
    outs, offs = [], []
    for a, n in zip(at, lens):
        s = slice(a, a + n)
        o, e = ref.attention(q16[s].cpu(), k16[s].cpu(), v16[s].cpu(), d ** -0.5, True)
        outs.append(o)
        offs.append(e)
    want, off = torch.cat(outs), torch.cat(offs)
    ref.check(ref.unpack(whole, total, heads * d).view(-1, heads, d), want, off, torch.float16, "whole prompts")

    # the same prompts in chunks: 50 and 100 tokens, then the rest but three
    # single tokens, then those
    pages = torch.arange(2 * 9, dtype=torch.int32).view(2, 9).flip(0).contiguous().cuda()
    kc, vc = (torch.full((18, kv_heads, page, d), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    done, got = [0, 0], torch.zeros(total, hidden, device="cuda")
    plan = [[50, 100], [17, 30]] + [[1, 1]] * 3
    for step in plan:
        rows = torch.cat([torch.arange(at[b] + done[b], at[b] + done[b] + c) for b, c in enumerate(step)]).cuda()
        xs = x[rows].contiguous()
        done = [a + c for a, c in zip(done, step)]
        st, kl = i32(torch, ref.starts(step)), i32(torch, done)
        q, k, v = front(xs)
        q16 = b1.qkv_rope_paged(q, k, v, kc, vc, st, kl, pages, qw, kw, rope=rope)
        packed = b1.attention_paged(q16, kc, vc, st, kl, pages, packed=True)
        got[rows] = back(packed, xs)
    assert done == lens
    # the linears of few rows sum in another order than those of many, so an
    # operand may round to its fp16 neighbour: a value then moves by one fp16
    # step, and y, a sum of heads * d such operands times +-0.05 at most, by
    # far less than 2 % of its own size in the 2-norm
    err = float((got - y).double().norm() / (y - x).double().norm())
    say(f"chunks against whole prompts: {err:.2e}")
    assert err < 0.02


def test_captured_decode_step(torch, b1):
    """One step of several sequences over a paged cache captured once and
    replayed while the lengths in device memory grow, with eager work between
    the replays; the sequences share the pages of a common prefix."""
    from bonsai_b1 import synth
    hidden, heads, kv_heads, d, page, n = 768, 12, 3, 64, 16, 3  # the linears read multiples of 384
    width = (heads + 2 * kv_heads) * d
    x = normal(torch, 30, n, hidden)
    w_norm = 1.0 + normal(torch, 31, hidden, spread=0.2)
    wqkv, wo = synth.device_packed_weights(width, hidden, 32), synth.device_packed_weights(hidden, heads * d, 33)
    rope = table(torch, 2048, d)
    split = [heads * d, kv_heads * d, kv_heads * d]
    prefix, most = 60, 80  # pages; 960 shared keys
    pages = torch.empty(n, most, dtype=torch.int32)
    pages[:, :prefix] = torch.arange(prefix)
    for b in range(n):
        pages[b, prefix:] = prefix + b * (most - prefix) + torch.arange(most - prefix).flip(0)
    pages = pages.cuda()
    total = prefix + n * (most - prefix)
    kc, vc = (normal(torch, s, total, kv_heads, page, d).half() for s in (34, 35))
    start, first = i32(torch, [0, 1, 2, 3]), [960, 975, 1100]
    lens = i32(torch, [m + 1 for m in first])

    def step(k_cache, v_cache, ws):
        h, packed = b1.rms_norm(x, w_norm, add=x, packed=True)
        q, k, v = b1.linear_packed_f16(packed, wqkv, hidden, width, n).split(split, 1)
        q16 = b1.qkv_rope_paged(q, k, v, k_cache, v_cache, start, lens, pages, rope=rope)
        out = b1.attention_paged(q16, k_cache, v_cache, start, lens, pages, packed=True, workspace=ws)
        return h, b1.linear_packed_f16(out, wo, heads * d, hidden, n)

    ws, ws2 = (torch.empty(64 << 20, dtype=torch.uint8, device="cuda") for _ in range(2))
    kg, vg, ke, ve = kc.clone(), vc.clone(), kc.clone(), vc.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(kc, vc, ws)  # what the library allocates once
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            h, y = step(kg, vg, ws)
        for turn in range(5):
            graph.replay()
            stream.synchronize()
            he, ye = step(ke, ve, ws2)
            stream.synchronize()
            assert bool(ye.isfinite().all()), f"step {turn}"
            assert torch.equal(h, he) and torch.equal(y, ye), f"step {turn}"
            assert torch.equal(kg, ke) and torch.equal(vg, ve), f"step {turn}"
            lens += 1
            x.mul_(0.75)
        stream.synchronize()
    # the shared pages are as they were, the steps' places are not
    assert torch.equal(kg[:prefix], kc[:prefix]) and not torch.equal(kg[prefix:], kc[prefix:])
    del graph


def test_rms_norm_of_more_wide_rows_than_a_launch(torch, b1):
    """Rows of 1024 threads: 2^22 of them would be 2^32 threads at once."""
    rows, h = (1 << 22) + 3, 4128
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    if free < rows * h * 6 + (4 << 30):
        pytest.skip("needs 108 GB of free device memory")
    x = torch.empty((rows, h), dtype=torch.float32, device="cuda")
    some = torch.tensor([0, 1, (1 << 21) - 1, 1 << 21, (1 << 21) + 1, rows - 4, rows - 1], device="cuda")
    x.fill_(1.0)
    x[some] = normal(torch, 40, len(some), h)
    packed = b1.rms_norm(x, None, 1e-6, packed=True)
    want, off = norm_ref(torch, x[some], None, 1e-6)
    del x
    got = packed.view(torch.float16).view(rows, h)[some].contiguous().view(torch.uint8).flatten()
    ref.check(ref.unpack(got, len(some), h), want, off, torch.float16, "rows")
    del packed, got
    torch.cuda.empty_cache()
