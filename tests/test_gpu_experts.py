"""GPU checks of the mixture-of-experts operators (route, linear_experts,
combine_experts), alone and as a block's MLP, against float64."""
import math
import sys

import pytest

from tests import attention_ref as ref
from tests import experts_ref as moe

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


# ---- the router ------------------------------------------------------------


def check_routes(torch, r, logits, top_k, **how):
    expert, weight, off = moe.route(logits, top_k, **how)
    experts = logits.shape[1]
    assert torch.equal(r.expert.cpu(), expert), "experts"
    ref.check(r.weight, weight, off, torch.float32, "weights")
    start, order, place = moe.layout(expert, experts)
    assert torch.equal(r.start.cpu(), start), "start"
    assert torch.equal(r.order.cpu(), order), "order"
    assert torch.equal(r.place.cpu(), place), "place"


@pytest.mark.parametrize("score,with_bias,renormalize,scale", [
    ("softmax", False, True, 1.0), ("softmax", False, False, 1.0), ("softmax", True, True, 0.5),
    ("softmax", True, False, 1.0), ("sigmoid", False, False, 1.0), ("sigmoid", True, True, 2.5)])
@pytest.mark.parametrize("tokens,experts,top_k,t", [
    (1, 1, 1, "fp32"), (1, 128, 8, "fp32"), (3, 2, 2, "bf16"), (17, 64, 6, "fp16"), (64, 65, 5, "fp32"),
    (65, 128, 8, "bf16"), (257, 20, 3, "fp16"), (700, 256, 8, "fp32"), (100, 300, 4, "fp32"),
    (90, 1000, 10, "bf16"), (70, 1024, 64, "fp32"), (5, 513, 33, "fp16")])
def test_route(torch, b1, tokens, experts, top_k, t, score, with_bias, renormalize, scale):
    say(f"route {tokens} {experts} {top_k} {t} {score} {with_bias} {renormalize}")
    dtype = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[t]
    logits = normal(torch, tokens + experts, tokens, experts, spread=2.0).to(dtype)
    bias = normal(torch, 5, experts, spread=0.2) if with_bias else None
    r = b1.route(logits, top_k, score=score, bias=bias, renormalize=renormalize, scale=scale)
    check_routes(torch, r, logits, top_k, score=score, bias=bias, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens", [16, 160])
def test_route_of_unusual_rows(torch, b1, score, with_bias, renormalize, tokens):
    """Ties, experts that are off, rows that are all off, the type's lowest
    value, infinities and NaN; a strided table of logits."""
    say(f"route unusual {score} {with_bias} {renormalize} {tokens}")
    experts, k = 70, 4
    wide = normal(torch, 9, tokens, experts + 9, spread=2.0)
    x = wide[:, 3:3 + experts]
    low = torch.finfo(torch.float32).min
    x[0] = 1.25                      # every expert alike
    x[1] = -math.inf                 # no expert at all
    x[2] = -math.inf
    x[2, [7, 66]] = torch.tensor([0.5, 0.75], device="cuda")  # fewer than top_k
    x[3, 5] = math.nan
    x[4] = math.nan
    x[5, 64:] = low
    x[6] = low
    x[7] = low
    x[7, 69] = 3.0
    x[8] = torch.where(torch.arange(experts, device="cuda") % 2 == 0, 0.0, -0.0)  # zeros of both signs
    x[9, 11] = math.inf
    x[10, :66] = -math.inf           # exactly top_k left
    x[11] = -100.0
    x[11, 3] = -99.0
    x[12] = 200.0                    # scores that saturate
    x[13, ::3] = -math.inf
    x[14] = x[14].round()            # many ties
    bias = None
    if with_bias:
        bias = normal(torch, 5, experts, spread=0.25).mul(4).round().div(16)  # ties among score + bias too
        bias[13] = -math.inf
    r = b1.route(x, k, score=score, bias=bias, renormalize=renormalize)
    check_routes(torch, r, x, k, score=score, bias=bias, renormalize=renormalize)
    if with_bias:
        bias[2] = math.nan
        r = b1.route(x, k, score=score, bias=bias, renormalize=renormalize)
        check_routes(torch, r, x, k, score=score, bias=bias, renormalize=renormalize)


@pytest.mark.parametrize("off", [-math.inf, -4.0])
@pytest.mark.parametrize("experts", [6, 40, 100, 200, 400, 900])
@pytest.mark.parametrize("tokens", [9, 90])
def test_route_far_behind_a_logit_that_is_not_chosen(torch, b1, tokens, experts, off):
    """Renormalized softmax weights depend on the chosen logits alone, however
    far below the largest one they lie, which the bias turns off or puts
    behind.  The bound: differences of at most `spread` to the largest chosen
    logit, rounded (half a step each), an exponential (2 steps), a sum of four
    (3 half steps), in numerator and denominator, and a division."""
    say(f"route far behind {tokens} {experts} {off}")
    k, peak = 4, experts // 3
    far = torch.tensor([80.0, 87.5, 95.0, 103.0, 104.0, 120.0, 300.0, 1000.0, 3e38], device="cuda")
    x = normal(torch, experts, tokens, experts)
    x[:, peak] = far[torch.arange(tokens, device="cuda") % len(far)]
    # steps of 2^-10 tell the others apart: their scores are below 1e-30
    rank = torch.randperm(experts, generator=torch.Generator().manual_seed(experts))
    bias = -rank.float() / 1024
    bias[peak] = off
    chosen = torch.argsort(bias, descending=True)[:k]
    assert peak not in chosen.tolist()
    r = b1.route(x, k, bias=bias.cuda())
    expert = chosen.int().expand(tokens, k)
    assert torch.equal(r.expert.cpu(), expert)
    z = x.cpu().double()[:, chosen]
    z = z - z.amax(1, keepdim=True)
    want = z.exp() / z.exp().sum(1, keepdim=True)
    spread = -z.amin(1, keepdim=True)
    ref.check(r.weight, want, want * (2 * spread + 16) * ref.U32, torch.float32, "weights")
    for got, at in zip((r.start, r.order, r.place), moe.layout(expert, experts)):
        assert torch.equal(got.cpu(), at)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [6, 100, 200, 400, 900])
@pytest.mark.parametrize("tokens", [7, 70])
def test_route_never_chooses_what_a_bias_turns_off(torch, b1, tokens, experts, score):
    """An expert whose bias is -inf has no rows, whatever the logits are: NaN
    and infinities among them, its own or others'."""
    say(f"route off by bias {tokens} {experts} {score}")
    on = [1, experts // 2, experts - 1]
    off = [e for e in range(experts) if e not in on]
    bias = torch.full((experts,), -math.inf, device="cuda")
    bias[on] = 0.0
    x = normal(torch, 1, tokens, experts)
    x[0, on[1]] = math.inf
    x[1] = math.nan
    x[2, off[0]] = math.nan
    x[3, [on[0], off[1]]] = math.inf
    x[4, off[-1]] = math.inf
    x[5, off] = math.inf
    r = b1.route(x, 4, score=score, bias=bias)
    expert = r.expert.cpu()
    assert bool((expert[:, 3] == -1).all()) and expert[:, :3].sort(1).values.tolist() == [on] * tokens
    for got, at in zip((r.start, r.order, r.place), moe.layout(expert, experts)):
        assert torch.equal(got.cpu(), at)
    nan = torch.zeros(tokens, dtype=torch.bool)
    nan[[1, 2] + ([0, 3, 4, 5] if score == "softmax" else [])] = True
    weight = r.weight.cpu()
    assert torch.equal(weight[:, :3].isnan(), nan[:, None].expand(tokens, 3)) and bool((weight[:, 3] == 0).all())


@pytest.mark.parametrize("tokens", [1, 32, 33, 1000, 4099])
@pytest.mark.parametrize("experts,k", [(1, 1), (2, 2), (3, 1), (8, 8)])
def test_route_of_experts_that_all_tokens_want(torch, b1, tokens, experts, k):
    """Every lane of a wave places a row of the same few experts, turn after
    turn: in an expert's rows the slots still ascend."""
    say(f"route all alike {tokens} {experts} {k}")
    logits = torch.zeros(tokens, experts, device="cuda")
    r = b1.route(logits, k)
    expert = torch.arange(k, dtype=torch.int32).expand(tokens, k)
    assert torch.equal(r.expert.cpu(), expert)
    for got, at in zip((r.start, r.order, r.place), moe.layout(expert, experts)):
        assert torch.equal(got.cpu(), at)


def same_routes(torch, a, b):
    for name in ("expert", "start", "order", "place"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert torch.equal(a.weight.nan_to_num(7.0), b.weight.nan_to_num(7.0))


def blank_routes(torch, b1, tokens, experts, k):
    def i32(*shape):
        return torch.full(shape, -77, dtype=torch.int32, device="cuda")
    return b1.Routes(i32(tokens, k), torch.full((tokens, k), 3.0, device="cuda"), i32(experts + 1), i32(tokens * k),
                     i32(tokens, k))


def test_route_with_and_without_a_workspace(torch, b1):
    """One work-group alone gives what the many give; a workspace that is too
    small is as none."""
    logits = normal(torch, 3, 1000, 96).to(torch.bfloat16)
    want = b1.route(logits, 5)
    for size in (16, 1 << 20):
        got = blank_routes(torch, b1, 1000, 96, 5)
        ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        assert b1.route(logits, 5, out=got, workspace=ws) is got
        same_routes(torch, got, want)


def test_route_of_no_tokens(torch, b1):
    r = b1.route(torch.empty(0, 12, device="cuda"), 3)
    assert r.start.tolist() == [0] * 13 and r.order.numel() == 0


def test_route_of_many_tokens(torch, b1):
    """Popular experts, more tokens than a work-group's share is small."""
    tokens, experts, k = 30011, 128, 8
    logits = normal(torch, 8, tokens, experts) + normal(torch, 9, experts, spread=3.0)
    r = b1.route(logits, k)
    expert = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.expert.long(), expert)
    flat = expert.flatten()
    order = torch.sort(flat, stable=True).indices
    assert torch.equal(r.order.long(), order)
    assert torch.equal(r.place.flatten()[order], torch.arange(tokens * k, dtype=torch.int32, device="cuda"))
    assert torch.equal(r.start[1:].long(), torch.bincount(flat, minlength=experts).cumsum(0)) and int(r.start[0]) == 0


# ---- the experts' linears --------------------------------------------------


def routes_of(torch, b1, expert, experts, weight=None):
    """A Routes of expert ids [tokens, top_k] (host)."""
    start, order, place = moe.layout(expert, experts)
    if weight is None:
        weight = torch.rand(expert.shape, generator=torch.Generator().manual_seed(4)) * (expert >= 0)
    return b1.Routes(*(t.cuda().contiguous() for t in (expert.int(), weight.float(), start, order, place)))


def spread_out(torch, tokens, experts, k, seed, counts=None):
    """Expert ids [tokens, k], each row without repeats; counts: about how
    often each expert is wanted."""
    g = torch.Generator().manual_seed(seed)
    want = torch.rand(tokens, experts, generator=g).log().neg().log().neg()
    if counts is not None:
        want = want + torch.tensor(counts, dtype=torch.float32).clamp(min=1e-9).log()
    return want.topk(k, 1).indices.int()


def run_linear(torch, b1, unpack, expert, experts, in_dim, out_dim, rows, act, packed, seed=0, **more):
    """Runs linear_experts over rows of known filling and compares every row."""
    from bonsai_b1 import synth
    tokens, k = expert.shape
    n = tokens * k
    r = routes_of(torch, b1, expert, experts)
    used = int(r.start[-1])
    have = tokens if rows == "tokens" else n
    a = b1.pack_act_f16(normal(torch, 11 + seed, have, in_dim))
    w = synth.device_packed_weights(experts * out_dim, in_dim, 12 + seed)
    nf = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    cols = out_dim // 2 if act == "swiglu" else out_dim
    if packed:
        ldp = cols + 40
        buf = torch.full(((n * ldp + 64) * 2,), 0x3c, dtype=torch.uint8, device="cuda")
        first = 32
        view = buf[first * 2:]
        y = b1.linear_experts(a, w, r, in_dim, out_dim, act=act, rows=rows, packed=view, ldp=ldp, nonfinite=nf,
                              bad=bad, **more)
        assert y is view
        got = ref.unpack(buf, n, cols, ldp, first)
        kept = buf.view(torch.float16)[first:first + n * ldp].view(n, ldp)
        filling = torch.full((1,), 0x3c3c, dtype=torch.int16).view(torch.float16).item()
        assert bool((kept[:, cols:] == filling).all()), "columns behind the range"
        assert bool((kept[used:] == filling).all()), "rows behind the last"
    else:
        out = torch.full((n, out_dim + 4), 7.5, device="cuda")
        y = b1.linear_experts(a, w, r, in_dim, out_dim, act=act, rows=rows, out=out[:, :out_dim], nonfinite=nf,
                              bad=bad, **more)
        got = out[:, :out_dim]
        assert bool((out[:, out_dim:] == 7.5).all()), "columns behind the row"
        assert bool((out[used:] == 7.5).all()), "rows behind the last"
    want, off = moe.experts(ref.unpack(a, have, in_dim), unpack(w, experts * out_dim, in_dim).cpu()
                            .view(experts, out_dim, in_dim), r.start.cpu(), r.order.cpu(), k, rows == "tokens", act)
    ref.check(got[:used], want, off, torch.float16 if packed else torch.float32, "rows")
    assert int(nf) == 0 and int(bad) == 0
    return r, a, w


@pytest.mark.parametrize("rows", ["tokens", "routes"])
@pytest.mark.parametrize("act,packed", [("none", False), ("none", True), ("gelu_tanh", True), ("swiglu", True)])
@pytest.mark.parametrize("tokens,experts,k,in_dim,out_dim", [
    (1, 8, 2, 64, 64), (1, 128, 8, 512, 192), (5, 4, 1, 256, 128), (23, 5, 3, 320, 256), (16, 1, 1, 1088, 64),
    (64, 16, 4, 768, 448), (61, 3, 2, 2048, 320), (300, 4, 2, 576, 384), (200, 33, 6, 128, 576),
    (900, 2, 1, 192, 448)])
def test_linear_experts(torch, b1, unpack, tokens, experts, k, in_dim, out_dim, rows, act, packed):
    say(f"linear_experts {tokens} {experts} {k} {in_dim} {out_dim} {rows} {act} {packed}")
    run_linear(torch, b1, unpack, spread_out(torch, tokens, experts, k, tokens), experts, in_dim, out_dim, rows, act,
               packed)


@pytest.mark.parametrize("rows", ["tokens", "routes"])
@pytest.mark.parametrize("act,packed", [("none", False), ("none", True), ("gelu_tanh", True), ("swiglu", True)])
@pytest.mark.parametrize("shape", moe.KERNELS)
def test_linear_experts_by_each_kernel(torch, b1, unpack, shape, rows, act, packed):
    """Every kernel that the dispatch knows; the CPU tests hold its shapes."""
    tokens, experts, k, in_dim, out_dim = shape
    say(f"linear_experts kernel {shape} {rows} {act} {packed}")
    run_linear(torch, b1, unpack, spread_out(torch, tokens, experts, k, tokens), experts, in_dim, out_dim, rows, act,
               packed)


@pytest.mark.parametrize("rows", ["tokens", "routes"])
@pytest.mark.parametrize("act,packed", [("none", False), ("none", True), ("gelu_tanh", True), ("swiglu", True)])
@pytest.mark.parametrize("shape", list(moe.KERNELS) + [(1, 128, 8, 2048, 192), (300, 20, 3, 1344, 1408)])
def test_linear_experts_lose_no_product(torch, b1, unpack, shape, rows, act, packed):
    """Activations of +-1, 2, 3 and scales of 2^-5, 2^-4, 2^-3: every partial sum
    is a multiple of 2^-5 below 2^13, exact in fp32 in any order, so that a
    single product lost or taken twice shows at any width.  Rows are equal to
    the definition's, plain packed rows to their rounding; behind an activation
    only its own steps count."""
    from bonsai_b1 import synth
    tokens, experts, k, in_dim, out_dim = shape
    say(f"linear_experts exact {shape} {rows} {act} {packed}")
    r = routes_of(torch, b1, spread_out(torch, tokens, experts, k, tokens), experts)
    n = tokens * k
    have = tokens if rows == "tokens" else n
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens + in_dim)
    a = torch.randint(1, 4, (have, in_dim), generator=g, device="cuda").float()
    a *= torch.randint(0, 2, a.shape, generator=g, device="cuda") * 2 - 1
    w = synth.device_packed_weights(experts * out_dim, in_dim, 12).view(-1, 6)
    w[:, :2] = (2.0 ** torch.randint(-5, -2, (len(w), 1), generator=g, device="cuda")).half().view(torch.uint8)
    w = w.flatten()
    cols = out_dim // 2 if act == "swiglu" else out_dim
    y = b1.linear_experts(b1.pack_act_f16(a), w, r, in_dim, out_dim, act=act, rows=rows, packed=packed or None)
    got = ref.unpack(y, n, cols) if packed else y
    order = r.order.cpu()
    want, _ = moe.experts(a.cpu(), unpack(w, experts * out_dim, in_dim).cpu().view(experts, out_dim, in_dim),
                          r.start.cpu(), order, k, rows == "tokens")
    assert bool((want.abs() < 2 ** 13).all()) and torch.equal(want * 32, (want * 32).round())
    if act == "none":
        assert torch.equal(got.cpu(), want.to(torch.float16 if packed else torch.float32))
        return
    want, off = moe.activation(want, torch.zeros_like(want), act)
    ref.check(got, want, off, torch.float16, "rows")


@pytest.mark.parametrize("tokens,experts,k,in_dim,out_dim", [
    (20, 20, 2, 192, 2497), (100, 20, 3, 1088, 2303), (2721, 5, 3, 192, 131), (512, 20, 1, 1088, 2345),
    (2829, 3, 3, 320, 333), (6000, 2, 1, 64, 2111)])
def test_linear_experts_by_tiles_of_odd_widths(torch, b1, unpack, tokens, experts, k, in_dim, out_dim):
    say(f"linear_experts odd tiles {tokens} {experts} {k} {in_dim} {out_dim}")
    run_linear(torch, b1, unpack, spread_out(torch, tokens, experts, k, 5), experts, in_dim, out_dim, "tokens", "none",
               False)


@pytest.mark.parametrize("counts", [
    [1, 0, 0, 0, 0], [0, 0, 0, 0, 1], [0, 1, 0, 1, 0], [4000, 1, 1, 1, 1], [1, 1, 1, 1, 300]])
@pytest.mark.parametrize("tokens,in_dim,out_dim", [(60, 192, 2496), (2721, 192, 128), (4243, 320, 320)])
def test_linear_experts_by_tiles_of_uneven_groups(torch, b1, unpack, tokens, in_dim, out_dim, counts):
    say(f"linear_experts uneven tiles {tokens} {in_dim} {out_dim} {counts}")
    expert = spread_out(torch, tokens, 5, 1, 3, counts)
    expert[5::97] = -1
    run_linear(torch, b1, unpack, expert, 5, in_dim, out_dim, "tokens", "swiglu", True)
    run_linear(torch, b1, unpack, expert, 5, in_dim, out_dim - 1, "routes", "none", False)


@pytest.mark.parametrize("out_dim", [1, 2, 15, 63, 65, 100, 129, 191, 193, 257, 1003])
@pytest.mark.parametrize("tokens", [2, 40, 400])
def test_linear_experts_of_odd_widths(torch, b1, unpack, out_dim, tokens):
    say(f"linear_experts odd {out_dim} {tokens}")
    run_linear(torch, b1, unpack, spread_out(torch, tokens, 3, 2, 5), 3, 192, out_dim, "tokens", "none", False)


@pytest.mark.parametrize("in_dim", [2112, 4096, 4160, 8192])
@pytest.mark.parametrize("tokens", [3, 150])
def test_linear_experts_of_wide_inputs(torch, b1, unpack, in_dim, tokens):
    say(f"linear_experts wide {in_dim} {tokens}")
    run_linear(torch, b1, unpack, spread_out(torch, tokens, 3, 2, 5), 3, in_dim, 128, "routes", "swiglu", True)
    run_linear(torch, b1, unpack, spread_out(torch, tokens, 3, 2, 6), 3, in_dim, 70, "tokens", "none", False)


@pytest.mark.parametrize("tokens", [9, 77, 512])
@pytest.mark.parametrize("counts", [
    [1, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 1], [0, 1, 0, 0, 1, 0], [1000, 1, 1, 1, 1, 1], [1, 1, 1, 1, 1, 100]])
def test_linear_experts_of_uneven_groups(torch, b1, unpack, tokens, counts):
    """All rows with one expert, empty experts first, last and between."""
    say(f"linear_experts uneven {tokens} {counts}")
    expert = spread_out(torch, tokens, 6, 1, 3, counts)
    run_linear(torch, b1, unpack, expert, 6, 320, 192, "tokens", "swiglu", True)
    run_linear(torch, b1, unpack, expert, 6, 320, 200, "routes", "none", False)


@pytest.mark.parametrize("tokens,experts", [(40, 6), (300, 3), (30, 900)])
def test_linear_experts_of_tokens_without_routes(torch, b1, unpack, tokens, experts):
    """Slots of no expert: fewer rows than slots, the rest left as it was."""
    say(f"linear_experts holes {tokens} {experts}")
    expert = spread_out(torch, tokens, experts, 2, 3)
    expert[::3, 1] = -1
    expert[1::5] = -1
    run_linear(torch, b1, unpack, expert, experts, 128, 64, "tokens", "gelu_tanh", True)
    run_linear(torch, b1, unpack, expert, experts, 128, 68, "routes", "none", False)
    expert[:] = -1  # no rows at all
    run_linear(torch, b1, unpack, expert, experts, 128, 68, "tokens", "none", False)


@pytest.mark.parametrize("tokens,experts", [(6, 8), (500, 3)])
def test_linear_experts_counts_what_is_not_finite(torch, b1, tokens, experts):
    from bonsai_b1 import synth
    k, n, top_k = 256, 96, 2
    expert = spread_out(torch, tokens, experts, top_k, 2)
    r = routes_of(torch, b1, expert, experts)
    a = normal(torch, 1, tokens, k)
    a[3, 5] = math.inf
    w = synth.device_packed_weights(experts * n, k, 3)
    nf = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = b1.linear_experts(b1.pack_act_f16(a), w, r, k, n, nonfinite=nf)
    rows = r.place[3].long()
    assert not bool(y[rows].isfinite().any())
    keep = torch.ones(len(y), dtype=torch.bool, device="cuda")
    keep[rows] = False
    assert bool(y[keep].isfinite().all()) and int(nf) == top_k * n


def bad_starts(torch, routes, experts):
    yield "descending", [routes - i for i in range(experts + 1)]
    yield "negative", [-5] + [0] * (experts - 1) + [routes]
    yield "too far", [0] * experts + [routes + 9]
    yield "far between", [0, 1 << 30] + [3] * (experts - 2) + [routes]
    yield "extremes", [-(1 << 31)] + [(1 << 31) - 1] * experts


@pytest.mark.parametrize("tokens,experts,k", [(5, 6, 2), (300, 3, 2), (40, 130, 3), (9000, 2, 1), (3000, 300, 2)])
def test_bad_indices(torch, b1, tokens, experts, k):
    """Starts out of order or range make the call's rows NaN, an order entry
    or a place out of range its row; nothing else is touched, and `bad` says
    so.  Rows that no group holds stay as they were."""
    from bonsai_b1 import synth
    in_dim, n = 192, 64
    expert = spread_out(torch, tokens, experts, k, 1)
    good = routes_of(torch, b1, expert, experts)
    routes = tokens * k
    a = b1.pack_act_f16(normal(torch, 1, tokens, in_dim))
    w = synth.device_packed_weights(experts * n, in_dim, 3)
    fine = b1.linear_experts(a, w, good, in_dim, n)

    def call(r, **how):
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        guard = torch.full((routes + 16, n), 7.5, device="cuda")
        b1.linear_experts(a, w, r, in_dim, n, out=guard[8:8 + routes], bad=bad, **how)
        assert bool((guard[:8] == 7.5).all()) and bool((guard[8 + routes:] == 7.5).all())
        return guard[8:8 + routes], int(bad)

    for what, values in bad_starts(torch, routes, experts):
        say(f"bad starts {what} {tokens} {experts}")
        r = b1.Routes(good.expert, good.weight, torch.tensor(values, dtype=torch.int32, device="cuda"), good.order,
                      good.place)
        y, bad = call(r)
        assert bad >= 1 and bool((y.isnan() | (y == 7.5)).all()), what
        p = torch.full((routes + 16, n), 0x3c, dtype=torch.float16, device="cuda")
        b1.linear_experts(a, w, r, in_dim, n, packed=p[8:8 + routes].view(torch.uint8).flatten())
        assert bool((p[:8] == 0x3c).all()) and bool((p[8 + routes:] == 0x3c).all())
    for value in (-1, routes, (1 << 31) - 1, -(1 << 31)):
        say(f"bad order {value} {tokens} {experts}")
        order = good.order.clone()
        order[3] = value
        y, bad = call(b1.Routes(good.expert, good.weight, good.start, order, good.place))
        keep = torch.arange(routes, device="cuda") != 3
        assert bad >= 1 and bool(y[3].isnan().all()) and torch.equal(y[keep], fine[keep])
    for value in (-2, routes, (1 << 31) - 1, -(1 << 31)):
        say(f"bad place {value} {tokens} {experts}")
        place = good.place.clone()
        place[2, k - 1] = value
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        r = b1.Routes(good.expert, good.weight, good.start, good.order, place)
        out, want = b1.combine_experts(fine, r, bad=bad), b1.combine_experts(fine, good)
        keep = torch.arange(tokens, device="cuda") != 2
        assert int(bad) >= 1 and bool(out[2].isnan().all()) and torch.equal(out[keep], want[keep])


@pytest.mark.parametrize("act,packed", [("none", False), ("none", True), ("gelu_tanh", True), ("swiglu", True)])
@pytest.mark.parametrize("tokens,experts,k,in_dim,out_dim", [
    (40, 3, 2, 192, 256), (30, 900, 2, 128, 64), (200, 33, 6, 128, 576), (512, 20, 1, 1088, 2368),
    (2721, 5, 3, 192, 128), (6000, 2, 1, 64, 2112), (3000, 300, 2, 192, 64)])
def test_bad_indices_leave_no_row(torch, b1, tokens, experts, k, in_dim, out_dim, act, packed):
    """Starts out of order or range make every row NaN, an order entry out of
    range its row, in every kind of output; columns and rows around them stay
    as they were."""
    from bonsai_b1 import synth
    good = routes_of(torch, b1, spread_out(torch, tokens, experts, k, 1), experts)
    routes = tokens * k
    a = b1.pack_act_f16(normal(torch, 1, tokens, in_dim))
    w = synth.device_packed_weights(experts * out_dim, in_dim, 3)
    cols = out_dim // 2 if act == "swiglu" else out_dim

    def call(r):
        bad = torch.zeros(1, dtype=torch.int32, device="cuda")
        dtype = torch.float16 if packed else torch.float32
        guard = torch.full((routes + 16, cols + 8), 7.5, dtype=dtype, device="cuda")
        inside = guard[8:8 + routes]
        if packed:
            b1.linear_experts(a, w, r, in_dim, out_dim, act=act, bad=bad,
                              packed=inside.view(torch.uint8).flatten(), ldp=cols + 8)
        else:
            b1.linear_experts(a, w, r, in_dim, out_dim, bad=bad, out=inside[:, :cols])
        assert bool((guard[:8] == 7.5).all()) and bool((guard[8 + routes:] == 7.5).all())
        assert bool((inside[:, cols:] == 7.5).all())
        return inside[:, :cols], int(bad)

    fine, bad = call(good)
    assert bad == 0 and bool(fine.isfinite().all())
    for what, values in bad_starts(torch, routes, experts):
        say(f"bad starts {what} {tokens} {experts} {act} {packed}")
        y, bad = call(b1.Routes(good.expert, good.weight, torch.tensor(values, dtype=torch.int32, device="cuda"),
                                good.order, good.place))
        assert bad >= 1 and bool(y.isnan().all()), what
    for value in (-1, routes, -(1 << 31)):
        order = good.order.clone()
        order[[0, routes - 1]] = value
        y, bad = call(b1.Routes(good.expert, good.weight, good.start, order, good.place))
        assert bad == 2 and bool(y[[0, routes - 1]].isnan().all())
        assert torch.equal(y[1:-1], fine[1:-1])


def test_no_rows(torch, b1):
    r = b1.route(torch.empty(0, 4, device="cuda"), 2)
    w = torch.zeros(4 * 64 * 2 * 6, dtype=torch.uint8, device="cuda")
    empty = torch.empty(0, dtype=torch.uint8, device="cuda")
    assert b1.linear_experts(empty, w, r, 64, 64).shape == (0, 64)
    b1.linear_experts(empty, w, r, 64, 64, act="swiglu", packed=True)
    assert b1.combine_experts(torch.empty(0, 8, device="cuda"), r).shape == (0, 8)


# ---- the weighted sum ------------------------------------------------------


@pytest.mark.parametrize("tokens,experts,k,h", [(1, 4, 1, 4), (1, 128, 8, 2048), (7, 5, 3, 100), (33, 16, 8, 1028),
                                                (300, 4, 2, 64), (5, 80, 64, 4100), (64, 128, 8, 2048)])
@pytest.mark.parametrize("how", ["plain", "residual", "in place", "strided", "holes"])
def test_combine(torch, b1, tokens, experts, k, h, how):
    say(f"combine {tokens} {experts} {k} {h} {how}")
    expert = spread_out(torch, tokens, experts, k, tokens)
    if how == "holes":
        expert[::2, k - 1] = -1
        expert[1::4] = -1
    r = routes_of(torch, b1, expert, experts)
    y, x = normal(torch, 1, tokens * k, h), normal(torch, 2, tokens, h, spread=3.0)
    if how == "holes":
        y[int(r.start[-1]):] = math.nan  # rows of nobody
    residual = None if how == "plain" else x
    want, off = moe.combine(y.cpu(), r.weight.cpu(), r.place.cpu(), residual)
    out = None
    if how == "in place":
        out = x
    elif how == "strided":
        y = torch.cat([y, y], 1)[:, :h]
        residual = torch.cat([x, x, x], 1)[:, h:2 * h]
        out = torch.full((tokens, h + 8), 7.5, device="cuda")[:, 4:4 + h]
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = b1.combine_experts(y, r, residual=residual, out=out, bad=bad)
    assert out is None or got is out
    ref.check(got, want, off, torch.float32, how)
    assert int(bad) == 0
    if how == "strided" and tokens > 1:
        assert bool((out.as_strided((tokens, 4), (h + 8, 1), 0) == 7.5).all())


# ---- a block's MLP ---------------------------------------------------------


def block(b1, x, w_norm, w_router, w_up, w_down, experts, k, h, f, ws=None, bias=None):
    """norm -> router -> up with SwiGLU -> down -> residual + weighted sum."""
    a = b1.rms_norm(x, w_norm, packed=True)
    logits = b1.linear_packed_f16(a, w_router, h, experts, x.shape[0])
    r = b1.route(logits, k, bias=bias, score="sigmoid" if bias is not None else "softmax", workspace=ws)
    up = b1.linear_experts(a, w_up, r, h, 2 * f, act="swiglu", packed=True)
    y = b1.linear_experts(up, w_down, r, f, h, rows="routes")
    return a, logits, r, up, y, b1.combine_experts(y, r, residual=x)


@pytest.mark.parametrize("tokens,balanced", [(1, False), (9, True), (130, False), (700, True)])
def test_each_step_of_a_block(torch, b1, unpack, tokens, balanced):
    """Every operator of a block's mixture of experts, element by element,
    against float64 on the operands that it read."""
    from bonsai_b1 import synth
    say(f"block {tokens} {balanced}")
    experts, k, h, f = 12, 3, 768, 320
    x = normal(torch, 1, tokens, h)
    w_norm = 1.0 + normal(torch, 2, h, spread=0.2)
    w_router = synth.device_packed_weights(experts, h, 3)
    w_up, w_down = (synth.device_packed_weights(experts * n, d, s) for n, d, s in ((2 * f, h, 4), (h, f, 5)))
    bias = normal(torch, 6, experts, spread=0.1) if balanced else None
    a, logits, r, up, y, out = block(b1, x, w_norm, w_router, w_up, w_down, experts, k, h, f, bias=bias)
    check_routes(torch, r, logits, k, score="sigmoid" if balanced else "softmax", bias=bias)
    start, order = r.start.cpu(), r.order.cpu()
    a16 = ref.unpack(a, tokens, h)
    want, off = moe.experts(a16, unpack(w_up, experts * 2 * f, h).cpu().view(experts, 2 * f, h), start, order, k, True,
                            "swiglu")
    up16 = ref.unpack(up, tokens * k, f)
    ref.check(up16, want, off, torch.float16, "up")
    want, off = moe.experts(up16, unpack(w_down, experts * h, f).cpu().view(experts, h, f), start, order, k, False)
    ref.check(y, want, off, torch.float32, "down")
    want, off = moe.combine(y.cpu(), r.weight.cpu(), r.place.cpu(), x)
    ref.check(out, want, off, torch.float32, "sum")


@pytest.mark.parametrize("tokens", [4, 600])
def test_a_block_captured_and_replayed(torch, b1, tokens):
    """Captured once, replayed over other inputs (so other routes), with eager
    work of the same operators between the replays; a second graph with its
    own workspace replayed on another stream meanwhile."""
    from bonsai_b1 import synth
    say(f"graph {tokens}")
    experts, k, h, f = 16, 2, 384, 192
    w_norm = 1.0 + normal(torch, 2, h, spread=0.2)
    w_router = synth.device_packed_weights(experts, h, 3)
    w_up, w_down = (synth.device_packed_weights(experts * n, d, s) for n, d, s in ((2 * f, h, 4), (h, f, 5)))

    def step(x, ws):
        return block(b1, x, w_norm, w_router, w_up, w_down, experts, k, h, f, ws=ws)

    xs = [normal(torch, 20 + i, tokens, h) for i in range(2)]
    wss = [torch.empty(1 << 20, dtype=torch.uint8, device="cuda") for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i]):
            step(xs[i], wss[i])
            streams[i].synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[i]):
                outs.append(step(xs[i], wss[i]))
            graphs.append(g)
    torch.cuda.synchronize()
    for turn in range(5):
        for i in range(2):
            xs[i].copy_(normal(torch, 40 + 2 * turn + i, tokens, h))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = step(xs[i], wss[2])
            torch.cuda.synchronize()
            same_routes(torch, outs[i][2], want[2])
            for j in (0, 1, 3, 4, 5):
                assert torch.equal(outs[i][j], want[j]), f"turn {turn}, graph {i}, output {j}"
    del graphs


def test_a_capture_without_a_workspace(torch, b1):
    """Nothing is allocated while a stream is captured: one work-group routes."""
    logits = normal(torch, 3, 500, 40)
    want = b1.route(logits, 4)
    got = blank_routes(torch, b1, 500, 40, 4)
    stream = torch.cuda.Stream()  # with no workspace of the library's
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            b1.route(logits, 4, out=got)
        for turn in range(3):
            logits.copy_(normal(torch, 30 + turn, 500, 40))
            g.replay()
            stream.synchronize()
            want = b1.route(logits, 4)
            stream.synchronize()
            same_routes(torch, got, want)
    del g


def test_large_kernels_captured(torch, b1):
    """Kernels with more than 64 KB of LDS ask for it at every call, a captured
    one too: 128-row tiles, one work-group that routes over 1024 experts."""
    from bonsai_b1 import synth
    say("large kernels captured")
    tokens, experts, k, in_dim, out_dim = 2829, 3, 3, 320, 320
    logits, wide = normal(torch, 1, tokens, experts), normal(torch, 2, 20, 1024)
    acts = b1.pack_act_f16(normal(torch, 3, tokens, in_dim))
    w = synth.device_packed_weights(experts * out_dim, in_dim, 4)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def step():
        r = b1.route(logits, k, workspace=ws)
        return r, b1.linear_experts(acts, w, r, in_dim, out_dim), b1.route(wide, 6)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            got = step()
        for turn in range(3):
            logits.copy_(normal(torch, 10 + turn, tokens, experts))
            wide.copy_(normal(torch, 20 + turn, 20, 1024))
            g.replay()
            stream.synchronize()
            want = step()
            stream.synchronize()
            same_routes(torch, got[0], want[0])
            same_routes(torch, got[2], want[2])
            assert torch.equal(got[1], want[1])
    del g


@pytest.mark.parametrize("tokens,real", [(8, 5), (200, 77), (64, 0)])
def test_padded_batch(torch, b1, tokens, real):
    """Tokens whose experts are all off have no rows and get their residual;
    the others come out as without them."""
    from bonsai_b1 import synth
    say(f"padded batch {tokens} {real}")
    experts, k, h, f = 6, 2, 256, 64
    x, logits = normal(torch, 1, tokens, h), normal(torch, 2, tokens, experts)
    logits[real:] = -math.inf
    up_w, down_w = (synth.device_packed_weights(experts * n, d, s) for n, d, s in ((2 * f, h, 4), (h, f, 5)))
    acts = b1.pack_act_f16(x)
    r = b1.route(logits, k)
    assert int(r.start[-1]) == real * k and bool((r.order[real * k:] == -1).all())
    up = torch.full((tokens * k * f * 2 + 16,), 255, dtype=torch.uint8, device="cuda")  # NaN where nothing is written
    b1.linear_experts(acts, up_w, r, h, 2 * f, act="swiglu", packed=up)
    y = torch.full((tokens * k, h), math.nan, device="cuda")
    b1.linear_experts(up, down_w, r, f, h, rows="routes", out=y)
    out = b1.combine_experts(y, r, residual=x)
    assert torch.equal(out[real:], x[real:]) and bool(out.isfinite().all())
    assert bool(y[real * k:].isnan().all())


def test_calls_on_another_stream(torch, b1):
    """stream=: results, and outputs that belong to that stream."""
    from bonsai_b1 import synth
    x = normal(torch, 1, 200, 384)
    w = synth.device_packed_weights(8 * 128, 384, 2)
    logits = normal(torch, 3, 200, 8)
    a = b1.pack_act_f16(x)
    r = b1.route(logits, 2)
    y = b1.linear_experts(a, w, r, 384, 128)
    out = b1.combine_experts(y, r)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    r2 = b1.route(logits, 2, stream=s)
    y2 = b1.linear_experts(a, w, r2, 384, 128, stream=s)
    out2 = b1.combine_experts(y2, r2, stream=s)
    s.synchronize()
    same_routes(torch, r2, r)
    assert torch.equal(y, y2) and torch.equal(out, out2)


def test_rows_past_32_bit_offsets(torch, b1, unpack):
    """Down projections of rows whose bytes pass 2^32, in and out."""
    from bonsai_b1 import synth
    torch.cuda.empty_cache()
    tokens, experts, k, in_dim, out_dim = 300000, 3, 1, 8192, 4096
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    say("rows past 32-bit offsets")
    n = tokens * k
    ends = [0, 100000, 100003, n]
    r = b1.Routes(torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), torch.ones(tokens, 1, device="cuda"),
                  torch.tensor(ends, dtype=torch.int32, device="cuda"),
                  torch.arange(n, dtype=torch.int32, device="cuda"),
                  torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1))
    a = torch.empty(n * in_dim, dtype=torch.float16, device="cuda").normal_()
    w = synth.device_packed_weights(experts * out_dim, in_dim, 2)
    y = b1.linear_experts(a.view(torch.uint8), w, r, in_dim, out_dim, rows="routes")
    w64 = unpack(w, experts * out_dim, in_dim).cpu().view(experts, out_dim, in_dim)
    for row, e in ((0, 0), (99999, 0), (100001, 1), (100003, 2), (262143, 2), (262144, 2), (n - 1, 2)):
        one = a[row * in_dim:(row + 1) * in_dim].view(torch.uint8)
        want, off = moe.linear(ref.unpack(one, 1, in_dim), w64[e])
        ref.check(y[row:row + 1], want, off, torch.float32, f"row {row}")
    out = b1.combine_experts(y, r)
    assert torch.equal(out, y)
    del a, y, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens,experts,in_dim,out_dim", [
    (262143, 1024, 8192, 64), (262143, 1000, 8192, 256), (32767, 1024, 65536, 64), (16384, 1024, 65536, 63)])
def test_token_rows_past_31_bit_offsets(torch, b1, unpack, tokens, experts, in_dim, out_dim):
    """Up projections over tokens whose rows take up to 2^32 bytes, the most
    that is accepted: the same rows as from activations gathered beforehand,
    and some of them against float64."""
    from bonsai_b1 import synth
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    say(f"token rows past 31-bit offsets {tokens} {experts} {in_dim} {out_dim}")
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    expert = torch.randint(0, experts, (tokens, 1), generator=g, device="cuda", dtype=torch.int32)
    order = torch.argsort(expert.flatten(), stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(tokens, device="cuda")
    start = torch.bincount(expert.flatten(), minlength=experts).cumsum(0)
    r = b1.Routes(expert, torch.ones(tokens, 1, device="cuda"), torch.cat([start.new_zeros(1), start]).int(),
                  order.int(), place.int().view(tokens, 1))
    a = torch.empty(tokens, in_dim, dtype=torch.float16, device="cuda").normal_(generator=g)
    assert 1 << 31 <= 2 * a.numel() < 1 << 32
    w = synth.device_packed_weights(experts * out_dim, in_dim, 2)
    y = b1.linear_experts(a.view(torch.uint8), w, r, in_dim, out_dim)
    gathered = torch.empty_like(a)
    for at in torch.arange(tokens, device="cuda").split(1 << 15):
        gathered[at] = a[order[at]]
    assert torch.equal(y, b1.linear_experts(gathered.view(torch.uint8), w, r, in_dim, out_dim, rows="routes"))
    for t in (0, 1, tokens // 2 - 1, tokens // 2, tokens // 2 + 1, tokens - 1):
        e, row = int(expert[t]), int(place[t])
        w64 = unpack(w.view(experts, -1)[e], out_dim, in_dim).cpu()
        want, off = moe.linear(ref.unpack(a[t].view(torch.uint8), 1, in_dim), w64)
        ref.check(y[row:row + 1], want, off, torch.float32, f"token {t}")
    del a, gathered, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens,experts", [(41, 8), (41, 1), (2050, 2)])
def test_swiglu_of_far_negative_gates(torch, b1, tokens, experts):
    """Gates from -80 to -100, where the hardware's reciprocal passes through
    its smallest numbers to 0: with values as large as inputs of fp16 make them
    here (2^22) the result is a zero of the value's other sign."""
    say(f"swiglu far gates {tokens} {experts}")
    in_dim, f = 64, 64
    a = torch.zeros(tokens, in_dim, device="cuda")
    a[:, 0] = 80.0 + 0.5 * (torch.arange(tokens, device="cuda") % 41)
    # gates -a[0], values +-2^15 a[0]
    w = torch.zeros(experts, 2 * f, in_dim // 32, 6, dtype=torch.uint8, device="cuda")
    scale = torch.ones(experts, 2 * f, in_dim // 32, 1, device="cuda")
    scale[:, f:] = 2.0 ** 15
    w[..., :2] = scale.half().view(torch.uint8)
    w[:, f:, :, 2:] = 255
    w[:, f + 1::2, :, 2:] = 0
    expert = torch.arange(tokens, dtype=torch.int32).view(-1, 1) % experts
    r = routes_of(torch, b1, expert, experts)
    nf = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = b1.linear_experts(b1.pack_act_f16(a), w.flatten(), r, in_dim, 2 * f, act="swiglu", packed=True, nonfinite=nf)
    got = ref.unpack(y, tokens, f)
    assert bool((got == 0).all()) and int(nf) == 0
    assert bool(got[:, ::2].signbit().all()) and not bool(got[:, 1::2].signbit().any())


def test_the_most_routes(torch, b1):
    """2^24 - 1 routes, the most that is accepted, nearly all of one expert:
    the router's 16-bit counts of its work-groups full, and launches of close to
    2^32 threads.  Whole activations and scales: rows are exact."""
    tokens, in_dim, out_dim = (1 << 24) - 1, 64, 4
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    say("the most routes")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    logits = torch.zeros(tokens, 2, device="cuda")
    other = torch.randint(0, tokens, (1000,), generator=g, device="cuda")
    logits[other, 1] = 1.0
    r = b1.route(logits, 1)
    expert = (logits[:, 1] > 0).int()
    assert torch.equal(r.expert.flatten(), expert) and bool((r.weight == 1).all())
    order = torch.argsort(expert, stable=True)
    first = tokens - int(expert.sum())
    assert r.start.tolist() == [0, first, tokens] and torch.equal(r.order.long(), order)
    assert torch.equal(r.place.flatten()[order], torch.arange(tokens, dtype=torch.int32, device="cuda"))
    a = torch.randint(-3, 4, (tokens, in_dim), generator=g, device="cuda", dtype=torch.int8).half()
    w = torch.randint(0, 256, (2, out_dim, in_dim // 32, 6), generator=g, device="cuda", dtype=torch.uint8)
    w[..., :2] = torch.ones(2, out_dim, in_dim // 32, 1, device="cuda").half().view(torch.uint8)
    y = b1.linear_experts(a.view(torch.uint8), w.flatten(), r, in_dim, out_dim)
    bits = torch.arange(8, device="cuda", dtype=torch.uint8)
    sign = 2.0 * ((w[..., 2:, None] >> bits) & 1).float().view(2, out_dim, in_dim) - 1.0
    c = torch.arange(in_dim, device="cuda")  # column c of a row is stored here
    stored = c // 32 * 32 + 2 * (c % 16) + c % 32 // 16
    for e, (lo, hi) in enumerate(((0, first), (first, tokens))):
        for at in torch.arange(lo, hi, device="cuda").split(1 << 21):
            x = a[order[at]][:, stored].float()
            want = torch.stack([(x * sign[e, n]).sum(1) for n in range(out_dim)], 1)
            assert torch.equal(y[at], want)
    x = normal(torch, 2, tokens, out_dim)
    out = b1.combine_experts(y, r, residual=x)
    assert torch.equal(out[order], y + x[order])
    del a, y, x, out
    torch.cuda.empty_cache()


def test_combine_of_more_than_32_bits_of_threads(torch, b1):
    """Tokens and columns whose work-groups have over 2^32 threads in all."""
    tokens, h = (1 << 23) + 3, 1028
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    if free < 90 << 30:
        pytest.skip("needs 90 GB of free device memory")
    say("combine of more than 32 bits of threads")
    place = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device="cuda").view(tokens, 1)
    r = b1.Routes(torch.zeros_like(place), torch.ones(tokens, 1, device="cuda"),
                  torch.tensor([0, tokens], dtype=torch.int32, device="cuda"), place.flatten(), place)
    y = torch.empty(tokens, h, device="cuda").normal_()
    out = torch.full((tokens, h), math.nan, device="cuda")
    assert b1.combine_experts(y, r, out=out) is out
    for at in torch.arange(tokens, device="cuda").split(1 << 20):
        assert torch.equal(out[at], y[tokens - 1 - at])
    del y, out
    torch.cuda.empty_cache()
