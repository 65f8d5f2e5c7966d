"""The router against the definition in 64 bits: the same experts in the same order, and weights that are off by the rounding to fp32 (2^-24 of the
value; sums and exponentials in 64 bits are off by less than 2^-40 of it)."""
import math

import pytest
import torch

import kudnn_b200 as kb

CODE = {torch.float32: kb.F32, torch.float16: kb.F16, torch.bfloat16: kb.BF16}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def route(x, w, top, bias=None, sigmoid=False, normalise=True, scale=1.0, stream=None):
    tokens, experts = x.shape[0], w.shape[0]
    desc = kb.make_route_desc(tokens, experts, x.shape[1], top, CODE[x.dtype], router_dtype=CODE[w.dtype], normalise=normalise, scale=scale,
                              score=kb.SCORE_SIGMOID if sigmoid else kb.SCORE_SOFTMAX, x_ld=x.stride(0), w_ld=w.stride(0))
    weights = torch.full((tokens, top), -7.0, device="cuda")
    ids = torch.full((tokens, top), -7, dtype=torch.int32, device="cuda")
    kb.route(desc, x, w, weights, ids, bias, stream=stream)
    return weights, ids


def definition(x, w, top, bias=None, sigmoid=False, normalise=True, scale=1.0):
    logits = x.double() @ w.double().t()
    out = torch.zeros(w.shape[0], dtype=torch.bool, device="cuda") if bias is None else torch.isneginf(bias)
    if sigmoid:
        score = 1 / (1 + torch.exp(-logits))
    else:
        score = torch.softmax(logits.masked_fill(out, -math.inf), dim=1)
    key = (score if bias is None else score + bias.double()).masked_fill(out, -math.inf)
    key, ids = torch.sort(key, dim=1, descending=True, stable=True)
    key, ids = key[:, :top], ids[:, :top]
    none = ~(key > -math.inf)
    p = score.gather(1, ids).masked_fill(none, 0.0)
    if normalise:
        total = p.sum(dim=1, keepdim=True)
        p = torch.where(total != 0, p / total, torch.zeros_like(p))
    return p * scale, ids.masked_fill(none, -1).int()


def check(got, want):
    weights, ids = got
    p, names = want
    assert torch.equal(ids, names)
    assert torch.all((weights.double() - p).abs() <= (2.0 ** -24 + 2.0 ** -40) * p.abs() + 2.0 ** -149)


def operands(tokens, experts, hidden, dtype, router, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, hidden), generator=gen, device="cuda").to(dtype)
    return x, (torch.randn((experts, hidden), generator=gen, device="cuda") * 2 * hidden ** -0.5).to(router)


SIZES = [(1, 1, 1, 1), (1, 2, 7, 2), (3, 8, 64, 3), (5, 9, 130, 4), (4, 60, 511, 6), (33, 64, 4096, 8), (2, 128, 2050, 64), (130, 33, 1000, 5),
         (257, 5, 33, 2), (300, 64, 1000, 8), (271, 150, 130, 64), (513, 1024, 70, 3),
         (769, 5, 33, 2), (800, 64, 1000, 8), (783, 150, 130, 64), (801, 1024, 70, 3),
         (1, 256, 7168, 8), (6, 1000, 300, 64), (2, 1024, 128, 33)]


@gpu
@pytest.mark.parametrize("dtype,router", [(d, r) for d in TYPES for r in TYPES])
@pytest.mark.parametrize("tokens,experts,hidden,top", SIZES)
def test_choices(cuda_device, dtype, router, tokens, experts, hidden, top):
    x, w = operands(tokens, experts, hidden, dtype, router)
    gen = torch.Generator(device="cuda").manual_seed(3)
    bias = torch.randn(experts, generator=gen, device="cuda") * 0.1
    check(route(x, w, top), definition(x, w, top))
    check(route(x, w, top, normalise=False, scale=2.5), definition(x, w, top, normalise=False, scale=2.5))
    check(route(x, w, top, bias), definition(x, w, top, bias))
    check(route(x, w, top, bias, sigmoid=True, scale=0.75), definition(x, w, top, bias, sigmoid=True, scale=0.75))


@gpu
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("left", [0, 1, 3, 20])
def test_experts_that_are_taken_out(cuda_device, sigmoid, left):
    x, w = operands(6, 40, 200, torch.bfloat16, torch.float32)
    bias = torch.full((40,), -math.inf, device="cuda")
    bias[torch.randperm(40)[:left]] = 0.25
    got = route(x, w, 8, bias, sigmoid=sigmoid)
    check(got, definition(x, w, 8, bias, sigmoid=sigmoid))
    assert bool(((got[1] >= 0).sum(dim=1) == min(left, 8)).all())


@gpu
@pytest.mark.parametrize("sigmoid", [False, True])
def test_equal_scores_go_to_the_lower_index(cuda_device, sigmoid):
    x, w = operands(5, 4, 777, torch.float16, torch.float32)
    order = torch.tensor([2, 0, 1, 0, 3, 2, 2, 1, 0, 3, 3, 0], device="cuda")
    check(route(x, w[order], 9, sigmoid=sigmoid), definition(x, w[order], 9, sigmoid=sigmoid))
    flat = torch.zeros((70, 777), device="cuda")
    assert torch.equal(route(x, flat, 64, sigmoid=sigmoid)[1], torch.arange(64, device="cuda", dtype=torch.int32).expand(5, 64))


@gpu
def test_scores_that_fp32_cannot_tell_apart(cuda_device):
    """Logits of 4096 + i 2^-13: their sums in 32 bits are equal."""
    w = torch.zeros((50, 512), device="cuda")
    w[:, 3] = 4096.0
    w[:, 500] = torch.randperm(50, device="cuda") * 2.0 ** -13
    x = torch.ones((3, 512), dtype=torch.bfloat16, device="cuda")
    got = route(x, w, 10)
    assert torch.equal(got[1][0], torch.argsort(w[:, 500], descending=True)[:10].int())
    check(got, definition(x, w, 10))


@gpu
def test_values_that_are_no_numbers(cuda_device):
    """An expert whose key is NaN takes no part; other tokens are not touched; far logits underflow to scores of zero."""
    x, w = operands(4, 12, 64, torch.float32, torch.float32)
    clean = definition(x, w, 4)
    bad = x.clone()
    bad[2, 5] = float("nan")
    weights, ids = route(bad, w, 4)
    keep = [0, 1, 3]
    check((weights[keep], ids[keep]), (clean[0][keep], clean[1][keep]))
    assert bool((ids[2] == -1).all()) and bool((weights[2] == 0).all())
    one = w.clone()
    one[7, 3] = float("nan")
    weights, ids = route(x, one, 11)
    rest = [e for e in range(12) if e != 7]
    p, names = definition(x, w[rest], 11)
    check((weights, ids), (p, torch.tensor(rest, device="cuda", dtype=torch.int32)[names.long()]))
    far = torch.zeros((1, 64), device="cuda")
    far[0, 0] = 1e4
    ladder = torch.zeros((6, 64), device="cuda")
    ladder[:, 0] = torch.tensor([0.0, 3.0, 1.0, 3.0, 2.0, -1.0])
    check(route(far, ladder, 6), definition(far, ladder, 6))


@gpu
@pytest.mark.parametrize("tokens", [6, 800])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("taken_out", [[], [3], [3, 7]])
def test_scores_that_are_no_numbers_come_first_where_asked_for(cuda_device, tokens, sigmoid, normalise, taken_out):
    """nan_first: a token with a NaN, one with an infinity (whose softmax is NaN), and an expert whose row holds a NaN; an expert that is taken
    out stays out.  The other tokens' ids and weights are those of the call without it."""
    x, w = operands(tokens, 12, 64, torch.bfloat16, torch.float32)
    x[2, 5], x[4, 9] = float("nan"), float("inf")
    bias = torch.zeros(12, device="cuda")
    bias[taken_out] = -math.inf
    for broken in (None, 7):
        if broken is not None:
            w[broken, 3] = float("nan")
        logits = x.double() @ w.double().t()
        out, nan = torch.isneginf(bias), torch.isnan(logits)
        score = 1 / (1 + torch.exp(-logits)) if sigmoid else torch.softmax(logits.masked_fill(out | nan, -math.inf), dim=1)
        score = score.masked_fill(nan, float("nan"))
        key = torch.where(torch.isnan(score), torch.full_like(score, 9.0), score).masked_fill(out, -math.inf)
        ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :4]
        p = score.gather(1, ids)
        p = p / p.sum(dim=1, keepdim=True) if normalise else p
        desc = kb.make_route_desc(tokens, 12, 64, 4, kb.BF16, normalise=normalise, nan_first=True, score=kb.SCORE_SIGMOID if sigmoid else kb.SCORE_SOFTMAX)
        weights, names = torch.full((tokens, 4), -7.0, device="cuda"), torch.full((tokens, 4), -7, dtype=torch.int32, device="cuda")
        kb.route(desc, x, w, weights, names, bias)
        assert torch.equal(names, ids.int())
        assert torch.equal(torch.isnan(weights), torch.isnan(p)) and bool(torch.isnan(weights[2]).any())
        there = ~torch.isnan(p)
        assert torch.all((weights.double() - p)[there].abs() <= (2.0 ** -24 + 2.0 ** -40) * p[there].abs() + 2.0 ** -149)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 0), (2, 3), (4, 4), (3, 1)])
def test_pitch_and_alignment(cuda_device, dtype, offset, extra):
    x0, w0 = operands(9, 20, 301, dtype, dtype)

    def moved(t):
        ld = t.shape[1] + extra
        store = torch.full((offset + t.shape[0] * ld,), float("nan"), dtype=t.dtype, device="cuda")
        view = store[offset:].view(t.shape[0], ld)[:, :t.shape[1]]
        view.copy_(t)
        return view

    check(route(moved(x0), moved(w0), 5), definition(x0, w0, 5))


@gpu
def test_streams_graphs_and_no_tokens(cuda_device):
    x, w = operands(17, 64, 1024, torch.bfloat16, torch.float32)
    other, _ = operands(17, 64, 1024, torch.bfloat16, torch.float32, seed=4)
    want = [route(t, w, 8) for t in (x, other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for t, s in zip((x, other), streams):
            with torch.cuda.stream(s):
                got.append(route(t, w, 8, stream=s.cuda_stream))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, v in zip(got, want) for a, b in zip(g, v))
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = route(held, w, 8, stream=torch.cuda.current_stream().cuda_stream)
    held.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[1]))
    assert route(x[:0], w, 8)[0].shape == (0, 8)


def desc(**more):
    return kb.make_route_desc(more.pop("tokens", 2), more.pop("experts", 8), more.pop("hidden", 16), more.pop("top", 2), more.pop("dtype", kb.BF16), **more)


@pytest.mark.parametrize("d,status", [
    (desc(tokens=-1), 2), (desc(hidden=0), 1), (desc(hidden=2 ** 31), 1), (desc(tokens=2 ** 30), 1), (desc(experts=0), 1), (desc(experts=1025), 1),
    (desc(top=0), 2), (desc(top=9), 2), (desc(experts=100, top=65), 1), (desc(dtype=kb.E4M3), 1), (desc(router_dtype=kb.S8), 1), (desc(score=2), 1),
    (desc(scale=float("nan")), 2), (desc(x_ld=-1), 2),
])
def test_descriptors_that_are_refused(d, status):
    with pytest.raises(kb.KudnnError) as e:
        kb.route(d, 16, 16, 16, 16)
    assert e.value.status == status


@pytest.mark.parametrize("place,wrong", [(place, wrong) for place in range(5) for wrong in (None, 17) if (place, wrong) != (4, None)])
def test_calls_that_are_refused(place, wrong):
    """On the host, ahead of any device: the addresses are made up."""
    operands = [16] * 5
    operands[place] = wrong
    with pytest.raises(kb.KudnnError) as e:
        kb.route(desc(), *operands)
    assert e.value.status == 2


def test_the_longest_rows():
    """Steps of up to 2048 elements are taken while they end within a row, in 32 bits: rows that such a sum could pass 2^31 for are refused."""
    for hidden, status in ((2 ** 31 - 1025, 1), (2 ** 31 - 2049, 1), (2 ** 31 - 4096, 1), (2 ** 31 - 4097, 2)):
        with pytest.raises(kb.KudnnError) as e:
            kb.route(desc(hidden=hidden), None, 16, 16, 16)
        assert e.value.status == status


@gpu
@pytest.mark.parametrize("tokens", [768, 769, 2000])
@pytest.mark.parametrize("experts,top", [(1, 1), (8, 2), (16, 4), (32, 8), (96, 6)])
def test_prompts_with_few_experts(cuda_device, tokens, experts, top):
    x, w = operands(tokens, experts, 264, torch.bfloat16, torch.float32)
    check(route(x, w, top), definition(x, w, top))
