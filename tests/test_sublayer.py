"""The torch operators layernorm, route and experts and their modules, alone and together as a decoder's sublayer x + experts(layernorm(x))."""
import pytest
import torch

import kudnn_b200 as kb
from kudnn_b200 import torch_ops
from tests.test_experts import experts64

ops = torch.ops.kudnn_b200
gpu = pytest.mark.gpu


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_fake_implementations_propagate_shapes_without_a_device():
    y, mean, variance = ops.layernorm(meta(2, 5, 300), meta(300), meta(300))
    assert y.shape == (2, 5, 300) and y.dtype == torch.bfloat16 and mean.shape == variance.shape == (2, 5) and mean.dtype == torch.float32
    dx, dscale, dshift = ops.layernorm_backward(meta(5, 300), meta(5, 300), None, meta(5), meta(5), 1e-5, torch.float32)
    assert dx.shape == (5, 300) and dscale.shape == dshift.shape == (300,) and dscale.dtype == torch.float32
    weights, ids = ops.route(meta(5, 300), meta(8, 300, dtype=torch.float32), 3)
    assert weights.shape == ids.shape == (5, 3) and weights.dtype == torch.float32 and ids.dtype == torch.int32
    assert ops.experts(meta(5, 300), weights, ids, meta(8, 400, 300), meta(8, 300, 200)).shape == (5, 300)


def block(eight_bit, few, hidden=512, ffn=384, count=16, top=4, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    router = torch.randn(count, hidden, generator=gen, device="cuda") * 0.1
    gate_up = (torch.randn(count, 2 * ffn, hidden, generator=gen, device="cuda") * hidden ** -0.5).to(dtype)
    down = (torch.randn(count, hidden, ffn, generator=gen, device="cuda") * ffn ** -0.5).to(dtype)
    return torch_ops.Experts(router, gate_up, down, top, eight_bit=eight_bit, few=few), (router, gate_up, down, top)


@pytest.mark.parametrize("wrong", [
    dict(dy=torch.zeros(5, 300, dtype=torch.bfloat16)), dict(mean=torch.zeros(5)), dict(variance=torch.zeros(5)), dict(scale=torch.zeros(300)),
    dict(x=torch.zeros(5, 300, dtype=torch.bfloat16)), dict(param_dtype=torch.float16), dict(param_dtype=torch.int32), dict(dy=meta(5, 299)),
    dict(mean=meta(5)), dict(scale=meta(300)),
])
def test_gradients_across_devices_or_types_are_refused_before_any_launch(wrong):
    """The operator's own body, with tensors that have no memory: a host address must not reach a kernel."""
    given = dict(dy=meta(5, 300), x=meta(5, 300), scale=None, mean=meta(5, dtype=torch.float32), variance=meta(5, dtype=torch.float32), eps=1e-5,
                 param_dtype=torch.float32)
    with pytest.raises(ValueError, match="layernorm"):
        torch_ops.layernorm_backward._init_fn(**{**given, **wrong})


@pytest.mark.parametrize("more", [dict(few=65), dict(few=-1), dict(few=4, top=17)])
def test_experts_refuse_more_tokens_than_the_kernels_take(more):
    with pytest.raises(ValueError):
        torch_ops.Experts(meta(20, 64, dtype=torch.float32), meta(20, 64, 64), meta(20, 64, 32), more.get("top", 2), few=more["few"])


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("shape", [(0, 300), (3, 300), (5, 300)])
def test_shapes_on_either_side_of_few(eight_bit, shape):
    experts = torch_ops.Experts(meta(6, 300, dtype=torch.float32), meta(6, 400, 300), meta(6, 300, 200), 2, eight_bit=eight_bit, few=3)
    y = experts(meta(*shape))
    assert y.shape == shape and y.dtype == torch.bfloat16


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("tokens", [0, 3])
def test_a_module_without_few_keeps_to_the_way_of_many(eight_bit, tokens):
    """Not even no tokens go to the kernels for few: without `few` any top is allowed, also one that those refuse."""
    from torch.utils._python_dispatch import TorchDispatchMode

    called = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            called.append(func.name())
            return func(*args, **(kwargs or {}))

    experts = torch_ops.Experts(meta(20, 300, dtype=torch.float32), meta(20, 400, 300), meta(20, 300, 200), 17, eight_bit=eight_bit)
    with Record():
        y = experts(meta(tokens, 300))
    assert y.shape == (tokens, 300) and "kudnn_b200::grouped" in called
    assert "kudnn_b200::route" not in called and "kudnn_b200::experts" not in called


@gpu
@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("few,top", [(0, 17), (8, 4)])
def test_no_tokens(cuda_device, eight_bit, few, top):
    experts, _ = block(eight_bit, few, count=20, top=top)
    y = experts(torch.empty((2, 0, 512), dtype=torch.bfloat16, device="cuda"))
    assert y.shape == (2, 0, 512) and y.dtype == torch.bfloat16


@gpu
@pytest.mark.parametrize("tokens", [1, 7, 64, 65])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_experts_of_few_tokens(cuda_device, tokens, eight_bit):
    """Norm of the error over the norm of the result: 2^-9 for the rounding of 16-bit results, and for e4m3 weights 2^-4 / sqrt(3) for each of two
    products' weights, the first one's error with a slope of up to 1.1 in both gate and up: 3.6 % (1.1^2 + 1 + 1)^(1/2) = 6.5 %.  65 tokens take
    the way of many, whose limits are 2^-7 and 9.4 %."""
    experts, parts = block(eight_bit, 64)
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(1, tokens, 512, generator=gen, device="cuda").bfloat16()
    y, want = experts(x), experts64(x, *parts)
    off = torch.linalg.vector_norm(y.double() - want) / torch.linalg.vector_norm(want)
    assert y.shape == x.shape and y.dtype == x.dtype
    assert off <= ((0.094 if eight_bit else 2.0 ** -7) if tokens > 64 else 0.065 if eight_bit else 2.0 ** -9)
    assert torch.equal(experts(x), y)


@gpu
def test_many_tokens_and_few_of_zero_take_the_way_they_took(cuda_device):
    few, _ = block(True, 8)
    plain, _ = block(True, 0)
    x = torch.randn(24, 512, device="cuda").bfloat16()
    assert torch.equal(few(x), plain(x))
    assert torch.equal(few(x[:4].float()), plain(x[:4].float()))  # tokens of 32 bits are not of the kernels' types


@gpu
@pytest.mark.parametrize("eight_bit", [False, True])
def test_tokens_whose_scores_are_no_numbers_stay_visible_either_way(cuda_device, eight_bit):
    """A token with a NaN or an infinity has a softmax of NaN, and so its answer is NaN, by the kernels for few tokens as by those for many; the
    others are as without it but for their rounding, twice 2^-8: with other experts chosen the weights are cut elsewhere, and sums are taken in
    another order.  A router that holds a NaN has no softmax for any token."""
    few, _ = block(eight_bit, 64)
    many, _ = block(eight_bit, 0)
    x = torch.randn(6, 512, device="cuda").bfloat16()
    clean = few(x)
    x[1, 5], x[4, 300] = float("nan"), float("inf")
    bad = torch.tensor([False, True, False, False, True, False], device="cuda")
    for experts in (few, many):
        y = experts(x)
        assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all())
    got, want = few(x)[~bad].double(), clean[~bad].double()
    assert torch.linalg.vector_norm(got - want) <= 2.0 ** -7 * torch.linalg.vector_norm(want)
    for experts in (few, many):
        experts.router[3, 17] = float("nan")
        assert bool(torch.isnan(experts(x)).all())


@gpu
@pytest.mark.parametrize("eight_bit", [False, True])
def test_a_sublayer(cuda_device, eight_bit):
    """x + experts(layernorm(x)) of one to 64 tokens, eager and captured; against 64 bits on the normalised rows as they were rounded."""
    experts, parts = block(eight_bit, 64, hidden=768, ffn=320)
    norm = torch_ops.LayerNorm(768, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        norm.inner.weight.normal_(1.0, 0.1)
        norm.inner.bias.normal_(0.0, 0.1)
        for tokens in (1, 5, 64):
            x = torch.randn(tokens, 768, device="cuda").bfloat16()
            z = norm(x)
            exact = torch.nn.functional.layer_norm(x.double(), (768,), norm.inner.weight.double(), norm.inner.bias.double(), norm.inner.eps)
            assert torch.all((z.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 1e-5)
            y, want = x + experts(z), x.double() + experts64(z, *parts)
            off = torch.linalg.vector_norm(y.double() - want) / torch.linalg.vector_norm(want)
            assert off <= (0.065 if eight_bit else 2.0 ** -8)
            held, other = x.clone(), torch.randn(tokens, 768, device="cuda").bfloat16()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                experts(norm(held))
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = held + experts(norm(held))
            for t in (other, x):
                held.copy_(t)
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, t + experts(norm(t)))


@gpu
@pytest.mark.parametrize("dtype,kind", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("shape", [(3, 40, 130), (65, 1024), (7,), (2, 0, 12)])
def test_gradients_of_the_module(cuda_device, dtype, kind, shape):
    """Against torch's in 64 bits: results and gradients of 16 bits are rounded once (2^-8, 2^-11), and 10^-5 of the largest for sums in fp32."""
    norm = torch_ops.LayerNorm(shape[-1], device="cuda", dtype=kind)
    with torch.no_grad():
        norm.inner.weight.normal_(1.0, 0.2)
        norm.inner.bias.normal_(0.0, 0.2)
    x = (torch.randn(shape, device="cuda") * 2 + 1).to(dtype).requires_grad_()
    dy = torch.randn(shape, device="cuda").to(dtype)
    norm(x).backward(dy)
    x64, w64, b64 = [t.detach().double().requires_grad_() for t in (x, norm.inner.weight, norm.inner.bias)]
    torch.nn.functional.layer_norm(x64, shape[-1:], w64, b64, norm.inner.eps).backward(dy.double())
    for got, want in ((x.grad, x64.grad), (norm.inner.weight.grad, w64.grad), (norm.inner.bias.grad, b64.grad)):
        most = float(want.abs().max()) if want.numel() else 0.0
        assert got.shape == want.shape and torch.all((got.double() - want).abs() <= torch.finfo(got.dtype).eps / 2 * want.abs() + 1e-5 * most)


@gpu
def test_what_takes_no_gradient(cuda_device):
    x = torch.randn(5, 64, device="cuda", requires_grad=True)
    y, mean, variance = ops.layernorm(x)
    assert y.requires_grad and not mean.requires_grad and not variance.requires_grad
    y.sum().backward()
    assert float(x.grad.abs().max()) <= 1e-5  # the rows' sums do not depend on x
    plain = torch.nn.LayerNorm(64, elementwise_affine=False, device="cuda")
    assert torch.allclose(torch_ops.LayerNorm.from_torch(plain)(x), plain(x), atol=1e-5)
    with pytest.raises(ValueError):
        torch_ops.LayerNorm.from_torch(torch.nn.LayerNorm((4, 64)))


@gpu
def test_a_captured_training_step(cuda_device):
    """Forward and backward in one graph, after eager passes whose graphs are gone."""
    norm = torch_ops.LayerNorm(520, device="cuda")
    x = torch.randn(33, 520, device="cuda")
    dy = torch.randn(33, 520, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            norm.zero_grad(set_to_none=True)
            norm(x).backward(dy)
    torch.cuda.current_stream().wait_stream(side)
    want = norm.inner.weight.grad.clone()
    norm.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm(x).backward(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm.inner.weight.grad, want)


@gpu
@pytest.mark.parametrize("wrong", [
    lambda x, r, p, i, u, d: ops.layernorm(x.double()), lambda x, r, p, i, u, d: ops.layernorm(x, r[0, :32]), lambda x, r, p, i, u, d: ops.layernorm(x, x[0].half()),
    lambda x, r, p, i, u, d: ops.layernorm(x, r[0], x[0]), lambda x, r, p, i, u, d: ops.layernorm(x, r[0].cpu()),
    lambda x, r, p, i, u, d: ops.route(x, r[:, :32], 2), lambda x, r, p, i, u, d: ops.route(x, r, 2, r[:, 0].half()), lambda x, r, p, i, u, d: ops.route(x[0], r, 2),
    lambda x, r, p, i, u, d: ops.route(x, r, 2, None, "other"), lambda x, r, p, i, u, d: ops.route(x, r.cpu(), 2), lambda x, r, p, i, u, d: ops.route(x, r, 9),
    lambda x, r, p, i, u, d: ops.route(x, r, 0), lambda x, r, p, i, u, d: ops.experts(x.float(), p, i, u, d), lambda x, r, p, i, u, d: ops.experts(x, p.half(), i, u, d),
    lambda x, r, p, i, u, d: ops.experts(x, p, i.long(), u, d), lambda x, r, p, i, u, d: ops.experts(x, p[:, :1], i, u, d),
    lambda x, r, p, i, u, d: ops.experts(x, p, i, u, d.half()), lambda x, r, p, i, u, d: ops.experts(x, p, i, u[:, :-2], d),
    lambda x, r, p, i, u, d: ops.experts(x, p, i, u, d, r, r), lambda x, r, p, i, u, d: ops.experts(x, p, i, u.to(torch.float8_e4m3fn), d.to(torch.float8_e4m3fn)),
    lambda x, r, p, i, u, d: ops.experts(x, p.cpu(), i, u, d),
    lambda x, r, p, i, u, d: ops.experts(x.repeat(20, 1), p.repeat(20, 1), i.repeat(20, 1), u, d),
])
def test_refusals(cuda_device, wrong):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    r = torch.zeros(8, 64, device="cuda")
    u, d = torch.zeros(8, 64, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 64, 32, dtype=torch.bfloat16, device="cuda")
    with pytest.raises((TypeError, ValueError, kb.KudnnError)):
        wrong(x, r, torch.ones(4, 2, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), u, d)


@gpu
def test_a_wait_that_runs_out_is_reported(cuda_device):
    """No weights are copied from the second step of K on: the waits give up after a moment, both kernels end, and the next call is right again."""
    experts, _ = block(False, 64)
    x = torch.randn(3, 512, device="cuda").bfloat16()
    want = experts(x)
    torch.cuda.synchronize()
    kb.experts_check()
    kb.experts_set_wait(2000000, 1)
    try:
        experts(x)
        with pytest.raises(kb.KudnnError) as e:
            kb.experts_check(torch.cuda.current_stream().cuda_stream)
        assert e.value.status == 5
    finally:
        kb.experts_set_wait()
    assert torch.equal(experts(x), want)
    kb.experts_check(torch.cuda.current_stream().cuda_stream)


@gpu
def test_no_thread_takes_a_report_from_another(cuda_device):
    """Two threads whose waits ran out: each learns of it, once, whichever looks first."""
    import threading

    experts, _ = block(False, 64)
    x = torch.randn(3, 512, device="cuda").bfloat16()
    ran, looked, seen = threading.Barrier(2), threading.Barrier(2), {}

    def work(name):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            experts(x)
            stream.synchronize()
            ran.wait(60)
            for turn in range(2):
                if name == "second":
                    looked.wait(60)
                try:
                    kb.experts_check(stream.cuda_stream)
                    seen[name, turn] = 0
                except kb.KudnnError as e:
                    seen[name, turn] = e.status
                if name == "first":
                    looked.wait(60)

    torch.cuda.synchronize()
    kb.experts_set_wait(2000000, 1)
    try:
        threads = [threading.Thread(target=work, args=(name,)) for name in ("first", "second")]
        for t in threads:
            t.start()
        for t in threads:
            t.join(120)
    finally:
        kb.experts_set_wait()
    assert seen == {("first", 0): 5, ("first", 1): 0, ("second", 0): 5, ("second", 1): 0}
    with pytest.raises(kb.KudnnError):
        kb.experts_check()
    kb.experts_check()


@gpu
@pytest.mark.parametrize("dtype,kind", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
def test_operators_of_layer_normalisation_meet_the_contract_of_custom_operators(cuda_device, dtype, kind):
    x, w, b = torch.randn(3, 5, 72, device="cuda").to(dtype), torch.randn(72, device="cuda").to(kind), torch.randn(72, device="cuda").to(kind)
    _, mean, variance = ops.layernorm(x, w, b)
    torch.library.opcheck(ops.layernorm.default, [t.clone().requires_grad_() for t in (x, w, b)] + [1e-5])
    torch.library.opcheck(ops.layernorm.default, (x.transpose(0, 1)[..., :-1], None, b[:-1], 1e-5))
    torch.library.opcheck(ops.layernorm_backward.default, (torch.randn_like(x), x, w, mean, variance, 1e-5, kind))


@gpu
def test_operators_of_experts_meet_the_contract_of_custom_operators(cuda_device):
    x, r = torch.randn(5, 64, device="cuda").bfloat16(), torch.randn(8, 64, device="cuda")
    u, d = torch.randn(8, 64, 64, device="cuda").bfloat16(), torch.randn(8, 64, 32, device="cuda").bfloat16()
    torch.library.opcheck(ops.route.default, (x, r, 3, None, "sigmoid", False, 2.0, True))
    p, ids = ops.route(x, r, 3)
    for t in (x, torch.randn(64, 5, device="cuda").bfloat16().t()):
        torch.library.opcheck(ops.experts.default, (t, p, ids, u, d))


@gpu
@pytest.mark.parametrize("eight_bit", [False, True])
def test_a_sublayer_traces_as_one_graph(cuda_device, eight_bit):
    experts, _ = block(eight_bit, 64)
    norm = torch_ops.LayerNorm(512, device="cuda", dtype=torch.bfloat16)

    def run(x):
        return x + experts(norm(x))

    with torch.no_grad():
        for tokens in (1, 5, 64):
            x = torch.randn(tokens, 512, device="cuda").bfloat16()
            assert torch.equal(torch.compile(run, backend="aot_eager", fullgraph=True)(x), run(x))


@gpu
@pytest.mark.parametrize("frozen", range(7))
def test_gradients_beside_frozen_tensors(cuda_device, frozen):
    """Bit i of `frozen`: x, the scale, the shift take no gradient; the others' are those of the call with all three."""
    made = [torch.randn(7, 40, device="cuda"), torch.randn(40, device="cuda"), torch.randn(40, device="cuda")]
    dy = torch.randn(7, 40, device="cuda")
    every = [t.clone().requires_grad_() for t in made]
    some = [t.clone().requires_grad_((frozen >> i & 1) == 0) for i, t in enumerate(made)]
    for tensors in (every, some):
        ops.layernorm(*tensors)[0].backward(dy)
    for i, (a, b) in enumerate(zip(every, some)):
        assert b.grad is None if (frozen >> i & 1) != 0 else torch.equal(a.grad, b.grad)
