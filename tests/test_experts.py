"""The torch operators kudnn_b200::quantize and ::grouped, and the feed-forward block of experts that runs them together."""
import collections
import types

import pytest
import torch

import kudnn_b200 as kb
from kudnn_b200 import torch_ops

ops = torch.ops.kudnn_b200
gpu = pytest.mark.gpu


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_fake_implementations_propagate_shapes_without_a_device():
    q, s = ops.quantize(meta(5, 300))
    assert q.shape == (5, 300) and q.dtype == torch.float8_e4m3fn and q.stride() == (304, 1)
    assert s.shape == (5, 3) and s.dtype == torch.float32 and s.stride() == (1, 5)
    q, s = ops.quantize(meta(5, 600), True, meta(9, dtype=torch.int32))
    assert q.shape == (9, 300) and s.shape == (9, 3)
    q, s = ops.quantize(meta(200, 300), block_rows=128)
    assert q.shape == (200, 300) and s.shape == (2, 3) and s.stride() == (3, 1)
    e = meta(7, 300, dtype=torch.float8_e4m3fn)
    assert ops.grouped(e, meta(4, 64, 300, dtype=torch.float8_e4m3fn)).dtype == torch.bfloat16
    y = ops.grouped(meta(7, 300), meta(4, 64, 300), out_dtype=torch.float32)
    assert y.shape == (7, 64) and y.dtype == torch.float32


@pytest.fixture
def bfloat16_by_default():
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    yield
    torch.set_default_dtype(before)


@pytest.mark.parametrize("more", [dict(), dict(block_rows=128)])
def test_scales_hold_32_bits_whatever_the_default_type(bfloat16_by_default, monkeypatch, more):
    """On the host: what the operator hands to the library, whose kernel writes 4 bytes per scale."""
    got = {}

    class _Nothing:
        cuda_stream = 0

        def __init__(self, *args):
            pass

        def __enter__(self):
            return self

        def __exit__(self, *args):
            pass

    monkeypatch.setattr(torch_ops, "_on", _Nothing)
    monkeypatch.setattr(torch.cuda, "current_stream", _Nothing)
    monkeypatch.setattr(torch_ops.capi, "quantize", lambda desc, x, q, scale, index, stream: got.update(desc=desc, q=q, scale=scale))
    x = torch.zeros(200, 300)
    q, scale = torch_ops.quantize._init_fn(x, **more)
    fake = ops.quantize(meta(200, 300), **more)
    assert got["scale"] is scale and scale.dtype == torch.float32 and scale.numel() * 4 <= scale.untyped_storage().nbytes()
    for own, other in zip((q, scale), fake):
        assert (own.dtype, own.shape, own.stride()) == (other.dtype, other.shape, other.stride())
    assert got["desc"].s_row == scale.stride(0) and got["desc"].s_col == scale.stride(1) and got["desc"].q_ld == q.stride(0)


@gpu
def test_quantize_under_another_default_type(cuda_device, bfloat16_by_default):
    x = torch.randn(37, 520, device="cuda", dtype=torch.float32)
    for block_rows in (1, 128):
        made = torch_ops._quantized(x, 37, 520, block_rows)[1]
        assert made.dtype == torch.float32 and made.untyped_storage().nbytes() == 4 * made.numel()  # before anything is launched
        q, scale = ops.quantize(x, block_rows=block_rows)
        torch.set_default_dtype(torch.float32)
        q2, scale2 = ops.quantize(x, block_rows=block_rows)
        torch.set_default_dtype(torch.bfloat16)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale, scale2)


class _Recorded:
    def __init__(self, desc):
        self.closed = False

    def close(self):
        self.closed = True


def test_created_products_are_bounded_and_captured_ones_stay(monkeypatch):
    capturing = [False]
    monkeypatch.setattr(torch_ops.capi, "Grouped", _Recorded)
    monkeypatch.setattr(torch_ops, "_GROUPED", collections.OrderedDict())
    monkeypatch.setattr(torch_ops, "_MAX_GROUPED", 3)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    cuda = torch.device("cuda", 0)

    def handle(key):
        return torch_ops._grouped_handle(cuda, key, lambda: None)

    capturing[0] = True
    first = handle("a")
    capturing[0] = False
    second = handle("b")
    assert handle("a") is first and handle("b") is second
    for key in "cdefg":
        handle(key)
        assert len(torch_ops._GROUPED) == 3
    assert handle("a") is first and handle("b") is not second
    torch_ops.clear_cache()
    assert first.closed and not torch_ops._GROUPED


def test_dropped_primitives_are_destroyed_without_the_lock(monkeypatch):
    """Destroying one waits for the device, and the lock holds up the calls of all other threads."""
    locked = []

    class Watched:
        def __init__(self, desc):
            self.graphs = 0

        def prepack(self, b, stream=None):
            pass

        def close(self):
            locked.append(torch_ops._LOCK.locked())

        __del__ = close

    for name in ("Grouped", "Linear"):
        monkeypatch.setattr(torch_ops.capi, name, Watched)
    for name in ("_GROUPED", "_HANDLES"):
        monkeypatch.setattr(torch_ops, name, collections.OrderedDict())
    monkeypatch.setattr(torch_ops, "_MAX_GROUPED", 2)
    monkeypatch.setattr(torch_ops, "_MAX_HANDLES", 2)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=1))
    weight = torch.zeros(8, 16)
    for m in range(1, 5):
        torch_ops._grouped_handle(torch.device("cuda", 0), m, lambda: None)
        torch_ops._handle(m, 8, 16, torch.zeros(m, 16), weight, None, 0, 1.0, None, 0)
    assert locked == [False] * 4
    torch_ops.clear_cache()
    assert not torch_ops._GROUPED and not torch_ops._HANDLES and len(locked) >= 8 and not any(locked)


@gpu
def test_operators_against_their_definition(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(37, 520, generator=gen, device="cuda").bfloat16()
    w = torch.randn(3, 264, 520, generator=gen, device="cuda").bfloat16() * 0.05
    bias = torch.randn(3, 264, generator=gen, device="cuda")
    offsets = torch.tensor([0, 10, 10, 37], device="cuda")
    y = ops.grouped(x, w, offsets, bias=bias, act=kb.ACT_RELU, act_alpha=0.0, out_dtype=torch.float32)
    for g, (lo, hi) in enumerate(((0, 10), (10, 10), (10, 37))):
        want = torch.relu(x[lo:hi].double() @ w[g].double().t() + bias[g].double())
        limit = (520 / 8 + 8) * 2.0 ** -23 * (x[lo:hi].double().abs() @ w[g].double().abs().t() + bias[g].double().abs())
        assert torch.all((y[lo:hi].double() - want).abs() <= limit)
    # 8-bit operands of the quantiser's own making, dense
    q, s = ops.quantize(x)
    qw, sw = ops.quantize(w[0], block_rows=128)
    y = ops.grouped(q, qw, None, s, sw, out_dtype=torch.float32)
    a = q.double() * s.double().repeat_interleave(128, 1)[:, :520]
    b = qw.double() * sw.double().repeat_interleave(128, 0)[:264].repeat_interleave(128, 1)[:, :520]
    assert torch.all((y.double() - a @ b.t()).abs() <= (520 / 8 + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t()))
    # views: rows at a pitch, transposed weights, no rows
    wide = torch.randn(37, 600, generator=gen, device="cuda").bfloat16()
    t = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.allclose(ops.grouped(wide[:, :520], t, offsets).float(), ops.grouped(wide[:, :520].contiguous(), w, offsets).float(), atol=2e-2, rtol=2e-2)
    assert ops.grouped(x[:0], w, torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 264)
    assert ops.quantize(x[:0])[0].shape == (0, 520)


@gpu
@pytest.mark.parametrize("wrong", [
    lambda x, w, o: ops.grouped(x.float(), w.float(), o), lambda x, w, o: ops.grouped(x, w.half(), o), lambda x, w, o: ops.grouped(x, w[:, :, :-8], o),
    lambda x, w, o: ops.grouped(x, w, None), lambda x, w, o: ops.grouped(x, w, o[:-1]), lambda x, w, o: ops.grouped(x, w, o.float()),
    lambda x, w, o: ops.grouped(x, w, o.cpu()), lambda x, w, o: ops.grouped(x, w, o, x_scale=torch.ones(4, 1, device="cuda")),
    lambda x, w, o: ops.grouped(x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn), o),
    lambda x, w, o: ops.grouped(x, w, o, bias=torch.ones(64, device="cuda")), lambda x, w, o: ops.grouped(x, w, o, out_dtype=torch.float64),
    lambda x, w, o: ops.quantize(x.double()), lambda x, w, o: ops.quantize(x[0]), lambda x, w, o: ops.quantize(x[:, :63], True),
    lambda x, w, o: ops.quantize(x, False, o.long()), lambda x, w, o: ops.quantize(x, block_rows=64), lambda x, w, o: ops.quantize(x, True, None, 128),
])
def test_refusals(cuda_device, wrong):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 64, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises((TypeError, ValueError)):
        wrong(x, w, torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda"))


def meta_experts(eight_bit, hidden=300, ffn=200, experts=6):
    return torch_ops.Experts(meta(experts, hidden, dtype=torch.float32), meta(experts, 2 * ffn, hidden), meta(experts, hidden, ffn), 2,
                             eight_bit=eight_bit)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("shape", [(0, 300), (2, 0, 300), (5, 300)])
def test_experts_propagate_shapes_of_any_number_of_tokens(eight_bit, shape):
    y = meta_experts(eight_bit)(meta(*shape))
    assert y.shape == shape and y.dtype == torch.bfloat16


MOVES = [lambda b: b.half(), lambda b: b.to(torch.bfloat16), lambda b: b.double(), lambda b: b.type(torch.float16)]


@pytest.mark.parametrize("move", MOVES)
def test_casts_of_the_experts_leave_8_bit_weights_scales_and_the_router(move):
    block = meta_experts(True)
    before = {name: (t.dtype, t.shape, t.stride()) for name, t in block.named_buffers()}
    assert before["down"] == (torch.float8_e4m3fn, (6, 300, 200), (300 * 208, 208, 1))
    move(block)
    assert {name: (t.dtype, t.shape, t.stride()) for name, t in block.named_buffers()} == before
    block = move(meta_experts(False))
    assert block.router.dtype == torch.float32 and block.down.dtype == block.gate_up.dtype != torch.float32


def experts64(x, router, gate_up, down, top):
    tokens = x.reshape(-1, x.shape[-1])
    p = torch.softmax(tokens.double() @ router.double().t(), dim=1)
    p, chosen = torch.topk(p, top, dim=1)
    p = p / p.sum(dim=1, keepdim=True)
    y = torch.zeros(tokens.shape, dtype=torch.float64, device=x.device)
    for e in range(router.shape[0]):
        t, slot = (chosen == e).nonzero(as_tuple=True)
        h = tokens[t].double() @ gate_up[e].double().t()
        gate, up = h.chunk(2, dim=1)
        y.index_add_(0, t, (torch.nn.functional.silu(gate) * up @ down[e].double().t()) * p[t, slot][:, None])
    return y.view(x.shape)


@gpu
@pytest.mark.parametrize("tokens", [1, 7, 300])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_experts(cuda_device, tokens, eight_bit):
    """Norm of the error over the norm of the result.  bf16: the values between the products, the gated ones, the second product and the sum
    are each rounded to 2^-9: 2^-7 in all.  8 bits: the two operands of either product are each off by 2^-4 at most, 3.6 % in the square mean;
    the first product's error (5.1 %) enters the gated value twice with a slope of up to 1.1, so 7.9 %, and with the second product's two
    operands 9.4 %."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    hidden, ffn, experts, top = 512, 384, 16, 4
    x = torch.randn(1, tokens, hidden, generator=gen, device="cuda").bfloat16()
    router = torch.randn(experts, hidden, generator=gen, device="cuda") * 0.1
    gate_up = (torch.randn(experts, 2 * ffn, hidden, generator=gen, device="cuda") * hidden ** -0.5).bfloat16()
    down = (torch.randn(experts, hidden, ffn, generator=gen, device="cuda") * ffn ** -0.5).bfloat16()
    block = torch_ops.Experts(router, gate_up, down, top, eight_bit=eight_bit)
    y = block(x)
    want = experts64(x, router, gate_up, down, top)
    assert y.shape == x.shape and y.dtype == x.dtype
    off = torch.linalg.vector_norm(y.double() - want) / torch.linalg.vector_norm(want)
    assert off <= (0.094 if eight_bit else 2.0 ** -7)
    assert torch.equal(block(x), y)


@gpu
@pytest.mark.parametrize("eight_bit", [False, True])
def test_experts_without_tokens(cuda_device, eight_bit):
    w = torch.ones(4, 64, 32, dtype=torch.bfloat16, device="cuda")
    block = torch_ops.Experts(torch.ones(4, 32, device="cuda"), w, w.transpose(1, 2)[:, :, :32].contiguous(), 2, eight_bit=eight_bit)
    assert block(torch.ones(3, 0, 32, dtype=torch.bfloat16, device="cuda")).shape == (3, 0, 32)


@gpu
def test_experts_keep_their_results_when_they_are_moved(cuda_device):
    gen = torch.Generator(device="cuda").manual_seed(2)
    gate_up = (torch.randn(6, 400, 300, generator=gen, device="cuda") * 0.05).bfloat16()
    down = (torch.randn(6, 300, 200, generator=gen, device="cuda") * 0.05).bfloat16()
    block = torch_ops.Experts(torch.randn(6, 300, generator=gen, device="cuda"), gate_up, down, 2, eight_bit=True)
    x = torch.randn(9, 300, generator=gen, device="cuda").bfloat16()
    want = block(x)
    for move in MOVES + [lambda b: b.cpu().to("cuda"), lambda b: b.to("cuda", torch.bfloat16)]:
        move(block)
        assert torch.equal(block(x), want)


@gpu
def test_experts_in_a_graph(cuda_device):
    """The sizes of the groups stay on the device: one captured graph serves other tokens."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    hidden, ffn, experts, top = 256, 256, 8, 2
    router = torch.randn(experts, hidden, generator=gen, device="cuda") * 0.2
    gate_up = (torch.randn(experts, 2 * ffn, hidden, generator=gen, device="cuda") * hidden ** -0.5).bfloat16()
    down = (torch.randn(experts, hidden, ffn, generator=gen, device="cuda") * ffn ** -0.5).bfloat16()
    block = torch_ops.Experts(router, gate_up, down, top, eight_bit=True)
    x = torch.randn(24, hidden, generator=gen, device="cuda").bfloat16()
    other = torch.randn(24, hidden, generator=gen, device="cuda").bfloat16()
    want = block(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x)
    x.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
