"""The block of experts for few tokens, against its definition in 64 bits.

Tolerances: a sum of K products in fp32 is off by at most b(K) = (K / 8 + 16) 2^-23 of the sum of their magnitudes (the tensor cores add 16 products
at a time and cut what lies below; 16 warps' sums follow).  gate and up are off by that; h by 1.1 |off gate| |up| (the slope of silu) +
|silu(gate)| |off up|, and by 2^-17 of it for its two 16-bit halves; y by what that and b(ffn) make of it through the absolute weights, times the
token's weight, 2^-20 for the sum over the experts, and by half a step of its type."""
import pytest
import torch

import kudnn_b200 as kb

CODE = {torch.float16: kb.F16, torch.bfloat16: kb.BF16, torch.float8_e4m3fn: kb.E4M3}
KINDS = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)]
gpu = pytest.mark.gpu


def b(k):
    return (k / 8 + 16) * 2.0 ** -23


def up_blocks(scale, n, k):
    return scale.repeat_interleave(128, dim=-2)[..., :n, :].repeat_interleave(128, dim=-1)[..., :k]


def to_e4m3(w):
    """e4m3 weights at a pitch of 16 bytes, NaN between the rows, and scales per 128 x 128."""
    groups, n, k = w.shape
    ld = -(-k // 16) * 16
    scale = torch.rand((groups, -(-n // 128), -(-k // 128)), device="cuda") + 0.5
    q = torch.full((groups, n, ld), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    q[:, :, :k] = (w.float() / up_blocks(scale, n, k)).to(torch.float8_e4m3fn)
    return q[:, :, :k], scale


class Block:
    """Operands of one call; wide: fp64 copies of the weights as the kernels understand them."""

    def __init__(self, tokens, experts, top, hidden, ffn, dtype, eight, seed=0, ids=None, loud=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.tokens, self.experts, self.top, self.hidden, self.ffn = tokens, experts, top, hidden, ffn
        self.x = (torch.randn((tokens, hidden), generator=gen, device="cuda") * loud).to(dtype)
        gate_up = (torch.randn((experts, 2 * ffn, hidden), generator=gen, device="cuda") * hidden ** -0.5).to(dtype)
        down = (torch.randn((experts, hidden, ffn), generator=gen, device="cuda") * ffn ** -0.5).to(dtype)
        self.scales = (None, None)
        if eight:
            (gate_up, s0), (down, s1) = to_e4m3(gate_up), to_e4m3(down)
            self.scales = (s0, s1)
        self.gate_up, self.down = gate_up, down
        if ids is None:
            ids = torch.rand((tokens, experts), generator=gen, device="cuda").argsort(dim=1)[:, :top].int()
        self.ids = ids.contiguous()
        self.p = torch.rand((tokens, top), generator=gen, device="cuda") + 0.1

    def wide(self, which, e):
        w, scale = ((self.gate_up, self.scales[0]), (self.down, self.scales[1]))[which]
        v = w[e].double()
        return v if scale is None else v * up_blocks(scale[e].double(), *v.shape)

    def run(self, x=None, y=None, stream=None, workspace=None):
        x = self.x if x is None else x
        y = torch.full((self.tokens, self.hidden), -7.0, dtype=x.dtype, device="cuda") if y is None else y
        strides = [None if s is None else s.stride() for s in self.scales]
        desc = kb.make_experts_desc(self.tokens, self.hidden, self.ffn, self.experts, self.top, CODE[x.dtype], weight_dtype=CODE[self.gate_up.dtype],
                                    x_ld=x.stride(0), y_ld=y.stride(0), gate_up_strides=self.gate_up.stride(), down_strides=self.down.stride(),
                                    gate_up_scale_strides=strides[0], down_scale_strides=strides[1])
        size = kb.experts_workspace(desc)
        space = torch.full((max(size, 4) // 4 + 8,), float("nan"), device="cuda") if workspace is None else workspace
        kb.experts(desc, x, self.p, self.ids, self.gate_up, self.down, y, space, size, *self.scales, stream=stream)
        if workspace is None:
            assert bool(torch.isnan(space[size // 4:]).all()), "written beyond the workspace"
        return y

    def definition(self):
        """y and by how much a result may be off."""
        x = self.x.double()
        y, off = [torch.zeros((self.tokens, self.hidden), dtype=torch.float64, device="cuda") for _ in range(2)]
        size = torch.zeros_like(y)
        for e in sorted(set(self.ids.reshape(-1).tolist())):
            if not 0 <= e < self.experts:
                continue
            here = self.ids == e
            t = here.any(dim=1).nonzero()[:, 0]
            p = (self.p.double() * here).sum(dim=1)[t][:, None]
            w, d = self.wide(0, e), self.wide(1, e)
            both, around = x[t] @ w.t(), b(self.hidden) * (x[t].abs() @ w.abs().t())
            gate, up = both.chunk(2, dim=1)
            off_gate, off_up = around.chunk(2, dim=1)
            silu = torch.nn.functional.silu(gate)
            h = silu * up
            off_h = 1.1 * off_gate * (up.abs() + off_up) + silu.abs() * off_up + (2.0 ** -17 + 2.0 ** -21) * h.abs()
            y.index_add_(0, t, p * (h @ d.t()))
            off.index_add_(0, t, p.abs() * ((off_h + b(self.ffn) * (h.abs() + off_h)) @ d.abs().t()))
            size.index_add_(0, t, p.abs() * (h @ d.t()).abs())
        info = torch.finfo(self.x.dtype)
        return y, off + 2.0 ** -20 * size + (info.eps / 2) * (1 + 2 ** -10) * (y.abs() + off) + info.tiny * info.eps / 2

    def check(self, got=None):
        got = self.run() if got is None else got
        y, off = self.definition()
        assert torch.all((got.double() - y).abs() <= off), float(((got.double() - y).abs() / off).max())


# tokens, experts, top, hidden, ffn
SIZES = [(1, 1, 1, 8, 8), (1, 4, 2, 64, 32), (2, 3, 3, 16, 1), (3, 8, 2, 40, 24), (5, 6, 2, 300, 200), (1, 8, 8, 1024, 704), (8, 8, 2, 2048, 136),
         (9, 16, 4, 512, 384), (17, 16, 3, 301, 203), (33, 32, 8, 1024, 352), (64, 8, 2, 520, 136), (64, 60, 6, 640, 1408), (2, 128, 8, 4096, 256),
         (64, 1, 1, 256, 2048), (40, 200, 16, 128, 64), (12, 4, 2, 5120, 96), (4, 1000, 16, 64, 72),
         (35, 3, 2, 9536, 16), (3, 2, 1, 4784, 24), (64, 5, 3, 2376, 40), (9, 2, 2, 2360, 64)]


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(cuda_device, dtype, eight, size):
    block = Block(*size, dtype, eight)
    got = block.run()
    block.check(got)
    assert torch.equal(block.run(), got)


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_tokens_and_places_without_experts(cuda_device, dtype, eight):
    """ids outside of the experts take no part, whatever their weights; tokens without any get zeros; experts that nobody chose are not read."""
    ids = torch.tensor([[3, -1, 5], [-1, -1, -1], [0, 5, 3], [8, 2 ** 31 - 1, -2 ** 31], [5, 3, 9]], dtype=torch.int32, device="cuda")
    block = Block(5, 8, 3, 256, 192, dtype, eight, ids=ids)
    for e in (1, 2, 4, 6, 7):
        block.gate_up[e].view(torch.uint8 if eight else torch.int16).fill_(0x7f if eight else 0x7fff)
        block.down[e].view(torch.uint8 if eight else torch.int16).fill_(0x7f if eight else 0x7fff)
    clean = block.p.clone()
    block.p[(ids < 0) | (ids >= 8)] = float("nan")
    got = block.run()
    block.p = clean
    block.check(got)
    assert bool((got[1] == 0).all()) and bool((got[3] == 0).all())
    block.ids = torch.full_like(ids, -1)
    assert bool((block.run() == 0).all())


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_an_expert_named_twice_counts_with_both_weights(cuda_device, dtype, eight):
    ids = torch.tensor([[1, 1, 2, 1], [0, 0, 0, 0], [3, 2, 3, 2]] * 5, dtype=torch.int32, device="cuda")
    Block(15, 4, 4, 320, 160, dtype, eight, ids=ids).check()


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("experts", [1, 2])
def test_all_tokens_to_the_same_experts(cuda_device, dtype, eight, experts):
    ids = torch.arange(experts, dtype=torch.int32, device="cuda").expand(64, experts)
    Block(64, 9, experts, 384, 320, dtype, eight, ids=ids).check()


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("hidden,ffn", [(256, 128), (264, 72), (250, 130), (300, 200)])
def test_pitch_alignment_and_layout(cuda_device, dtype, eight, hidden, ffn):
    """x and y anywhere, NaN around; weights at a pitch, off their 16-byte boundaries, and contiguous along the other axis."""
    block = Block(6, 5, 2, hidden, ffn, dtype, eight)
    for offset, extra in ((0, 8), (1, 0), (4, 12), (8, 3)):
        store = torch.full((offset + 6 * (hidden + extra) + 8,), float("nan"), dtype=dtype, device="cuda")
        x = store[offset:offset + 6 * (hidden + extra)].view(6, hidden + extra)[:, :hidden]
        x.copy_(block.x)
        out = torch.full_like(store, 3.0)
        y = out[offset:offset + 6 * (hidden + extra)].view(6, hidden + extra)[:, :hidden]
        block.check(block.run(x=x, y=y))
        y.fill_(3.0)
        assert bool((out == 3.0).all())
    one = block.gate_up, block.down
    nothing = torch.full((1,), 0x7f, dtype=torch.uint8, device="cuda").view(one[0].dtype) if eight else torch.full((1,), float("nan"), dtype=dtype, device="cuda")
    for offset, extra in ((0, 16), (16, 32), (1, 0), (8, 5)):
        def moved(w):
            g, n, k = w.shape
            ld = (-(-k // 16) * 16 if extra else k) + extra
            store = nothing.expand(offset + g * n * ld + 32).clone()
            view = store[offset:offset + g * n * ld].view(g, n, ld)[:, :, :k]
            view.copy_(w)
            return view
        block.gate_up, block.down = moved(one[0]), moved(one[1])
        block.check()
    block.gate_up, block.down = [w.transpose(1, 2).contiguous().transpose(1, 2) for w in one]
    block.check()
    if eight:
        block.gate_up, block.down = one
        block.scales = tuple(s.permute(2, 0, 1).contiguous().permute(1, 2, 0) for s in block.scales)
        block.check()


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("tokens", [1, 3, 8, 13, 40])
@pytest.mark.parametrize("hidden", [1, 7, 8, 65, 130, 250, 301])
def test_tokens_that_end_inside_16_bytes(cuda_device, dtype, eight, tokens, hidden):
    """Rows of x on 16-byte boundaries whose last elements fill a part of 16 bytes only, NaN behind them, the last row at its storage's end;
    weights that are streamed."""
    block = Block(tokens, 5, 2, hidden, 72, dtype, eight)
    block.gate_up, block.down = pitched(block.gate_up, 16), pitched(block.down, 16)
    ld = -(-hidden // 8) * 8
    store = torch.full(((tokens - 1) * ld + hidden,), float("nan"), dtype=dtype, device="cuda")
    x = torch.as_strided(store, (tokens, hidden), (ld, 1))
    x.copy_(block.x)
    block.check(block.run(x=x))


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_in_place(cuda_device, dtype, eight):
    block = Block(7, 8, 2, 512, 256, dtype, eight)
    want = block.run()
    x = block.x.clone()
    assert torch.equal(block.run(x=x, y=x), want)


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
def test_values_that_are_no_numbers(cuda_device, dtype, eight):
    """They reach the results that the definition gives them to, and no others."""
    block = Block(9, 6, 2, 264, 136, dtype, eight, ids=torch.tensor([[t % 6, (t + 1) % 6] for t in range(9)], dtype=torch.int32, device="cuda"))
    want = block.run()
    block.x[4, 17] = float("nan")
    block.x[6, 30] = float("inf")
    got = block.run()
    clean = [t for t in range(9) if t not in (4, 6)]
    assert torch.equal(got[clean], want[clean]) and bool(torch.isnan(got[4]).all()) and not bool(torch.isfinite(got[6]).any())
    block.x[4, 17] = block.x[6, 30] = 0.0
    # one weight of expert 2's down: its row of y for the tokens of expert 2
    bits = block.down.view(torch.uint8) if eight else block.down
    bits[2, 100, 70] = 0x7f if eight else float("nan")
    got = block.run()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[(block.ids == 2).any(dim=1), 100] = True
    assert torch.equal(torch.isnan(got), bad)
    # and of its gate: everything of those tokens
    bits[2, 100, 70] = 0
    bits = block.gate_up.view(torch.uint8) if eight else block.gate_up
    bits[2, 135, 263] = 0xff if eight else float("nan")
    got = block.run()
    assert torch.equal(torch.isnan(got).all(dim=1), (block.ids == 2).any(dim=1)) and torch.equal(torch.isnan(got).any(dim=1), (block.ids == 2).any(dim=1))


@gpu
@pytest.mark.parametrize("dtype,eight", KINDS)
@pytest.mark.parametrize("loud", [300.0, 2.0 ** -9])
def test_gated_values_beyond_the_range_of_16_bits(cuda_device, dtype, eight, loud):
    """h of 10^5 and more, or of 10^-6: it is held in 32 bits or as two halves that carry as much."""
    block = Block(3, 4, 2, 256, 192, dtype, eight, loud=loud)
    block.p *= 1.0 / loud ** 2 if loud > 1 else 1.0
    x = block.x.double()
    if loud > 1:
        assert max(float((x @ block.wide(0, e).t()).abs().max()) for e in range(4)) ** 2 / 4 > 65504
    block.check()


def pitched(w, extra, offset=0):
    """w at a pitch of its rows that is a multiple of 16 bytes where `offset` is 0 and `extra` such a number of elements."""
    g, n, k = w.shape
    ld = -(-k // 16) * 16 + extra
    store = torch.zeros((offset + g * n * ld,), dtype=w.dtype, device="cuda")
    view = store[offset:].view(g, n, ld)[:, :, :k]
    view.copy_(w)
    return view


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 6, 12, 20, 64])
@pytest.mark.parametrize("offset", [0, 1])
def test_infinite_weights(cuda_device, dtype, tokens, offset):
    """As the definition has it, by the kernels that stream (offset 0) and by the general ones: an infinity in down, times values that are not
    zero, is an infinity of the product's sign; two of unlike signs are NaN; one in up's rows makes h infinite."""
    block = Block(tokens, 3, 2, 264, 136, dtype, False, seed=tokens)
    block.ids = torch.tensor([[t % 3, (t + 1) % 3] for t in range(tokens)], dtype=torch.int32, device="cuda")
    if tokens == 64:
        block.ids[:, :] = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    block.down[0, 100, 70] = float("inf")
    block.down[0, 263, 135] = float("-inf")
    block.down[1, 7, 3], block.down[1, 7, 4] = float("inf"), float("inf")
    block.gate_up[2, 136 + 50, 9] = float("inf")
    block.gate_up, block.down = pitched(block.gate_up, 0, offset), pitched(block.down, 0, offset)
    y, off = block.definition()
    got = block.run().double()
    assert bool(torch.isinf(y).any())
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    assert torch.equal(torch.isposinf(got), torch.isposinf(y)) and torch.equal(torch.isneginf(got), torch.isneginf(y))
    finite = torch.isfinite(y)
    assert bool(finite.any()) or tokens == 1
    clean = torch.isfinite(off) & finite
    assert torch.all((got - y)[clean].abs() <= off[clean])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1])
def test_infinite_weights_times_values_without_a_lower_half(cuda_device, dtype, offset):
    """h = 64 * 2 exactly: its upper half is all of it, its lower half is zero."""
    block = Block(1, 1, 1, 8, 8, dtype, False)
    block.x.fill_(0.0)
    block.x[0, 0] = 2.0
    block.gate_up.fill_(0.0)
    block.gate_up[0, 2, 0], block.gate_up[0, 8 + 2, 0] = 32.0, 1.0
    block.down.fill_(1.0)
    block.down[0, 5, 2], block.down[0, 6, 2] = float("inf"), float("-inf")
    block.p.fill_(0.5)
    block.gate_up, block.down = pitched(block.gate_up, 0, offset), pitched(block.down, 0, offset)
    want = torch.full((1, 8), 64.0, device="cuda")
    want[0, 5], want[0, 6] = float("inf"), float("-inf")
    assert torch.equal(block.run().float(), want)


@gpu
@pytest.mark.parametrize("offset", [0, 1])
def test_gated_values_next_to_the_largest(cuda_device, offset):
    """h = 2^64 (2^64 - 2^55): below fp32's largest value, but nearer to 2^128 than to bf16's largest.  Times 2^-126 it is 4 - 2^-7, which bf16
    rounds to 4."""
    block = Block(1, 1, 1, 8, 8, torch.bfloat16, False)
    block.x.fill_(0.0)
    block.x[0, 0], block.x[0, 1] = 2.0 ** 64, 2.0 ** 55
    block.gate_up.fill_(0.0)
    block.gate_up[0, 2, 0] = 1.0
    block.gate_up[0, 8 + 2, 0], block.gate_up[0, 8 + 2, 1] = 1.0, -1.0
    block.down.fill_(0.0)
    block.down[0, 5, 2], block.down[0, 6, 2] = 2.0 ** -126, -(2.0 ** -120)
    block.p.fill_(1.0)
    block.gate_up, block.down = pitched(block.gate_up, 0, offset), pitched(block.down, 0, offset)
    want = torch.zeros((1, 8), device="cuda")
    want[0, 5], want[0, 6] = 4.0, -256.0
    assert torch.equal(block.run().float(), want)


@gpu
def test_streams_and_graphs(cuda_device):
    """Two calls at once, each with a workspace; one captured and replayed on other tokens, ids and weights: the same bits as alone."""
    blocks = [Block(6, 32, 4, 512, 384, torch.bfloat16, False, seed=s) for s in (1, 2)]
    blocks[1].gate_up, blocks[1].down = blocks[0].gate_up, blocks[0].down
    want = [block.run() for block in blocks]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    for _ in range(10):
        got = []
        for block, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                space = torch.empty(1 << 16, device="cuda")
                got.append((block.run(stream=s.cuda_stream, workspace=space), space))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for (g, _), w in zip(got, want))
    block, other = blocks
    space = torch.empty(1 << 16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.run(stream=torch.cuda.current_stream().cuda_stream, workspace=space)
    block.x.copy_(other.x)
    block.ids.copy_(other.ids)
    block.p.copy_(other.p)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[1])


@gpu
def test_calls_of_all_sizes_side_by_side(cuda_device):
    """Launches that share SMs with their successors, of CTA pairs and of whole SMs, on four streams at once: the same bits as alone."""
    sizes = [(1, 16, 8, 2048, 1408, False), (4, 16, 4, 1024, 2048, False), (64, 16, 4, 1024, 512, False), (12, 16, 4, 2048, 512, True)]
    blocks = [Block(*size[:5], torch.bfloat16, size[5], seed=i) for i, size in enumerate(sizes)]
    want = [block.run() for block in blocks]
    for block, y in zip(blocks, want):
        block.check(y)
    spaces = [torch.empty(1 << 21, device="cuda") for _ in blocks]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    for _ in range(15):
        got = []
        for block, s, space in zip(blocks, streams, spaces):
            with torch.cuda.stream(s):
                got.append([block.run(stream=s.cuda_stream, workspace=space) for _ in range(2)])
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for pair, w in zip(got, want) for g in pair)
    kb.experts_check()


def desc(**more):
    sizes = [more.pop(name, v) for name, v in (("tokens", 2), ("hidden", 16), ("ffn", 8), ("experts", 4), ("top", 2), ("dtype", kb.BF16))]
    return kb.make_experts_desc(*sizes, **more)


@pytest.mark.parametrize("d,status", [
    (desc(tokens=-1), 2), (desc(tokens=65), 1), (desc(top=17, experts=20), 1), (desc(top=0), 2), (desc(experts=0), 2), (desc(experts=1025), 1),
    (desc(hidden=0), 1), (desc(ffn=0), 1), (desc(ffn=2 ** 30), 1), (desc(dtype=kb.F32), 1), (desc(weight_dtype=kb.F16), 1), (desc(y_ld=15), 2),
    (desc(x_ld=-1), 2), (desc(down_strides=(8, -8, 1)), 2),
])
def test_descriptors_that_are_refused(d, status):
    with pytest.raises(kb.KudnnError) as e:
        kb.experts(d, *[16] * 7, 10 ** 9)
    assert e.value.status == status
    with pytest.raises(kb.KudnnError):
        kb.experts_workspace(d)


@pytest.mark.parametrize("place", range(7))
@pytest.mark.parametrize("wrong", [None, 17])
def test_calls_that_are_refused(place, wrong):
    """On the host, ahead of any device: the addresses are made up."""
    operands = [16] * 7
    operands[place] = wrong
    with pytest.raises(kb.KudnnError) as e:
        kb.experts(desc(), *operands, 10 ** 9)
    assert e.value.status == 2


@pytest.mark.parametrize("call", [
    lambda: kb.experts(desc(), *[16] * 7, kb.experts_workspace(desc()) - 1), lambda: kb.experts(desc(), *[16] * 6, 24, 10 ** 9),
    lambda: kb.experts(desc(), *[16] * 7, 10 ** 9, 16, 16), lambda: kb.experts(desc(weight_dtype=kb.E4M3), *[16] * 7, 10 ** 9, 16),
    lambda: kb.experts(desc(weight_dtype=kb.E4M3), *[16] * 7, 10 ** 9, 16, 18), lambda: kb.experts(desc(weight_dtype=kb.E4M3), *[16] * 7, 10 ** 9),
])
def test_scales_and_workspaces_that_are_refused(call):
    with pytest.raises(kb.KudnnError) as e:
        call()
    assert e.value.status == 2
