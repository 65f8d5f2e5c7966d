"""Quantisation to e4m3 with a scale per block, against the definition in 64 bits.

Tolerances: q * scale is v rounded to three bits after the leading one, so it is off by at most 1/16 of |v|, or by half of the smallest
step 2^-9 where v / scale lies below 2^-6; both in units of the block's scale, with 2^-20 more for the fp32 arithmetic (v * (448 / most)
has two roundings, the scale one) and, behind a gate, 2^-18 for the approximate exponential and reciprocal of 16-bit inputs.
Without a gate every step is one correctly rounded fp32 operation, so q and scale are compared bit by bit with the same steps in torch.
"""
import numpy as np
import pytest
import torch

import kudnn_b200 as kb
from kudnn_b200 import capi

CODE = {torch.float32: kb.F32, torch.float16: kb.F16, torch.bfloat16: kb.BF16}
gpu = pytest.mark.gpu


def pitch(k):
    return -(-k // 16) * 16


def run(x, rows, k, gate=False, index=None, q_ld=None, s_by_row=False, block_rows=1, stream=None):
    """q as floats and the scales [rows or blocks of rows, blocks of columns]; q's memory holds 0x55 where nothing is written."""
    q_ld = q_ld or pitch(k)
    blocks_k, scale_rows = -(-k // 128), -(-rows // block_rows)
    store = torch.full((rows, q_ld), 0x55, dtype=torch.uint8, device=x.device)
    scale = torch.full((scale_rows, blocks_k) if s_by_row else (blocks_k, scale_rows), -1.0, device=x.device)
    desc = kb.make_quantize_desc(rows, k, CODE[x.dtype], gate=gate, x_rows=x.shape[0], x_ld=x.stride(0), q_ld=q_ld,
                                 block_rows=block_rows, scale_strides=(blocks_k, 1) if s_by_row else (1, scale_rows))
    kb.quantize(desc, x, store, scale, index, stream=stream)
    torch.cuda.synchronize()
    assert bool((store[:, k:] == 0x55).all()), "written beyond the columns"
    return store[:, :k].view(torch.float8_e4m3fn), scale if s_by_row else scale.t()


def in_fp32(v, block_rows=1):
    """The definition, one rounding per step, v [rows, k] in fp32."""
    rows, k = v.shape
    rb, kbs = -(-rows // block_rows), -(-k // 128)
    full = torch.zeros((rb * block_rows, kbs * 128), device=v.device)
    full[:rows, :k] = v
    blocks = full.view(rb, block_rows, kbs, 128)
    most = blocks.abs().amax(dim=(1, 3)).clamp(min=1e-30)
    largest = torch.full_like(most, 448.0)  # a tensor: torch multiplies by the rounded reciprocal of a scalar divisor
    q = (blocks * (largest / most)[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(rb * block_rows, -1)[:rows, :k], most / largest


def same(got, want):
    q, s = got
    q2, s2 = want
    assert torch.equal(torch.isnan(s), torch.isnan(s2)) and torch.equal(torch.nan_to_num(s, nan=0.0), torch.nan_to_num(s2, nan=0.0))
    q, q2 = q.float(), q2.float()
    assert torch.equal(torch.isnan(q), torch.isnan(q2)) and torch.equal(torch.nan_to_num(q, nan=0.0), torch.nan_to_num(q2, nan=0.0))


def values(rows, k, dtype, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x[:, :: max(1, k // 3)] *= 40.0
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 127), (5, 129), (8, 4096), (1, 16), (33, 384), (70, 1000), (257, 2050), (1031, 641)])
def test_rows(cuda_device, dtype, rows, k):
    x = values(rows, k, dtype)
    same(run(x, rows, k), in_fp32(x.float()))
    same(run(x, rows, k, s_by_row=True), in_fp32(x.float()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (128, 128), (129, 257), (300, 100), (1, 640), (256, 2048)])
def test_blocks_of_weights(cuda_device, dtype, rows, k):
    x = values(rows, k, dtype)
    same(run(x, rows, k, block_rows=128), in_fp32(x.float(), 128))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 8), (2, 128), (9, 11008), (70, 1000), (257, 130)])
def test_gate(cuda_device, dtype, rows, k):
    x = values(rows, 2 * k, dtype)
    q, scale = run(x, rows, k, gate=True)
    v = x[:, :k].double() * torch.sigmoid(x[:, :k].double()) * x[:, k:].double()
    blocks_k = -(-k // 128)
    full = torch.zeros((rows, blocks_k * 128), dtype=torch.float64, device="cuda")
    full[:, :k] = v
    want = full.view(rows, blocks_k, 128).abs().amax(dim=2).clamp(min=1e-30) / 448.0
    assert torch.all((scale.double() - want).abs() <= 2.0 ** -18 * want)
    s = scale.double().repeat_interleave(128, dim=1)[:, :k]
    off = (q.double() * s - v).abs()
    assert torch.all(off <= torch.maximum(v.abs() / 16, s * 2.0 ** -10) * (1 + 2.0 ** -18) + 448 * s * 2.0 ** -20)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 16])
def test_gate_keeps_the_bits_of_the_scale(cuda_device, dtype, k):
    """A gate and an up per row, so that the scale is silu(gate) * up / 448.  In units of 2^-24: the exponential 4 (2 in the last place), its
    product with the gate, the sum with 1, the product with the inverse, that with up and the scale's division 1 each, the inverse 2."""
    far = 60.0 if dtype == torch.float16 else 87.0  # e^-87 is a normal number, and times up above 1e-30, below which nothing is scaled up
    gate = torch.linspace(-far, 40.0, 3001, device="cuda").to(dtype)
    gate = gate[gate != 0]
    up = torch.full_like(gate, 1e4 if dtype == torch.float16 else 1e36)
    x = torch.cat([gate[:, None].expand(-1, k), up[:, None].expand(-1, k)], dim=1).contiguous()
    _, scale = run(x, x.shape[0], k, gate=True)
    want = (gate.double() * torch.sigmoid(gate.double()) * up.double()).abs() / 448.0
    assert torch.all((scale[:, 0].double() - want).abs() <= 11 * 2.0 ** -24 * want)


@gpu
@pytest.mark.parametrize("rows,k", [(1, 256), (40, 4099), (77, 640)])
@pytest.mark.parametrize("gate", [False, True])
def test_index(cuda_device, rows, k, gate):
    tokens = 13
    x = values(tokens, 2 * k if gate else k, torch.bfloat16)
    index = torch.randint(0, tokens, (rows,), device="cuda", dtype=torch.int32)
    got, want = run(x, rows, k, gate=gate, index=index), run(x, tokens, k, gate=gate)
    same(got, (want[0].view(torch.uint8)[index.long()].view(torch.float8_e4m3fn), want[1][index.long()]))


@gpu
def test_index_outside_of_x_gives_zeros(cuda_device):
    x = values(4, 300, torch.float16)
    index = torch.tensor([3, -1, 4, 2 ** 31 - 1, 0], device="cuda", dtype=torch.int32)
    q, scale = run(x, 5, 300, index=index)
    want = in_fp32(x.float())
    for r, t in ((0, 3), (4, 0)):
        assert torch.equal(q[r].float(), want[0][t].float()) and torch.equal(scale[r], want[1][t])
    for r in (1, 2, 3):
        assert bool((q[r].float() == 0).all()) and bool((scale[r] == in_fp32(torch.zeros((1, 128), device="cuda"))[1]).all())


@gpu
@pytest.mark.parametrize("offset,ld", [(0, 300), (1, 301), (3, 307), (8, 304)])
def test_pitch_and_alignment(cuda_device, offset, ld):
    rows, k = 19, 290
    base = values(rows, ld, torch.bfloat16).reshape(-1)
    base = torch.cat([torch.full((offset,), float("nan"), dtype=torch.bfloat16, device="cuda"), base])
    x = base[offset:].view(rows, ld)[:, :k]
    for q_ld in (290, 291, 304):
        same(run(x, rows, k, q_ld=q_ld), in_fp32(x.float()))


@gpu
def test_extremes(cuda_device):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros((8, 256), device="cuda")
    x[1, 5] = nan                      # the block becomes NaN, its neighbour stays
    x[1, 200] = 2.0
    x[2, 7], x[2, 8] = inf, 3.0        # infinite scale, zeros and NaN
    x[3, :128] = 1e-35                 # below the least magnitude that is scaled up
    x[4, 0], x[4, 1] = 3.4e38, -3.4e38
    x[5, :] = -0.0
    x[6, 0], x[6, 1] = 1e-30, 5e-31
    x[7, 0], x[7, 1], x[7, 2] = -448.0, 1.0 / 512, 1.0 / 1024   # a scale of one: the smallest steps, a tie to even
    same(run(x, 8, 256), in_fp32(x))
    q, scale = run(x, 8, 256)
    assert bool(torch.isnan(q[1, :128].float()).all()) and q[1, 200].float() == 448.0
    assert torch.isinf(scale[2, 0]) and torch.isnan(q[2, 7].float()) and q[2, 8].float() == 0.0
    assert q[7, 0].float() == -448.0 and q[7, 1].float() == 2.0 ** -9 and q[7, 2].float() == 0.0 and scale[7, 0] == 1.0


@gpu
def test_on_another_stream_and_in_a_graph(cuda_device):
    x = values(64, 1024, torch.bfloat16)
    want = in_fp32(x.float())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    same(run(x, 64, 1024, stream=side.cuda_stream), want)
    q = torch.empty((64, 1024), dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty((8, 64), device="cuda")
    desc = kb.make_quantize_desc(64, 1024, kb.BF16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kb.quantize(desc, x, q, scale, stream=torch.cuda.current_stream().cuda_stream)
    y = values(64, 1024, torch.bfloat16, seed=7)
    x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    same((q, scale.t()), in_fp32(y.float()))


@gpu
def test_large_offsets(cuda_device):
    """Rows whose elements lie beyond 2^31."""
    rows, k = 70000, 128
    ld = 1 << 15
    x = torch.zeros((rows, ld), dtype=torch.bfloat16, device="cuda")
    x[:, :k] = values(rows, k, torch.bfloat16)
    same(run(x[:, :k], rows, k), in_fp32(x[:, :k].float()))


def desc(**more):
    base = dict(rows=4, k=256, dtype=kb.BF16)
    extra = {key: more.pop(key) for key in list(more) if key in ("gate", "x_rows", "block_rows", "x_ld", "q_ld", "scale_strides")}
    d = kb.make_quantize_desc(base["rows"], base["k"], base["dtype"], **extra)
    for key, v in more.items():
        setattr(d, key, v)
    return d


@pytest.mark.parametrize("more,status", [
    (dict(rows=-1), 2), (dict(k=0), 1), (dict(k=1 << 31), 1), (dict(x_dtype=kb.S8), 1), (dict(x_dtype=kb.E4M3), 1),
    (dict(block_rows=64), 1), (dict(block_rows=128, gate=True), 1), (dict(block_rows=128, x_rows=9), 1), (dict(q_ld=255), 2),
    (dict(s_row=0), 2), (dict(s_col=0), 2), (dict(s_col=-1), 2), (dict(x_ld=-1), 2), (dict(), 0), (dict(x_rows=9), 0), (dict(block_rows=128), 0),
])
def test_refusals(more, status):
    import ctypes
    assert kb.library().kudnn_b200_quantize_validate(ctypes.byref(desc(**more))) == status


def test_null_pointers_and_rows_without_index_are_refused():
    x = np.zeros((4, 256), dtype=np.uint16)
    with pytest.raises(kb.KudnnError) as e:
        kb.quantize(desc(), x, None, None)
    assert e.value.status == 2
    with pytest.raises(kb.KudnnError) as e:
        kb.quantize(desc(block_rows=128), x, x, x, index=x)   # an index goes with a scale per row
    assert e.value.status == 1
    d = desc()
    d.x_rows = 5
    with pytest.raises(kb.KudnnError) as e:
        kb.quantize(d, x, x, x)
    assert e.value.status == 2
    d = desc()
    d.rows = d.x_rows = 0
    kb.quantize(d, None, None, None)            # no rows: nothing to do
    assert capi.library().kudnn_b200_quantize_validate(None) == 2


def test_addresses_between_elements_are_refused():
    at = 1 << 20
    for x, scale, index in ((at + 1, at, at), (at, at + 2, at), (at, at, at + 1)):
        with pytest.raises(kb.KudnnError) as e:
            kb.quantize(desc(), x, at, scale, index)
        assert e.value.status == 2


@pytest.mark.parametrize("strides,status", [((1, 4), 0), ((1, 3), 2), ((1, 1), 2), ((2, 1), 0), ((3, 2), 0), ((1, 2), 2), ((2, 3), 0)])
def test_scales_that_share_memory_are_refused(strides, status):
    """4 rows, 2 blocks of columns; held against all addresses."""
    import ctypes
    shared = len({r * strides[0] + c * strides[1] for r in range(4) for c in range(2)}) < 8
    assert shared == (status != 0)
    assert kb.library().kudnn_b200_quantize_validate(ctypes.byref(desc(scale_strides=strides))) == status
