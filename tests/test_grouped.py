"""Products by group and block-scaled 8-bit products against the definition in 64 bits.

Tolerance of an element, from S = sum over k of |a||b| (scales included) and the sum's exact value y: the fp32 additions, counted as one
cut of 2^-23 of S for every eight products and eight more for scales and bias, carried through the activation (whose slope is at most
1.13, its approximations within 2^-18 of the value and 2^-20 of the argument), and half a unit of the result's last place.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import kudnn_b200 as kb

CODE = {"f32": kb.F32, "f16": kb.F16, "bf16": kb.BF16, "e4m3": kb.E4M3}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of the value; bf16: 2^-9, doubled at a power of two
LEAST = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
ACTS = {"none": kb.ACT_NONE, "relu": kb.ACT_RELU, "silu": kb.ACT_SWISH, "gelu_tanh": kb.ACT_GELU_TANH, "gelu_erf": kb.ACT_GELU_ERF,
        "sigmoid": kb.ACT_SIGMOID, "tanh": kb.ACT_TANH}
gpu = pytest.mark.gpu


def pitch(k, dtype):
    size = 1 if dtype == "e4m3" else 2
    return -(-k * size // 16) * 16 // size


def act64(v, act):
    if act == "relu":
        return torch.relu(v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(v, approximate="tanh")
    if act == "gelu_erf":
        return torch.nn.functional.gelu(v)
    if act == "sigmoid":
        return torch.sigmoid(v)
    if act == "tanh":
        return torch.tanh(v)
    return v


def cleaned(offsets, rows):
    """Offsets as the operator reads them: within [0, rows], never descending."""
    out = []
    for v in offsets:
        v = min(max(int(v), 0), rows)
        out.append(max(v, out[-1]) if out else v)
    return out


class Problem:
    def __init__(self, rows, n, k, dtype, sizes=None, out=None, act="none", bias=None, seed=0, a_ld=None, b_major="k", b_ld=None, c_ld=None,
                 offsets=None, wide_offsets=False, a_scale_by_row=False, guard=True):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.rows, self.n, self.k, self.dtype, self.act = rows, n, k, dtype, act
        self.out = out or ("bf16" if dtype == "e4m3" else dtype)
        if sizes is not None:
            offsets = [sum(sizes[:g]) for g in range(len(sizes) + 1)]
        self.groups = len(offsets) - 1 if offsets is not None else 1
        self.ends = cleaned(offsets, rows) if offsets is not None else [0, rows]
        self.offsets = None if offsets is None else torch.tensor(offsets, dtype=torch.int64 if wide_offsets else torch.int32, device="cuda")
        a_ld, b_ld, c_ld = a_ld or pitch(k, dtype), b_ld or pitch(k if b_major == "k" else n, dtype), c_ld or n

        def operand(count, columns, ld, std):
            x = torch.randn((count, ld), generator=gen, device="cuda") * std
            if dtype != "e4m3":
                return x.to(TORCH[dtype])[:, :columns]
            return (x / std * 60).clamp(-448, 448).to(TORCH[dtype])[:, :columns]

        self.a = operand(max(rows, 1), k, a_ld, 1.0)[:rows]
        b_rows, b_columns = (n, k) if b_major == "k" else (k, n)
        self.b = operand(self.groups * b_rows, b_columns, b_ld, 0.05)
        if b_major == "k":
            self.b_strides = (n * b_ld, b_ld, 1)
        else:
            self.b_strides = (k * b_ld, 1, b_ld)
        self.b3 = torch.as_strided(self.b, (self.groups, n, k), self.b_strides)
        self.bn, self.bk = -(-n // 128), -(-k // 128)
        self.a_scale = self.b_scale = None
        if dtype == "e4m3":
            by = (rows, self.bk) if a_scale_by_row else (self.bk, rows)
            self.a_scale = torch.rand(by, generator=gen, device="cuda") * 0.02 + 0.001
            self.b_scale = torch.rand((self.groups, self.bn, self.bk), generator=gen, device="cuda") * 0.002 + 0.0001
        self.as_view = None if self.a_scale is None else (self.a_scale if a_scale_by_row else self.a_scale.t())
        self.bias = None if bias is None else torch.randn((self.groups, n), generator=gen, device="cuda").to(TORCH[bias])
        self.store = torch.full((max(rows, 1), c_ld), 77.0, dtype=TORCH[self.out], device="cuda")
        self.c = self.store[:rows, :n]
        self.desc = kb.make_grouped_desc(
            rows, n, k, CODE[dtype], groups=self.groups, c_dtype=CODE[self.out],
            offsets_dtype=0 if offsets is None else kb.S64 if wide_offsets else kb.S32, a_strides=(a_ld, 1), b_strides=self.b_strides,
            c_strides=(c_ld, 1), a_scale_strides=(self.bk, 1) if a_scale_by_row else (1, max(rows, 1)), has_bias=bias is not None,
            bias_dtype=None if bias is None else CODE[bias], act=ACTS[act], act_alpha=0.0 if act == "relu" else 1.0)

    def run(self, kernel=kb.KERNEL_AUTO, stream=None):
        op = kb.Grouped(self.desc)
        op.force_kernel(kernel)
        op.run(self.a, self.b, self.c, offsets=self.offsets, a_scale=self.a_scale, b_scale=self.b_scale, bias=self.bias, stream=stream)
        op.check(stream)
        self.kernel = op.last_kernel
        assert bool((self.store[:, self.n:] == 77.0).all()), "written beyond the columns"
        return self

    def exact(self):
        y = torch.zeros((self.rows, self.n), dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(y)
        for g in range(self.groups):
            lo, hi = self.ends[g], self.ends[g + 1]
            if lo == hi:
                continue
            a, b = self.a[lo:hi].double(), self.b3[g].double()
            if self.dtype == "e4m3":
                a = a * self.as_view[lo:hi].double().repeat_interleave(128, 1)[:, :self.k]
                b = b * self.b_scale[g].double().repeat_interleave(128, 0)[:self.n].repeat_interleave(128, 1)[:, :self.k]
            v, s = a @ b.t(), a.abs() @ b.abs().t()
            if self.bias is not None:
                v = v + self.bias[g].double()
                s = s + self.bias[g].double().abs()
            r = act64(v, self.act)
            y[lo:hi] = r
            sums = (self.k / 8 + 8) * 2.0 ** -23 * s
            tol[lo:hi] = 1.13 * sums + HALF_ULP[self.out] * (r.abs() + 1.13 * sums) + LEAST[self.out]
            if self.act != "none":
                tol[lo:hi] += 2.0 ** -18 * r.abs() + 2.0 ** -20 * v.abs()
        return y, tol

    def aligned(self):
        size = 1 if self.dtype == "e4m3" else 2
        return all(s * size % 16 == 0 for s in (self.a.stride(0), self.b_strides[0], self.b_strides[1])) and (self.b_strides[2] == 1 or self.k == 1)

    def check(self, kernel=kb.KERNEL_AUTO, stream=None):
        self.run(kernel, stream)
        if self.aligned() and kernel == kb.KERNEL_AUTO:
            assert self.kernel == kb.KERNEL_TC
        y, tol = self.exact()
        got = self.c.double()
        off = (got - y).abs()
        bad = ~(off <= tol)
        assert not bool(bad.any()), "%d of %d off, the first at %s: %r for %r, tolerance %r" % (
            int(bad.sum()), bad.numel(), tuple(bad.nonzero()[0].tolist()), got[bad][0].item(), y[bad][0].item(), tol[bad][0].item())
        return self


OPERANDS = ["bf16", "f16", "e4m3"]


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 128, 130, 255, 256, 257, 600])
@pytest.mark.parametrize("n,k", [(128, 128), (200, 640), (1000, 1000), (56, 48)])
def test_one_group(cuda_device, dtype, m, n, k):
    Problem(m, n, k, dtype).check()


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 16), (7, 1, 300), (3, 129, 127), (40, 257, 129), (200, 8, 4100), (5, 4097, 264), (1, 2048, 8192)])
def test_odd_sizes(cuda_device, dtype, m, n, k):
    Problem(m, n, k, dtype).check()
    Problem(m, n, k, dtype, sizes=[0, m, 0]).check()


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
@pytest.mark.parametrize("sizes", [
    [1], [0, 0, 3, 0], [1] * 8, [5, 0, 300, 17, 0, 0, 64, 1], [256, 512, 1], [700, 1, 1, 1, 1, 0, 90], [0] * 63 + [9],
    [i % 7 for i in range(130)], [33] * 31 + [1000],
])
def test_ragged_groups(cuda_device, dtype, sizes):
    rows = sum(sizes)
    Problem(rows, 264, 400, dtype, sizes=sizes, bias="f32", act="silu").check()
    Problem(rows, 128, 1024, dtype, sizes=sizes, wide_offsets=True, out="f32").check()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("offsets", [
    [0, 0, 0, 0], [3, 9, 9, 20], [0, 40, 10, 30], [-5, 7, 1000, 8], [50, 50, 50, 50], [60, 20, 10, 0], [0, 5, 2 ** 31 - 1, -2 ** 31],
])
def test_rows_that_no_group_holds_and_offsets_out_of_order(cuda_device, dtype, offsets):
    Problem(50, 200, 272, dtype, offsets=offsets, act="sigmoid").check()
    Problem(50, 200, 272, dtype, offsets=[v * 2 ** 20 if abs(v) > 100 else v for v in offsets], wide_offsets=True, act="sigmoid").check()


@gpu
def test_most_groups(cuda_device):
    sizes = [(g * 7) % 3 for g in range(1024)]
    Problem(sum(sizes), 24, 48, "bf16", sizes=sizes).check()
    p = Problem(1, 24, 48, "bf16", sizes=[0] * 1023 + [1]).check()
    assert p.desc.groups == 1024


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", sorted(ACTS))
def test_results_bias_and_activation(cuda_device, dtype, out, act):
    for bias in ("f32", "f16", "bf16"):
        Problem(75, 136, 320, dtype, sizes=[20, 0, 55], out=out, act=act, bias=bias).check()


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
@pytest.mark.parametrize("more", [dict(a_ld=416), dict(b_ld=448), dict(c_ld=300), dict(c_ld=301), dict(a_scale_by_row=True), dict(b_major="n"),
                                  dict(a_ld=401), dict(b_ld=403), dict(a_ld=400, b_ld=400)])
def test_layouts(cuda_device, dtype, more):
    for m in (3, 90, 300):
        Problem(m, 264, 400, dtype, sizes=[m // 3, m - m // 3], **more).check()


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
def test_the_general_kernel(cuda_device, dtype):
    for m, n, k in ((1, 100, 100), (70, 136, 320), (129, 65, 1000)):
        p = Problem(m, n, k, dtype, sizes=[m // 2, m - m // 2], bias="f32", act="gelu_tanh").check(kb.KERNEL_SIMT)
        assert p.kernel == kb.KERNEL_SIMT


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
def test_fp32_results_of_the_general_kernel_keep_their_bits(cuda_device, dtype):
    """128 products add up, then 64 of these sums.  An addition is off by 0.42 * 2^-24 of the running sum in the square mean, and that is half
    of the last one on average: 0.3 * 2^-24 * sqrt(128 + 64) = 4.1 * 2^-24 in the norm.  Twice that is the limit."""
    p = Problem(130, 200, 8192, dtype, out="f32", sizes=[60, 70]).check(kb.KERNEL_SIMT)
    y, _ = p.exact()
    assert torch.linalg.vector_norm(p.c.double() - y) <= 8.2 * 2.0 ** -24 * torch.linalg.vector_norm(y)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_what_is_not_finite_stays_in_its_row_or_column(cuda_device, dtype):
    p = Problem(300, 264, 400, dtype, sizes=[100, 0, 200])
    p.a[40, 3] = float("nan")
    p.b3[2, 200, 399] = float("nan")
    if dtype == "e4m3":
        p.a_scale.t()[299, 1] = float("inf")
    else:
        p.a[299, 7] = float("inf")
    p.run()
    fine = torch.isfinite(p.c.float())
    want = torch.ones_like(fine)
    want[40] = False
    want[100:, 200] = False
    want[299] = False
    assert torch.equal(fine, want)


@gpu
def test_no_rows(cuda_device):
    Problem(0, 64, 64, "bf16", sizes=[0, 0]).run()
    Problem(0, 64, 64, "e4m3").run()


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
@pytest.mark.parametrize("m,k", [(3, 8192), (50, 2000), (100, 8192), (700, 8192), (1, 520)])
def test_fp32_results_keep_their_bits(cuda_device, dtype, m, k):
    """256 products at most add up in the tensor cores before fp32 registers take over: 16 cuts of up to 2^-23, half of it on average, of sums
    that are half of the last one on average, 2^-21 in the norm; as much again for the fp32 additions."""
    p = Problem(m, 384, k, dtype, sizes=[m - m // 3, m // 3], out="f32").check()
    y, _ = p.exact()
    assert torch.linalg.vector_norm(p.c.double() - y) <= 2.0 ** -20 * torch.linalg.vector_norm(y)


@gpu
@pytest.mark.parametrize("dtype", OPERANDS)
def test_the_same_bits_every_time(cuda_device, dtype):
    p = Problem(16, 512, 4096, dtype)
    first = p.run().c.clone()
    for _ in range(5):
        assert torch.equal(p.run().c, first)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_streams_and_graphs(cuda_device, dtype):
    problems = [Problem(m, 520, 1024, dtype, sizes=[m // 4, 0, m - m // 4], seed=m) for m in (4, 60, 700)]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    ops = [kb.Grouped(p.desc) for p in problems]
    for _ in range(3):
        for p, op, s in zip(problems, ops, streams):
            op.run(p.a, p.b, p.c, offsets=p.offsets, a_scale=p.a_scale, b_scale=p.b_scale, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for p in problems:
        y, tol = p.exact()
        assert bool(((p.c.double() - y).abs() <= tol).all())
    # a graph whose group sizes change between replays
    p, op = problems[1], kb.Grouped(problems[1].desc)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run(p.a, p.b, p.c, offsets=p.offsets, a_scale=p.a_scale, b_scale=p.b_scale, stream=torch.cuda.current_stream().cuda_stream)
    for offsets in ([0, 15, 15, 60], [0, 0, 60, 60], [0, 1, 2, 50]):
        p.offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
        p.ends = offsets
        graph.replay()
        torch.cuda.synchronize()
        y, tol = p.exact()
        assert bool(((p.c.double() - y).abs() <= tol).all())


@gpu
def test_the_first_run_of_a_handle_may_be_captured(cuda_device):
    p = Problem(33, 136, 256, "e4m3", sizes=[3, 30])
    y, tol = p.exact()
    op = kb.Grouped(p.desc)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="thread_local")
        op.run(p.a, p.b, p.c, offsets=p.offsets, a_scale=p.a_scale, b_scale=p.b_scale, stream=stream.cuda_stream)
        graph.capture_end()
    for _ in range(3):
        p.c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bool(((p.c.double() - y).abs() <= tol).all())
    op.check()


@gpu
def test_rows_that_share_memory(cuda_device):
    """Operands broadcast with a stride of zero."""
    p = Problem(20, 72, 96, "bf16", sizes=[5, 15])
    want = p.a[:1].double() @ p.b3[1].double().t()
    p.desc.a_sm = 0
    p.run()
    assert p.kernel == kb.KERNEL_SIMT
    limit = (96 / 8 + 8) * 2.0 ** -23 * (p.a[:1].double().abs() @ p.b3[1].double().abs().t()) + 2.0 ** -8 * want.abs()
    assert bool(((p.c[5:].double() - want).abs() <= limit).all())


@gpu
def test_large_offsets(cuda_device):
    """Rows of a and c, and weights, whose elements lie beyond 2^31."""
    p = Problem(3000, 128, 256, "bf16", sizes=[2990, 10], a_ld=1 << 20, c_ld=1 << 20)
    p.check()
    big = Problem(9, 128, 128, "e4m3", sizes=[4, 5], b_ld=1 << 24)
    big.check()


@gpu
def test_out_of_device_memory(cuda_device):
    p = Problem(4, 64, 64, "bf16")
    kb.debug_fail_allocation(0)
    try:
        with pytest.raises(kb.KudnnError) as e:
            p.run()
        assert e.value.status == 3
    finally:
        kb.debug_fail_allocation(-1)
    p.check()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("m", [1, 40, 100, 500])
def test_a_wait_that_runs_out(cuda_device, dtype, m):
    """Loads that never come: the kernel gives up, reports it and leaves the device usable."""
    p = Problem(m, 256, 2048, dtype)
    op = kb.Grouped(p.desc)
    op.set_wait(20_000_000, 3)
    op.run(p.a, p.b, p.c, a_scale=p.a_scale, b_scale=p.b_scale)
    with pytest.raises(kb.KudnnError) as e:
        op.check()
    assert e.value.status == 5
    op.set_wait(0)
    op.run(p.a, p.b, p.c, a_scale=p.a_scale, b_scale=p.b_scale)
    op.check()
    y, tol = p.exact()
    assert bool(((p.c.double() - y).abs() <= tol).all())


@gpu
def test_forced_tensor_cores_refuse_what_they_do_not_take(cuda_device):
    p = Problem(20, 64, 100, "bf16", a_ld=101)
    with pytest.raises(kb.KudnnError) as e:
        p.run(kb.KERNEL_TC)
    assert e.value.status == 1


def small(**more):
    d = kb.make_grouped_desc(8, 256, 256, more.pop("dtype", kb.E4M3), groups=more.pop("groups", 4), offsets_dtype=more.pop("offsets_dtype", kb.S32))
    for key, v in more.items():
        setattr(d, key, v)
    return d


@pytest.mark.parametrize("more,status", [
    (dict(), 0), (dict(rows=0), 0), (dict(dtype=kb.BF16, has_bias=1, bias_dtype=kb.F16, act=kb.ACT_SWISH), 0), (dict(groups=1, offsets_dtype=0), 0),
    (dict(rows=-1), 2), (dict(n=0), 1), (dict(k=0), 1), (dict(groups=0), 2), (dict(groups=1025), 1), (dict(rows=1 << 31), 1), (dict(n=1 << 31), 1),
    (dict(dtype=kb.F32), 1), (dict(dtype=kb.S8), 1), (dict(c_dtype=kb.E4M3), 1), (dict(has_bias=1, bias_dtype=kb.S32), 1), (dict(act=1), 1),
    (dict(offsets_dtype=kb.F32), 1), (dict(offsets_dtype=0), 2), (dict(a_sm=-1), 2), (dict(b_scale_sk=-1), 2), (dict(c_sm=0), 2), (dict(c_sn=0), 2),
])
def test_refusals(more, status):
    d = small(**more)
    assert kb.library().kudnn_b200_grouped_validate(ctypes.byref(d)) == status
    if status != 0:
        with pytest.raises(kb.KudnnError) as e:
            kb.Grouped(d)
        assert e.value.status == status


def test_pointers_that_do_not_match_the_descriptor_are_refused():
    x = np.zeros(16, dtype=np.float32)
    op = kb.Grouped(small())
    every = dict(offsets=x, a_scale=x, b_scale=x)
    for wrong in (dict(every, offsets=None), dict(every, a_scale=None), dict(every, b_scale=None), dict(every, bias=x)):
        with pytest.raises(kb.KudnnError) as e:
            op.run(x, x, x, **wrong)
        assert e.value.status == 2
    for a, b, c in ((None, x, x), (x, None, x), (x, x, None)):
        with pytest.raises(kb.KudnnError) as e:
            op.run(a, b, c, **every)
        assert e.value.status == 2
    op = kb.Grouped(small(dtype=kb.BF16))
    with pytest.raises(kb.KudnnError) as e:
        op.run(x, x, x, **every)  # scales of operands that have none
    assert e.value.status == 2
    for kernel in (kb.KERNEL_GEMV_FMA, 9):
        with pytest.raises(kb.KudnnError) as e:
            op.force_kernel(kernel)
        assert e.value.status == 2
    empty = kb.Grouped(small(rows=0))
    empty.run(None, None, None, **every)  # no rows: nothing to do
    assert kb.library().kudnn_b200_grouped_validate(None) == 2
    assert math.isclose(small().act_alpha, 1.0)


def test_addresses_between_elements_are_refused():
    """A load from one would fault."""
    at = 1 << 20
    op = kb.Grouped(small(offsets_dtype=kb.S64, has_bias=1, bias_dtype=kb.F16))
    every = dict(a=at, b=at, c=at, offsets=at, a_scale=at, b_scale=at, bias=at)
    for name, off in (("c", 1), ("offsets", 4), ("a_scale", 2), ("b_scale", 1), ("bias", 1)):
        with pytest.raises(kb.KudnnError) as e:
            op.run(**dict(every, **{name: at + off}))
        assert e.value.status == 2
    op = kb.Grouped(small(dtype=kb.BF16))
    for name, off in (("a", 1), ("b", 1), ("c", 1), ("offsets", 2)):
        with pytest.raises(kb.KudnnError) as e:
            op.run(**dict(dict(a=at, b=at, c=at, offsets=at), **{name: at + off}))
        assert e.value.status == 2


@pytest.mark.parametrize("c_sm,c_sn,status", [
    (256, 1, 0), (255, 1, 2), (1, 8, 0), (1, 7, 2), (1, 1, 2), (0, 1, 2), (1, 0, 2), (2, 16, 0), (2, 15, 0), (6, 4, 2), (257, 8, 0), (255, 8, 0),
])
def test_results_that_share_memory_are_refused(c_sm, c_sn, status):
    """8 x 256 of them; held against all addresses."""
    shared = len({r * c_sm + n * c_sn for r in range(8) for n in range(256)}) < 8 * 256
    assert shared == (status != 0)
    d = small(c_sm=c_sm, c_sn=c_sn)
    assert kb.library().kudnn_b200_grouped_validate(ctypes.byref(d)) == status
    one = small(rows=1, c_sm=0)
    assert kb.library().kudnn_b200_grouped_validate(ctypes.byref(one)) == 0
