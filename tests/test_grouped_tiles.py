"""Every instance of the tensor-core kernel for products by group, whatever tile the sizes would choose: rows of a tile, the operand on the
M side, and how the blocks of K add up (in tensor memory; in registers with scales; in registers every four blocks, for fp32 results).

Reference and tolerance are those of tests/test_grouped.py.
"""
import pytest
import torch

import kudnn_b200 as kb
from tests.test_grouped import ACTS, Problem

gpu = pytest.mark.gpu

# operands, results that an instance is asked for, rows of a tile, rows on the M side
SCALED = [("e4m3", None, 32, False), ("e4m3", None, 64, False), ("e4m3", None, 128, False), ("e4m3", None, 256, False), ("e4m3", None, 256, True)]
PLAIN = [(dtype, dtype, rows, False) for dtype in ("bf16", "f16") for rows in (32, 64, 128, 256)]
DRAINED = [("bf16", "f32", rows, False) for rows in (32, 64, 128, 256)]  # K of more than four blocks of 64
INSTANCES = SCALED + PLAIN + DRAINED


def name_of(instance):
    return "%s-%s-%d%s" % (instance[0], instance[1] or "any", instance[2], "m" if instance[3] else "")


instances = pytest.mark.parametrize("instance", INSTANCES, ids=name_of)


class Tiled(Problem):
    """A problem on one instance."""

    def __init__(self, instance, rows, n, k, out=None, **more):
        dtype, own, self.tile, self.on_m = instance
        super().__init__(rows, n, k, dtype, out=own or out, **more)

    def run(self, kernel=kb.KERNEL_AUTO, stream=None):
        op = kb.Grouped(self.desc)
        op.force_tile(self.tile, self.on_m)
        op.run(self.a, self.b, self.c, offsets=self.offsets, a_scale=self.a_scale, b_scale=self.b_scale, bias=self.bias, stream=stream)
        op.check(stream)
        self.kernel, (rows, on_m, self.splits) = op.last_kernel, op.last_tile
        assert (rows, on_m) == (self.tile, self.on_m)
        assert bool((self.store[:, self.n:] == 77.0).all()), "written beyond the columns"
        return self


@gpu
@pytest.mark.parametrize("instance,out", [(i, out) for i in INSTANCES for out in ("f32", "f16", "bf16") if i[1] in (None, out)],
                         ids=lambda v: v if isinstance(v, str) else name_of(v))
@pytest.mark.parametrize("c_ld", [264, 268, 301])  # rows on 32 bytes, on 8 or 16, on none
def test_results_bias_and_activation(cuda_device, instance, out, c_ld):
    sizes = [5, 0, 270, 33, 1]
    for act in sorted(ACTS):
        Tiled(instance, 309, 264, 528, out=out, sizes=sizes, act=act, bias="f32", c_ld=c_ld).check()
    for bias in (None, "f16", "bf16"):
        Tiled(instance, 309, 264, 528, out=out, sizes=sizes, bias=bias, c_ld=c_ld, act="silu").check()


@gpu
@instances
@pytest.mark.parametrize("n", [1, 31, 127, 129, 255, 257, 385, 500])
def test_cut_columns(cuda_device, instance, n):
    for k in (328, 520, 1100):
        Tiled(instance, 300, n, k, sizes=[100, 200], bias="f32").check()


@gpu
@instances
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 33, 63, 65, 127, 129, 255, 257, 511, 513, 1000])
def test_rows(cuda_device, instance, m):
    Tiled(instance, m, 200, 640).check()
    Tiled(instance, m, 200, 640, sizes=[0, m // 3, 0, m - m // 3], wide_offsets=True).check()


@gpu
@instances
@pytest.mark.parametrize("k", [1, 16, 127, 128, 129, 250, 257, 1024, 4100])
def test_lengths_of_k(cuda_device, instance, k):
    Tiled(instance, 150, 260, k, sizes=[20, 130], a_scale_by_row=k % 2 == 0).check()


@gpu
@instances
@pytest.mark.parametrize("offsets", [[0, 0, 0, 0], [3, 9, 9, 290], [0, 300, 10, 30], [-5, 7, 1000, 8], [60, 20, 10, 0], [0, 5, 2 ** 31 - 1, -2 ** 31]])
def test_rows_that_no_group_holds(cuda_device, instance, offsets):
    Tiled(instance, 300, 200, 528, offsets=offsets, act="sigmoid").check()
    Tiled(instance, 300, 300, 528, offsets=offsets, c_ld=305).check()


@gpu
@instances
def test_many_items_and_bands(cuda_device, instance):
    """More items than CTAs, and more row tiles of a group than one raster band has."""
    tile = instance[2]
    Tiled(instance, 18 * tile + 5, 2500, 640, sizes=[17 * tile + 3, 0, tile + 2]).check()
    Tiled(instance, 700, 1500, 640, sizes=[i % 14 for i in range(107)] + [8]).check()


@gpu
@pytest.mark.parametrize("instance", SCALED + DRAINED, ids=name_of)
def test_fp32_results_keep_their_bits(cuda_device, instance):
    """The norm of the error as in test_grouped.py."""
    p = Tiled(instance, 300, 384, 8192, sizes=[200, 100], out="f32").check()
    y, _ = p.exact()
    assert torch.linalg.vector_norm(p.c.double() - y) <= 2.0 ** -20 * torch.linalg.vector_norm(y)


@gpu
@instances
def test_what_is_not_finite_stays_in_its_row_or_column(cuda_device, instance):
    p = Tiled(instance, 300, 264, 528, sizes=[100, 0, 200])
    p.a[40, 3] = float("nan")
    p.b3[2, 200, 527] = float("nan")
    if p.dtype == "e4m3":
        p.a_scale.t()[299, 1] = float("inf")
    else:
        p.a[299, 7] = float("inf")
    p.run()
    want = torch.ones_like(p.c, dtype=torch.bool)
    want[40] = False
    want[100:, 200] = False
    want[299] = False
    assert torch.equal(torch.isfinite(p.c.float()), want)


@gpu
@instances
def test_the_same_bits_every_time(cuda_device, instance):
    p = Tiled(instance, 600, 2000, 1024, sizes=[590, 10])
    first = p.run().c.clone()
    for _ in range(5):
        assert torch.equal(p.run().c, first)


@gpu
@instances
def test_a_wait_that_runs_out(cuda_device, instance):
    p = Tiled(instance, 500, 600, 2048)
    op = kb.Grouped(p.desc)
    op.force_tile(p.tile, p.on_m)
    op.set_wait(20_000_000, 3)
    op.run(p.a, p.b, p.c, a_scale=p.a_scale, b_scale=p.b_scale)
    with pytest.raises(kb.KudnnError) as e:
        op.check()
    assert e.value.status == 5 and op.last_tile[:2] == (p.tile, p.on_m)
    p.check()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("splits,n,k", [(1, 18944, 1024), (2, 8960, 1024), (4, 4608, 2048), (4, 11008, 4096)])
def test_cuts_of_k(cuda_device, dtype, splits, n, k):
    for m, more in ((1, dict()), (13, dict(c_ld=n + 1)), (32, dict(bias="f32", act="gelu_erf"))):
        p = Tiled((dtype, None, 32, False), m, n, k, **more).check()
        assert p.splits == splits


@gpu
@pytest.mark.parametrize("dtype,out,rows,n,k,sizes,tile,on_m", [
    ("e4m3", "bf16", 40, 2000, 1000, None, 32, False), ("e4m3", "bf16", 300, 4097, 520, None, 64, False),
    ("e4m3", "bf16", 1000, 2300, 1000, None, 128, False), ("e4m3", "bf16", 2048, 4096, 512, None, 256, True),
    ("e4m3", "f32", 700, 2300, 520, [100, 0, 90, 80, 150, 80, 100, 100], 256, False),
    ("bf16", "bf16", 1, 2048, 8192, None, 256, False), ("bf16", "bf16", 1000, 300, 640, [4] * 250, 32, False),
    ("bf16", "bf16", 2400, 300, 640, [40] * 60, 64, False), ("bf16", "f32", 775, 1294, 1972, [60] * 12 + [55], 128, False),
    ("bf16", "f32", 2048, 4096, 512, None, 256, False),
])
def test_the_tile_that_the_sizes_choose(cuda_device, dtype, out, rows, n, k, sizes, tile, on_m):
    """Of 148 SMs."""
    p = Problem(rows, n, k, dtype, sizes=sizes, out=out).check()
    op = kb.Grouped(p.desc)
    op.run(p.a, p.b, p.c, offsets=p.offsets, a_scale=p.a_scale, b_scale=p.b_scale)
    assert op.last_tile[:2] == (tile, on_m)


def test_refusals():
    eight = kb.Grouped(kb.make_grouped_desc(8, 256, 256, kb.E4M3))
    sixteen = kb.Grouped(kb.make_grouped_desc(8, 256, 256, kb.BF16))
    for op, rows, on_m, status in ((eight, 16, False, 2), (eight, 512, False, 2), (eight, 128, True, 1), (sixteen, 256, True, 1)):
        with pytest.raises(kb.KudnnError) as e:
            op.force_tile(rows, on_m)
        assert e.value.status == status
    eight.force_tile(256, True)
    eight.force_tile(0)
    assert eight.last_tile == (0, False, 0)
    assert kb.library().kudnn_b200_grouped_last_tile(None, None, None, None) == 2
