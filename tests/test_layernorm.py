"""Layer normalisation and its gradient, against the definition in 64 bits.

Tolerances, u = 2^-24: a sum of n values in fp32 is off by at most d u times the sum of their magnitudes, where d is how many additions stand
behind one another.  A thread adds up to 32 values of a row (axis / 512 in the general kernel), 9 exchanges follow: d = 48 + axis / 512 covers
that and the roundings of each summand.  From there, for every element,
  mean      d u mean|x|
  variance  (d + 4) u v + (off mean)^2
  xh        off mean * r + |xh| (off v / (2 v) + 6 u)
  y         |scale| (off xh) + 2 u (|scale xh| + |shift|) + half a step of y's type
  dx        (d + 16) u r (|g| + mean|g| + |xh| mean|g xh|) + half a step; the statistics are given, so xh is off by 5 u |xh| only
  dscale    (e + 8) u sum|dy xh|, dshift e u sum|dy|, e = rows / 100 + 100: a CTA's rows one after the other (at least 148 CTAs or as many as
            rows, of four rows at a time or one), then an eighth of at most 592 sets, 8 of those, 4 warps
and half a step of subnormal results."""
import pytest
import torch

import kudnn_b200 as kb

CODE = {torch.float32: kb.F32, torch.float16: kb.F16, torch.bfloat16: kb.BF16}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
EPS = 1e-5
gpu = pytest.mark.gpu


def half_step(dtype, v):
    info = torch.finfo(dtype)
    return info.eps / 2 * v.abs() + info.tiny * info.eps / 2


def values(rows, axis, dtype, seed=0, mean=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, axis), generator=gen, device="cuda")
    x[:, :: max(1, axis // 3)] *= 20.0
    return (x + mean).to(dtype)


def params(axis, dtype, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (1 + 0.2 * torch.randn(axis, generator=gen, device="cuda")).to(dtype), (0.3 * torch.randn(axis, generator=gen, device="cuda")).to(dtype)


def place(t, offset, ld, fill):
    """t at a pitch of ld elements, `offset` elements behind a 512-byte boundary, in memory full of `fill`."""
    rows, axis = t.shape
    store = torch.full((offset + rows * ld + 8,), fill, dtype=t.dtype, device=t.device)
    view = store[offset:offset + rows * ld].view(rows, ld)[:, :axis]
    view.copy_(t)
    return store, view


def forward(x, scale=None, shift=None, mean=None, variance=None, out=None, stream=None, eps=EPS):
    rows, axis = x.shape
    given = mean is not None
    y = torch.empty((rows, axis), dtype=x.dtype, device="cuda") if out is None else out
    kind = x.dtype if scale is None and shift is None else (scale if scale is not None else shift).dtype
    desc = kb.make_layernorm_desc(rows, axis, CODE[x.dtype], param_dtype=CODE[kind], has_scale=scale is not None, has_shift=shift is not None,
                                  given_stats=given, eps=eps, x_ld=x.stride(0), y_ld=y.stride(0))
    if not given:
        mean, variance = torch.full((rows,), -7.0, device="cuda"), torch.full((rows,), -7.0, device="cuda")
    kb.layernorm(desc, x, y, scale, shift, mean, variance, stream=stream)
    return y, mean, variance


def backward(x, dy, scale, mean, variance, out=None, wanted=(True, True, True), given=False, kind=None, stream=None, eps=EPS):
    rows, axis = x.shape
    kind = kind or (x.dtype if scale is None else scale.dtype)
    dx = torch.empty((rows, axis), dtype=x.dtype, device="cuda") if out is None else out
    dscale, dshift = [torch.full((axis,), -7.0, device="cuda").to(kind) for _ in range(2)]
    desc = kb.make_layernorm_desc(rows, axis, CODE[x.dtype], param_dtype=CODE[kind], has_scale=scale is not None, given_stats=given, eps=eps,
                                  x_ld=x.stride(0), dy_ld=dy.stride(0), dx_ld=dx.stride(0))
    size = kb.layernorm_backward_workspace(desc)
    space = torch.full((size // 4 + 3 * axis + 64,), float("nan"), device="cuda")
    kb.layernorm_backward(desc, x, dy, scale, mean, variance, *[t if w else None for t, w in zip((dx, dscale, dshift), wanted)], space, size, stream=stream)
    if stream is None:
        assert bool(torch.isnan(space[size // 4:]).all()), "written beyond the workspace"
    return dx, dscale, dshift


def check_forward(got, x, scale, shift, mean=None, variance=None, eps=EPS):
    y, m, v = got
    axis = x.shape[1]
    d = 48 + axis / 512
    x = x.double()
    a = torch.ones(axis, dtype=torch.float64, device="cuda") if scale is None else scale.double()
    b = torch.zeros(axis, dtype=torch.float64, device="cuda") if shift is None else shift.double()
    if mean is None:
        m64, v64 = x.mean(dim=1), x.var(dim=1, unbiased=False)
        off_m = d * U * x.abs().mean(dim=1) + 1e-44
        off_v = (d + 4) * U * v64 + off_m ** 2
        assert torch.all((m.double() - m64).abs() <= off_m)
        assert torch.all((v.double() - v64).abs() <= off_v + 1e-44)
    else:
        m64, v64 = mean.double(), variance.double()
        off_m, off_v = torch.zeros_like(m64), torch.zeros_like(v64)
    r = (1 / (v64 + eps).sqrt())[:, None]
    xh = (x - m64[:, None]) * r
    off = off_m[:, None] * r + xh.abs() * (off_v[:, None] * r * r / 2 + 6 * U)
    want = xh * a + b
    assert torch.all((y.double() - want).abs() <= a.abs() * off + 2 * U * ((a * xh).abs() + b.abs()) + half_step(y.dtype, want) * (1 + 2 ** -10))


def check_backward(got, x, dy, scale, mean, variance, given=False, eps=EPS):
    dx, dscale, dshift = got
    rows, axis = x.shape
    d, e = 48 + axis / 512, rows / 100 + 100
    x, dy = x.double(), dy.double()
    a = torch.ones(axis, dtype=torch.float64, device="cuda") if scale is None else scale.double()
    r = (1 / (variance.double() + eps).sqrt())[:, None]
    xh, g = (x - mean.double()[:, None]) * r, dy * a
    along = (g * xh).mean(dim=1, keepdim=True)
    want = r * g if given else r * (g - g.mean(dim=1, keepdim=True) - xh * along)
    size = g.abs() if given else g.abs() + g.abs().mean(dim=1, keepdim=True) + xh.abs() * (g * xh).abs().mean(dim=1, keepdim=True)
    assert torch.all((dx.double() - want).abs() <= (d + 16) * U * r * size + half_step(dx.dtype, want) * (1 + 2 ** -10))
    for t, terms, more in ((dscale, dy * xh, 8), (dshift, dy, 0)):
        want = terms.sum(dim=0)
        assert torch.all((t.double() - want).abs() <= (e + more) * U * terms.abs().sum(dim=0) + half_step(t.dtype, want) * (1 + 2 ** -10))


SHAPES = [(1, 1), (5, 2), (3, 7), (4, 8), (9, 9), (33, 64), (2, 127), (700, 128), (7, 255), (129, 256), (6, 257), (5000, 72), (12, 513), (257, 1000),
          (3, 1024), (40, 1025), (8, 1040), (311, 2050), (70, 4096), (37, 4099), (1300, 1028), (6, 8192), (9, 8195), (3, 16384), (5, 20001),
          (2, 32768), (2, 40000)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,axis", SHAPES)
def test_forward(cuda_device, dtype, rows, axis):
    x = values(rows, axis, dtype)
    for kind in {dtype, torch.float32}:
        scale, shift = params(axis, kind)
        check_forward(forward(x, scale, shift), x, scale, shift)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,axis", SHAPES)
def test_backward(cuda_device, dtype, rows, axis):
    x, dy = values(rows, axis, dtype), values(rows, axis, dtype, seed=5, mean=0.1)
    for kind in {dtype, torch.float32}:
        scale, _ = params(axis, kind)
        mean, variance = x.double().mean(dim=1).float(), x.double().var(dim=1, unbiased=False).float()
        check_backward(backward(x, dy, scale, mean, variance), x, dy, scale, mean, variance)


@gpu
@pytest.mark.parametrize("rows,axis", [(1, 130), (70, 130), (2500, 40), (33, 2050), (20, 5000)])
def test_without_parameters_and_with_given_statistics(cuda_device, rows, axis):
    x, dy = values(rows, axis, torch.bfloat16), values(rows, axis, torch.bfloat16, seed=5)
    scale, shift = params(axis, torch.float32)
    check_forward(forward(x), x, None, None)
    check_forward(forward(x, scale), x, scale, None)
    check_forward(forward(x, None, shift), x, None, shift)
    mean, variance = torch.linspace(-1, 1, rows, device="cuda"), torch.linspace(0.5, 9, rows, device="cuda")
    kept = mean.clone(), variance.clone()
    check_forward(forward(x, scale, shift, mean, variance), x, scale, shift, mean, variance)
    check_backward(backward(x, dy, scale, mean, variance, given=True), x, dy, scale, mean, variance, given=True)
    check_backward(backward(x, dy, None, mean, variance), x, dy, None, mean, variance)
    assert torch.equal(mean, kept[0]) and torch.equal(variance, kept[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("axis", [5, 65, 384, 1000, 2048])
@pytest.mark.parametrize("offset,ld", [(0, 0), (1, 0), (3, 1), (4, 4), (7, 8), (8, 3)])
def test_pitch_and_alignment(cuda_device, dtype, axis, offset, ld):
    """Rows that begin anywhere, NaN between them; nothing but the rows is written."""
    rows, ld = 45, axis + ld
    x0, dy0 = values(rows, axis, dtype), values(rows, axis, dtype, seed=5)
    (_, x), (_, dy) = place(x0, offset, ld, float("nan")), place(dy0, offset, ld, float("nan"))
    scale, shift = params(axis, dtype)
    store, y = place(torch.zeros_like(x0), offset, ld, 3.0)
    y, mean, variance = forward(x, scale, shift, out=y)
    check_forward((y, mean, variance), x0, scale, shift)
    y.fill_(3.0)
    assert bool((store == 3.0).all())
    store, dx = place(torch.zeros_like(x0), offset, ld, 3.0)
    got = backward(x, dy, scale, mean, variance, out=dx)
    check_backward(got, x0, dy0, scale, mean, variance)
    dx.fill_(3.0)
    assert bool((store == 3.0).all())
    # results that begin elsewhere than the rows
    check_forward(forward(x, scale, shift), x0, scale, shift)
    check_backward(backward(x, dy0, scale, mean, variance), x0, dy0, scale, mean, variance)


@gpu
@pytest.mark.parametrize("axis", [100, 1030, 4096, 40000])
def test_in_place(cuda_device, axis):
    x, dy = values(300, axis, torch.bfloat16), values(300, axis, torch.bfloat16, seed=5)
    scale, shift = params(axis, torch.bfloat16)
    y, mean, variance = forward(x, scale, shift)
    same = x.clone()
    assert torch.equal(forward(same, scale, shift, out=same)[0], y)
    dx, dscale, dshift = backward(x, dy, scale, mean, variance)
    for take in (0, 1):
        pair = [x.clone(), dy.clone()]
        got = backward(*pair, scale, mean, variance, out=pair[take])
        assert torch.equal(pair[take], dx) and torch.equal(got[1], dscale) and torch.equal(got[2], dshift)


@gpu
@pytest.mark.parametrize("rows,axis", [(3000, 96), (400, 2050)])
def test_the_gradients_that_are_wanted(cuda_device, rows, axis):
    x, dy = values(rows, axis, torch.float16), values(rows, axis, torch.float16, seed=5)
    scale, _ = params(axis, torch.float32)
    _, mean, variance = forward(x, scale)
    whole = backward(x, dy, scale, mean, variance, out=torch.full_like(x, -7.0))
    for wanted in ((True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, False, False)):
        got = backward(x, dy, scale, mean, variance, out=torch.full_like(x, -7.0), wanted=wanted)
        for g, w, flag in zip(got, whole, wanted):
            assert torch.equal(g, w) if flag else bool((g == -7.0).all())


@gpu
def test_rows_do_not_reach_into_others(cuda_device):
    """Infinities, NaN and constant rows stay where they are; the type's largest values do not overflow where fp32 holds their squares."""
    x = values(9, 523, torch.bfloat16)
    x[2, 5], x[4, 7], x[6] = float("nan"), float("inf"), 3.0
    scale, shift = params(523, torch.bfloat16)
    y, mean, variance = forward(x, scale, shift)
    clean = [r for r in range(9) if r not in (2, 4)]
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[4]).all())
    check_forward((y[clean], mean[clean], variance[clean]), x[clean], scale, shift)
    assert bool((variance[6] == 0).all()) and torch.allclose(y[6].float(), shift.float())
    far = torch.tensor([[6e4, -6e4] * 40], device="cuda").half()
    check_forward(forward(far), far, None, None)


@gpu
def test_no_rows(cuda_device):
    x = torch.empty((0, 77), device="cuda")
    scale, shift = params(77, torch.float32)
    assert forward(x, scale, shift)[0].shape == (0, 77)
    _, dscale, dshift = backward(x, x, scale, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"))
    assert bool((dscale == 0).all()) and bool((dshift == 0).all())


@gpu
def test_gradients_against_differences(cuda_device):
    """The derivative of sum(w y) along random directions, by differences of the fp32 forward pass.  A difference over +-h is off by
    h^2 |f'''| / 6, here below 1e-3 of the derivative's scale for h = 2^-7, and by the forward pass's rounding, 2^-20 of sum|w y| over h."""
    rows, axis, h = 6, 150, 2.0 ** -7
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, w, dirx = [torch.randn((rows, axis), generator=gen, device="cuda") for _ in range(3)]
    scale, shift = params(axis, torch.float32)
    dira, dirb = [torch.randn(axis, generator=gen, device="cuda") for _ in range(2)]

    def loss(t, a, b):
        return float((forward(t, a, b)[0].double() * w.double()).sum())

    y, mean, variance = forward(x, scale, shift)
    dx, dscale, dshift = backward(x, w, scale, mean, variance)
    size = float((w * y).abs().sum())
    for grad, direction, up, down in ((dx, dirx, loss(x + h * dirx, scale, shift), loss(x - h * dirx, scale, shift)),
                                      (dscale, dira, loss(x, scale + h * dira, shift), loss(x, scale - h * dira, shift)),
                                      (dshift, dirb, loss(x, scale, shift + h * dirb), loss(x, scale, shift - h * dirb))):
        along = float((grad.double() * direction.double()).sum())
        assert abs((up - down) / (2 * h) - along) <= 1e-3 * float((grad * direction).abs().sum()) + 2.0 ** -20 * size / h


@gpu
def test_streams_graphs_and_repetition(cuda_device):
    """Two streams at once, and a captured pass on other values: the same bits as alone."""
    sets = [(values(900, 1026, torch.bfloat16, seed=s), values(900, 1026, torch.bfloat16, seed=s + 9)) for s in (1, 2)]
    scale, shift = params(1026, torch.float32)

    def both(x, dy, stream):
        y, mean, variance = forward(x, scale, shift, stream=stream)
        return (y,) + backward(x, dy, scale, mean, variance, stream=stream)

    want = [both(x, dy, torch.cuda.current_stream().cuda_stream) for x, dy in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        got = []
        for (x, dy), s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(both(x, dy, s.cuda_stream))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    x, dy = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(x, dy, torch.cuda.current_stream().cuda_stream)
    for k in (1, 0):
        x.copy_(sets[k][0])
        dy.copy_(sets[k][1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want[k]))


def desc(**more):
    return kb.make_layernorm_desc(more.pop("rows", 4), more.pop("axis", 8), more.pop("dtype", kb.BF16), **more)


@pytest.mark.parametrize("d,status", [
    (desc(rows=-1), 2), (desc(axis=0), 1), (desc(axis=2 ** 31), 1), (desc(dtype=kb.S8, param_dtype=kb.S8), 1), (desc(param_dtype=kb.F16), 1),
    (desc(eps=-1.0), 2), (desc(eps=float("nan")), 2), (desc(eps=float("inf")), 2), (desc(y_ld=7), 2), (desc(dx_ld=7), 2), (desc(x_ld=-8), 2),
])
def test_descriptors_that_are_refused(d, status):
    with pytest.raises(kb.KudnnError) as e:
        kb.layernorm(d, 16, 16)
    assert e.value.status == status
    with pytest.raises(kb.KudnnError):
        kb.layernorm_backward_workspace(d)


def test_flags_of_the_reference_that_are_refused():
    d = desc()
    d.flags |= 8  # a fused relu
    with pytest.raises(kb.KudnnError) as e:
        kb.layernorm(d, 16, 16)
    assert e.value.status == 1


@pytest.mark.parametrize("call", [
    lambda: kb.layernorm(desc(), None, 16), lambda: kb.layernorm(desc(), 16, None), lambda: kb.layernorm(desc(), 17, 16),
    lambda: kb.layernorm(desc(), 16, 17), lambda: kb.layernorm(desc(has_scale=True), 16, 16), lambda: kb.layernorm(desc(), 16, 16, 16),
    lambda: kb.layernorm(desc(has_shift=True), 16, 16), lambda: kb.layernorm(desc(), 16, 16, None, 16),
    lambda: kb.layernorm(desc(has_scale=True, param_dtype=kb.F32), 16, 16, 18), lambda: kb.layernorm(desc(given_stats=True), 16, 16),
    lambda: kb.layernorm(desc(), 16, 16, None, None, 18, 16),
    lambda: kb.layernorm_backward(desc(), 16, None, None, 16, 16, 16), lambda: kb.layernorm_backward(desc(), 16, 16, None, None, 16, 16),
    lambda: kb.layernorm_backward(desc(), 16, 16, None, 16, None, 16), lambda: kb.layernorm_backward(desc(), 16, 16, None, 16, 16, 17),
    lambda: kb.layernorm_backward(desc(), 16, 16, None, 16, 16, 16, 16), lambda: kb.layernorm_backward(desc(), 16, 16, None, 16, 16, 16, 16, 16, 16, 8),
    lambda: kb.layernorm_backward(desc(), 16, 16, None, 16, 16, 16, 16, 16, 18, 4 * 2 * 8 * 4),
    lambda: kb.layernorm_backward(desc(), 16, 16, None, 16, 16, 16, 17, 16, 16, 4 * 2 * 8 * 4),
])
def test_calls_that_are_refused(call):
    """On the host, ahead of any device: the addresses are made up."""
    with pytest.raises(kb.KudnnError) as e:
        call()
    assert e.value.status == 2


def test_workspace_grows_with_the_rows_up_to_a_bound():
    sizes = [kb.layernorm_backward_workspace(desc(rows=rows, axis=100)) for rows in (0, 1, 7, 592, 10 ** 6)]
    assert sizes == [0, 800, 5600, 473600, 473600]


@pytest.mark.parametrize("unused", [dict(dx_ld=0, dy_ld=0), dict(dx_ld=0)])
def test_pitches_that_a_forward_call_does_not_use_may_be_zero(unused):
    """On the host: refused for its y (misaligned), not for a dx that it does not write."""
    with pytest.raises(kb.KudnnError, match="aligned"):
        kb.layernorm(desc(**unused), 16, 17)
    with pytest.raises(kb.KudnnError, match="overlap"):
        kb.layernorm(desc(y_ld=0), 16, 16)


def test_pitches_that_a_gradient_does_not_use_may_be_zero():
    assert kb.layernorm_backward_workspace(desc(y_ld=0)) == 4 * 2 * 8 * 4
    with pytest.raises(kb.KudnnError, match="aligned"):
        kb.layernorm_backward(desc(y_ld=0), 16, 16, None, 16, 16, 17)
    with pytest.raises(kb.KudnnError, match="workspace"):  # dx is not wanted
        kb.layernorm_backward(desc(y_ld=0, dx_ld=0), 16, 16, None, 16, 16, None, 16)
    with pytest.raises(kb.KudnnError, match="overlap"):
        kb.layernorm_backward(desc(dx_ld=0), 16, 16, None, 16, 16, 16)


@gpu
def test_results_with_only_the_pitches_that_they_use(cuda_device):
    x, dy = values(5, 24, torch.float32), values(5, 24, torch.float32, seed=5)
    y, mean, variance = forward(x)
    want = backward(x, dy, None, mean, variance)
    again, dx, dscale, dshift = torch.empty_like(x), torch.empty_like(x), torch.empty(24, device="cuda"), torch.empty(24, device="cuda")
    kb.layernorm(kb.make_layernorm_desc(5, 24, kb.F32, eps=EPS, dy_ld=0, dx_ld=0), x, again)
    assert torch.equal(again, y)
    d = kb.make_layernorm_desc(5, 24, kb.F32, eps=EPS, y_ld=0)
    size = kb.layernorm_backward_workspace(d)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    kb.layernorm_backward(d, x, dy, None, mean, variance, dx, dscale, dshift, space, size)
    assert all(torch.equal(a, b) for a, b in zip((dx, dscale, dshift), want))
    d.dx_ld = 0
    dscale.zero_(), dshift.zero_()
    kb.layernorm_backward(d, x, dy, None, mean, variance, None, dscale, dshift, space, size)
    assert torch.equal(dscale, want[1]) and torch.equal(dshift, want[2])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,axis", [(5, 130), (40, 4096), (3, 8195), (2, 40000)])
def test_means_far_above_the_deviation(cuda_device, dtype, rows, axis):
    x = values(rows, axis, dtype, mean=1000.0)
    scale, shift = params(axis, torch.float32)
    got = forward(x, scale, shift)
    check_forward(got, x, scale, shift)
    dy = values(rows, axis, dtype, seed=5, mean=0.1)
    check_backward(backward(x, dy, scale, got[1], got[2]), x, dy, scale, got[1], got[2])


@gpu
def test_elements_beyond_2_to_the_31(cuda_device):
    """Two rows further apart than 32 bits count: x, y, dy and dx."""
    ld, axis = 2 ** 31 + 9, 1027
    near = values(2, axis, torch.float16)
    store, out = [torch.empty(ld + axis, dtype=torch.float16, device="cuda") for _ in range(2)]
    x, y = [torch.as_strided(t, (2, axis), (ld, 1)) for t in (store, out)]
    x.copy_(near)
    scale, shift = params(axis, torch.float32)
    _, mean, variance = got = forward(x, scale, shift, out=y)
    check_forward(got, near, scale, shift)
    dy = values(2, axis, torch.float16, seed=5)
    y.copy_(dy)
    check_backward(backward(x, y, scale, mean, variance, out=y), near, dy, scale, mean, variance)
