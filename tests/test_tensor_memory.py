"""Launches that cut K over clusters, on several streams at a time: none may keep tensor memory while it waits for its cluster."""
import pytest
import torch

import kudnn_b200 as kb

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("linears", [1, 2, 4])
def test_cut_launches_on_several_streams(cuda_device, monkeypatch, capfd, linears):
    """Products by group and linear ones whose CTAs are small enough to share an SM, but not its tensor memory."""
    monkeypatch.setenv("KUDNN_B200_TC_SPLITS", "4")
    monkeypatch.setenv("KUDNN_B200_DEBUG", "1")
    gen = torch.Generator(device="cuda").manual_seed(5)
    k = 2048
    x = torch.randn(24, k, generator=gen, device="cuda").bfloat16()
    jobs = []
    for i in range(4):
        n = 2304 - 256 * i
        w = (torch.randn(n, k, generator=gen, device="cuda") * 0.05).bfloat16()
        y = torch.empty(24, n, dtype=torch.bfloat16, device="cuda")
        if i < linears:
            op = kb.Linear(kb.make_desc(24, n, k, kb.BF16))
            op.force_kernel(kb.KERNEL_TC)
            jobs.append((op, (x, w, y), w, y))
        else:
            q, qw = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
            one = torch.ones(1, device="cuda")
            op = kb.Grouped(kb.make_grouped_desc(24, n, k, kb.E4M3, a_scale_strides=(0, 0), b_scale_strides=(0, 0, 0)))
            jobs.append((op, (q, qw, y, None, one, one), qw, y))
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(100):
        for (op, args, _, _), s in zip(jobs, streams):
            op.run(*args, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert "k splits 4," in capfd.readouterr().err
    for op, args, w, y in jobs:
        op.check()
        a, b = args[0].double(), w.double()
        limit = (k / 8 + 8) * 2.0 ** -23 * (a.abs() @ b.abs().t()) + 2.0 ** -8 * (a @ b.t()).abs()
        assert torch.all((y.double() - a @ b.t()).abs() <= limit)
