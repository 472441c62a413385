"""Layer norm where its persistent kernels take their other paths, held to the
bounds of test_layer_norm_gpu: rows enough for several rows side by side in a
CTA-wide group, for a second turn of the loop with its look-ahead, for both at
odd counts; captured in a graph; on two streams at once."""

import pytest
import torch
from test_layer_norm_gpu import check, run

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,D,dtype,rdtype", [
    # a CTA a row, several rows a turn (from 2368 rows of 256 vectors on, 4736 of 128, 9472 of 64)
    (2401, 2048, BF16, None), (2401, 2048, BF16, F32), (2401, 2048, BF16, BF16), (4801, 1024, BF16, None),
    (9601, 512, BF16, F32), (2401, 1024, F32, None), (2401, 1024, F32, F32), (4801, 512, F32, None),
    # just below those counts: one row a turn, many turns
    (2367, 2048, BF16, None), (2367, 2048, BF16, F32), (2367, 1024, F32, F32),
    # a warp a row or less, second turns (from 28416 rows of 32 vectors on, 56832 of 16, 113664 of 8)
    (29001, 256, BF16, None), (60001, 128, BF16, None), (60001, 128, BF16, F32), (120001, 64, BF16, BF16),
    (29001, 128, F32, None), (60001, 64, F32, F32),
    # two and four vectors a thread, CTAs of 512, odd widths, over several turns
    (2001, 4096, BF16, None), (2001, 8192, BF16, F32), (2001, 4096, F32, None), (601, 16384, BF16, None),
    (601, 8192, F32, F32), (3001, 1001, BF16, None), (3001, 1001, F32, F32), (1501, 4095, BF16, F32), (401, 9001, BF16, None)])
def test_many_rows(gdn2, rows, D, dtype, rdtype):
    got, want = run(gdn2, (rows, D), dtype, F32, rdtype, seed=rows + D)
    if dtype == F32:  # the weights' gradients are sums of `rows` terms: rounding errors grow with their root
        for n in ("dw", "db"):
            err = float((got.pop(n).double() - want[n]).norm() / want[n].norm())
            assert err <= 5e-6 * max(1.0, rows / 3000) ** 0.5, (n, err)
    check(got, want)


def test_same_bits_twice_are_the_right_ones(gdn2):
    got, want = run(gdn2, (5000, 512), BF16, F32, F32)
    again, _ = run(gdn2, (5000, 512), BF16, F32, F32)
    check(got, want)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("rows,D", [(5, 2048), (300, 1001), (40000, 128)])
def test_graph_capture(gdn2, rows, D):
    """Forward and backward captured in a CUDA graph and replayed on new inputs."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x, res, dy, ds = r(rows, D).bfloat16(), r(rows, D), r(rows, D).bfloat16(), r(rows, D)
    w, b = r(D), r(D)

    def step(x, w, b, res, dy, ds):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, res)]
        out = gdn2.layer_norm(*leaves[:3], residual=leaves[3])
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (dy, ds))]

    want = step(x, w, b, res, dy, ds)
    static = [torch.zeros_like(t) for t in (x, w, b, res, dy, ds)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*static)
    for s, t in zip(static, (x, w, b, res, dy, ds)):
        s.copy_(t)
    g.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_two_streams_at_once(gdn2):
    """Calls in flight on two streams do not share scratch memory."""
    data = [torch.randn(4000, 1000 + 24 * i, device="cuda").bfloat16() for i in range(2)]

    def step(x):
        x = x.detach().requires_grad_()
        w = torch.ones(x.shape[1], device="cuda", requires_grad=True)
        y = gdn2.layer_norm(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), y.detach())]

    want = [step(x) for x in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[] for _ in data]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
