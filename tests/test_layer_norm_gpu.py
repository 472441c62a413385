"""GPU parity of layer norm, forward and backward, against its formula in 64 bits.

Tolerances (relative 2-norm): a bf16 result is rounded once, at most its unit
roundoff 2^-8 (8 significant bits); fp32 results are sums of at most a few thousand terms in fp32 and an
rsqrt of two ulp: below 5e-6.  Where x lies on a large mean, the differences
s - mean lose the bits that the mean takes from them: bounds scale with it.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = {torch.bfloat16: 2.0 ** -8, torch.float32: 5e-6}


def formula(x, w, b, eps, r, dy, ds, rdtype):
    """Outputs and gradients by the closed formulas, in float64."""
    s = x.double()
    if r is not None:
        s = (x.float() + r.float()).to(rdtype).double()  # what is stored
    mean = s.mean(-1, keepdim=True)
    var = ((s - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    hat = (s - mean) * rstd
    y = hat * (1 if w is None else w.double()) + (0 if b is None else b.double())
    d = dy.double() * (1 if w is None else w.double())
    dx = rstd * (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double()
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    return dict(y=y, s=s, dx=dx, dr=dx, dx_terms=rstd * d, dw=flat(dy.double() * hat).sum(0), db=flat(dy.double()).sum(0))


def rel(a, e):
    a, e = a.detach().double().cpu(), e.detach().double().cpu()
    assert a.shape == e.shape and torch.isfinite(a).all()
    return float((a - e).norm() / e.norm()) if e.norm() > 0 else float(a.norm())


def run(gdn2, shape, dtype, wdtype, rdtype=None, affine="wb", seed=0, mean=0.5, eps=1e-5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    D = shape[-1]
    x = (r(*shape) + mean).to(dtype).requires_grad_()
    w = (1 + 0.3 * r(D)).to(wdtype).requires_grad_() if "w" in affine else None
    b = (0.3 * r(D)).to(wdtype).requires_grad_() if "b" in affine else None
    res = r(*shape).to(rdtype).requires_grad_() if rdtype is not None else None
    dy, ds = r(*shape).to(dtype), r(*shape).to(rdtype) if rdtype is not None else None
    out = gdn2.layer_norm(x, w, b, eps=eps, residual=res)
    leaves = {n: t for n, t in (("dx", x), ("dw", w), ("db", b), ("dr", res)) if t is not None}
    outs, cots = ((out,), (dy,)) if res is None else (out, (dy, ds))
    grads = torch.autograd.grad(outs, list(leaves.values()), cots)
    got = dict(zip(leaves, grads), y=outs[0])
    if res is not None:
        got["s"] = outs[1]
    want = formula(*(None if t is None else t.detach() for t in (x, w, b)), eps,
                   None if res is None else res.detach(), dy, ds, rdtype)
    return got, want


def check(got, want, k=1.0):
    for n, t in got.items():
        assert rel(t, want[n]) <= k * TOL[t.dtype], f"{n}: {rel(t, want[n]):.2e} ({t.dtype})"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,D", [
    (1, 2), (3, 7), (5, 64), (300, 64), (17, 128), (1, 2048), (33, 2048), (129, 100), (40, 1001), (9, 4096), (7, 4608),
    (6, 8192), (3, 8200), (2, 16384), (2, 32768), (2, 32767), (2, 12289), (1000, 72)])
def test_shapes(gdn2, rows, D, dtype):
    got, want = run(gdn2, (rows, D), dtype, torch.float32, seed=rows + D)
    if D == 2:  # hat is nearly +-1 and dx cancels to eps / var of its terms rstd dy w: held against those
        dx, terms = got.pop("dx"), want["dx_terms"]
        assert float((dx.double() - want["dx"]).norm()) <= TOL[torch.float32] * float(terms.norm()) + \
            (TOL[dtype] * float(want["dx"].norm()) if dtype == torch.bfloat16 else 0.0)
    check(got, want)


@pytest.mark.parametrize("dtype,wdtype,rdtype", [
    (torch.bfloat16, torch.float32, None), (torch.bfloat16, torch.bfloat16, None),
    (torch.bfloat16, torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16),
    (torch.float32, torch.float32, torch.float32), (torch.float32, torch.bfloat16, None)])
@pytest.mark.parametrize("shape", [(2, 50, 256), (4, 3, 5, 64), (31, 333), (2000, 1024)])
@pytest.mark.parametrize("affine", ["wb", "w", "b", ""])
def test_types_and_residuals(gdn2, shape, dtype, wdtype, rdtype, affine):
    check(*run(gdn2, shape, dtype, wdtype, rdtype, affine))


def test_large_mean(gdn2):
    """Rows on a mean of 1000 times their spread: two passes keep the spread's bits (x itself holds 2^-24 of the mean)."""
    got, want = run(gdn2, (50, 640), torch.float32, torch.float32, mean=1000.0)
    check(got, want, 1000 * 2 ** -24 / 5e-6 + 1)


def test_one_element_and_constant_rows(gdn2):
    """No spread: y is the bias and nothing flows to x; eps keeps it finite."""
    for x in (torch.randn(4, 1, device="cuda"), torch.full((4, 37), 3.0, device="cuda")):
        x.requires_grad_()
        b = torch.randn(x.shape[1], device="cuda")
        y = gdn2.layer_norm(x, torch.ones_like(b), b)
        (dx,) = torch.autograd.grad(y.sum() * 2, x)
        assert torch.equal(y, b.expand_as(y)) and dx.abs().max() < 1e-2


def test_rows_do_not_mix(gdn2):
    """A NaN row and an inf row leave the others (and only them) as they were."""
    for D in (64, 100, 2048):
        x = torch.randn(40, D, device="cuda").bfloat16()
        y = gdn2.layer_norm(x)
        x2 = x.clone()
        x2[3, 5], x2[17, 1] = float("nan"), float("inf")
        y2 = gdn2.layer_norm(x2)
        keep = [i for i in range(40) if i not in (3, 17)]
        assert torch.equal(y[keep], y2[keep]) and not torch.isfinite(y2[3]).any()


def test_empty_strided_and_unaligned(gdn2):
    w = torch.randn(96, device="cuda", requires_grad=True)
    x = torch.zeros(0, 96, device="cuda", requires_grad=True)
    y = gdn2.layer_norm(x, w, w.detach())
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 96) and not dw.any()
    x = torch.randn(50, 200, device="cuda").bfloat16()
    for view in (x[:, 3:99], x[::2, 8:104], x[:, 96:192].t().contiguous().t()):
        assert torch.equal(gdn2.layer_norm(view, w.detach()), gdn2.layer_norm(view.clone(
            memory_format=torch.contiguous_format), w.detach()))
    flat = torch.randn(1 + 64 * 128, device="cuda").bfloat16()  # a contiguous tensor off the 16-byte grid
    assert rel(gdn2.layer_norm(flat[1:].view(64, 128)), gdn2.layer_norm(flat[1:].view(64, 128).clone())) <= 1e-3


def test_unused_outputs(gdn2):
    """Only one of (y, s) used: the other's cotangent counts as zero."""
    x = torch.randn(20, 256, device="cuda").bfloat16().requires_grad_()
    r = torch.randn(20, 256, device="cuda").requires_grad_()
    w = torch.ones(256, device="cuda", requires_grad=True)
    y, s = gdn2.layer_norm(x, w, residual=r)
    dx, dr = torch.autograd.grad(s.sum(), (x, r), retain_graph=True)
    assert torch.equal(dr, torch.ones_like(dr)) and torch.equal(dx, torch.ones_like(dx))
    dy = torch.randn_like(y)
    want = formula(x.detach(), w.detach(), None, 1e-5, r.detach(), dy, None, torch.float32)
    (dr,) = torch.autograd.grad(y, r, dy)
    assert rel(dr, want["dr"]) <= TOL[torch.float32]


def test_same_bits_twice(gdn2):
    a, _ = run(gdn2, (5000, 512), torch.bfloat16, torch.float32, torch.float32)
    b, _ = run(gdn2, (5000, 512), torch.bfloat16, torch.float32, torch.float32)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_gradients_against_differences(gdn2):
    """Central differences along random directions: third-order terms of a step of 1e-2 and fp32 rounding, 1e-3."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    t = dict(x=r(12, 200), w=r(200), b=r(200), r=r(12, 200))
    t = {n: x.requires_grad_() for n, x in t.items()}
    dy, ds = r(12, 200).double(), r(12, 200).double()

    def loss(t):
        y, s = gdn2.layer_norm(t["x"], t["w"], t["b"], residual=t["r"])
        return (y.double() * dy).sum() + (s.double() * ds).sum()

    grads = dict(zip(t, torch.autograd.grad(loss(t), list(t.values()))))
    for n in t:
        u = r(*t[n].shape)
        with torch.no_grad():
            slope = float((loss({**t, n: t[n] + 1e-2 * u}) - loss({**t, n: t[n] - 1e-2 * u})) / 2e-2)
        mine, size = float((grads[n].double() * u.double()).sum()), float(grads[n].double().norm())
        assert abs(slope - mine) <= 1e-3 * size, (n, slope, mine)


def test_module_and_refusals(gdn2):
    m = gdn2.LayerNorm(128).cuda()
    ref = torch.nn.LayerNorm(128).cuda()
    ref.load_state_dict(m.state_dict())
    x = torch.randn(9, 128, device="cuda")
    assert rel(m(x), ref(x).double()) <= TOL[torch.float32]
    z = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    for err, a, kw in [
        (TypeError, z(4, 8, dt=torch.float16), {}), (ValueError, z(4, 32769), {}), (ValueError, z(4, 0), {}),
        (ValueError, z(4, 8), dict(weight=z(9))), (TypeError, z(4, 8), dict(weight=z(8, dt=torch.float64))),
        (TypeError, z(4, 8), dict(weight=z(8), bias=z(8, dt=torch.bfloat16))),
        (ValueError, z(4, 8), dict(residual=z(4, 9))), (TypeError, z(4, 8), dict(residual=z(4, 8, dt=torch.bfloat16))),
        (ValueError, z(4, 8), dict(weight=torch.zeros(8))),
    ]:
        with pytest.raises(err):
            gdn2.layer_norm(a, **kw)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        gdn2.layer_norm(torch.zeros(4, 8))
