"""GPU parity of the linear attention with a decay for each head against a
token-by-token restatement in 64 bits, differentiated by autograd.

Tolerances (relative 2-norm), from the roundings of each path:
* bf16 outputs and gradients: three roundings to bf16 (the decayed scores, the
  state operand, the result), each at most 2^-9 and 2^-9 / sqrt(3) in the rms;
  together 2^-9 = 2.0e-3 in the rms.  Twice that.
* fp32 results (everything of the fp32 path, and the final state and the
  initial state's gradient of the bf16 path): sums of a few hundred terms in
  fp32, or of products whose operands carry 16 bits or more: below 1e-5.
* the gradient of g is a difference of sums: its error is held against the
  magnitude of the terms, not of the difference.  Each term carries three
  roundings (the decayed scores and both states of a product), one rounding to
  8 significant bits being 1.7e-3 in the rms: together 2.9e-3, and twice that.
"""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.bfloat16: 4e-3, torch.float32: 1e-5}
STATE_TOL = 1e-5


def reference(q, k, v, g, scale, h0, lens):
    """o and the final states of sequences lying one after the other in each row; float64, differentiable."""
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    group = HV // H
    o, hts = [], []
    for b in range(B):
        at, rows = 0, []
        for n, L in enumerate(lens if lens is not None else [T]):
            S = (torch.zeros(HV, K, V, dtype=torch.double) if h0 is None
                 else h0[n if lens is not None else b])
            for t in range(at, at + L):
                if g is not None:
                    gt = g if g.ndim == 1 else g[b, t]
                    S = S * torch.exp(gt)[:, None, None]
                kt, qt = (x[b, t].repeat_interleave(group, 0) for x in (k, q))
                S = S + kt[:, :, None] * v[b, t][:, None, :]
                rows.append(scale * torch.einsum("hkv,hk->hv", S, qt))
            at += L
            hts.append(S)
        o.append(torch.stack(rows) if rows else torch.zeros(0, HV, V, dtype=torch.double))
    return torch.stack(o), torch.stack(hts) if hts else torch.zeros(0, HV, K, V, dtype=torch.double)


def rel(x, ref):
    x, ref = x.detach().double().cpu(), ref.detach().double()
    assert x.shape == ref.shape
    assert torch.isfinite(x).all()
    n = ref.norm()
    return float((x - ref).norm() / n) if n > 0 else float((x - ref).norm())


def make(seed, B, T, H, HV, K, V, dtype, decay, h0=False, N=None, strong=False):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    d = dict(q=r(B, T, H, K).to(dtype), k=r(B, T, H, K).to(dtype), v=r(B, T, HV, V).to(dtype), g=None, h0=None)
    if decay == "token":
        d["g"] = (-torch.nn.functional.softplus(r(B, T, HV)) * (8.0 if strong else 0.3)).to(dtype)
    elif decay == "head":
        d["g"] = -0.5 * torch.rand(HV, generator=gen) - 0.001
    if h0:
        d["h0"] = r(B if N is None else N, HV, K, V)
    d["do"], d["dht"] = r(B, T, HV, V).to(dtype), r(B if N is None else N, HV, K, V)
    return d


def run_both(gdn2, d, lens=None, scale=None, final=True, use_dht=True):
    names = [n for n in ("q", "k", "v", "g", "h0") if d[n] is not None]
    ref = {n: d[n].double().requires_grad_() for n in names}
    sc = d["q"].shape[-1] ** -0.5 if scale is None else scale
    o, ht = reference(ref["q"], ref["k"], ref["v"], ref.get("g"), sc, ref.get("h0"), lens)
    outs, cots = [o], [d["do"].double()]
    if use_dht:
        outs, cots = outs + [ht], cots + [d["dht"].double()]
    grads = torch.autograd.grad(outs, list(ref.values()), cots, allow_unused=True)
    want = dict(o=o, ht=ht, **{"d" + n: (x if x is not None else torch.zeros_like(ref[n]))
                               for n, x in zip(names, grads)})
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0).cuda()
    own = {n: d[n].cuda().requires_grad_() for n in names}
    o, ht = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own.get("g"), scale=scale,
                                   initial_state=own.get("h0"), output_final_state=final, cu_seqlens=cu)
    outs, cots = [o], [d["do"].cuda()]
    if use_dht:
        outs, cots = outs + [ht], cots + [d["dht"].cuda()]
    grads = torch.autograd.grad(outs, list(own.values()), cots)
    got = dict(o=o, ht=ht, **{"d" + n: x for n, x in zip(names, grads)})
    with torch.no_grad():  # nothing kept for a backward: the prompt's form, with and without the final state
        got["o_p"], got["ht_p"] = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own.get("g"), scale=scale,
                                                         initial_state=own.get("h0"), output_final_state=True,
                                                         cu_seqlens=cu)
        got["o_n"], none = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own.get("g"), scale=scale,
                                                  initial_state=own.get("h0"), cu_seqlens=cu)
        assert none is None
    want.update(o_p=want["o"], ht_p=want["ht"], o_n=want["o"])
    assert gdn2._lib.device_fault_read() == 0
    return got, want


def dg_mass(d, want):
    """The size of what dg adds up, per element: |q . dq| + |k . dk| at each token, summed over a chunk."""
    m = (d["q"].double() * want["dq"]).sum(-1).abs().mean() + (d["k"].double() * want["dk"]).sum(-1).abs().mean()
    return float(m)


def check(got, want, d, dtype, names=("o", "ht", "dq", "dk", "dv", "dg", "dh0", "o_p", "ht_p", "o_n")):
    for n in names:
        if n not in got or got[n] is None:
            continue
        tol = STATE_TOL if n in ("ht", "ht_p", "dh0") else TOL[dtype]
        if n == "dg":
            err = (got[n].detach().double().cpu() - want[n]).norm() / want[n].numel() ** 0.5
            ref = want[n].norm() / want[n].numel() ** 0.5
            scale = max(float(ref), dg_mass(d, want) * (1.0 if d["g"].ndim == 3 else want["dq"].shape[1] ** 0.5))
            t = 6e-3 if dtype == torch.bfloat16 else TOL[dtype]
            assert float(err) <= t * scale, f"dg: {float(err):.3e} of {scale:.3e}"
        else:
            assert rel(got[n], want[n]) <= tol, f"{n}: {rel(got[n], want[n]):.3e} > {tol}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(gdn2, T, dtype):
    d = make(T, 2, T, 2, 2, 128, 128, dtype, "token", h0=True)
    check(*run_both(gdn2, d), d, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K,V,H,HV,decay", [
    (64, 64, 1, 1, "token"), (64, 128, 2, 4, "head"), (128, 64, 2, 2, "none"), (128, 128, 1, 3, "token"),
    (64, 64, 3, 6, "none"), (128, 64, 2, 8, "token"), (64, 128, 1, 1, "token"), (128, 128, 2, 2, "head")])
def test_heads_dims_decays(gdn2, K, V, H, HV, decay, dtype):
    d = make(K + V + HV, 2, 150, H, HV, K, V, dtype, decay, h0=HV % 2 == 0)
    check(*run_both(gdn2, d), d, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[0, 1, 64, 0, 130, 7], [5], [0, 0, 3], [1] * 9, [129, 127, 0], [257, 1, 64, 0]])
@pytest.mark.parametrize("h0", [False, True])
def test_packed(gdn2, lens, h0, dtype):
    d = make(len(lens), 1, sum(lens), 2, 4, 64, 128, dtype, "token", h0=h0, N=len(lens))
    check(*run_both(gdn2, d, lens=lens), d, dtype)


@pytest.mark.parametrize("lens", [
    [40, 1, 0, 129, 1310, 3, 128, 256, 64, 17, 300, 0, 5, 127, 2, 90, 33, 1, 200, 11, 130, 7, 65, 18],  # one is cut
    [130, 1, 0, 200, 90] * 8])  # none is
def test_packed_more_work_than_one_turn(gdn2, lens):
    """More segments and heads than CTAs, of unlike lengths."""
    d = make(31, 1, sum(lens), 4, 8, 64, 64, torch.bfloat16, "token", h0=True, N=len(lens))
    check(*run_both(gdn2, d, lens=lens), d, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strong_decays_and_resets(gdn2, dtype):
    """Decays down to e^-40 a token, and -inf: the state is forgotten, later tokens keep full precision."""
    d = make(3, 2, 200, 2, 2, 64, 64, dtype, "token", h0=True, strong=True)
    for t in (0, 1, 40, 41, 64, 130, 199):
        d["g"][:, t, 0] = -float("inf")
    d["g"][:, 20, 1] = -float("inf")
    ref = {n: d[n].double() for n in ("q", "k", "v", "g", "h0")}
    o, ht = reference(ref["q"], ref["k"], ref["v"], ref["g"], 64 ** -0.5, ref["h0"], None)
    own = {n: d[n].cuda().requires_grad_() for n in ref}
    og, htg = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own["g"], initial_state=own["h0"],
                                     output_final_state=True)
    assert rel(og, o) <= TOL[dtype] and rel(htg, ht) <= STATE_TOL
    grads = torch.autograd.grad([og, htg], list(own.values()), [d["do"].cuda(), d["dht"].cuda()])
    # gradients against a finite decay that is as good as -inf (autograd of exp(-inf) times 0 is not defined)
    d["g"] = d["g"].clamp(min=-300.0)
    _, want = run_both(gdn2, d)
    got = dict(zip(("dq", "dk", "dv", "dg", "dh0"), grads))
    check(got, want, d, dtype, names=("dq", "dk", "dv", "dg", "dh0"))
    assert torch.equal(got["dh0"][:, 0], torch.zeros_like(got["dh0"][:, 0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_single_token_without_state_has_zero_decay_gradient(gdn2, dtype):
    """No decay acts on a first token: its gradient is exactly zero, not a difference of roundings."""
    d = make(5, 3, 1, 2, 2, 128, 64, dtype, "token")
    got, _ = run_both(gdn2, d)
    assert torch.equal(got["dg"], torch.zeros_like(got["dg"]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_views_and_expanded_cotangents(gdn2, dtype):
    """q, k, v as views of one projection (and of an odd, unaligned one), g with swapped strides, an expanded do."""
    B, T, H, HV, K, V = 2, 140, 2, 4, 64, 128
    d = make(6, B, T, H, HV, K, V, dtype, "token")
    want = gdn2.chunk_linear_attn(*(d[n].cuda() for n in ("q", "k", "v", "g")))[0]
    for extra in (0, 8, 3):
        flat = torch.cat([d["q"].flatten(2), d["k"].flatten(2), d["v"].flatten(2),
                          torch.full((B, T, extra), float("nan"), dtype=dtype)], -1).cuda()
        q, k, v, _ = flat.split([H * K, H * K, HV * V, extra], dim=-1)
        g = d["g"].transpose(0, 2).contiguous().cuda().transpose(0, 2)
        o, _ = gdn2.chunk_linear_attn(q.unflatten(-1, (H, K)), k.unflatten(-1, (H, K)), v.unflatten(-1, (HV, V)), g)
        assert torch.equal(o, want)
    v1 = d["v"].cuda().requires_grad_()
    o, _ = gdn2.chunk_linear_attn(d["q"].cuda(), d["k"].cuda(), v1, d["g"].cuda())
    (a,) = torch.autograd.grad(o.sum(), v1, retain_graph=True)
    (b,) = torch.autograd.grad(o, v1, torch.ones_like(o))
    assert torch.equal(a, b)
    qe = d["q"][:, :, :1].cuda().expand(B, T, H, K)  # a broadcast head
    o, _ = gdn2.chunk_linear_attn(qe, d["k"].cuda(), d["v"].cuda(), d["g"].cuda())
    assert torch.equal(o, gdn2.chunk_linear_attn(qe.contiguous(), d["k"].cuda(), d["v"].cuda(), d["g"].cuda())[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_stays_in_its_sequence(gdn2, dtype):
    lens = [100, 90, 110]
    d = make(7, 1, sum(lens), 2, 2, 128, 128, dtype, "token", h0=True, N=3)
    clean, _ = run_both(gdn2, d, lens=lens)
    for n in ("q", "k", "v"):
        d[n][:, 100:190] = float("nan")
    d["g"][:, 100:190] = float("nan")
    d["do"][:, 100:190] = float("inf")
    cu = torch.tensor([0, 100, 190, 300]).cuda()
    own = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v", "g", "h0")}
    o, ht = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own["g"], initial_state=own["h0"],
                                   output_final_state=True, cu_seqlens=cu)
    grads = torch.autograd.grad([o, ht], list(own.values()), [d["do"].cuda(), d["dht"].cuda()])
    got = dict(o=o, ht=ht, **{"d" + n: x for n, x in zip(own, grads)})
    for n, x in got.items():
        for part in ((slice(0, 100), slice(190, 300)) if n not in ("ht", "dh0") else (slice(0, 1), slice(2, 3))):
            a, b = (y[:, part] if n not in ("ht", "dh0") else y[part] for y in (x, clean[n]))
            assert torch.equal(a, b), n


def test_rows_outside_of_every_sequence_get_zeros(gdn2):
    d = make(8, 1, 150, 2, 2, 64, 64, torch.bfloat16, "token")
    cu = torch.tensor([10, 80, 140]).cuda()
    own = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v", "g")}
    o, _ = gdn2.chunk_linear_attn(*own.values(), cu_seqlens=cu)
    grads = torch.autograd.grad(o, list(own.values()), d["do"].cuda())
    for x in (o, *grads):
        assert torch.isfinite(x).all()
        assert not x[:, :10].any() and not x[:, 140:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_empty(gdn2, dtype):
    d = make(9, 2, 0, 2, 2, 64, 64, dtype, "token", h0=True)
    own = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v", "g", "h0")}
    o, ht = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own["g"], initial_state=own["h0"],
                                   output_final_state=True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(ht, own["h0"])
    grads = torch.autograd.grad(ht, list(own.values()), d["dht"].cuda())
    assert torch.equal(grads[4].cpu(), d["dht"]) and all(x.numel() == 0 for x in grads[:4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_sequence_in_segments(gdn2, dtype):
    """Few heads over a long axis, where the work is split over time: against the token-serial form."""
    T = 5000 if dtype == torch.bfloat16 else 1500
    d = make(10, 1, T, 1, 2, 128, 128, dtype, "token", h0=True)
    d["g"] = (d["g"].float() * 0.02).to(dtype)  # memory over thousands of tokens
    q, k, v, g, h0 = (d[n].cuda() for n in ("q", "k", "v", "g", "h0"))
    o, ht = gdn2.chunk_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True)
    o2, ht2 = gdn2.fused_recurrent_linear_attn(q.float(), k.float(), v.float(), g, initial_state=h0,
                                               output_final_state=True)
    assert rel(o, o2.double().cpu()) <= TOL[dtype] and rel(ht, ht2.double().cpu()) <= STATE_TOL


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_split_in_two_calls(gdn2, dtype):
    """A prompt in one call, and in two joined by the state."""
    d = make(11, 2, 333, 2, 2, 128, 64, dtype, "head")
    q, k, v, g = (d[n].cuda() for n in ("q", "k", "v", "g"))
    o, ht = gdn2.chunk_linear_attn(q, k, v, g, output_final_state=True)
    o1, h1 = gdn2.chunk_linear_attn(q[:, :101], k[:, :101], v[:, :101], g, output_final_state=True)
    o2, h2 = gdn2.chunk_linear_attn(q[:, 101:], k[:, 101:], v[:, 101:], g, initial_state=h1, output_final_state=True)
    assert rel(torch.cat([o1, o2], 1), o.double().cpu()) <= 2 * TOL[dtype]
    assert rel(h2, ht.double().cpu()) <= 2 * STATE_TOL


def test_same_bits_twice_and_on_another_stream(gdn2):
    d = make(12, 2, 400, 2, 4, 128, 128, torch.bfloat16, "head", h0=True)
    def once():
        own = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v", "g", "h0")}
        o, ht = gdn2.chunk_linear_attn(own["q"], own["k"], own["v"], own["g"], initial_state=own["h0"],
                                       output_final_state=True)
        return [o, ht, *torch.autograd.grad([o, ht], list(own.values()), [d["do"].cuda(), d["dht"].cuda()])]
    first = once()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        second = once()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_gradients_against_differences(gdn2):
    """Central differences of the fp32 path along random directions (o and the final
    state are linear in q, k, v, h0, so those are exact up to rounding: sums of 1e4
    products at 1e-6 against slopes of their size; in g the step's third order, 1e-4)."""
    d = make(13, 2, 130, 2, 4, 64, 64, torch.float32, "token", h0=True)
    own = {n: d[n].cuda().requires_grad_() for n in ("q", "k", "v", "g", "h0")}
    do, dht = d["do"].cuda().double(), d["dht"].cuda().double()

    def loss(x):
        o, ht = gdn2.chunk_linear_attn(x["q"], x["k"], x["v"], x["g"], initial_state=x["h0"], output_final_state=True)
        return (o.double() * do).sum() + (ht.double() * dht).sum()

    grads = dict(zip(own, torch.autograd.grad(loss(own), list(own.values()))))
    gen = torch.Generator(device="cuda").manual_seed(1)
    for n in own:
        u = torch.randn(own[n].shape, device="cuda", generator=gen)
        eps = 1e-2 if n == "g" else 0.5
        with torch.no_grad():
            up, down = (loss({**own, n: own[n] + s * eps * u}) for s in (1, -1))
        slope = float((up - down) / (2 * eps))
        mine = float((grads[n].double() * u.double()).sum())
        size = float(grads[n].double().norm())  # the slope's standard deviation over directions
        assert abs(slope - mine) <= 2e-3 * size, (n, slope, mine, size)


# ---------------------------------------------------------------------------
# the token-serial form
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K,V,H,HV,decay,T", [
    (128, 128, 2, 2, "token", 1), (64, 64, 1, 1, "none", 1), (64, 128, 2, 4, "head", 5), (128, 64, 1, 3, "token", 17),
    (128, 128, 2, 2, "none", 3)])
def test_recurrent(gdn2, K, V, H, HV, decay, T, dtype):
    d = make(T + K, 3, T, H, HV, K, V, dtype, decay, h0=True)
    x = {n: d[n].double() if d[n] is not None else None for n in ("q", "k", "v", "g", "h0")}
    o, ht = reference(x["q"], x["k"], x["v"], x["g"], K ** -0.5, x["h0"], None)
    y = {n: d[n].cuda() if d[n] is not None else None for n in x}
    og, htg = gdn2.fused_recurrent_linear_attn(y["q"], y["k"], y["v"], y["g"], initial_state=y["h0"],
                                               output_final_state=True)
    assert rel(og, o) <= TOL[dtype] and rel(htg, ht) <= STATE_TOL
    assert torch.equal(y["h0"].cpu(), d["h0"])  # not in place
    o0, none = gdn2.fused_recurrent_linear_attn(y["q"], y["k"], y["v"], y["g"])
    assert none is None
    o0r, _ = reference(x["q"], x["k"], x["v"], x["g"], K ** -0.5, None, None)
    assert rel(o0, o0r) <= TOL[dtype]


def test_recurrent_packed_in_place(gdn2):
    lens = [3, 0, 1, 9]
    d = make(20, 1, sum(lens), 2, 4, 128, 64, torch.bfloat16, "token", h0=True, N=4)
    x = {n: d[n].double() for n in ("q", "k", "v", "g", "h0")}
    o, ht = reference(x["q"], x["k"], x["v"], x["g"], 128 ** -0.5, x["h0"], lens)
    h0 = d["h0"].cuda()
    cu = torch.tensor([0] + lens).cumsum(0).cuda()
    og, htg = gdn2.fused_recurrent_linear_attn(*(d[n].cuda() for n in ("q", "k", "v", "g")), initial_state=h0,
                                               inplace_final_state=True, cu_seqlens=cu)
    assert htg is h0 and rel(og, o) <= TOL[torch.bfloat16] and rel(htg, ht) <= STATE_TOL


def test_recurrent_pool(gdn2):
    """Slots in any order; a slot outside the pool is padding; other slots stay as they were."""
    N, slots = 5, 9
    d = make(21, N, 1, 2, 2, 64, 128, torch.bfloat16, "token")
    pool = torch.randn(slots, 2, 64, 128)
    idx = torch.tensor([7, -1, 0, slots, 3])
    keep = [0, 2, 4]
    x = {n: d[n].double()[keep] for n in ("q", "k", "v", "g")}
    o, ht = reference(x["q"], x["k"], x["v"], x["g"], 64 ** -0.5, pool[idx[keep]].double(), None)
    for dt in (torch.int32, torch.int64):
        p = pool.cuda()
        og, pg = gdn2.fused_recurrent_linear_attn(*(d[n].cuda() for n in ("q", "k", "v", "g")), initial_state=p,
                                                  inplace_final_state=True, ssm_state_indices=idx.cuda().to(dt))
        assert pg is p
        assert rel(og[keep], o) <= TOL[torch.bfloat16] and rel(p[idx[keep].cuda()], ht) <= STATE_TOL
        assert not og[[1, 3]].any()
        rest = [i for i in range(slots) if i not in idx[keep].tolist()]
        assert torch.equal(p[rest].cpu(), pool[rest])


def test_recurrent_pool_beyond_32_bits(gdn2):
    """Element offsets above 2^31 in a large pool."""
    slots, HV, K, V = 8300, 16, 128, 128
    assert (slots - 1) * HV * K * V > 2 ** 31
    d = make(22, 1, 1, 16, HV, K, V, torch.bfloat16, "token")
    pool = torch.empty(slots, HV, K, V, device="cuda")
    last = torch.randn(HV, K, V)
    pool[-1] = last.cuda()
    x = {n: d[n].double() for n in ("q", "k", "v", "g")}
    o, ht = reference(x["q"], x["k"], x["v"], x["g"], K ** -0.5, last[None].double(), None)
    og, _ = gdn2.fused_recurrent_linear_attn(*(d[n].cuda() for n in ("q", "k", "v", "g")), initial_state=pool,
                                             inplace_final_state=True,
                                             ssm_state_indices=torch.tensor([slots - 1], device="cuda"))
    assert rel(og, o) <= TOL[torch.bfloat16] and rel(pool[-1:], ht) <= STATE_TOL


def test_prompt_then_decode(gdn2):
    """The chunkwise form's state continued token by token equals one long call."""
    d = make(23, 2, 205, 2, 2, 128, 128, torch.bfloat16, "token")
    q, k, v, g = (d[n].cuda() for n in ("q", "k", "v", "g"))
    o, ht = gdn2.chunk_linear_attn(q, k, v, g, output_final_state=True)
    o1, S = gdn2.chunk_linear_attn(q[:, :200], k[:, :200], v[:, :200], g[:, :200], output_final_state=True)
    tail = []
    for t in range(200, 205):
        sl = slice(t, t + 1)
        x, S = gdn2.fused_recurrent_linear_attn(q[:, sl], k[:, sl], v[:, sl], g[:, sl], initial_state=S,
                                                inplace_final_state=True)
        tail.append(x)
    assert rel(torch.cat([o1, *tail], 1), o.double().cpu()) <= 2 * TOL[torch.bfloat16]
    assert rel(S, ht.double().cpu()) <= 2 * STATE_TOL


def test_graph_capture(gdn2):
    """A decode step captured in a CUDA graph and replayed on new inputs."""
    d = make(24, 4, 1, 2, 2, 128, 128, torch.bfloat16, "token", h0=True)
    y = {n: d[n].cuda() for n in ("q", "k", "v", "g", "h0")}
    want, wS = gdn2.fused_recurrent_linear_attn(y["q"], y["k"], y["v"], y["g"], initial_state=y["h0"],
                                                output_final_state=True)
    S = torch.zeros_like(y["h0"])
    static = {n: torch.zeros_like(y[n]) for n in ("q", "k", "v", "g")}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, _ = gdn2.fused_recurrent_linear_attn(*static.values(), initial_state=S, inplace_final_state=True)
    S.copy_(y["h0"])
    for n in static:
        static[n].copy_(y[n])
    g.replay()
    assert torch.equal(o, want) and torch.equal(S, wS)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals(gdn2):
    f, r = gdn2.chunk_linear_attn, gdn2.fused_recurrent_linear_attn
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    q, v = z(2, 8, 2, 64), z(2, 8, 4, 128)
    ok = z(2, 8, 4, dt=torch.float32)
    S = z(2, 4, 64, 128, dt=torch.float32)
    bad = [
        (ValueError, dict(k=z(2, 8, 2, 128))), (ValueError, dict(v=z(2, 8, 3, 128))), (ValueError, dict(v=z(2, 9, 4, 128))),
        (ValueError, dict(q=z(2, 8, 2, 96), k=z(2, 8, 2, 96))), (ValueError, dict(v=z(2, 8, 4, 32))),
        (TypeError, dict(k=q.float())), (TypeError, dict(q=q.half(), k=q.half(), v=v.half())),
        (ValueError, dict(g=ok[:, :, :2])), (TypeError, dict(g=ok.double())),
        (TypeError, dict(initial_state=S.bfloat16())), (ValueError, dict(initial_state=S[:1])),
        (ValueError, dict(initial_state=S.transpose(2, 3))),
        (ValueError, dict(cu_seqlens=torch.tensor([0, 8], device="cuda"))),
        (ValueError, dict(g=ok.cpu())),
    ]
    for fn, (err, kw) in itertools.product((f, r), bad):
        with pytest.raises(err):
            fn(**{**dict(q=q, k=q, v=v), **kw})
    with pytest.raises(ValueError):
        r(q, q, v, inplace_final_state=True)
    with pytest.raises(ValueError):
        r(q, q, v, initial_state=S, ssm_state_indices=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        r(q, q, v, initial_state=S, inplace_final_state=True,
          ssm_state_indices=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        r(q, q, v, initial_state=z(2, 4, 128, 64, dt=torch.float32).transpose(2, 3), inplace_final_state=True)
