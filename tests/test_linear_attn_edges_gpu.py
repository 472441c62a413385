"""Calls of linear attention and layer norm at the edges of what they take: rows
and batches that no sequence covers, offsets out of order, tensors off the
16-byte grid, index types, other ways of differentiating."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rand(seed, *shape, dtype=F32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


# ---------------------------------------------------------------------------
# offsets that decrease
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,repeats", [(8192, 5), (1000, 3), (130, 9)])
def test_decreasing_offsets_stay_in_the_workspace(gdn2, dtype, T, repeats):
    """Overlapping sequences have more chunks and segments than the buffers hold: what follows the buffers stays as it was."""
    L, lib = gdn2._lib, gdn2._lib.load()
    H, K, V = 1, 64, 64
    cu = torch.tensor([0, T] * repeats + [0, T], device="cuda")
    N = len(cu) - 1
    q, k, v, do = (rand(i, 1, T, H, K, dtype=dtype) for i in range(4))
    g, h0, dht = -0.1 * rand(5, 1, T, H).abs(), rand(6, N, H, K, V), rand(7, N, H, K, V)
    guard = 4 << 20

    def room(n):  # n bytes and a guard after them
        t = torch.zeros(n + guard, dtype=torch.uint8, device="cuda")
        t[n:] = 0xA5
        return t

    def out(shape, dt):
        n = torch.Size(shape).numel() * dt.itemsize
        return room(n), n

    o, ht, dq, dk, dv = out(q.shape, dtype), out(h0.shape, F32), out(q.shape, dtype), out(q.shape, dtype), out(q.shape, dtype)
    dg, dh0 = out(g.shape, F32), out(h0.shape, F32)
    st = dict(q_b=T * K, q_t=K, q_h=K, k_b=T * K, k_t=K, k_h=K, v_b=T * V, v_t=V, v_h=V, g_b=T, g_t=1, g_h=1)
    a = L.LinearAttnArgs(B=1, T=T, H=H, HV=H, K=K, V=V, N=N, cu_seqlens=L.ptr(cu), scale=0.125,
                         flags=L.HAS_H0 | L.STORE_FINAL | L.SAVE_FOR_BWD, dtype=L.BF16 if dtype == BF16 else L.F32,
                         dtype_g=L.F32, decay=L.DECAY_TOKEN, q=L.ptr(q), k=L.ptr(k), v=L.ptr(v), g=L.ptr(g), h0=L.ptr(h0),
                         ht=L.ptr(ht[0]), o=L.ptr(o[0]), **st)
    gr = L.LinearAttnGrads(dout=L.ptr(do), dht=L.ptr(dht), dq=L.ptr(dq[0]), dk=L.ptr(dk[0]), dv=L.ptr(dv[0]),
                           dg=L.ptr(dg[0]), dh0=L.ptr(dh0[0]))
    n = lib.gdn2_linear_attn_workspace_size(a)
    nb = lib.gdn2_linear_attn_bwd_workspace_size(a)
    ws, bws = (room(n), n), (room(nb), nb)
    stream = L.stream_ptr(q.device)
    assert lib.gdn2_linear_attn_fwd(a, L.ptr(ws[0]), n, stream) == 0
    assert lib.gdn2_linear_attn_bwd(a, gr, L.ptr(ws[0]), n, L.ptr(bws[0]), nb, stream) == 0
    torch.cuda.synchronize()
    assert L.device_fault_read() == 0
    for t, size in (o, ht, dq, dk, dv, dg, dh0, ws, bws):
        assert (t[size:] == 0xA5).all()


# ---------------------------------------------------------------------------
# rows that no sequence covers
# ---------------------------------------------------------------------------
def dirty(*like):
    """Leaves NaN in the memory that the next allocations of these sizes get."""
    for t in like:
        for _ in range(3):
            torch.full_like(t, float("nan"))


def small(dtype, B=1, T=60, H=2, HV=4, K=64, V=128):
    return (rand(1, B, T, H, K, dtype=dtype), rand(2, B, T, H, K, dtype=dtype), rand(3, B, T, HV, V, dtype=dtype),
            -0.2 * rand(4, B, T, HV).abs())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offsets", [[7, 20, 20, 50], [0, 30], [60, 60], [10, 11]])
def test_recurrent_rows_outside_of_every_sequence_get_zeros(gdn2, dtype, offsets):
    q, k, v, g = small(dtype)
    cu = torch.tensor(offsets, device="cuda")
    want, _ = gdn2.chunk_linear_attn(q, k, v, g, cu_seqlens=cu)
    first, last = offsets[0], offsets[-1]
    pool = rand(5, len(offsets), 4, 64, 128)
    slots = torch.arange(len(offsets) - 1, device="cuda")
    for kw in (dict(), dict(initial_state=pool.clone(), inplace_final_state=True, ssm_state_indices=slots),
               dict(initial_state=pool.clone(), inplace_final_state=True, ssm_state_indices=slots - 1)):
        dirty(v)
        o, _ = gdn2.fused_recurrent_linear_attn(q, k, v, g, cu_seqlens=cu, **kw)
        assert torch.isfinite(o).all() and not o[:, :first].any() and not o[:, last:].any()
        if not kw:
            assert (o.float() - want.float()).abs().max() <= 2.0 ** -6 * max(float(want.abs().max()), 1.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_batches_with_states(gdn2, dtype):
    """No batch, no tokens: states of no elements have no address, which is no error."""
    q, k, v, g = (t[:0] for t in small(dtype))
    h0 = torch.zeros(0, 4, 64, 128, device="cuda")
    for f in (gdn2.chunk_linear_attn, gdn2.fused_recurrent_linear_attn):
        o, ht = f(q, k, v, g, initial_state=h0, output_final_state=True)
        assert o.shape == v.shape and ht.shape == h0.shape
    leaves = [t.clone().requires_grad_() for t in (q, k, v, g, h0)]
    o, ht = gdn2.chunk_linear_attn(*leaves[:4], initial_state=leaves[4], output_final_state=True)
    grads = torch.autograd.grad([o, ht], leaves, [torch.ones_like(o), torch.ones_like(ht)])
    assert all(x.shape == t.shape for x, t in zip(grads, leaves))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pool_without_slots(gdn2, dtype):
    """Every sequence is padding: zeros."""
    q, k, v, g = small(dtype, B=3, T=1)
    pool = torch.zeros(0, 4, 64, 128, device="cuda")
    dirty(v)
    o, p = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=pool, inplace_final_state=True,
                                            ssm_state_indices=torch.full((3,), -1, device="cuda"))
    assert p is pool and not o.any()


# ---------------------------------------------------------------------------
# no sequences
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("decay", ["token", "head"])
def test_tokens_but_no_sequences(gdn2, dtype, decay):
    """cu_seqlens of one offset: every row lies outside, o and all gradients are zeros."""
    q, k, v, g = small(dtype)
    g = g if decay == "token" else g[0, 0].clone()
    cu = torch.tensor([0], device="cuda")
    h0 = torch.zeros(0, 4, 64, 128, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v, g, h0)]
    dirty(v)
    o, ht = gdn2.chunk_linear_attn(*leaves[:4], initial_state=h0, output_final_state=True, cu_seqlens=cu)
    assert ht.shape == h0.shape and not o.any()
    dirty(q, k, v, g)
    grads = torch.autograd.grad([o, ht], leaves, [torch.ones_like(o), torch.ones_like(ht)])
    assert all(not x.any() and x.shape == t.shape for x, t in zip(grads, leaves))
    with torch.no_grad():
        dirty(v)
        assert not gdn2.chunk_linear_attn(q, k, v, g, cu_seqlens=cu)[0].any()
        dirty(v)
        o, ht = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True, cu_seqlens=cu)
        assert not o.any() and ht.shape == h0.shape


# ---------------------------------------------------------------------------
# the mixer's padding mask
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("T", [40, 90])
def test_mixer_mask(gdn2, T, side):
    """A padded batch against its sequences run alone, then a decode step on its states.  fp32
    throughout: sums of at most 256 terms in another order, five in a row, stay below 1e-5."""
    torch.manual_seed(0)
    layer = gdn2.LinearAttention(hidden_size=256, head_dim=64, num_heads=2, num_v_heads=4, layer_idx=0).cuda().eval()
    x, nxt = rand(1, 3, T, 256), rand(2, 3, 1, 256)
    lens = [T, T - 29, 1]
    mask = torch.zeros(3, T, dtype=torch.int64, device="cuda")
    for i, n in enumerate(lens):
        mask[i, slice(T - n, T) if side == "left" else slice(0, n)] = 1

    def close(a, b):
        assert float((a - b).norm()) <= 1e-5 * float(b.norm())

    with torch.no_grad():
        cache = gdn2.LayerCache()
        o, none, same = layer(x, mask, cache, True)  # the older mixer's order of arguments
        assert none is None and same is cache and not o[mask == 0].any()
        for m in (mask.bool(), mask.float()):
            assert torch.equal(layer(x, attention_mask=m)[0], o)
        step = layer(nxt, attention_mask=torch.cat([mask, mask.new_ones(3, 1)], 1), past_key_values=cache, use_cache=True)[0]
        for i in range(3):
            alone = gdn2.LayerCache()
            close(o[i][mask[i] == 1], layer(x[i:i + 1, mask[i] == 1], past_key_values=alone, use_cache=True)[0][0])
            close(step[i], layer(nxt[i:i + 1], past_key_values=alone, use_cache=True)[0][0])
            close(cache[0]["recurrent_state"][i], alone[0]["recurrent_state"][0])
    # training: nothing flows to padding
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(layer.train()(leaf, attention_mask=mask)[0].square().sum(), leaf)
    assert not dx[mask == 0].any()
    for i in range(3):
        one = x[i:i + 1, mask[i] == 1].clone().requires_grad_()
        close(dx[i][mask[i] == 1], torch.autograd.grad(layer(one)[0].square().sum(), one)[0][0])
    for bad in (mask[0], mask[:2], mask[:, :-1], mask[:, None]):
        with pytest.raises(ValueError):
            layer(x, attention_mask=bad)
    with pytest.raises(ValueError):
        layer(x[:1], attention_mask=mask[:1], cu_seqlens=torch.tensor([0, T], device="cuda"))


# ---------------------------------------------------------------------------
# other ways of differentiating
# ---------------------------------------------------------------------------
def test_forward_mode_is_refused(gdn2):
    """No tangent is computed: a dual input is an error, as for chunk_gdn2, and not a result without one."""
    import torch.autograd.forward_ad as fwd
    q, k, v, g = small(BF16)
    h0 = rand(9, 1, 4, 64, 128)
    x, w, b, r = rand(10, 20, 64), rand(11, 64), rand(12, 64), rand(13, 20, 64)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for i in range(5):
            a = [dual(t) if i == j else t for j, t in enumerate((q, k, v, g, h0))]
            for f in (gdn2.chunk_linear_attn, gdn2.fused_recurrent_linear_attn):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    f(*a[:4], initial_state=a[4])
        for i in range(4):
            a = [dual(t) if i == j else t for j, t in enumerate((x, w, b, r))]
            with pytest.raises((RuntimeError, NotImplementedError)):
                gdn2.layer_norm(a[0], a[1], a[2], residual=a[3])


def test_second_derivatives_are_refused(gdn2):
    """The gradients are not differentiable: asking for their gradient is an error, not a missing term."""
    q, k, v, g = (t.requires_grad_() for t in small(BF16))
    o, _ = gdn2.chunk_linear_attn(q, k, v, g)
    (dq,) = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().square().sum() + q.float().sum(), q)
    x, w = rand(10, 20, 64).requires_grad_(), rand(11, 64).requires_grad_()
    (dx,) = torch.autograd.grad(gdn2.layer_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.square().sum() + x.sum(), x)


def test_a_state_updated_in_place_counts_as_changed(gdn2):
    """A state that another function saved for its backward, then updated in place, is an error in that backward."""
    q, k, v, g = small(BF16, T=1)
    pool = rand(14, 1, 4, 64, 128)
    w = torch.ones((), device="cuda", requires_grad=True)
    y = (w * pool).sum()  # saves the pool
    before = pool._version
    gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=pool, inplace_final_state=True)
    assert pool._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=torch.zeros_like(pool), inplace_final_state=True)


# ---------------------------------------------------------------------------
# tensors off the 16-byte grid
# ---------------------------------------------------------------------------
def off_grid(t):
    """The same values in a contiguous tensor whose first element lies off the 16-byte grid."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    x = flat[1:].view(t.shape)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_states_and_cotangents_off_the_grid(gdn2, dtype):
    q, k, v, g = small(dtype, B=2)
    h0, do, dht = rand(6, 2, 4, 64, 128), rand(7, *v.shape, dtype=dtype), rand(8, 2, 4, 64, 128)

    def once(f):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, g)] + [f(h0).detach().requires_grad_()]
        o, ht = gdn2.chunk_linear_attn(*leaves[:4], initial_state=leaves[4], output_final_state=True)
        return [o, ht, *torch.autograd.grad([o, ht], leaves, [f(do), f(dht)])]

    for a, b in zip(once(lambda t: t), once(off_grid)):
        assert torch.equal(a, b)
    a = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True)
    b = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=off_grid(h0), output_final_state=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with pytest.raises(ValueError):  # an update in place has to stay where it is
        gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=off_grid(h0), inplace_final_state=True)


def test_backward_through_a_cat_at_an_odd_place(gdn2):
    q, k, v, g = small(BF16)
    v.requires_grad_()
    o, _ = gdn2.chunk_linear_attn(q, k, v, g)
    weight = rand(9, o.numel(), dtype=BF16)
    (want,) = torch.autograd.grad(o, v, weight.view(o.shape), retain_graph=True)
    joined = torch.cat([torch.zeros(3, device="cuda", dtype=BF16), o.flatten()])
    (dv,) = torch.autograd.grad(joined, v, torch.cat([weight[:3], weight]))
    assert torch.equal(dv, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_sequence_with_an_odd_batch_step(gdn2, dtype):
    """A dimension of one element may have any step: it is never taken."""
    q, k, v, g = small(dtype)
    n = 4 * 64 * 128
    h0 = rand(6, n + 2).as_strided((1, 4, 64, 128), (n + 1, 64 * 128, 128, 1))
    want = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0.clone(), output_final_state=True)
    got = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    o, ht = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, inplace_final_state=True)
    assert ht is h0 and torch.equal(o, want[0]) and torch.equal(h0, want[1])


def test_an_expanded_state_is_not_updated_in_place(gdn2):
    """Sequences that share memory cannot each have a state there; reading it for all of them is fine."""
    q, k, v, g = small(BF16, B=3, T=1)
    h0 = rand(6, 1, 4, 64, 128).expand(3, 4, 64, 128)
    want = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0.clone(), output_final_state=True)
    got = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    half = rand(7, 4 * 4 * 64 * 128).as_strided((3, 4, 64, 128), (2 * 64 * 128, 64 * 128, 128, 1))  # half of each overlaps
    for bad in (h0, half):
        with pytest.raises(ValueError):
            gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=bad, inplace_final_state=True)


# ---------------------------------------------------------------------------
# types of slots
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("itype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_slot_types(gdn2, itype):
    q, k, v, g = small(BF16, B=4, T=1)
    pool = rand(5, 9, 4, 64, 128)
    idx = torch.tensor([7, 100, 0, 3], device="cuda")
    want = pool.clone()
    ow, _ = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=want, inplace_final_state=True,
                                             ssm_state_indices=idx.int())
    o, _ = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=pool, inplace_final_state=True,
                                            ssm_state_indices=idx.to(itype))
    assert torch.equal(o, ow) and torch.equal(pool, want)


def test_slots_beyond_32_bits_are_padding(gdn2):
    q, k, v, g = small(BF16, B=3, T=1)
    pool = rand(5, 4, 4, 64, 128)
    keep = pool.clone()
    idx = torch.tensor([2 ** 32, -2 ** 32 + 1, 2 ** 63 - 1], device="cuda")
    o, _ = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=pool, inplace_final_state=True, ssm_state_indices=idx)
    assert not o.any() and torch.equal(pool, keep)


# ---------------------------------------------------------------------------
# under a compiler
# ---------------------------------------------------------------------------
@pytest.mark.filterwarnings("error:Dynamo does not know how to trace")
def test_traced_callers_run_the_operators_as_they_are(gdn2):
    """A traced caller breaks its graph at these functions, as at the gated delta rule's."""
    q, k, v, g = small(BF16)
    q.requires_grad_()
    w = rand(11, 128)

    def f(q, k, v, g, w):
        o, ht = gdn2.chunk_linear_attn(q * 1.0, k, v, g, output_final_state=True)
        r, _ = gdn2.fused_recurrent_linear_attn(q.detach(), k, v, g)
        return gdn2.layer_norm(o.float(), w) + r.float(), ht

    want, want_ht = f(q, k, v, g, w)
    got, ht = torch.compile(f, backend="eager")(q, k, v, g, w)
    assert torch.equal(got, want) and torch.equal(ht, want_ht)
    assert torch.equal(*(torch.autograd.grad(x.sum(), q)[0] for x in (got, want)))


# ---------------------------------------------------------------------------
# strong decays
# ---------------------------------------------------------------------------
def test_decays_after_a_strong_burst_keep_their_bits(gdn2):
    """64 tokens of decay -140 put the chunk's running sum near -9000, where floats are 2^-10 apart;
    the factors between the tokens after them must not notice.

    One nonzero term per value, operands of 1: an output is then its factor, rounded once to bf16 where
    it goes through a product's operand (2^-8 of it at most) and not at all in the decays' gradient.  The factor
    itself: 2^-22 from the exponential, differences of sums held to 2^-31 of 9000, an exponent of at
    most 13 rounded a few times (2^-23 of it each): below 2e-5."""
    T, H, K = 128, 32, 64
    gen = torch.Generator().manual_seed(0)
    g = torch.empty(1, T, H)
    g[:, :64] = -140 + torch.rand(1, 64, H, generator=gen)
    g[:, 64:] = -0.2 * torch.rand(1, 64, H, generator=gen)
    G = g[0].double().cumsum(0)
    one = torch.zeros(1, T, H, K)
    one[..., 0] = 1.0
    dev = lambda t: t.bfloat16().cuda().requires_grad_()  # noqa: E731

    # the pairs (127, j): o of a value at j, and dv_j of a cotangent at 127
    only = torch.zeros(1, T, H, K)
    only[:, 127, :, 0] = 1.0
    q, k, v, gl = dev(one), dev(one), dev(one), g.cuda().requires_grad_()
    o, ht = gdn2.chunk_linear_attn(q, k, v, gl, scale=1.0, output_final_state=True)
    dv, dk = torch.autograd.grad(o, (v, k), only.bfloat16().cuda(), retain_graph=True)
    want = (G[127] - G[64:]).exp()
    for name, x in (("dv", dv), ("dk", dk)):
        err = (x[0, 64:, :, 0].detach().double().cpu() - want).abs() / want
        assert float(err.max()) <= 2.0 ** -8 + 2e-5, (name, float(err.max()))

    # the final state's cotangent and one key at 100: dg of every later token is that term's value
    key = torch.zeros(1, T, H, K)
    key[:, 100, :, 0] = 1.0
    dht = torch.zeros(1, H, K, K)
    dht[..., 0, 0] = 1.0
    k = dev(key)
    o, ht = gdn2.chunk_linear_attn(q, k, v, gl, scale=1.0, output_final_state=True)
    (dg,) = torch.autograd.grad(ht, gl, dht.cuda())
    want = (G[127] - G[100]).exp()
    err = (dg[0, 101:].double().cpu() - want).abs() / want
    assert float(err.max()) <= 2e-5, float(err.max())
    err = (ht[0, :, 0, 0].detach().double().cpu() - want).abs() / want
    assert float(err.max()) <= 2e-5, float(err.max())


# ---------------------------------------------------------------------------
# the chunkwise form in a graph, and on two streams at once
# ---------------------------------------------------------------------------
def step(gdn2, q, k, v, g, h0, do, dht, cu=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, h0)]
    o, ht = gdn2.chunk_linear_attn(*leaves[:4], initial_state=leaves[4], output_final_state=True, cu_seqlens=cu)
    return [o.detach(), ht.detach(), *torch.autograd.grad((o, ht), leaves, (do, dht))]


def inputs(dtype, T, N, HV=4, seed=0, B=1):
    H, K, V = 2, 64, 128
    return [*(t.clone() for t in small(dtype, B=B, T=T, H=H, HV=HV)), rand(seed + 20, N, HV, K, V),
            rand(seed + 21, B, T, HV, V, dtype=dtype), rand(seed + 22, N, HV, K, V)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,offsets", [(300, None), (5000, None), (400, [0, 130, 130, 131, 390])])
def test_chunkwise_graph_capture(gdn2, dtype, T, offsets):
    """A training step captured in a CUDA graph and replayed on new inputs, and new offsets."""
    N = 1 if offsets is None else len(offsets) - 1
    x = inputs(dtype, T, N)
    cu = None if offsets is None else torch.tensor(offsets, device="cuda")
    want = step(gdn2, *x, cu)
    static = [torch.zeros_like(t) for t in x]
    scu = None if cu is None else torch.linspace(0, T, N + 1, device="cuda").long()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(gdn2, *static, scu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(gdn2, *static, scu)
    for s, t in zip(static, x):
        s.copy_(t)
    if cu is not None:
        scu.copy_(cu)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert gdn2._lib.device_fault_read() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_two_streams_at_once(gdn2, dtype):
    """Calls in flight on two streams do not share scratch memory."""
    data = [inputs(dtype, 700 + 300 * i, 1, seed=i) for i in range(2)]
    want = [step(gdn2, *x) for x in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[] for _ in data]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(gdn2, *data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    assert gdn2._lib.device_fault_read() == 0


def test_long_fp32_prompt(gdn2):
    """Many chunks of the fp32 form against the token-serial one: sums of some hundred terms in another order."""
    T = 20000
    q, k, v, g = small(F32, T=T, H=1, HV=1)
    g = g * 0.02
    h0 = rand(6, 1, 1, 64, 128)
    o, ht = gdn2.chunk_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True)
    o2, ht2 = gdn2.fused_recurrent_linear_attn(q, k, v, g, initial_state=h0, output_final_state=True)
    for a, b in ((o, o2), (ht, ht2)):
        assert float((a - b).norm()) <= 1e-5 * float(b.norm())


def test_backward_after_the_initial_state_was_updated(gdn2):
    """The backward does not read the initial state, so a decode step on it in between is no matter."""
    q, k, v, g = small(BF16, T=100)
    h0 = rand(6, 1, 4, 64, 128)
    for dtype in (BF16, F32):
        leaves = [t.to(dtype).requires_grad_() for t in (q, k, v)] + [g.clone().requires_grad_()]
        S = h0.clone()
        want = torch.autograd.grad(gdn2.chunk_linear_attn(*leaves, initial_state=S)[0].float().square().sum(), leaves)
        o, _ = gdn2.chunk_linear_attn(*leaves, initial_state=S)
        gdn2.fused_recurrent_linear_attn(*(t.detach()[:, :1] for t in leaves), initial_state=S, inplace_final_state=True)
        S.zero_()
        got = torch.autograd.grad(o.float().square().sum(), leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_heads_before_tokens(gdn2, dtype):
    """q, k, v laid out [B, H, T, D] in memory, and with the batch innermost of the three."""
    x = [t.requires_grad_() for t in small(dtype, B=3, T=150)]
    o, _ = gdn2.chunk_linear_attn(*x)
    do = rand(9, *o.shape, dtype=dtype)
    want = [o, *torch.autograd.grad(o, x, do), gdn2.fused_recurrent_linear_attn(*x)[0]]
    for order in ((0, 2, 1, 3), (2, 1, 0, 3), (1, 0, 2, 3)):
        back = [order.index(i) for i in range(4)]
        y = [t.detach().permute(order).contiguous().permute(back).requires_grad_() for t in x[:3]] + [x[3]]
        assert not y[0].is_contiguous()
        o, _ = gdn2.chunk_linear_attn(*y)
        got = [o, *torch.autograd.grad(o, y, do), gdn2.fused_recurrent_linear_attn(*y)[0]]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# infinities
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_an_infinite_value_is_infinite_in_the_state(gdn2, dtype):
    """Infinite values in a column: k (+-inf) in that column of the final state, and nothing of it in the others."""
    q, k, v, g = small(dtype, T=300)
    k = torch.where(k == 0, torch.ones_like(k), k)
    v = v.clone()
    v[0, 290, 1, 5], v[0, 130, 2, 70] = float("inf"), -float("inf")
    g = 0.01 * g  # far from underflow over the whole length
    clean = v.clone()
    clean[0, 290, 1, 5] = clean[0, 130, 2, 70] = 0.0
    _, want = gdn2.chunk_linear_attn(q, k, clean, g, output_final_state=True)
    _, ht = gdn2.chunk_linear_attn(q, k, v, g, output_final_state=True)
    want = want.clone()
    want[0, 1, :, 5] = float("inf") * k[0, 290, 0].sign().float()
    want[0, 2, :, 70] = -float("inf") * k[0, 130, 1].sign().float()
    assert torch.equal(ht, want)
