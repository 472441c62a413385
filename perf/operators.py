"""Measured cases of the linear-attention and layer-norm operators.

Each case is one call (or one training step: forward and backward) of

* ``chunk_linear_attn``            prompts and training, a decay for each head;
* ``fused_recurrent_linear_attn``  one token per sequence on kept states;
* ``layer_norm``                   with and without a residual stream.

``run`` makes the package's calls where ``own`` is true; otherwise it computes
the same values in elementary torch operations in 32 bits.  ``exact`` computes
them from the definitions in 64 bits.
"""

import math
import random

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
_DTYPES = {"bf16": BF16, "fp32": F32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a chat turn's short prompt, one sequence: latency counts; fixed decays, the state is kept for decoding
        dict(name="prompt_short", op="prompt", B=1, T=77, H=16, HV=16, K=128, V=128, seqs=0, decay="fixed",
             h0=False, fused=True, dtype="bf16"),
        # a serving batch of ragged prompts packed into one row, continued from kept states (some empty, some of one token)
        dict(name="prompt_packed", op="prompt", B=1, T=9001, H=16, HV=16, K=128, V=128, seqs=23, decay="token",
             h0=True, fused=True, dtype="bf16"),
        # one long document: few heads, a long axis
        dict(name="prompt_long", op="prompt", B=1, T=65536, H=16, HV=16, K=128, V=128, seqs=0, decay="token",
             h0=False, fused=False, dtype="bf16"),
        # the training shape of the repository's chunk benchmark, decays learned for each token
        dict(name="train_4x4096", op="train", B=4, T=4096, H=16, HV=16, K=128, V=128, seqs=0, decay="token",
             h0=False, fused=False, dtype="bf16"),
        # grouped value heads, fixed decays, an odd length, smaller keys; truncated back-propagation through a state
        dict(name="train_grouped", op="train", B=3, T=1511, H=4, HV=16, K=64, V=128, seqs=0, decay="fixed",
             h0=True, fused=False, dtype="bf16"),
        # an fp32 run of a small model (the package's fp32 path), decays learned for each token
        dict(name="train_fp32", op="train", B=2, T=1000, H=4, HV=4, K=64, V=64, seqs=0, decay="token",
             h0=False, fused=False, dtype="fp32"),
        # decoding for a handful of users: latency counts
        dict(name="decode_4", op="decode", N=4, slots=6, H=16, HV=16, K=128, V=128, decay="token", dtype="bf16"),
        # decoding for the repository's 256-sequence batch, states in a pool
        dict(name="decode_256", op="decode", N=256, slots=300, H=16, HV=16, K=128, V=128, decay="token", dtype="bf16"),
        # the norm before a block while decoding: a few rows, forward only
        dict(name="norm_rows_33", op="norm", rows=33, D=2048, residual=False, train=False, dtype="bf16", wdtype="fp32"),
        # add and norm of a training step: bf16 branch onto the fp32 residual stream of the hybrid model
        dict(name="norm_residual_16384", op="norm", rows=16384, D=2048, residual=True, train=True, dtype="bf16",
             wdtype="fp32"),
        # the norm of each head's output in a training step of the shape above
        dict(name="norm_heads_262144", op="norm", rows=262144, D=128, residual=False, train=True, dtype="bf16",
             wdtype="fp32"),
        # an odd width in fp32
        dict(name="norm_odd_fp32", op="norm", rows=3001, D=1001, residual=False, train=True, dtype="fp32",
             wdtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "decode", "norm", "norm"])
    if op == "norm":
        D = rng.choice([64, 128, 2048, 4608, _log_int(rng, 17, 8192), 8 * _log_int(rng, 8, 1024)])
        rows = _log_int(rng, 1, max(2, (1 << 25) // D))
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        return dict(op="norm", rows=rows, D=D, residual=rng.random() < 0.4, train=rng.random() < 0.7, dtype=dtype,
                    wdtype=rng.choice(["fp32", dtype]))
    K, V = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (128, 64)])
    H = rng.choice([1, 2, 3, 4, 8, 16])
    HV = H * rng.choice([1, 1, 1, 2, 4])
    decay = rng.choice(["token", "token", "fixed", "none"])
    if op == "decode":
        N = _log_int(rng, 1, max(1, 4096 // HV))
        return dict(op="decode", N=N, slots=N + rng.randint(0, N), H=H, HV=HV, K=K, V=V, decay=decay,
                    dtype=rng.choice(["bf16", "bf16", "fp32"]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    most = (1 << 20 if op == "prompt" else 1 << 18) // (1 if dtype == "bf16" else 4)  # tokens times heads
    longest = 65536 if op == "prompt" else 8192
    T = min(_log_int(rng, 1, longest), most // HV)
    seqs, B = 0, 1
    if rng.random() < 0.35 and T > 8:
        seqs = _log_int(rng, 1, min(T, 64))
    else:
        B = _log_int(rng, 1, max(1, min(64, most // (HV * T))))
    return dict(op=op, B=B, T=T, H=H, HV=HV, K=K, V=V, seqs=seqs, decay=decay, h0=rng.random() < 0.4,
                fused=rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """Ragged lengths of a packed row: fixed by the case; one sequence in eight is empty or a single token."""
    r = random.Random("%d of %d" % (case["seqs"], case["T"]))
    n, left = case["seqs"], case["T"]
    share = [0.0 if r.random() < 0.125 else math.exp(r.uniform(-2.0, 2.0)) for _ in range(n)]
    if sum(share) == 0.0:
        share[0] = 1.0
    lens = [int(left * s / sum(share)) if s else r.randint(0, 1) for s in share]
    while sum(lens) > left:
        lens[lens.index(max(lens))] -= sum(lens) - left
    lens[lens.index(max(lens))] += left - sum(lens)
    return lens


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if case["op"] == "norm":
        rows, D, wd = case["rows"], case["D"], _DTYPES[case["wdtype"]]
        s = dict(case=case, x=(randn(rows, D) + 0.5 * randn(D)).to(dt), w=(1 + 0.2 * randn(D)).to(wd),
                 b=(0.2 * randn(D)).to(wd))
        if case["residual"]:
            s["r"] = 2 * randn(rows, D)  # the residual stream is kept in fp32
        if case["train"]:
            s["dy"] = randn(rows, D).to(dt)
            if case["residual"]:
                s["ds"] = randn(rows, D)
        return s

    H, HV, K, V = case["H"], case["HV"], case["K"], case["V"]
    B, T = (case["N"], 1) if case["op"] == "decode" else (case["B"], case["T"])
    if case.get("fused") or case["op"] == "decode":  # views of one projection's output
        proj = randn(B, T, 2 * H * K + HV * V).to(dt)
        q, k, v = proj.split([H * K, H * K, HV * V], dim=-1)
        q, k, v = q.unflatten(-1, (H, K)), k.unflatten(-1, (H, K)), v.unflatten(-1, (HV, V))
    else:
        q, k, v = randn(B, T, H, K).to(dt), randn(B, T, H, K).to(dt), randn(B, T, HV, V).to(dt)
    s = dict(case=case, q=q, k=k, v=v, g=None, h0=None, cu=None)
    if case["decay"] == "fixed":  # a slope for each head, from slow to fast
        s["g"] = torch.log1p(-torch.exp2(torch.linspace(-9, -2, HV, device=dev)))
    elif case["decay"] == "token":  # learned: heads from slow to fast, tokens around their head's
        rate = torch.exp2(torch.linspace(-7, 0, HV, device=dev))
        s["g"] = (-rate * torch.nn.functional.softplus(randn(B, T, HV))).to(dt)
    if case["op"] == "decode":
        s["pool"] = randn(case["slots"], HV, K, V)
        s["slot"] = torch.randperm(case["slots"], device=dev, generator=gen)[: case["N"]].to(torch.int32)
        return s
    N = B
    if case["seqs"]:
        N = case["seqs"]
        s["lens"] = _lengths(case)
        s["cu"] = torch.tensor([0] + s["lens"], device=dev).cumsum(0)
    if case["h0"]:
        s["h0"] = randn(N, HV, K, V)
    if case["op"] == "train":
        s["do"] = randn(B, T, HV, V).to(dt)
        if case["h0"]:
            s["dht"] = randn(N, HV, K, V)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _segment_sums(g):
    """x[..., i, j] = g[j+1] + ... + g[i] for i >= j, -inf above the diagonal."""
    n = g.shape[-1]
    low = torch.ones(n, n, dtype=torch.bool, device=g.device).tril()
    x = g.unsqueeze(-1).expand(*g.shape, n).masked_fill(~low.tril(-1), 0.0)
    return torch.cumsum(x, dim=-2).masked_fill(~low, -math.inf)


def _plain_chunk(q, k, v, g, h0, cu, lens, final):
    dt, scale, C = q.dtype, q.shape[-1] ** -0.5, 64
    HV, group = v.shape[2], v.shape[2] // q.shape[2]
    g = torch.zeros(v.shape[:3], device=v.device) if g is None else g.float().expand(v.shape[:3])
    q, k, v = q.float() * scale, k.float(), v.float()
    if cu is not None:  # packed rows as a padded batch
        pos = torch.arange(max(lens), device=q.device)
        at = cu[:-1, None] + pos
        inside = at < cu[1:, None]
        at = at.clamp(max=q.shape[1] - 1)
        q, k, v = (x[0][at].masked_fill(~inside[..., None, None], 0.0) for x in (q, k, v))
        g = g[0][at].masked_fill(~inside[..., None], 0.0)
    N, T, _, K = q.shape
    V, pad = v.shape[-1], (-T) % C
    q, k = (x.repeat_interleave(group, dim=2) for x in (q, k))

    def chunks(x):
        x = torch.nn.functional.pad(x, (0,) * (2 * (x.ndim - 2)) + (0, pad))
        return x.unflatten(1, (-1, C)).movedim(3, 1)  # [N, HV, chunks, C, ...]

    q, k, v, g = chunks(q), chunks(k), chunks(v), chunks(g)
    inside_chunk = torch.exp(_segment_sums(g))
    G = torch.cumsum(g, -1)
    rest = inside_chunk[..., -1, :]  # the decay from each token to its chunk's end
    o = ((q @ k.transpose(-1, -2)) * inside_chunk) @ v
    adds = (k * rest[..., None]).transpose(-1, -2) @ v
    # a state before each chunk, and one after the last
    first = torch.zeros_like(adds[:, :, :1]) if h0 is None else h0.float().unsqueeze(2)
    adds = torch.cat([first, adds], 2)
    between = torch.exp(_segment_sums(torch.nn.functional.pad(G[..., -1], (1, 0))))
    S = (between @ adds.flatten(-2)).unflatten(-1, (K, V))
    o = o + torch.exp(G)[..., None] * (q @ S[:, :, :-1])
    o = o.movedim(1, 3).flatten(1, 2)[:, :T]
    if cu is not None:
        at = torch.arange(int(sum(lens)), device=o.device)
        n = torch.searchsorted(cu, at, right=True) - 1
        o = o[n, at - cu[n]].unsqueeze(0)
    return o.to(dt), (S[:, :, -1] if final else None)


def _plain_decode(q, k, v, g, pool, slot):
    dt, group, scale = q.dtype, v.shape[2] // q.shape[2], q.shape[-1] ** -0.5
    q, k = (x[:, 0].float().repeat_interleave(group, dim=1) for x in (q, k))
    S = pool[slot.long()]
    if g is not None:
        g = g.float() if g.ndim == 1 else g[:, 0].float()
        S = S * torch.exp(g)[..., None, None]
    S = S + k[..., :, None] * v[:, 0].float()[..., None, :]
    pool[slot.long()] = S
    o = (S * (q * scale)[..., :, None]).sum(-2)
    return o.to(dt).unsqueeze(1), pool


def _plain_norm(x, w, b, eps, r):
    s = x.float() if r is None else x.float() + r
    c = s - s.mean(-1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps) * w.float() + b.float()
    return (y.to(x.dtype), s) if r is not None else y.to(x.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _package():
    import importlib
    return importlib.import_module("gateddeltanet-2_b200")


def _norm(x, w, b, r):
    if own:
        return _package().layer_norm(x, w, b, eps=1e-5, residual=r)
    return _plain_norm(x, w, b, 1e-5, r)


def _attend(q, k, v, g, h0, s, final):
    if own:
        return _package().chunk_linear_attn(q, k, v, g, initial_state=h0, output_final_state=final,
                                            cu_seqlens=s["cu"])
    return _plain_chunk(q, k, v, g, h0, s["cu"], s.get("lens"), final)


def run(state):
    s, case = state, state["case"]
    if case["op"] == "decode":
        with torch.no_grad():
            if own:
                o, _ = _package().fused_recurrent_linear_attn(
                    s["q"], s["k"], s["v"], s["g"], initial_state=s["pool"], inplace_final_state=True,
                    ssm_state_indices=s["slot"])
            else:
                o, _ = _plain_decode(s["q"], s["k"], s["v"], s["g"], s["pool"], s["slot"])
        return {"o": o, "pool": s["pool"]}
    if case["op"] == "prompt":
        with torch.no_grad():
            o, ht = _attend(s["q"], s["k"], s["v"], s["g"], s["h0"], s, True)
        return {"o": o, "ht": ht}
    if case["op"] == "norm" and not case["train"]:
        with torch.no_grad():
            y = _norm(s["x"], s["w"], s["b"], s.get("r"))
        return dict(zip(("y", "s"), y)) if case["residual"] else {"y": y}
    names = ["x", "w", "b", "r"] if case["op"] == "norm" else ["q", "k", "v", "g", "h0"]
    if case.get("decay") == "fixed":
        names.remove("g")  # fixed decays are not learned
    leaves = {n: s[n].detach().requires_grad_() for n in names if s.get(n) is not None}
    if case["op"] == "norm":
        y = _norm(leaves["x"], leaves["w"], leaves["b"], leaves.get("r"))
        outs, douts = (y, (s["dy"], s["ds"])) if case["residual"] else ((y,), (s["dy"],))
        out = dict(zip(("y", "s"), outs))
    else:
        o, ht = _attend(leaves["q"], leaves["k"], leaves["v"], leaves.get("g", s["g"]), leaves.get("h0"), s, case["h0"])
        outs, douts = ((o, ht), (s["do"], s["dht"])) if case["h0"] else ((o,), (s["do"],))
        out = dict(zip(("o", "ht"), outs))
    grads = torch.autograd.grad(outs, list(leaves.values()), douts)
    out = {n: x.detach() for n, x in out.items()}
    out.update(("d" + n, x) for n, x in zip(leaves, grads))
    return out


def work(case):
    e = _DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        rows, D, we = case["rows"], case["D"], _DTYPES[case["wdtype"]].itemsize
        r = 4 if case["residual"] else 0
        if not case["train"]:
            return {"bytes": rows * D * (2 * e + 2 * r) + 2 * D * we, "flops": 8 * rows * D}
        # forward: x, r in, y, s out; backward: x (or s), dy, ds in, dx, dr out
        back = (r + e + r) + (e + r) if r else 3 * e
        return {"bytes": rows * D * (2 * e + 2 * r + back) + 5 * D * we, "flops": 20 * rows * D}
    H, HV, K, V = case["H"], case["HV"], case["K"], case["V"]
    if case["op"] == "decode":
        N = case["N"]
        g = N * HV * e if case["decay"] == "token" else 0
        return {"bytes": N * (2 * H * K + 2 * HV * V) * e + g + 2 * N * HV * K * V * 4, "flops": 5 * N * HV * K * V}
    rows, N = case["B"] * case["T"], case["seqs"] or case["B"]
    g = rows * HV * e if case["decay"] == "token" else 0
    state = N * HV * K * V * 4
    qk, vo = rows * H * K * e, rows * HV * V * e
    fwd = 2 * qk + 2 * vo + g + (state if case["h0"] else 0)
    if case["op"] == "prompt":
        return {"bytes": fwd + state, "flops": 4 * rows * HV * K * V}
    # backward: q, k, v, do, g, h0, dht in; dq, dk, dv, dg, dh0 out
    back = 4 * qk + 3 * vo + 2 * g + (3 * state if case["h0"] else 0)
    return {"bytes": fwd + (state if case["h0"] else 0) + back, "flops": 14 * rows * HV * K * V}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_tokens(s):
    """Token by token: S <- exp(g) S + k v^T, o = S^T q; all sequences side by side."""
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    g = torch.zeros(B, T, HV, device=q.device, dtype=torch.double) if s["g"] is None else s["g"].double().expand(B, T, HV)
    decay = g.exp()
    heads = torch.arange(HV, device=q.device) // (HV // H)
    starts, lens = ([0] * B, [T] * B) if s["cu"] is None else (s["cu"][:-1].tolist(), s["lens"])
    N = len(lens)
    S = torch.zeros(N, HV, K, V, device=q.device, dtype=torch.double) if s["h0"] is None else s["h0"].double()
    o = torch.zeros(B, T, HV, V, device=q.device, dtype=torch.double)
    order = sorted(range(N), key=lambda n: -lens[n])  # the longest first: the active ones are a prefix
    S = S[order].clone()
    row = torch.tensor([n if s["cu"] is None else 0 for n in order], device=q.device)
    start = torch.tensor([starts[n] for n in order], device=q.device)
    active = N
    for t in range(max(lens)):
        while active and lens[order[active - 1]] <= t:
            active -= 1
        b, at, A = row[:active], start[:active] + t, S[:active]
        A.mul_(decay[b, at][..., None, None]).add_(k[b, at][:, heads][..., :, None] * v[b, at][..., None, :])
        o[b, at] = torch.einsum("nhkv,nhk->nhv", A, q[b, at][:, heads]) * K ** -0.5
    back = torch.empty(N, dtype=torch.long, device=q.device)
    back[torch.tensor(order, device=q.device)] = torch.arange(N, device=q.device)
    return o, S[back]


def _exact_train(s):
    """Each sequence and head as a masked matrix, o = (q k^T * decays) v + decays q S0, differentiated."""
    case = s["case"]
    B, T, H, K = s["q"].shape
    HV, V = s["v"].shape[2:]
    spans = [(b, 0, T) for b in range(B)] if s["cu"] is None else []
    at = 0
    for n in s.get("lens", []):
        spans.append((0, at, at + n))
        at += n
    z = lambda x: torch.zeros(x.shape, device=x.device, dtype=torch.double)  # noqa: E731
    out = {"o": z(s["v"]), "dq": z(s["q"]), "dk": z(s["k"]), "dv": z(s["v"])}
    if case["decay"] == "token":
        out["dg"] = z(s["g"])
    if case["h0"]:
        out["ht"], out["dh0"] = z(s["h0"]), z(s["h0"])
    for n, (b, lo, hi) in enumerate(spans):
        low = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=s["q"].device).tril()
        for h in range(HV):
            hk = h // (HV // H)
            leaves = [s["q"][b, lo:hi, hk], s["k"][b, lo:hi, hk], s["v"][b, lo:hi, h]]
            leaves.append(torch.zeros(hi - lo, device=low.device) if s["g"] is None
                          else s["g"][b, lo:hi, h] if s["g"].ndim == 3 else s["g"][h].expand(hi - lo))
            if case["h0"]:
                leaves.append(s["h0"][n, h])
            leaves = [x.double().detach().requires_grad_() for x in leaves]
            q, k, v, g = leaves[:4]
            G = g.cumsum(0)
            D = (G[:, None] - G[None, :]).masked_fill(~low, -math.inf).exp()
            o = ((q @ k.T) * D) @ v
            outs, douts = [], []
            if case["h0"]:
                total = g.sum()
                o = o + G.exp()[:, None] * (q @ leaves[4])
                ht = total.exp() * leaves[4] + (k * (total - G).exp()[:, None]).T @ v
                out["ht"][n, h] = ht.detach()
                outs, douts = [ht], [s["dht"][n, h].double()]
            o = o * K ** -0.5
            out["o"][b, lo:hi, h] = o.detach()
            d = torch.autograd.grad([o] + outs, leaves, [s["do"][b, lo:hi, h].double()] + douts, allow_unused=True)
            out["dq"][b, lo:hi, hk] += d[0]
            out["dk"][b, lo:hi, hk] += d[1]
            out["dv"][b, lo:hi, h] = d[2]
            if "dg" in out:
                out["dg"][b, lo:hi, h] = d[3]
            if case["h0"]:
                out["dh0"][n, h] = d[4]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = (s[n].double() for n in ("x", "w", "b"))
        z = x + s["r"].double() if case["residual"] else x
        mean, var = z.mean(-1, keepdim=True), z.var(-1, unbiased=False, keepdim=True)
        hat = (z - mean) / (var + 1e-5).sqrt()
        out = {"y": hat * w + b}
        if case["residual"]:
            out["s"] = z
        if case["train"]:
            dy = s["dy"].double()
            dhat = dy * w
            dz = (dhat - dhat.mean(-1, keepdim=True) - hat * (dhat * hat).mean(-1, keepdim=True)) / (var + 1e-5).sqrt()
            if case["residual"]:
                dz = dz + s["ds"].double()
                out["dr"] = dz
            out.update(dx=dz, dw=(dy * hat).sum(0), db=dy.sum(0))
        return out
    if case["op"] == "decode":
        heads = torch.arange(case["HV"], device="cuda") // (case["HV"] // case["H"])
        s["q"], s["k"] = s["q"][:, :, heads], s["k"][:, :, heads]
        pool = s["pool"].double()
        s["h0"] = pool[s["slot"].long()]
        o, S = _exact_tokens(s)
        pool[s["slot"].long()] = S
        return {"o": o, "pool": pool}
    if case["op"] == "prompt":
        o, ht = _exact_tokens(s)
        return {"o": o, "ht": ht}
    return _exact_train(s)
