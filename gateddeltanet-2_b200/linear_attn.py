"""Linear attention with a decay for each head.

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,    o_t = scale * S_t^T q_t

``chunk_linear_attn`` is the chunkwise form (prompts and training, with
gradients), ``fused_recurrent_linear_attn`` the token-serial form (decoding on
kept states).  Layouts and conventions are those of ``chunk_gdn2`` and
``fused_recurrent_gdn2``; the state has no erase term and the decay is one
number per head, or per token and head.  Both run hand-written CUDA through
``gdn2_linear_attn_*``.
"""

from __future__ import annotations

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _strided(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself where the kernels can read it as it lies (contiguous
    innermost dimension, 16-byte aligned base and steps), else a copy."""
    per = 16 // x.element_size()
    sb, st, sh, sd = x.stride()
    B, T, H, _ = x.shape
    if (sd == 1 and (H == 1 or (sh > 0 and sh % per == 0)) and (T == 1 or (st > 0 and st % per == 0))
            and (B == 1 or (sb > 0 and sb % per == 0)) and x.data_ptr() % 16 == 0):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _steps(x: torch.Tensor):
    """Element steps of batch, token and head; a dimension of one element gets the step of a dense tensor."""
    sb, st, sh, _ = x.stride()
    B, T, H, D = x.shape
    if H == 1:
        sh = D
    if T == 1:
        st = H * sh if H > 1 else D
    if B == 1:
        sb = T * st
    return _lib._s3(sb, st, sh)


def _check(q, k, v, g, initial_state, cu_seqlens, states):
    if q.ndim != 4 or q.shape != k.shape:
        raise ValueError(f"q and k must have one shape [B, T, H, K]; got {tuple(q.shape)} and {tuple(k.shape)}.")
    B, T, H, K = q.shape
    if v.ndim != 4 or v.shape[:2] != q.shape[:2] or H == 0 or v.shape[2] % H or v.shape[2] == 0:
        raise ValueError(f"v must have shape [B, T, HV, V] with HV a multiple of H={H}; got {tuple(v.shape)} "
                         f"vs q {tuple(q.shape)}.")
    HV, V = v.shape[2:]
    if K not in (64, 128) or V not in (64, 128):
        raise ValueError(f"head dims K and V must be 64 or 128, got {K} and {V}.")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in _DTYPES:
        raise TypeError(f"q, k, v must all be bf16 or all fp32; got {q.dtype}, {k.dtype}, {v.dtype}.")
    if g is not None:
        if g.dtype not in _DTYPES:
            raise TypeError(f"g must be bf16 or fp32, got {g.dtype}.")
        if tuple(g.shape) not in ((HV,), (B, T, HV)):
            raise ValueError(f"g must have shape [HV] or [B, T, HV]; got {tuple(g.shape)} for B={B}, T={T}, HV={HV}.")
    N = B
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError(
                f"The batch size is expected to be 1 rather than {B} when using `cu_seqlens`. "
                f"Please flatten variable-length inputs before processing.")
        if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
            raise ValueError(f"cu_seqlens must be a vector of N + 1 offsets, got shape {tuple(cu_seqlens.shape)}.")
        N = cu_seqlens.shape[0] - 1
    if initial_state is not None:
        if initial_state.dtype != torch.float32:
            raise TypeError(f"initial_state must be in float32, got {initial_state.dtype}.")
        want = (N if states is None else states, HV, K, V)
        if tuple(initial_state.shape) != want:
            raise ValueError(f"initial_state must have shape {want}, got {tuple(initial_state.shape)}.")
    for name, x in (("k", k), ("v", v), ("g", g), ("initial_state", initial_state), ("cu_seqlens", cu_seqlens)):
        if x is not None and x.device != q.device:
            raise ValueError(f"{name} is on {x.device}, q on {q.device}.")
    return N


def _args(q, k, v, g, h0, ht, o, scale, N, cu, flags, slots=None, num_slots=0):
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    if g is None:
        gs, decay, gd = _lib._s3(0, 0, 0), _lib.DECAY_NONE, _lib.F32
    elif g.ndim == 1:
        gs, decay, gd = _lib._s3(0, 0, g.stride(0)), _lib.DECAY_HEAD, _DTYPES[g.dtype]
    else:
        gs, decay, gd = _lib._s3(*g.stride()), _lib.DECAY_TOKEN, _DTYPES[g.dtype]
    if h0 is not None:
        flags |= _lib.HAS_H0
    if ht is not None:
        flags |= _lib.STORE_FINAL
    ptr = _lib.ptr
    return _lib.LinearAttnArgs(
        B, T, H, HV, K, V, N, _steps(q), _steps(k), _steps(v), gs, ptr(cu), ptr(slots), num_slots,
        0 if h0 is None else h0.stride(0), 0 if ht is None else ht.stride(0), scale, flags, _DTYPES[q.dtype], gd,
        decay, q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(g), ptr(h0), ptr(ht), ptr(o))


def _cu(cu_seqlens):
    return None if cu_seqlens is None else cu_seqlens.to(torch.int64).contiguous()


class ChunkLinearAttnFunction(torch.autograd.Function):
    """Autograd wrapper over ``gdn2_linear_attn_fwd`` / ``gdn2_linear_attn_bwd``."""

    @staticmethod
    def forward(ctx, q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, N, grad):
        B, T, H, K = q.shape
        HV, V = v.shape[2:]
        q, k, v = _strided(q), _strided(k), _strided(v)
        h0 = None if initial_state is None else initial_state.contiguous()
        o = torch.empty(B, T, HV, V, device=q.device, dtype=q.dtype)
        ht = torch.empty(N, HV, K, V, device=q.device, dtype=torch.float32) if output_final_state else None
        save = grad and any(ctx.needs_input_grad)  # needs_input_grad alone is also set under no_grad
        lib = _lib.load()
        with _lib.on_device(q.device):
            args = _args(q, k, v, g, h0, ht, o, scale, N, cu_seqlens, _lib.SAVE_FOR_BWD if save else 0)
            size = lib.gdn2_linear_attn_workspace_size(args)
            ws = torch.empty(size, device=q.device, dtype=torch.uint8)
            _lib.check(lib.gdn2_linear_attn_fwd(args, ws.data_ptr(), size, _lib.stream_ptr(q.device)),
                       "gdn2_linear_attn_fwd")
        if save:
            ctx.save_for_backward(q, k, v, g, h0, cu_seqlens, ws)
            ctx.meta = (scale, N, ctx.needs_input_grad[3], ctx.needs_input_grad[5])
        return o, ht

    @staticmethod
    def backward(ctx, do, dht):
        q, k, v, g, h0, cu, ws = ctx.saved_tensors
        scale, N, want_dg, want_dh0 = ctx.meta
        do = do.contiguous()
        if dht is not None:
            dht = dht.contiguous()
        dq, dk, dv = (torch.empty(x.shape, device=x.device, dtype=x.dtype) for x in (q, k, v))
        dg = torch.empty(g.shape, device=q.device, dtype=g.dtype) if want_dg else None
        dh0 = torch.empty_like(h0) if want_dh0 else None
        ptr = _lib.ptr
        lib = _lib.load()
        with _lib.on_device(q.device):
            args = _args(q, k, v, g, h0, None, None, scale, N, cu, _lib.SAVE_FOR_BWD)
            size = lib.gdn2_linear_attn_bwd_workspace_size(args)
            bws = torch.empty(size, device=q.device, dtype=torch.uint8)
            grads = _lib.LinearAttnGrads(ptr(do), ptr(dht), ptr(dq), ptr(dk), ptr(dv), ptr(dg), ptr(dh0))
            _lib.check(lib.gdn2_linear_attn_bwd(args, grads, ws.data_ptr(), ws.numel(), bws.data_ptr(), size,
                                                _lib.stream_ptr(q.device)), "gdn2_linear_attn_bwd")
        return dq, dk, dv, dg, None, dh0, None, None, None, None


@torch.compiler.disable
def chunk_linear_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor | None = None,
    scale: float | None = None,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.LongTensor | None = None,
):
    r"""Chunkwise linear attention with a decay for each head.

    q, k: ``[B, T, H, K]``; v: ``[B, T, HV, V]``, HV a multiple of H (value
    head ``hv`` reads key head ``hv // (HV // H)``); K, V in {64, 128}; all
    bf16 or all fp32.  Strided views are read in place where their innermost
    dimension is contiguous and their steps are multiples of 16 bytes.
    ``g``: natural-log decays, ``[HV]`` (one per head), ``[B, T, HV]`` or None
    (no decay), bf16 or fp32; ``-inf`` forgets the state.  ``initial_state``:
    ``[N, HV, K, V]`` fp32.  With ``cu_seqlens`` the batch is one packed row
    of N sequences (empty ones allowed); rows outside of every sequence get
    zeros.  ``scale`` defaults to ``K ** -0.5``.

    Returns ``(o, final_state)``; ``final_state`` is None unless
    ``output_final_state``.  Differentiable in q, k, v, g and initial_state,
    through o and the final state.  With bf16 inputs o and the gradients of q,
    k, v, g carry bf16 operand rounding (fp32 accumulation); the final state
    and the gradient of the initial state keep fp32 accuracy.  A non-finite
    input may reach earlier outputs of its own chunk (at most 128 tokens), and
    nothing of other sequences.
    """
    N = _check(q, k, v, g, initial_state, cu_seqlens, None)
    _lib.require_device(q)
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return ChunkLinearAttnFunction.apply(q, k, v, g, float(scale), initial_state, output_final_state,
                                         _cu(cu_seqlens), N, torch.is_grad_enabled())


@torch.compiler.disable
def fused_recurrent_linear_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor | None = None,
    scale: float | None = None,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    inplace_final_state: bool = False,
    cu_seqlens: torch.LongTensor | None = None,
    ssm_state_indices: torch.Tensor | None = None,
):
    r"""Token-by-token linear attention (inference only, no gradients).

    Arguments as ``chunk_linear_attn``.  ``inplace_final_state`` writes the
    states back into ``initial_state`` (contiguous within a state), which is
    then also what is returned.  ``ssm_state_indices`` (``[N]``, with
    ``inplace_final_state``): sequence ``n`` reads and writes slot
    ``ssm_state_indices[n]`` of the pool ``initial_state`` ``[slots, HV, K,
    V]``; slots must differ, and a sequence whose slot is outside the pool
    (say -1, padding) is skipped and gets zero output.  Returns ``(o, final_state)``.
    """
    slots = None
    if ssm_state_indices is not None:
        if not inplace_final_state or initial_state is None or initial_state.ndim != 4:
            raise ValueError("ssm_state_indices needs a pool of states as initial_state and inplace_final_state=True")
        slots = initial_state.shape[0]
    N = _check(q, k, v, g, initial_state, cu_seqlens, slots)
    if inplace_final_state and initial_state is None:
        raise ValueError("inplace_final_state=True requires an initial_state")
    _lib.require_device(q)
    if ssm_state_indices is not None:
        if tuple(ssm_state_indices.shape) != (N,) or ssm_state_indices.device != q.device:
            raise ValueError(f"ssm_state_indices must be a vector of {N} slots on {q.device}")
        if ssm_state_indices.dtype != torch.int32 or not ssm_state_indices.is_contiguous():
            ssm_state_indices = ssm_state_indices.clamp(-1, 2 ** 31 - 1).to(torch.int32).contiguous()
    if scale is None:
        scale = q.shape[-1] ** -0.5
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    q, k, v = _strided(q.detach()), _strided(k.detach()), _strided(v.detach())
    h0 = initial_state
    if h0 is not None:
        h0 = h0.detach()
        if h0.stride()[1:] != (K * V, V, 1) or h0.stride(0) % 4 or h0.data_ptr() % 16:
            if inplace_final_state:
                raise ValueError("an initial_state that is updated in place must be contiguous within a state "
                                 "and 16-byte aligned")
            h0 = h0.contiguous()
    ht = None
    if inplace_final_state:
        ht = h0
    elif output_final_state:
        ht = torch.empty(N, HV, K, V, device=q.device, dtype=torch.float32)
    o = torch.empty(B, T, HV, V, device=q.device, dtype=q.dtype)
    with _lib.on_device(q.device):
        args = _args(q, k, v, g, h0, ht, o, float(scale), N, _cu(cu_seqlens), 0, ssm_state_indices, slots or 0)
        _lib.check(_lib.load().gdn2_linear_attn_recurrent_fwd(args, _lib.stream_ptr(q.device)),
                   "gdn2_linear_attn_recurrent_fwd")
    return o, (initial_state if inplace_final_state else ht)
