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
    through o and the final state (once, in reverse mode; forward-mode tangents are
    refused).  With bf16 inputs o and the gradients of q, k, v, g carry bf16
    operand rounding (fp32 accumulation); the final state and the gradient of
    the initial state are within 1e-5 of their size, 4e-6 as a rule (products of
    two bf16 terms per value).  A non-finite input may reach earlier outputs of
    its own chunk (at most 128 tokens), and nothing of other sequences; an
    infinite value stays one in the state unless a decay after it underflows
    (zero times it is NaN).
    """
    return _lib.ops().chunk_linear_attn(q, k, v, g, scale, initial_state, output_final_state, cu_seqlens)


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

    Arguments as ``chunk_linear_attn`` (rows outside of every sequence get zeros
    here too).  ``inplace_final_state`` writes the
    states back into ``initial_state`` (contiguous within a state), which is
    then also what is returned.  ``ssm_state_indices`` (``[N]``, with
    ``inplace_final_state``): sequence ``n`` reads and writes slot
    ``ssm_state_indices[n]`` of the pool ``initial_state`` ``[slots, HV, K,
    V]``; slots must differ, and a sequence whose slot is outside the pool
    (say -1, padding) is skipped and gets zero output.  Returns ``(o, final_state)``.
    """
    return _lib.ops().recurrent_linear_attn(q, k, v, g, scale, initial_state, output_final_state, inplace_final_state,
                                            cu_seqlens, ssm_state_indices)
