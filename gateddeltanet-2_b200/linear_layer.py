"""Linear-attention token mixer with a decay for each head.

The plain sibling of ``GatedDeltaNet2``: one projection to q, k, v, linear
attention (``chunk_linear_attn`` for training and prompts,
``fused_recurrent_linear_attn`` for up to 64 tokens outside training), a layer
norm of each head's output, a SiLU gate and the output projection.  Same
forward signature, return value and cache protocol as ``GatedDeltaNet2``: a
0-1 ``attention_mask`` [B, T] (0: padding) takes padding tokens out before the
projections, and their outputs are zeros.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .layer import _unpad
from .layer_norm import LayerNorm
from .linear_attn import chunk_linear_attn, fused_recurrent_linear_attn


class LinearAttention(nn.Module):
    """``decay``: "fixed" (a slope for each head, from slow to fast, not learned), "token" (learned
    for each token and head: ``-exp(A_log) * softplus(a_proj(x) + dt_bias)``) or "none"."""

    def __init__(
        self,
        hidden_size: int = 2048,
        head_dim: int = 128,
        num_heads: int = 16,
        num_v_heads: int | None = None,
        expand_v: float = 1,
        decay: str = "token",
        layer_idx: int | None = None,
        norm_eps: float = 1e-5,
        **kwargs,
    ):
        super().__init__()
        if decay not in ("fixed", "token", "none"):
            raise ValueError(f"decay must be 'fixed', 'token' or 'none', got {decay!r}")
        self.hidden_size, self.layer_idx, self.decay = hidden_size, layer_idx, decay
        self.num_heads = num_heads
        self.num_v_heads = num_v_heads if num_v_heads is not None else num_heads
        if self.num_v_heads % self.num_heads:
            raise ValueError(f"num_v_heads={self.num_v_heads} must be divisible by num_heads={self.num_heads}.")
        self.head_k_dim, self.head_v_dim = head_dim, int(head_dim * expand_v)
        self.key_dim = self.num_heads * self.head_k_dim
        self.value_dim = self.num_v_heads * self.head_v_dim
        self.qkv_proj = nn.Linear(hidden_size, 2 * self.key_dim + self.value_dim, bias=False)
        if decay == "token":
            self.a_proj = nn.Linear(hidden_size, self.num_v_heads, bias=False)
            self.A_log = nn.Parameter(torch.log(torch.empty(self.num_v_heads, dtype=torch.float32).uniform_(1, 16)))
            self.A_log._no_weight_decay = True
            dt = torch.exp(torch.rand(self.num_v_heads) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
            self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
            self.dt_bias._no_weight_decay = True
        elif decay == "fixed":
            slopes = torch.log1p(-torch.exp2(torch.linspace(-12, -5, self.num_v_heads)))
            self.register_buffer("slopes", slopes, persistent=False)
        self.g_proj = nn.Linear(hidden_size, self.value_dim, bias=False)
        self.o_norm = LayerNorm(self.head_v_dim, eps=norm_eps)
        self.o_proj = nn.Linear(self.value_dim, hidden_size, bias=False)
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.xavier_uniform_(m.weight, gain=2 ** -2.5)

    def forward(self, hidden_states, attention_mask=None, past_key_values=None, use_cache=False,
                output_attentions=False, cu_seqlens=None, **kwargs):
        B, T, _ = hidden_states.shape
        if attention_mask is not None:
            if attention_mask.ndim != 2 or attention_mask.shape[0] != B or attention_mask.shape[1] < T:
                raise ValueError(f"attention_mask must be a 0-1 matrix [batch, tokens] for padding, got "
                                 f"{tuple(attention_mask.shape)} for hidden states {tuple(hidden_states.shape)}")
            if cu_seqlens is not None:
                raise ValueError("attention_mask and cu_seqlens cannot be given together")
            indices, cu_seqlens = _unpad(attention_mask[:, -T:] if T else attention_mask[:, :0])
            hidden_states = hidden_states.flatten(0, 1).index_select(0, indices).unsqueeze(0)
        state = None
        if past_key_values is not None:
            if self.layer_idx is None:
                raise ValueError("a layer_idx is required to use a cache")
            if len(past_key_values) > self.layer_idx:
                state = past_key_values[self.layer_idx]["recurrent_state"]
        # strided views of one projection's output: the operators read them in place
        q, k, v = self.qkv_proj(hidden_states).split([self.key_dim, self.key_dim, self.value_dim], dim=-1)
        q, k = q.unflatten(-1, (self.num_heads, -1)), k.unflatten(-1, (self.num_heads, -1))
        v = v.unflatten(-1, (self.num_v_heads, -1))
        g = None
        if self.decay == "token":
            g = -self.A_log.float().exp() * F.softplus(self.a_proj(hidden_states).float() + self.dt_bias)
        elif self.decay == "fixed":
            g = self.slopes
        # The older mixer's switch.  Calls of 16 heads of 128, chunkwise and token-serial: 1 sequence of 4, 8, 64
        # tokens 10 and 7, 10 and 10, 10 and 53 us; 16 sequences of 8, 16, 64 tokens 27 and 16, 27 and 27, 28 and
        # 88 us; 256 sequences of 8, 16, 64 tokens 313 and 209, 313 and 362, 313 and 1271 us.
        if T <= 64 and not self.training and not torch.is_grad_enabled():
            o, state = fused_recurrent_linear_attn(q, k, v, g, initial_state=state, output_final_state=use_cache,
                                                   cu_seqlens=cu_seqlens)
        else:
            o, state = chunk_linear_attn(q, k, v, g, initial_state=state, output_final_state=use_cache,
                                         cu_seqlens=cu_seqlens)
        if past_key_values is not None:
            past_key_values.update(layer_idx=self.layer_idx, recurrent_state=state, offset=T)
        gate = self.g_proj(hidden_states).unflatten(-1, (self.num_v_heads, -1))
        o = self.o_norm(o) * F.silu(gate)
        o = self.o_proj(o.flatten(-2))
        if attention_mask is not None:
            o = o.new_zeros(B * T, o.shape[-1]).index_copy(0, indices, o.squeeze(0)).view(B, T, -1)
        return o, None, past_key_values
