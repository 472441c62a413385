"""CPU-side checks of the linear-attention and layer-norm entry points: invalid
arguments are refused before any launch, sizes of the workspaces, the model's
structure with these parts."""

import ctypes

import pytest
import torch


def _la(gdn2, **kw):
    L = gdn2._lib
    a = dict(B=2, T=100, H=2, HV=4, K=64, V=128, N=2, scale=0.125, flags=0, dtype=L.BF16, dtype_g=L.F32,
             decay=L.DECAY_NONE, q_b=12800, q_t=128, q_h=64, k_b=12800, k_t=128, k_h=64, v_b=51200, v_t=512, v_h=128)
    a.update(kw)
    return L.LinearAttnArgs(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(HV=3), 2), (dict(H=0), 2), (dict(B=-1), 2), (dict(N=3), 2), (dict(K=96), 4), (dict(V=32), 4),
    (dict(dtype=2), 3), (dict(decay=3), 7), (dict(decay=1, dtype_g=5), 3), (dict(flags=1), 7), (dict(flags=1 << 9), 7),
    (dict(HV=1 << 17, H=1 << 17), 2), (dict(T=1 << 31), 2), (dict(flags=1 << 4), 1), (dict(flags=1 << 5), 1), (dict(), 1)])
def test_invalid_linear_attn_args(gdn2, kw, code):
    lib = gdn2._lib.load()
    for call in (lambda a: lib.gdn2_linear_attn_fwd(a, None, 0, None),
                 lambda a: lib.gdn2_linear_attn_recurrent_fwd(a, None)):
        assert call(_la(gdn2, **kw)) == code


def test_linear_attn_alignment_workspace_and_flags(gdn2):
    L, lib = gdn2._lib, gdn2._lib.load()
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    ptrs = dict(q=p, k=p, v=p, o=p)
    assert lib.gdn2_linear_attn_fwd(_la(gdn2, **{**ptrs, "q": p + 2}), None, 0, None) == 5
    assert lib.gdn2_linear_attn_fwd(_la(gdn2, **ptrs, v_t=516), None, 0, None) == 5
    assert lib.gdn2_linear_attn_fwd(_la(gdn2, **ptrs, flags=L.SAVE_FOR_BWD), None, 0, None) == 6
    assert lib.gdn2_linear_attn_workspace_size(_la(gdn2, flags=L.SAVE_FOR_BWD)) >= 2 * 1 * 4 * 64 * 128 * 2
    assert lib.gdn2_linear_attn_workspace_size(_la(gdn2)) == 0  # one segment, nothing kept
    assert lib.gdn2_linear_attn_workspace_size(_la(gdn2, K=100)) == 0
    grads = L.LinearAttnGrads(dout=p, dq=p, dk=p, dv=p)
    assert lib.gdn2_linear_attn_bwd(_la(gdn2, **ptrs), grads, None, 0, None, 0, None) == 7  # no SAVE_FOR_BWD
    save = dict(flags=L.SAVE_FOR_BWD)
    assert lib.gdn2_linear_attn_bwd(_la(gdn2, **ptrs, **save), None, None, 0, None, 0, None) == 1
    assert lib.gdn2_linear_attn_bwd(_la(gdn2, **ptrs, **save), L.LinearAttnGrads(dout=p, dq=p, dk=p), None, 0, None, 0,
                                    None) == 1
    assert lib.gdn2_linear_attn_bwd(_la(gdn2, **ptrs, **save), L.LinearAttnGrads(dout=p, dq=p, dk=p, dv=p, dg=p), None,
                                    0, None, 0, None) == 7  # no decay, but its gradient
    assert lib.gdn2_linear_attn_bwd(_la(gdn2, **ptrs, **save), grads, None, 0, None, 0, None) == 6
    # pool slots belong to the recurrent form
    assert lib.gdn2_linear_attn_fwd(_la(gdn2, **ptrs, state_indices=p, num_slots=2), None, 0, None) == 7
    assert lib.gdn2_linear_attn_recurrent_fwd(_la(gdn2, **ptrs, state_indices=p, num_slots=-1), None) == 2
    assert lib.gdn2_linear_attn_recurrent_fwd(_la(gdn2, **ptrs, state_stride_in=2), None) == 5
    assert lib.gdn2_linear_attn_recurrent_fwd(_la(gdn2, **ptrs, **save), None) == 7
    # nothing to do
    assert lib.gdn2_linear_attn_fwd(_la(gdn2, B=0, N=0), None, 0, None) in (0, 6)


@pytest.mark.parametrize("kw,code", [
    (dict(D=0), 2), (dict(rows=-1), 2), (dict(D=32769), 4), (dict(dtype=7), 3), (dict(weight=16, dtype_weight=9), 3),
    (dict(residual=16, dtype=1, dtype_residual=0), 3), (dict(), 1), (dict(rows=0), 0)])
def test_invalid_layer_norm_args(gdn2, kw, code):
    L, lib = gdn2._lib, gdn2._lib.load()
    a = L.LayerNormArgs(**{**dict(rows=4, D=64, eps=1e-5, dtype=L.BF16, dtype_residual=L.F32, dtype_weight=L.F32), **kw})
    assert lib.gdn2_layer_norm_fwd(a, None) == code
    if code not in (0,):
        assert lib.gdn2_layer_norm_bwd(a, L.LayerNormGrads(), None, 0, None) == code
    assert (lib.gdn2_layer_norm_bwd_workspace_size(a) == 0) == (code in (2, 3, 4))


def test_layer_norm_bwd_workspace(gdn2):
    L, lib = gdn2._lib, gdn2._lib.load()
    a = L.LayerNormArgs(rows=4, D=64, dtype=L.BF16, dtype_weight=L.F32, mean=16, rstd=16)
    assert lib.gdn2_layer_norm_bwd(a, L.LayerNormGrads(dy=16, s=16, dx=16, dweight=16), None, 0, None) == 6


def test_ops_need_a_gpu(gdn2):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    x = torch.zeros(1, 8, 1, 64)
    for f in (gdn2.chunk_linear_attn, gdn2.fused_recurrent_linear_attn):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            f(x, x, x)
        with pytest.raises(ValueError):
            f(x, x[:, :4], x)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        gdn2.layer_norm(x)


def test_model_structure(gdn2):
    from gdn2_b200 import model as m
    with torch.device("meta"):
        net = m.GPT(m.HybridConfig(mixer="linear", norm="layer"))
    names = {n for n, _ in net.named_parameters()}
    for n in ("transformer.ln_f.bias", "transformer.h.0.norm_1.bias", "transformer.h.0.attn.qkv_proj.weight",
              "transformer.h.0.attn.A_log", "transformer.h.0.attn.o_norm.weight", "transformer.h.1.attn.attn.weight"):
        assert n in names, n


def test_more_states_than_a_grid_has_blocks(gdn2):
    """N * HV blocks walk the states: 2^31 of them are refused, not taken modulo 2^32."""
    lib = gdn2._lib.load()
    a = _la(gdn2, B=1, T=100, N=1 << 29, cu_seqlens=16)
    assert lib.gdn2_linear_attn_fwd(a, None, 0, None) == 2
    assert lib.gdn2_linear_attn_recurrent_fwd(a, None) == 2
    assert lib.gdn2_linear_attn_workspace_size(a) == 0
