"""4-bit weights: the format, and refusals on the host (nothing is launched)."""

import pytest
import torch
from torch import nn

from llms_b200 import _capi
from llms_b200.kernels import (Int4Attention, Int4FFN, Int4Linear, dequantize_grouped, int4_fused_gate_up_silu, int4_fused_qkv,
                               int4_linear, quantize_grouped)

BF = torch.bfloat16


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_quantize_is_within_half_a_step(group, dtype):
    W = torch.randn(37, 256).to(dtype)
    W[3] = 0
    w, s = quantize_grouped(W, group)
    assert w.shape == (37, 128) and w.dtype == torch.uint8 and s.shape == (37, 256 // group)
    assert s.dtype == (BF if dtype == torch.float32 else dtype)
    D = dequantize_grouped(w, s)
    step = s.float().repeat_interleave(group, 1)
    # half a step, and what the scale's own rounding takes from the largest weight
    assert ((D - W.float()).abs() <= step * (0.5 + 7 * torch.finfo(s.dtype).eps)).all()
    assert not D[3].any()
    low, high = w[0, 0] & 15, w[0, 0] >> 4
    assert D[0, 0] == (int(low) - 8) * s[0, 0].float() and D[0, 1] == (int(high) - 8) * s[0, 0].float()


def test_quantize_refuses():
    for W, g in ((torch.zeros(4, 96), 64), (torch.zeros(4, 128), 16), (torch.zeros(128), 32)):
        with pytest.raises(ValueError):
            quantize_grouped(W, g)
    with pytest.raises(ValueError):
        Int4Linear(96, 8, group=64)
    with pytest.raises(ValueError):
        Int4Linear.from_linear(nn.Linear(64, 8), group=32)  # a bias


def test_calls_refused():
    w, s = quantize_grouped(torch.randn(8, 128).to(BF), 64)
    x = torch.zeros(2, 128, dtype=BF)
    with pytest.raises(RuntimeError):
        int4_linear(x, w, s)  # no CPU path
    for a, b, c in ((x[:, :64], w, s), (x, w.int(), s), (x, w[0], s), (x, w, s[:, :1][:, :0]), (x, w, s[:4]), (x.float(), w, s.float()),
                    (x.half(), w, s), (x, w, s.repeat(1, 4)), (x, w[:, :48], s)):
        with pytest.raises(ValueError):
            int4_linear(a, b, c)
        with pytest.raises(ValueError):
            int4_fused_gate_up_silu(a, b, c, b, c)
    with pytest.raises(ValueError):
        int4_fused_gate_up_silu(x, w, s, w[:4], s[:4])
    with pytest.raises(ValueError):
        int4_fused_qkv(x, w, s, n_q=4, n_k=1)
    assert int4_linear(x[:0], w, s).shape == (0, 8)


def test_c_entry_points_refuse_before_any_launch():
    before = _capi.launch_count()
    p = 4096

    def call(x=p, ldx=256, w=p, ldw=128, s=p, lds=2, group=128, y=p, ldy=64, M=2, N=64, K=256, dtype=2, ws=None, n=0):
        a = _capi.lib.b200mm_linear_w4(x, ldx, w, ldw, s, lds, group, y, ldy, M, N, K, dtype, ws, n, None)
        b = _capi.lib.b200mm_gate_up_silu_w4(x, ldx, w, w, ldw, s, s, lds, group, y, ldy, M, N, K, dtype, ws, n, None)
        assert a == b
        return a

    OK, SHAPE, ALIGN, DTYPE, ARG, WORKSPACE = 0, 1, 2, 3, 5, 6
    assert call(dtype=0) == DTYPE and call(dtype=9) == DTYPE
    assert call(group=16) == SHAPE and call(group=256) == SHAPE and call(K=192, group=128) == SHAPE and call(K=0) == SHAPE
    assert call(N=0) == SHAPE and call(M=-1) == SHAPE and call(K=65536 + 128, ldx=1 << 17, ldw=1 << 16, lds=1 << 10) == SHAPE
    assert call(ldx=255) == SHAPE and call(ldw=112) == SHAPE and call(lds=1) == SHAPE and call(ldy=63) == SHAPE
    assert call(M=1 << 31) == SHAPE and call(N=(1 << 24) + 1, ldy=1 << 25) == SHAPE
    for n in ("x", "w", "s", "y"):
        assert call(**{n: None}) == ARG
    assert call(x=4104) == ALIGN and call(ldx=260) == ALIGN and call(w=4104) == ALIGN and call(ldw=136) == ALIGN
    assert call(M=0) == OK and call(M=0, x=None) == OK
    need = _capi.lib.b200mm_w4_workspace_size(4096, 64, 256, 1)
    assert need >= 2 * 64 * 256 * 2 and _capi.lib.b200mm_w4_workspace_size(1, 64, 256, 1) == 0
    assert call(M=4096) == WORKSPACE and call(M=4096, ws=4096, n=64) == WORKSPACE and call(M=4096, ws=4112, n=1 << 30) == WORKSPACE
    assert _capi.launch_count() == before


def test_modules_load_each_others_state():
    ffn = Int4FFN(128, 64, group=64)
    src = nn.Module()
    src.gate, src.up, src.down = nn.Linear(128, 64, bias=False), nn.Linear(128, 64, bias=False), nn.Linear(64, 128, bias=False)
    ffn.load_state_dict(Int4FFN.from_eager(src, group=64).state_dict())
    att = Int4Attention(hidden_size=128, num_heads=4, num_kv_heads=2, head_dim=32, rms_eps=1e-6, group=32)
    assert att.w_qkv.shape == (4 * 32 + 2 * 64, 64) and not hasattr(att, "W_qkv")
    lin = Int4Linear(128, 64, group=128)
    lin.load_state_dict(Int4Linear.from_linear(src.gate, group=128).state_dict())


def test_swaps_leave_4_bit_modules_alone():
    from llms_b200.kernels import Int8Attention, apply_int4_kernels, apply_int8_kernels, apply_triton_kernels
    from llms_b200.qwen3 import Qwen3Model, Qwen3Shape
    shape = Qwen3Shape(vocab_size=64, hidden_size=128, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
                       head_dim=64, intermediate_size=256, max_position_embeddings=32)
    m = apply_int4_kernels(Qwen3Model(shape), lm_head=True)
    blk = m.layers[0]
    kinds = [type(x) for x in (blk.attn, blk.ffn, blk.attn.o, blk.ffn.down, m.lm_head)]
    assert kinds == [Int4Attention, Int4FFN, Int4Linear, Int4Linear, Int4Linear]
    apply_triton_kernels(m), apply_int8_kernels(m), apply_int4_kernels(m, lm_head=True)
    assert [type(x) for x in (blk.attn, blk.ffn, blk.attn.o, blk.ffn.down, m.lm_head)] == kinds
    m8 = apply_int4_kernels(apply_int8_kernels(Qwen3Model(shape)))
    assert isinstance(m8.layers[0].attn, Int8Attention) and isinstance(m8.layers[0].attn.o, Int4Linear)
    assert m.alloc_cache(40, int8=True).capacity == 64 and m.alloc_cache(40).k[0].shape[2] == 40


def test_odd_addresses_are_refused():
    p = 4096
    for s, y in ((p + 1, p), (p, p + 1)):
        assert _capi.lib.b200mm_linear_w4(p, 256, p, 128, s, 2, 128, y, 64, 2, 64, 256, 2, None, 0, None) == 2
        assert _capi.lib.b200mm_gate_up_silu_w4(p, 256, p, p, 128, p, s, 2, 128, y, 64, 2, 64, 256, 2, None, 0, None) == 2


def test_4_bit_models_are_not_sharded():
    from llms_b200.kernels import apply_int4_kernels, apply_int8_kernels
    from llms_b200.qwen3 import Qwen3Model, Qwen3Shape
    from llms_b200.shard import shard_decode_model
    shape = Qwen3Shape(vocab_size=64, hidden_size=128, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
                       head_dim=64, intermediate_size=256, max_position_embeddings=32)
    for m in (apply_int4_kernels(Qwen3Model(shape)), apply_int4_kernels(apply_int8_kernels(Qwen3Model(shape)), o=False)):
        with pytest.raises(ValueError, match="4-bit"):
            shard_decode_model(m, 0, 1)


@pytest.mark.parametrize("hidden,heads,inter,head_dim,lm_head,group", [(128, 2, 160, 64, False, 128), (128, 2, 256, 48, False, 64), (192, 1, 256, 128, False, 128),
                                                                       (128, 2, 256, 64, True, 48)])
def test_a_refused_swap_changes_nothing(hidden, heads, inter, head_dim, lm_head, group):
    """Columns that the group does not divide, in a projection that comes after others."""
    from llms_b200.kernels import apply_int4_kernels
    from llms_b200.qwen3 import Qwen3Model, Qwen3Shape
    m = Qwen3Model(Qwen3Shape(vocab_size=64, hidden_size=hidden, num_hidden_layers=2, num_attention_heads=heads, num_key_value_heads=1,
                              head_dim=head_dim, intermediate_size=inter, max_position_embeddings=32))
    kinds = [type(x) for x in m.modules()]
    with pytest.raises(ValueError, match="group"):
        apply_int4_kernels(m, group=group, lm_head=lm_head)
    assert [type(x) for x in m.modules()] == kinds
    m.layers[1].attn.o = nn.Linear(heads * head_dim, hidden)
    with pytest.raises(ValueError):
        apply_int4_kernels(m, group=32, lm_head=lm_head)
    assert [type(x) for x in m.modules()] == kinds
