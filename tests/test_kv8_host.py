"""Refusals of the 8-bit KV cache calls, on the host: nothing is launched."""

import ctypes

import pytest
import torch

from llms_b200 import _capi
from llms_b200.kernels import Int8KV, Int8KVCache, int8_kv_append, int8_kv_decode_attn, int8_kv_expand, int8_kv_step


def _kv(rows=2, KV=2, S=128, D=64, dtype=torch.bfloat16):
    return Int8KV.alloc(rows=rows, num_kv_heads=KV, max_seq_len=S, head_dim=D, dtype=dtype, device="cpu")


def test_alloc_rounds_the_capacity_up():
    assert _kv(S=1).capacity == 64 and _kv(S=64).capacity == 64 and _kv(S=65).capacity == 128


@pytest.mark.parametrize("change", [
    {"kq": torch.zeros(2, 2, 128, 64), "vq": torch.zeros(2, 2, 128, 64)},                       # not int8
    {"kq": torch.zeros(2, 2, 100, 64, dtype=torch.int8), "vq": torch.zeros(2, 2, 100, 64, dtype=torch.int8)},
    {"kq": torch.zeros(2, 2, 128, 72, dtype=torch.int8), "vq": torch.zeros(2, 2, 128, 72, dtype=torch.int8)},
    {"vs": torch.zeros(2, 2, 3)},
    {"ks": torch.zeros(2, 2, 1), "vs": torch.zeros(2, 2, 1)},
    {"ks": torch.zeros(2, 2, 2, dtype=torch.float64), "vs": torch.zeros(2, 2, 2, dtype=torch.float64)},
    {"kt": torch.zeros(2, 2, 32, 64), "vt": torch.zeros(2, 2, 32, 64)},
    {"kt": torch.zeros(2, 2, 64, 64, dtype=torch.float64), "vt": torch.zeros(2, 2, 64, 64, dtype=torch.float64)},
    {"kq": torch.zeros(2, 2, 64, 128, dtype=torch.int8).transpose(2, 3),
     "vq": torch.zeros(2, 2, 64, 128, dtype=torch.int8).transpose(2, 3)},                      # tokens not contiguous
])
def test_storage_refused(change):
    kv = _kv()
    parts = {n: getattr(kv, n) for n in ("kq", "ks", "kt", "vq", "vs", "vt")}
    with pytest.raises(ValueError):
        Int8KV(**{**parts, **change})


def test_calls_refused():
    kv = _kv()
    q, k = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        int8_kv_append(kv, k, k, 0)  # a CPU cache
    with pytest.raises(RuntimeError):
        int8_kv_decode_attn(q, kv, 0, scale=0.1)
    with pytest.raises(RuntimeError):
        int8_kv_expand(kv, 5)
    for bad in (k[:, :1], k[..., :32], k.float(), k[:, :, 0]):
        with pytest.raises(ValueError):
            int8_kv_append(kv, bad, bad, 0)
    with pytest.raises(ValueError):
        int8_kv_append(kv, k, k.expand(2, 2, 2, 64), 0)
    with pytest.raises(ValueError):
        int8_kv_append(kv, torch.zeros(3, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 1, 64, dtype=torch.bfloat16), 0)
    for bad in (q[:, :3], q[..., :32], q.half(), q.expand(2, 4, 2, 64), q[0]):
        with pytest.raises(ValueError):
            int8_kv_decode_attn(bad, kv, 0, scale=0.1)
    with pytest.raises(ValueError):
        int8_kv_expand(kv, 129)
    with pytest.raises(ValueError):
        int8_kv_expand(kv, 1, batch=3)


def _c_cache(**kw):
    f = dict(kq=4096, ks=4096, kt=4096, vq=4096, vs=4096, vt=4096, q_sb=2 * 128 * 64, q_sh=128 * 64, s_sb=4, s_sh=2,
             t_sb=2 * 64 * 64, t_sh=64 * 64, S=128, KV=2, D=64, dtype=2, reserved=0)
    f.update(kw)
    return _capi.Kv8(**f)


OK, SHAPE, ALIGN, DTYPE, ARG, WORKSPACE = 0, 1, 2, 3, 5, 6


def _append(c, B=2, T=1, pos=0, stride=0, p=4096, ld=64):
    return _capi.lib.b200mm_kv8_append(ctypes.byref(c), p, 2 * ld, ld, ld, p, 2 * ld, ld, ld, B, T, pos, None, stride, None)


def _decode(c, B=2, H=4, pos=0, stride=0, scale=0.1, ws=4096, n=1 << 30, q=4096):
    return _capi.lib.b200mm_kv8_decode(ctypes.byref(c), q, H * 64, 64, 4096, H * 64, 64, B, H, pos, None, stride, scale,
                                       ws, n, None)


def test_c_entry_points_refuse_before_any_launch():
    before = _capi.launch_count()
    for bad, code in (({"dtype": 7}, DTYPE), ({"S": 100}, SHAPE), ({"S": 0}, SHAPE), ({"S": (1 << 24) + 64, "q_sh": 1 << 40}, SHAPE),
                      ({"D": 8}, SHAPE), ({"D": 272}, SHAPE), ({"D": 40}, SHAPE), ({"KV": 0}, SHAPE), ({"ks": None}, ARG),
                      ({"vt": None}, ARG), ({"q_sh": 64}, SHAPE), ({"q_sb": 0}, SHAPE), ({"t_sb": 0}, SHAPE), ({"s_sh": 1}, SHAPE),
                      ({"kq": 4097}, ALIGN), ({"q_sb": 2 * 128 * 64 + 8}, ALIGN), ({"t_sh": 64 * 64 + 4}, ALIGN)):
        c = _c_cache(**bad)
        assert _append(c) == code, bad
        assert _decode(c) == code, bad
        assert _capi.lib.b200mm_kv8_decode_workspace_size(ctypes.byref(c), 2, 4) == 0, bad
    c = _c_cache()
    assert _append(c, B=-1) == SHAPE and _append(c, T=-1) == SHAPE and _append(c, T=129) == SHAPE
    assert _append(c, pos=128) == SHAPE and _append(c, pos=127, T=2) == SHAPE and _append(c, pos=-2) == SHAPE
    assert _append(c, stride=2) == ARG and _append(c, p=None) == ARG and _append(c, p=4100) == ALIGN and _append(c, ld=68) == ALIGN
    assert _append(c, B=0) == OK and _append(c, T=0) == OK
    assert _decode(c, H=3) == SHAPE and _decode(c, H=0) == SHAPE and _decode(c, pos=128) == SHAPE
    assert _decode(c, scale=0.0) == ARG and _decode(c, scale=float("nan")) == ARG and _decode(c, q=None) == ARG
    assert _decode(c, q=4104) == ALIGN
    assert _decode(c, ws=None) == WORKSPACE and _decode(c, n=16) == WORKSPACE and _decode(c, ws=4096 + 16) == WORKSPACE
    assert _decode(c, B=0) == OK
    assert _capi.lib.b200mm_kv8_append(None, None, 0, 0, 0, None, 0, 0, 0, 1, 1, 0, None, 0, None) == ARG
    assert _capi.launch_count() == before


def test_rewind_takes_the_open_block_from_its_8_bit_values():
    kv = _kv(rows=1, KV=1, S=256)
    kv.length = 200
    kv.kq.copy_(torch.arange(256 * 64).remainder(255).sub(127).view(1, 1, 256, 64))
    kv.ks.fill_(0.5)
    kv.kt.fill_(7)
    kv.rewind(195)  # inside the last block: its tokens are there
    assert kv.length == 195 and (kv.kt == 7).all()
    kv.rewind(70)
    assert torch.equal(kv.kt[0, 0, :6], (kv.kq[0, 0, 64:70].float() * 0.5).bfloat16()) and (kv.kt[0, 0, 6:] == 7).all()
    with pytest.raises(ValueError):
        kv.rewind(71)


def test_model_cache_counts_and_seeks():
    c = Int8KVCache.alloc(num_layers=2, max_batch=1, num_kv_heads=1, max_seq_len=100, head_dim=64, dtype=torch.float16, device="cpu")
    assert c.capacity == 128 and c.cur_len == 0
    c.cur_len = 90
    c.seek(64)
    assert c.cur_len == 64 and [x.length for x in c.layers] == [64, 64]
    with pytest.raises(ValueError):
        c.seek(65)


def test_overlapping_rows_or_heads_and_odd_addresses_are_refused():
    n = 128 * 64
    for bad, code in (({"q_sb": n, "q_sh": n}, SHAPE), ({"q_sb": 2 * n - 16}, SHAPE), ({"s_sb": 3}, SHAPE),
                      ({"t_sb": 64 * 64, "t_sh": 64 * 64}, SHAPE), ({"q_sb": n, "q_sh": 2 * n - 16}, SHAPE),
                      ({"q_sh": 1 << 62, "q_sb": 1 << 62}, SHAPE), ({"ks": 4098}, ALIGN), ({"vs": 4097}, ALIGN)):
        c = _c_cache(**bad)
        assert _append(c) == code and _decode(c) == code, bad
    one_row = _c_cache(q_sb=0, s_sb=0, t_sb=0)
    assert _append(one_row, B=1, T=0) == OK and _decode(one_row, B=1, ws=None) == WORKSPACE
    heads_first = _c_cache(q_sb=n, q_sh=2 * n, s_sb=2, s_sh=4, t_sb=64 * 64, t_sh=2 * 64 * 64)
    assert _append(heads_first, T=0) == OK and _append(heads_first, B=3, T=0) == SHAPE
    c = _c_cache()
    assert _capi.lib.b200mm_kv8_append(ctypes.byref(c), 4096, 128, 64, 64, 4096, 128, 64, 64, 2, 1, 0, 4100, 1, None) == ALIGN
    assert _capi.lib.b200mm_kv8_decode(ctypes.byref(c), 4096, 256, 64, 4097, 256, 64, 2, 4, 0, None, 0, 0.1, 4096, 1 << 30,
                                       None) == ALIGN


def test_struct_layout():
    """llms_b200._capi.Kv8 has b200mm_kv8's layout (6 pointers, 7 int64, 4 int32)."""
    off = {n: getattr(_capi.Kv8, n).offset for n, _ in _capi.Kv8._fields_}
    names = ["kq", "ks", "kt", "vq", "vs", "vt", "q_sb", "q_sh", "s_sb", "s_sh", "t_sb", "t_sh", "S"]
    assert [off[n] for n in names] == list(range(0, 104, 8))
    assert [off[n] for n in ("KV", "D", "dtype", "reserved")] == [104, 108, 112, 116] and ctypes.sizeof(_capi.Kv8) == 120


def test_going_back_twice_refills_the_open_block():
    """A token that opened the next block took the place of the first one's
    tokens: going back to its border, and then further, finds them in 8 bits."""
    for how in ("rewind", "cur_len"):
        c = Int8KVCache.alloc(num_layers=1, max_batch=1, num_kv_heads=1, max_seq_len=128, head_dim=64, dtype=torch.float16,
                              device="cpu")
        kv = c.layers[0]
        kv.kq.fill_(3)
        kv.ks.fill_(0.5)
        c.cur_len = 65
        kv.kt.fill_(7)
        if how == "rewind":
            c.seek(64)
            assert (kv.kt == 7).all()
            c.seek(40)
        else:
            c.cur_len = 64
            c.cur_len = 40
        assert (kv.kt[0, 0, :40] == 1.5).all() and (kv.kt[0, 0, 40:] == 7).all(), how
        kv.kt[0, 0, :40] = 9
        c.seek(10)  # inside the block that is open now
        assert (kv.kt[0, 0, :40] == 9).all() and c.cur_len == 10 == kv.length


def _captured_step(max_positions, cache_of):
    """A GraphedDecodeStep without its graph (no GPU here): replays are counted."""
    import types

    from llms_b200.qwen3 import GraphedDecodeStep, Qwen3Model, Qwen3Shape
    model = Qwen3Model(Qwen3Shape(vocab_size=8, hidden_size=32, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=2,
                                  head_dim=16, intermediate_size=32, max_position_embeddings=max_positions))
    step = GraphedDecodeStep.__new__(GraphedDecodeStep)
    step.model, step.cache, step.replays = model, cache_of(model), 0

    def replay():
        step.replays += 1

    step.graph, step.logits = types.SimpleNamespace(replay=replay), torch.zeros(1, 1, 8)
    step.ids, step.pos = torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, dtype=torch.long)
    return step


@pytest.mark.parametrize("int8,size", [(True, 100), (False, 128)])
def test_a_captured_step_stays_inside_the_rope_tables(int8, size):
    """100 positions, and a cache that reaches further (8-bit: two blocks of 64)."""
    from llms_b200.qwen3 import GraphedDecodeStep
    step = _captured_step(100, lambda m: m.alloc_cache(size, int8=int8))
    ids = torch.ones(1, 1, dtype=torch.long)
    step.cache.cur_len = 99
    step(ids, 99)
    assert step.replays == 1 and step.cache.cur_len == 100 and step.pos.item() == 99
    for pos in (100, 127, 128, -1):
        with pytest.raises(ValueError):
            step(ids, pos)
    assert step.replays == 1
    with pytest.raises(ValueError, match="no room"):  # building it would run a step at 100
        GraphedDecodeStep(step.model, step.cache, 1)


def test_a_step_is_not_captured_on_a_full_16_bit_cache():
    from llms_b200.qwen3 import GraphedDecodeStep
    step = _captured_step(100, lambda m: m.alloc_cache(40))
    step.cache.cur_len = 40
    with pytest.raises(ValueError, match="no room"):
        GraphedDecodeStep(step.model, step.cache, 1)


def _inference_cache(model):
    with torch.inference_mode():
        return model.alloc_cache(192, int8=True)


def test_a_cache_of_inference_tensors_goes_back_outside_inference_mode():
    step = _captured_step(192, _inference_cache)
    c = step.cache
    c.cur_len = 150
    with torch.inference_mode():
        for layer in c.layers:
            layer.kq.fill_(3), layer.ks.fill_(0.5), layer.kt.fill_(7)
    step(torch.ones(1, 1, dtype=torch.long), 100)  # the block before the open one
    assert c.cur_len == 101 and step.replays == 1
    assert all((x.kt[:, :, :36] == 1.5).all() and (x.kt[:, :, 36:] == 7).all() for x in c.layers)
    c.cur_len = 20
    c.seek(10)
    c.layers[0].rewind(5)
    assert all((x.kt[:, :, :20] == 1.5).all() for x in c.layers)


def test_a_step_built_in_inference_mode_is_called_outside():
    with torch.inference_mode():
        step = _captured_step(64, lambda m: m.alloc_cache(64))
    step(torch.ones(1, 1, dtype=torch.long), 3)
    assert step.replays == 1 and step.ids.item() == 1 and step.pos.item() == 3


def test_a_refused_seek_leaves_every_layer_where_it_was():
    c = Int8KVCache.alloc(num_layers=3, max_batch=1, num_kv_heads=1, max_seq_len=128, head_dim=64, dtype=torch.float16, device="cpu")
    c.cur_len = 100
    c.layers[2].rewind(70)  # (a forward that failed between layers)
    for move in (lambda: c.seek(90), lambda: c.seek(-1), lambda: setattr(c, "cur_len", -1)):
        with pytest.raises(ValueError):
            move()
        assert [x.length for x in c.layers] == [100, 100, 70] and c.cur_len == 100
