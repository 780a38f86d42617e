"""Refusals of the log probability call, on the host: nothing is launched."""

import pytest
import torch

from llms_b200 import _capi
from llms_b200.kernels import b200_token_logprobs


def test_calls_refused():
    x, t = torch.zeros(2, 3, 50), torch.zeros(2, 3, dtype=torch.int64)
    for logits, tokens, top in ((x, t[0], 0), (x, t.int(), 0), (x, t, -1), (x, t, 51), (x.double(), t, 0), (x[..., :0], t, 0),
                                (torch.zeros(2, 3, 100), t, 65), (torch.tensor(1.0), torch.tensor(0), 0)):
        with pytest.raises(ValueError):
            b200_token_logprobs(logits, tokens, top=top)
    with pytest.raises(RuntimeError):
        b200_token_logprobs(x, t)  # no CPU path


def test_c_entry_point_refuses_before_any_launch():
    before = _capi.launch_count()
    p = 4096

    def call(x=p, ld=100, tok=p, lp=p, ent=p, ids=p, lps=p, M=2, V=100, top=4, dtype=2):
        return _capi.lib.b200mm_token_logprobs(x, ld, tok, lp, ent, ids, lps, M, V, top, dtype, None)

    OK, SHAPE, ALIGN, DTYPE, ARG = 0, 1, 2, 3, 5
    assert call(dtype=5) == DTYPE
    assert call(M=-1) == SHAPE and call(V=0) == SHAPE and call(ld=99) == SHAPE and call(M=1 << 27) == SHAPE
    assert call(V=(1 << 31) - 1, ld=1 << 31) == SHAPE
    assert call(top=-1) == SHAPE and call(top=65) == SHAPE and call(V=3, top=4) == SHAPE
    for n in ("x", "tok", "lp", "ent", "ids", "lps"):
        assert call(**{n: None}) == ARG, n
    assert call(x=4097) == ALIGN and call(x=4098, dtype=0) == ALIGN
    assert call(M=0) == OK
    assert _capi.launch_count() == before


def test_odd_addresses_are_refused():
    for bad in range(1, 6):
        p = [4096] * 6
        p[bad] += 2
        assert _capi.lib.b200mm_token_logprobs(p[0], 100, *p[1:], 2, 100, 4, 2, None) == 2, bad
