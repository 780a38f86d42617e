"""The low-memory decode operators together, as a model uses them: 4-bit
projections, the 8-bit KV cache (prompt, chunks, eager and captured steps), and
log probabilities of what came out.

Two references.  The projections: the same model with every weight the one that
its bits stand for, in float32, both on the 16-bit cache.  The cache: the same
modules on a plain cache that quantises by the formula and attends in 64 bits.
(Not one reference for both: a quantiser turns a difference of d before it into
a whole step with probability d / step, so activations that differ by a bf16
rounding, 0.3 %, come out of 8 bits 1 % apart, sqrt(0.1) of a 3 % step, whatever
the kernels do.)  The bar on the logits' norm, 2e-2, is the one that the swaps of
16-bit kernels meet in their models: activations rounded to bf16 through two
layers.  A logit is a sum of 2560 such roundings, so its error is close to
normal, with at most 2e-2 of the logits' rms as its deviation; over 1e5 logits
none lies beyond 6 deviations (2e-9 each): that bounds an element."""

import dataclasses

import pytest
import torch

from tests.conftest import bf16_check

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import llms_b200.kernels  # noqa: F401


def _models(group=128):
    """(a bf16 model on the kernels, the same weights on plain float32)."""
    from llms_b200.kernels import Int4Linear, apply_int4_kernels, dequantize_grouped
    from llms_b200.qwen3 import QWEN3_4B, Qwen3Model
    shape = dataclasses.replace(QWEN3_4B, num_hidden_layers=2, vocab_size=1000, max_position_embeddings=512)
    torch.manual_seed(0)
    m = Qwen3Model(shape).to("cuda", BF).eval()
    for name, p in m.named_parameters():
        if "norm" not in name:
            torch.nn.init.normal_(p, std=0.02)
    plain = Qwen3Model(shape).cuda().eval()
    plain.load_state_dict(m.state_dict())
    apply_int4_kernels(m, group=group, lm_head=True)
    with torch.no_grad():
        for a, b in zip(m.layers, plain.layers):
            b.attn.q.weight.data, b.attn.k.weight.data, b.attn.v.weight.data = dequantize_grouped(
                a.attn.w_qkv, a.attn.s_qkv).split([a.attn.n_q, a.attn.n_k, a.attn.n_k])
            b.ffn.gate.weight.data = dequantize_grouped(a.ffn.wg, a.ffn.sg)
            b.ffn.up.weight.data = dequantize_grouped(a.ffn.wu, a.ffn.su)
        for a, b in [(m.lm_head, plain.lm_head)] + [(getattr(getattr(x, o), n), getattr(getattr(y, o), n)) for x, y in
                                                    zip(m.layers, plain.layers) for o, n in (("attn", "o"), ("ffn", "down"))]:
            assert isinstance(a, Int4Linear)
            b.weight.data = dequantize_grouped(a.qweight, a.scale)
    return m, plain


def _plain_cache(layers):
    from llms_b200.kernels import Int8KVCache

    class PlainCache(Int8KVCache):
        def __init__(self):
            self.layers, self._len = [], 0
            self.k, self.v = [None] * layers, [None] * layers

        @staticmethod
        def _held(x):
            B, KV, T, D = x.shape
            p = torch.nn.functional.pad(x.double(), (0, 0, 0, -T % 64)).view(B, KV, -1, 64, D)
            s = (p.abs().amax((-2, -1), keepdim=True) / 127).float().double()
            return (torch.round(p / s.clamp(min=1e-300)) * s).view(B, KV, -1, D)[:, :, :T]

        def attend(self, q, k, v, i, start):
            whole = []
            for store, new in ((self.k, k), (self.v, v)):
                store[i] = new if start == 0 else torch.cat((store[i][:, :, :start], new), 2)
                x = self._held(store[i])
                if q.shape[2] > 1:
                    x[:, :, start:] = new.double()
                whole.append(x.repeat_interleave(q.shape[1] // x.shape[1], 1))
            T, L = q.shape[2], start + q.shape[2]
            sc = q.double() @ whole[0].transpose(-1, -2) * q.shape[-1] ** -0.5
            seen = torch.arange(start, L, device=q.device)[:, None] >= torch.arange(L, device=q.device)
            return (torch.softmax(sc.masked_fill(~seen, -torch.inf), -1) @ whole[1]).to(q.dtype)

    return PlainCache()


def _close(a, b):
    rms = b.float().square().mean().sqrt().item()
    bf16_check(a.float().cpu().numpy(), b.float().cpu().numpy(), max_abs=6 * 2e-2 * rms, rel_l2=2e-2)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_projections(group):
    """Prompt and steps of the 4-bit model, and of the weights it stands for."""
    m, plain = _models(group)
    ids = torch.randint(0, 1000, (2, 70), device="cuda")
    with torch.inference_mode():
        c, p = m.alloc_cache(100, max_batch=3), plain.alloc_cache(100, max_batch=3)
        _close(m(ids[:, :60], c, start_pos=0), plain(ids[:, :60], p, start_pos=0))
        for t in range(60, 64):
            _close(m(ids[:, t:t + 1], c), plain(ids[:, t:t + 1], p))


def test_prompt_and_steps():
    """A prompt that ends inside a block, eager steps across its end."""
    m, _ = _models()
    ids = torch.randint(0, 1000, (2, 70), device="cuda")
    with torch.inference_mode():
        c, p = m.alloc_cache(100, max_batch=3, int8=True), _plain_cache(2)
        _close(m(ids[:, :60], c, start_pos=0), m(ids[:, :60], p, start_pos=0))
        for t in range(60, 70):
            _close(m(ids[:, t:t + 1], c), m(ids[:, t:t + 1], p, start_pos=t))
    assert c.cur_len == 70 and all(x.length == 70 for x in c.layers)


def test_chunks_and_captured_steps():
    """A prompt in chunks, then one captured graph replayed at every position,
    and back to an earlier one."""
    from llms_b200.qwen3 import GraphedDecodeStep
    m, _ = _models(group=64)
    ids = torch.randint(0, 1000, (3, 140), device="cuda")
    with torch.inference_mode():
        c, p = m.alloc_cache(140, max_batch=3, int8=True), _plain_cache(2)
        for a, b in ((0, 50), (50, 81), (81, 126)):
            _close(m(ids[:, a:b], c), m(ids[:, a:b], p, start_pos=a))
        step = GraphedDecodeStep(m, c, 3)
        for t in list(range(126, 140)) + list(range(130, 133)):
            _close(step(ids[:, t:t + 1], t), m(ids[:, t:t + 1], p, start_pos=t))
        # the same by the same calls without the graph
        c2 = m.alloc_cache(140, max_batch=3, int8=True)
        for a, b in ((0, 50), (50, 81), (81, 126)):
            m(ids[:, a:b], c2)
        for t in range(126, 133):
            eager = m(ids[:, t:t + 1], c2)
        got = step(ids[:, 132:133], 132)
        # (rewinding within the open block keeps its tokens as they came)
        assert torch.equal(got, eager)
        with pytest.raises(ValueError):
            step(ids[:, :1], 135)  # past the tokens that are there
        with pytest.raises(ValueError):
            step(ids[:, :1], 192)  # past the capacity


def test_score():
    """Log probabilities of the prompt's own tokens, and of greedy continuations."""
    from llms_b200.kernels import b200_token_logprobs
    m, plain = _models(group=32)
    ids = torch.randint(0, 1000, (2, 40), device="cuda")
    with torch.inference_mode():
        r = m.score(ids, m.alloc_cache(64, max_batch=2, int8=True), top=5, start_pos=0)
        logits = m(ids, m.alloc_cache(64, max_batch=2, int8=True), start_pos=0)
        lp = torch.log_softmax(logits.double(), -1)
        assert r.logprob.shape == (2, 39) and r.top_ids.shape == (2, 39, 5)
        assert (r.logprob - lp[:, :-1].gather(-1, ids[:, 1:, None])[..., 0]).abs().max() <= 4e-4
        assert (r.top_logprobs - lp[:, :-1].gather(-1, r.top_ids)).abs().max() <= 4e-4
        assert (r.entropy - (-(lp.exp() * lp).sum(-1))[:, :-1]).abs().max() <= 4e-4
        assert torch.equal(r.top_ids[..., 0], logits[:, :-1].float().argmax(-1))
        c = m.alloc_cache(64, max_batch=2, int8=True)
        out = m(ids[:, :5], c, start_pos=0)[:, -1:]
        for _ in range(4):
            nxt = out.argmax(-1)
            s = b200_token_logprobs(out, nxt, top=3)
            assert (s.logprob >= s.top_logprobs[..., 0] - 1e-6).all()
            out = m(nxt, c)


@pytest.mark.parametrize("swap", ["none", "int8", "dense"])
def test_other_models_on_the_8_bit_cache(swap):
    """The eager model, int8 and 16-bit fused projections with the 8-bit cache."""
    from llms_b200.kernels import apply_int8_kernels, apply_triton_kernels
    from llms_b200.qwen3 import Qwen3Model
    _, plain = _models()
    m = Qwen3Model(plain.shape).cuda().eval()
    m.load_state_dict(plain.state_dict())
    m.to(BF)
    if swap == "int8":
        apply_int8_kernels(m)
    elif swap == "dense":
        apply_triton_kernels(m)
    ids = torch.randint(0, 1000, (1, 70), device="cuda")
    with torch.inference_mode():
        c, p = m.alloc_cache(128, int8=True), _plain_cache(2)
        _close(m(ids[:, :62], c, start_pos=0), m(ids[:, :62], p, start_pos=0))
        for t in range(62, 67):
            _close(m(ids[:, t:t + 1], c), m(ids[:, t:t + 1], p, start_pos=t))


def test_prewarm_takes_4_bit_modules():
    from llms_b200.kernels import prewarm_triton_kernels
    m, _ = _models()
    prewarm_triton_kernels(m, m_values=(1, 3))


def test_a_step_captured_at_a_border_and_replayed_before_it():
    """Building the step runs it once, which opens the block at the border;
    going back into the one before takes that one's tokens up again."""
    from llms_b200.qwen3 import GraphedDecodeStep
    m, _ = _models()
    ids = torch.randint(0, 1000, (2, 80), device="cuda")
    with torch.inference_mode():
        c, c2 = (m.alloc_cache(128, max_batch=2, int8=True) for _ in range(2))
        m(ids[:, :64], c), m(ids[:, :64], c2)  # (the same calls: a product's sums may differ with its rows)
        m(ids[:, 64:65], c2)
        step = GraphedDecodeStep(m, c, 2)
        c2.seek(60)
        for t in range(60, 70):
            assert torch.equal(step(ids[:, t:t + 1], t), m(ids[:, t:t + 1], c2))
        for a, b in zip(c.layers, c2.layers):
            assert torch.equal(a.kq[:, :, :70], b.kq[:, :, :70]) and torch.equal(a.vs, b.vs)


@pytest.mark.parametrize("o,down", [(True, True), (False, True), (True, False)])
def test_prewarm_takes_8_bit_modules_with_4_bit_outputs(o, down):
    from llms_b200.kernels import apply_int4_kernels, apply_int8_kernels, prewarm_triton_kernels
    from llms_b200.qwen3 import QWEN3_4B, Qwen3Model
    m = Qwen3Model(dataclasses.replace(QWEN3_4B, num_hidden_layers=1, vocab_size=1000)).to("cuda", BF)
    apply_int4_kernels(apply_int8_kernels(m), o=o, down=down)
    prewarm_triton_kernels(m, m_values=(1, 3))
