"""Log probabilities, entropy and top alternatives vs their definition in 64 bits.

Ids are compared exactly.  Numbers, with d = x - m <= 0: a term e^d is within
|d| 2^-23 + 2^-22 of itself (two roundings of the argument, the exponential),
which, weighted by the terms, is at most 2e-6 for entropies below 12.  l is summed
over at most 300 terms by one thread and 20 joins, each addition within 2^-24:
1.8e-5 in the worst case, all erring alike.  So log l is off by at most 2e-5,
e / l by 2e-5 of itself, and |e / l| <= entropy.  The last subtractions add 2^-23
of the value.  The bound: 2e-5 (1 + |value|)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import llms_b200.kernels  # noqa: F401


def _check(x, tokens, top):
    from llms_b200.kernels import b200_token_logprobs
    r = b200_token_logprobs(x, tokens, top=top)
    d = x.double()
    V = x.shape[-1]
    c = d - d.amax(-1, keepdim=True)  # (first: beside the type's lowest value the logarithm would be lost)
    lp = c - torch.log(torch.exp(c).sum(-1, keepdim=True))
    ok = (tokens >= 0) & (tokens < V)
    want = torch.where(ok, lp.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0], math.nan)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    dead = ~torch.isfinite(d.amax(-1)) | d.isnan().any(-1)
    want, ent = torch.where(dead, math.nan, want), torch.where(dead, math.nan, ent)

    def close(got, exp, what):
        exp = exp.to(got.device)
        assert torch.equal(got.isnan(), exp.isnan()), what
        inf = exp.isinf()
        assert torch.equal(got[inf].double(), exp[inf]), what
        ok = exp.isfinite()
        off = (got.double() - exp).abs()[ok] - (2e-5 * (1 + exp.abs()[ok]))
        assert off.numel() == 0 or off.max() <= 0, (what, off.max())

    close(r.logprob, want, "logprob")
    close(r.entropy, ent, "entropy")
    assert r.logprob.dtype == r.entropy.dtype == r.top_logprobs.dtype == FL and r.top_ids.dtype == torch.int64
    assert r.top_ids.shape == r.top_logprobs.shape == (*x.shape[:-1], top)
    # NaN first, then descending, equal ones by index
    f = torch.where(x.isnan(), math.inf, x.float() + 0.0)
    rank = torch.sort(f, dim=-1, descending=True, stable=True).indices
    nan_first = torch.sort(x.gather(-1, rank).isnan().int(), dim=-1, descending=True, stable=True).indices
    ids = rank.gather(-1, nan_first)[..., :top]
    assert torch.equal(r.top_ids, ids)
    close(r.top_logprobs, torch.where(dead[..., None], math.nan, lp.gather(-1, ids)), "top")
    return r


def _logits(M, V, dtype, seed=0, std=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, V, device="cuda", generator=g) * std
    x.scatter_add_(1, torch.randint(0, V, (M, 4), device="cuda", generator=g), torch.full((M, 4), 9.0, device="cuda"))
    return x.to(dtype), torch.randint(0, V, (M,), device="cuda", generator=g)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 64, 1000, 4097, 32000, 151936, 151937])
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_vocabularies(dtype, V):
    x, t = _logits(3, V, dtype, seed=V)
    for top in {0, 1, min(V, 5), min(V, 64)}:
        _check(x, t, top)


@pytest.mark.parametrize("M", [1, 2, 17, 64, 149, 700])
@pytest.mark.parametrize("top", [0, 20])
def test_rows(M, top):
    _check(*_logits(M, 50001, BF, seed=M), top)


def test_misaligned_rows_and_strides():
    x, t = _logits(6, 9001, BF, seed=1)
    big = torch.randn(6, 9100, device="cuda").to(BF)
    for off in range(9):
        v = big[:, off:off + 9001]
        v.copy_(x)
        _check(v, t, 9)
    _check(x.view(2, 3, 9001), t.view(2, 3), 4)
    _check(x.t().contiguous().t(), t, 4)
    _check(x[:1].expand(6, 9001), t, 4)


@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_masked_rows(dtype):
    """-inf, the type's lowest value, rows with one or no token left, fewer
    than asked for."""
    V = 20000
    x, t = _logits(12, V, dtype, seed=3)
    low = torch.finfo(dtype).min
    keep = torch.rand(V, device="cuda") < 0.1
    x[0][~keep] = -math.inf
    x[1][~keep] = low
    x[2] = -math.inf
    x[3] = low
    x[4] = -math.inf
    x[4, 12345] = 3.0
    x[5] = low
    x[5, 777] = 3.0
    x[6, 200:] = -math.inf
    x[7] = -math.inf
    x[7, ::1000] = 1.0
    x[8] = 0.0
    x[9] = torch.finfo(dtype).max
    x[10] = -0.0
    x[10, 5000:] = 0.0
    x[11, :] = torch.arange(V, device="cuda").to(dtype)
    t[4], t[0] = 12345, int(torch.nonzero(~keep)[0])
    for rows in (slice(0, 12), slice(2, 3), slice(4, 5), slice(8, 9)):  # several, and one row shared by a cluster
        for top in (1, 20, 64):
            _check(x[rows], t[rows], top)


def test_crowds_above_the_bound():
    """Thousands of large logits that a few threads hold: runs, strides of the
    kernel's own order, everything equal but a few."""
    V = 151936
    x, t = _logits(5, V, BF, seed=4)
    x[0, :40000] += 50
    x[1, -3000:] = 30
    n = V // 4096
    for i in range(n):
        x[2, 4096 * i:4096 * i + 32] = 40 + (torch.arange(32, device="cuda") % 7).to(BF)
        x[3, 4096 * i + 64:4096 * i + 160] = 40
    x[4] = 1.0
    x[4, 100000:100003] = 2.0
    for top in (1, 5, 33, 64):
        _check(x, t, top)
        for r in range(5):
            _check(x[r:r + 1], t[r:r + 1], top)


def test_nan_and_infinity():
    x, t = _logits(6, 5000, FL, seed=5)
    x[0, 17] = math.nan
    x[1, 18] = math.inf
    x[2, :] = math.nan
    x[3, 4999] = math.nan
    x[3, 0] = math.inf
    x[4, 3::2] = math.nan
    for top in (0, 1, 6):
        _check(x, t, top)


def test_tokens_outside_the_vocabulary():
    x, t = _logits(5, 1000, BF)
    t[1], t[2], t[3], t[4] = -1, 1000, -100, 999
    _check(x, t, 3)


def test_peaked_rows_keep_small_numbers():
    """One token that takes all but 1e-3 or 1e-6: its log probability and the
    entropy are small, and still right to 2^-22 absolute plus 1e-4 of themselves."""
    from llms_b200.kernels import b200_token_logprobs
    x = torch.zeros(2, 1001, device="cuda")
    x[0, 5], x[1, 6] = math.log(1e6), math.log(1e9)
    d = x.double()
    lp = torch.log_softmax(d, -1)
    r = b200_token_logprobs(x, torch.tensor([5, 6], device="cuda"), top=2)
    for got, want in ((r.logprob, lp[[0, 1], [5, 6]]), (r.entropy, -(lp.exp() * lp).sum(-1))):
        assert ((got.double() - want).abs() <= 2.0 ** -22 + 1e-4 * want.abs()).all()


def test_graph_streams_and_empty_calls():
    from llms_b200.kernels import b200_token_logprobs
    x, t = _logits(4, 30000, BF)
    want = b200_token_logprobs(x, t, top=7)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = b200_token_logprobs(x, t, top=7)
    y, u = _logits(4, 30000, BF, seed=9)
    x.copy_(y), t.copy_(u)
    g.replay()
    for a, b in zip(out, b200_token_logprobs(y, u, top=7)):
        assert torch.equal(a, b)
    assert not torch.equal(want.logprob, out.logprob)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        r = b200_token_logprobs(y, u, top=7)
    s.synchronize()
    assert torch.equal(r.top_ids, out.top_ids)
    e = b200_token_logprobs(x[:0], t[:0], top=3)
    assert e.top_ids.shape == (0, 3) and e.logprob.shape == (0,)


def test_offsets_past_32_bits():
    M, V = 15000, 151936  # 4.6 GB of bf16
    x = torch.zeros(M, V, dtype=BF, device="cuda")
    y, t = _logits(2, V, BF, seed=6)
    x[-2:] = y
    from llms_b200.kernels import b200_token_logprobs
    toks = torch.zeros(M, dtype=torch.int64, device="cuda")
    toks[-2:] = t
    r = b200_token_logprobs(x, toks, top=4)
    w = _check(y, t, 4)
    assert torch.equal(r.top_ids[-2:], w.top_ids)
    assert (r.logprob[-2:] - w.logprob).abs().max() <= 4e-5 and (r.logprob[:-2] + math.log(V)).abs().max() <= 4e-5
