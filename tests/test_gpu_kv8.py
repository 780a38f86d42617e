"""The 8-bit KV cache and its decode attention vs their formulas in 64 bits.

Stored bits are compared exactly.  Attention: an element may be off by
half a step of its own rounding, eps(dtype) / 2 |out|, plus 2^-11 sum_t p_t |v_t|:
the probabilities are rounded to 11 bits (2^-12 each), and the scores' fp32
sums and the exponentials stay well inside the other 2^-12 at these sizes
(scores of magnitude <= 64, each within 128 * 2^-24 of itself).  An fp16 number
below 2^-14 is rounded to a multiple of 2^-24 instead, by at most 2^-25; the
probabilities are held times 2^14 relative to their block's largest, which is
at most 1, and the sum they are divided by is at least 1 in that unit, so each
may also be off by 2^-39: 2^-39 sum_t |v_t|."""

import pytest
import torch

from tests.gpu_util import force_generic

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
PARTS = ("kq", "ks", "kt", "vq", "vs", "vt")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import llms_b200.kernels  # noqa: F401


def _alloc(rows, KV, S, D, dtype=BF):
    from llms_b200.kernels import Int8KV
    return Int8KV.alloc(rows=rows, num_kv_heads=KV, max_seq_len=S, head_dim=D, dtype=dtype, device="cuda")


def _tokens(B, KV, T, D, dtype=BF, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, KV, T, D, device="cuda", generator=g).to(dtype) for _ in range(2)]


def _store(x):
    """(B, KV, T, D) -> 8-bit values and scales by the formula, in 64 bits."""
    B, KV, T, D = x.shape
    n = -(-T // 64)
    p = torch.zeros(B, KV, n * 64, D, dtype=torch.float64, device=x.device)
    p[:, :, :T] = x.double()
    p = p.view(B, KV, n, 64, D)
    s = (p.abs().amax((-2, -1)) / 127).float()
    d = s.double()[..., None, None]
    q = torch.where(d > 0, torch.round(p / torch.where(d > 0, d, 1.0)), 0.0)
    return q.view(B, KV, n * 64, D)[:, :, :T].to(torch.int8), s


def _check_store(kv, k, v):
    T, n = k.shape[2], -(-k.shape[2] // 64)
    B = k.shape[0]
    for q, s, x in ((kv.kq, kv.ks, k), (kv.vq, kv.vs, v)):
        eq, es = _store(x)
        assert torch.equal(s[:B, :, :n], es)
        assert torch.equal(q[:B, :, :T], eq)


@pytest.mark.parametrize("T", [1, 5, 63, 64, 65, 200])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (FL, 128), (BF, 16), (HF, 48), (FL, 256), (BF, 256)])
def test_append_stores_the_formula(dtype, D, T):
    from llms_b200.kernels import int8_kv_append, int8_kv_expand
    kv = _alloc(2, 3, 256, D, dtype)
    k, v = _tokens(2, 3, T, D, dtype, seed=T)
    int8_kv_append(kv, k, v, 0)
    _check_store(kv, k, v)
    r = (T - 1) % 64 + 1
    assert torch.equal(kv.kt[:, :, :r], k[:, :, T - r:]) and torch.equal(kv.vt[:, :, :r], v[:, :, T - r:])
    assert not kv.kq[:, :, T:].any() and not kv.ks[:, :, -(-T // 64):].any()
    ek, ev = int8_kv_expand(kv, T)
    for e, q, s in ((ek, kv.kq, kv.ks), (ev, kv.vq, kv.vs)):
        assert torch.equal(e, (q[:, :, :T].float() * s.repeat_interleave(64, 2)[:, :, :T, None]).to(dtype))


@pytest.mark.parametrize("dtype", [BF, FL])
def test_append_at_the_borders_of_the_rounding(dtype):
    """Tokens on and next to halves of the scale, scales that are powers of
    two (true ties), tiny and subnormal ones, a zero block."""
    from llms_b200.kernels import int8_kv_append
    kv = _alloc(1, 1, 1024, 64, dtype)
    k = torch.zeros(1, 1, 1024, 64, dtype=torch.float64, device="cuda")
    j = torch.arange(64 * 64, device="cuda", dtype=torch.float64).view(64, 64)
    for i, (s, off) in enumerate([(1.0, 0.0), (0.25, 0.0), (0.37, 0.0), (0.37, 1e-7), (0.37, -1e-7), (2.0 ** -130, 0.0),
                                  (2.0 ** -60, 0.0), (1e37, 0.0), (1e-36, 0.0), (0.0, 0.0), (0.013, 0.0), (5.5, 0.0)]):
        blk = ((j.remainder(255) - 127) * 0.5 + off) * s
        blk[0, 0] = 127 * s
        k[0, 0, 64 * i:64 * i + 64] = blk
    k = k.to(dtype)
    int8_kv_append(kv, k, -k, 0)
    _check_store(kv, k, -k)
    assert kv.kq.abs().max() == 127


def test_infinities_and_nan_mark_their_block():
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn, int8_kv_expand
    kv = _alloc(1, 3, 256, 64)
    k, v = _tokens(1, 3, 200, 64)
    k[0, 0, 70, 3] = float("inf")
    v[0, 1, 130, 5] = float("nan")
    int8_kv_append(kv, k, v, 0)
    ek, ev = int8_kv_expand(kv, 200)
    assert ek[0, 0, 64:128].isnan().all() and ev[0, 1, 128:192].isnan().all()
    ek[0, 0, 64:128], ev[0, 1, 128:192] = 0, 0
    assert ek.isfinite().all() and ev.isfinite().all()
    q = torch.randn(1, 6, 1, 64, device="cuda").to(BF)
    out = int8_kv_decode_attn(q, kv, 199, scale=0.125)
    assert out[0, :4].isnan().all() and out[0, 4:].isfinite().all()
    assert int8_kv_decode_attn(q, kv, 63, scale=0.125).isfinite().all()


@pytest.mark.parametrize("cuts", [[1] * 130, [64, 64, 2], [1, 62, 1, 1, 65], [40, 90], [100, 28, 1, 1], [63, 1, 66]])
@pytest.mark.parametrize("dtype", [BF, FL])
def test_any_cut_of_a_prompt_stores_the_same(cuts, dtype):
    from llms_b200.kernels import int8_kv_append
    T = sum(cuts)
    k, v = _tokens(2, 2, T, 128, dtype, seed=3)
    k[:, :, 70:] *= 3  # the second block's scale grows inside it
    whole, parts = _alloc(2, 2, 192, 128, dtype), _alloc(2, 2, 192, 128, dtype)
    int8_kv_append(whole, k, v, 0)
    t = 0
    for n in cuts:
        int8_kv_append(parts, k[:, :, t:t + n], v[:, :, t:t + n], t)
        t += n
    for p in ("kq", "ks", "vq", "vs"):
        assert torch.equal(getattr(whole, p), getattr(parts, p))
    r = (T - 1) % 64 + 1
    assert torch.equal(whole.kt[:, :, :r], parts.kt[:, :, :r]) and torch.equal(whole.vt[:, :, :r], parts.vt[:, :, :r])


def test_tokens_of_the_last_block_can_be_written_again():
    """Another token in its place first (a larger one, which moves the scale),
    and a few positions back."""
    from llms_b200.kernels import int8_kv_append
    k, v = _tokens(1, 2, 100, 64, seed=5)
    kv, want = _alloc(1, 2, 128, 64), _alloc(1, 2, 128, 64)
    int8_kv_append(want, k, v, 0)
    int8_kv_append(kv, k[:, :, :99], v[:, :, :99], 0)
    int8_kv_append(kv, 100 * k[:, :, 99:], v[:, :, 99:], 99)
    int8_kv_append(kv, -k[:, :, 80:], 50 * v[:, :, 80:], 80)
    int8_kv_append(kv, k[:, :, 80:90], v[:, :, 80:90], 80)
    int8_kv_append(kv, k[:, :, 90:], v[:, :, 90:], 90)
    for p in PARTS:
        rows = 36 if p[1] == "t" else 100
        a, b = getattr(kv, p), getattr(want, p)
        assert torch.equal(a[:, :, :rows], b[:, :, :rows])


def test_ragged_positions_and_rows_that_are_not_there():
    from llms_b200.kernels import int8_kv_append
    pos = [0, 63, 64, 100, -1, 127, 128, -5]
    B, S = len(pos), 128
    kv = _alloc(B + 1, 2, S, 64)
    for p in PARTS:  # what is not written stays
        getattr(kv, p).copy_(torch.randint(1, 9, getattr(kv, p).shape, device="cuda"))
    k, v = _tokens(B, 2, 130, 64, seed=2)
    for b, p in enumerate(pos):
        if 0 < p < S:
            from llms_b200.kernels import Int8KV
            row = Int8KV(*(getattr(kv, n)[b:b + 1] for n in PARTS))
            int8_kv_append(row, k[b:b + 1, :, :p], v[b:b + 1, :, :p], 0)
    before = {p: getattr(kv, p).clone() for p in PARTS}
    nk, nv = _tokens(B, 2, 3, 64, seed=9)
    int8_kv_append(kv, nk, nv, torch.tensor(pos, device="cuda"))
    for b, p in enumerate(pos):
        if not 0 <= p < S:
            for n in PARTS:
                assert torch.equal(getattr(kv, n)[b], before[n][b])
            continue
        n = min(3, S - p)
        tk = torch.cat((k[b, :, :p], nk[b, :, :n]), 1)[None]
        eq, es = _store(tk)
        assert torch.equal(kv.kq[b, :, :p + n], eq[0]) and torch.equal(kv.ks[b, :, :es.shape[2]], es[0])
        assert torch.equal(kv.kq[b, :, p + n:], before["kq"][b, :, p + n:])
    for n in PARTS:
        assert torch.equal(getattr(kv, n)[B], before[n][B])


def _attend(q, kv, lens, scale):
    """The formula in 64 bits over the stored values: (out, sum p |v|, sum |v|)."""
    B, H, _, D = q.shape
    KV = kv.num_kv_heads
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    mass, every = torch.zeros_like(out), torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        j = -(-n // 64)
        for h in range(KV):
            k, v = (x[b, h, :n].double() * s[b, h, :j].double().repeat_interleave(64)[:n, None]
                    for x, s in ((kv.kq, kv.ks), (kv.vq, kv.vs)))
            hs = slice(h * H // KV, (h + 1) * H // KV)
            p = torch.softmax(q[b, hs, 0].double() @ k.T * scale, -1)
            out[b, hs], mass[b, hs], every[b, hs] = p @ v, p @ v.abs(), v.abs().sum(0)
    return out, mass, every


def _check_attn(got, q, kv, lens, scale):
    want, mass, every = _attend(q, kv, lens, scale)
    p, small = (1e-5, 0.0) if q.dtype == FL else (2.0 ** -11, 2.0 ** -39)
    tol = p * mass + small * every + torch.finfo(q.dtype).eps / 2 * want.abs()
    d = (got[:, :, 0].double() - want).abs()
    assert (d <= tol).all(), f"off by {(d - tol).max().item():.3e} beyond the bound at {(d - tol).argmax().item()}"


def _filled(B, KV, S, D, dtype=BF, seed=0):
    from llms_b200.kernels import int8_kv_append
    kv = _alloc(B, KV, S, D, dtype)
    k, v = _tokens(B, KV, S, D, dtype, seed=seed)
    int8_kv_append(kv, k, v, 0)
    return kv


@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 63, 64, 65, 129, 1000, 5003])
@pytest.mark.parametrize("B", [1, 3])
def test_lengths(B, L):
    from llms_b200.kernels import int8_kv_decode_attn
    kv = _filled(B, 8, L, 128, seed=L)
    q = torch.randn(B, 32, 1, 128, device="cuda").to(BF)
    _check_attn(int8_kv_decode_attn(q, kv, L - 1, scale=128 ** -0.5), q, kv, [L] * B, 128 ** -0.5)


@pytest.mark.parametrize("H,KV,D", [(8, 8, 128), (16, 1, 128), (32, 8, 64), (12, 4, 64), (20, 4, 128), (9, 1, 64), (7, 1, 128),
                                    (17, 1, 128), (4, 2, 32), (6, 2, 256), (3, 1, 16), (40, 2, 64)])
@pytest.mark.parametrize("dtype", [BF, HF, FL])
def test_groups_dims_and_types(H, KV, D, dtype):
    from llms_b200.kernels import int8_kv_decode_attn
    kv = _filled(2, KV, 300, D, dtype, seed=H + D)
    q = torch.randn(2, H, 1, D, device="cuda").to(dtype)
    pos = torch.tensor([299, 70], device="cuda")
    got = int8_kv_decode_attn(q, kv, pos, scale=D ** -0.5)
    _check_attn(got, q, kv, [300, 71], D ** -0.5)
    if dtype != FL:
        with force_generic():
            _check_attn(int8_kv_decode_attn(q, kv, pos, scale=D ** -0.5), q, kv, [300, 71], D ** -0.5)


@pytest.mark.parametrize("lens", [[0, 5, 0, 700, 64, 1, 0], [0, 0], [4096] * 3 + [1] * 40, [63, 64, 65, 3000, 0, 128] * 9])
def test_ragged_rows(lens):
    """Rows that are not there give zeros; lengths past the capacity stop at
    it; scales and values of blocks that hold no token (NaN here) do not count."""
    from llms_b200.kernels import int8_kv_decode_attn
    kv = _filled(len(lens), 2, max(max(lens), 64), 128, seed=1)
    for b, n in enumerate(lens):
        for s in (kv.ks, kv.vs):
            s[b, :, -(-n // 64):] = float("nan")
        kv.kq[b, :, n:], kv.vq[b, :, n:] = -128, 127
    q = torch.randn(len(lens), 8, 1, 128, device="cuda").to(BF)
    pos = torch.tensor([n - 1 if n != 4096 else 10 ** 9 for n in lens], device="cuda")
    got = int8_kv_decode_attn(q, kv, pos, scale=0.09)
    _check_attn(got, q, kv, lens, 0.09)
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()


def test_more_rows_than_one_launch_takes():
    from llms_b200.kernels import int8_kv_decode_attn
    B = 1030
    kv = _filled(B, 1, 64, 64, seed=4)
    lens = [(7 * b) % 65 for b in range(B)]
    q = torch.randn(B, 2, 1, 64, device="cuda").to(HF).to(BF)
    got = int8_kv_decode_attn(q, kv, torch.tensor(lens, device="cuda") - 1, scale=0.125)
    _check_attn(got, q, kv, lens, 0.125)


@pytest.mark.parametrize("spread", ["q large", "q small", "keys", "values", "one hot", "zero keys", "zero values", "zero q"])
def test_scales_far_apart(spread):
    """Queries near the ends of bf16's range, blocks whose scales differ by
    2^40, one token that takes all, zero blocks (the last one of them cut)."""
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn
    B, KV, L, D = 1, 2, 400, 128
    k, v = _tokens(B, KV, L, D, seed=6)
    q = torch.randn(B, 8, 1, D, device="cuda")
    scale = D ** -0.5
    if spread == "q large":
        q, scale = q * 2.0 ** 100, scale * 2.0 ** -100
    elif spread == "q small":
        q, scale = q * 2.0 ** -100, scale * 2.0 ** 100
    elif spread == "keys":
        k[:, :, 64:128] *= 2.0 ** -40
    elif spread == "values":
        v[:, :, 64:128] *= 2.0 ** 20
        v[:, :, 128:192] *= 2.0 ** -20
    elif spread == "zero keys":
        k[:, :, 64:128], k[:, :, 384:] = 0, 0
    elif spread == "zero values":
        v[:, :, 64:128], v[:, :, 384:] = 0, 0
    elif spread == "zero q":
        q[:, 1::2] = 0
    else:
        k[:, :, 200] = q[:, ::4, 0].to(BF) * 4
    q = q.to(BF)
    kv = _alloc(B, KV, L, D)
    int8_kv_append(kv, k, v, 0)
    _check_attn(int8_kv_decode_attn(q, kv, L - 1, scale=scale), q, kv, [L], scale)


def test_step_is_append_and_attention():
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn, int8_kv_step
    a, b = _filled(3, 2, 256, 128, seed=8), _filled(3, 2, 256, 128, seed=8)
    pos = torch.tensor([255, -1, 192], device="cuda")
    k, v = _tokens(3, 2, 1, 128, seed=11)
    q = torch.randn(3, 8, 1, 128, device="cuda").to(BF)
    got = int8_kv_step(q, k, v, a, pos, scale=0.1)
    int8_kv_append(b, k, v, pos)
    assert torch.equal(got, int8_kv_decode_attn(q, b, pos, scale=0.1))
    for p in PARTS:
        assert torch.equal(getattr(a, p), getattr(b, p))
    _check_attn(got, q, a, [256, 0, 193], 0.1)


def test_strides_views_and_other_orders():
    """Projections' layout (tokens before heads), unaligned views, head
    slices and rows of a larger cache, heads before rows."""
    from llms_b200.kernels import Int8KV, int8_kv_append, int8_kv_decode_attn
    big = _filled(4, 4, 192, 64, seed=3)
    part = Int8KV(*(getattr(big, n)[1:3, 1:3] for n in PARTS))
    x = torch.randn(2, 130, 3 * 2 * 64 + 3, device="cuda").to(BF)[:, :, 3:]
    k, v = (x[:, :, i * 128:i * 128 + 128].view(2, 130, 2, 64).transpose(1, 2) for i in (0, 1))
    before = big.kq.clone()
    int8_kv_append(part, k, v, 0)
    _check_store(part, k, v)
    rest = torch.ones(4, 4, dtype=torch.bool, device="cuda")
    rest[1:3, 1:3] = False
    assert torch.equal(big.kq[rest], before[rest])
    q = torch.randn(2, 1, 5, 65, device="cuda").to(BF)[:, :, :4, 1:].transpose(1, 2)
    _check_attn(int8_kv_decode_attn(q, part, 129, scale=0.125), q, part, [130] * 2, 0.125)
    turned = Int8KV(*(getattr(big, n).transpose(0, 1).contiguous().transpose(0, 1) for n in PARTS))
    q = torch.randn(4, 8, 1, 64, device="cuda").to(BF)
    assert torch.equal(int8_kv_decode_attn(q, turned, 100, scale=0.125), int8_kv_decode_attn(q, big, 100, scale=0.125))


def test_offsets_past_32_bits():
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn
    kv = _alloc(3, 8, 1 << 20, 128)  # 3.2 GB of keys
    k, v = _tokens(3, 8, 150, 128, seed=7)
    p0 = (1 << 20) - 192
    lens = [0, 0, 150]
    int8_kv_append(kv, k, v, torch.tensor([p0, -1, 0], device="cuda"))
    eq, es = _store(k)
    assert torch.equal(kv.kq[2, :, :150], eq[2]) and torch.equal(kv.ks[0, :, p0 // 64:p0 // 64 + 3], es[0])
    assert torch.equal(kv.kq[0, :, p0:p0 + 150], eq[0])
    q = torch.randn(3, 32, 1, 128, device="cuda").to(BF)
    got = int8_kv_decode_attn(q, kv, torch.tensor([-1, -1, 149], device="cuda"), scale=0.088)
    _check_attn(got, q, kv, lens, 0.088)
    # a whole long row: zeros but for its end (scores there against a crowd of zero scores)
    got = int8_kv_decode_attn(q, kv, torch.tensor([p0 + 149, -1, -1], device="cuda"), scale=0.088)
    want, mass = torch.zeros(32, 128, device="cuda").double(), torch.zeros(32, 128, device="cuda").double()
    for h in range(8):
        kk, vv = (x[0, h, p0:p0 + 150].double() * s[0, h, p0 // 64:p0 // 64 + 3].double().repeat_interleave(64)[:150, None]
                  for x, s in ((kv.kq, kv.ks), (kv.vq, kv.vs)))
        e = torch.exp(q[0, 4 * h:4 * h + 4, 0].double() @ kk.T * 0.088)
        z = e.sum(-1, keepdim=True) + p0
        want[4 * h:4 * h + 4], mass[4 * h:4 * h + 4] = e @ vv / z, e @ vv.abs() / z
    d = (got[0, :, 0].double() - want).abs()
    assert (d <= 2.0 ** -11 * mass + 2.0 ** -8 * want.abs()).all()


def test_graph_replayed_at_every_position():
    """One captured step, positions on the device; two graphs of the same
    shape replayed at once on two streams keep their own workspaces."""
    from llms_b200.kernels import int8_kv_step
    S = 130
    made = []
    for seed in (1, 2):
        kv = _alloc(2, 2, S, 128)
        q, k, v = (torch.zeros(2, h, 1, 128, dtype=BF, device="cuda") for h in (8, 2, 2))
        pos = torch.zeros(2, dtype=torch.int64, device="cuda")
        int8_kv_step(q, k, v, kv, pos, scale=0.1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = int8_kv_step(q, k, v, kv, pos, scale=0.1)
        ks, vs = _tokens(2, 2, S, 128, seed=seed)
        qs = torch.randn(S, 2, 8, 1, 128, device="cuda").to(BF)
        made.append((kv, q, k, v, pos, g, out, ks, vs, qs, torch.cuda.Stream(), []))
    for t in range(S):
        for kv, q, k, v, pos, g, out, ks, vs, qs, st, got in made:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                q.copy_(qs[t])
                k.copy_(ks[:, :, t:t + 1])
                v.copy_(vs[:, :, t:t + 1])
                pos.copy_(torch.tensor([t, t - 40], device="cuda"))
                if t < 40:
                    pos[1] = -1
                else:  # the second row runs 40 behind
                    k[1], v[1] = ks[1, :, t - 40:t - 39], vs[1, :, t - 40:t - 39]
                g.replay()
                got.append(out.clone())
    torch.cuda.synchronize()
    for kv, q, k, v, pos, g, out, ks, vs, qs, st, got in made:
        _check_store(kv, ks[:1], vs[:1])
        for t in (0, 1, 39, 40, 41, 63, 64, 65, 129):
            # the first row's scales at time t are those of its tokens so far
            now = _alloc(2, 2, S, 128)
            from llms_b200.kernels import int8_kv_append
            int8_kv_append(now, ks[:, :, :t + 1], vs[:, :, :t + 1], 0)
            if t >= 40:
                int8_kv_append(now, ks[:, :, :t - 39], vs[:, :, :t - 39], torch.tensor([-1, 0], device="cuda"))
            _check_attn(got[t], qs[t], now, [t + 1, max(0, t - 39)], 0.1)


def test_other_streams_and_repeated_calls():
    from llms_b200.kernels import int8_kv_decode_attn
    kv = _filled(4, 8, 2000, 128, seed=2)
    q = torch.randn(4, 32, 1, 128, device="cuda").to(BF)
    want = int8_kv_decode_attn(q, kv, 1999, scale=0.1)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(int8_kv_decode_attn(q, kv, 1999, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_gpu_refusals():
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn, int8_kv_step
    kv = _alloc(2, 2, 128, 64)
    q, k = torch.zeros(2, 4, 1, 64, dtype=BF, device="cuda"), torch.zeros(2, 2, 1, 64, dtype=BF, device="cuda")
    for pos in (128, -2, torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"),
                torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError):
            int8_kv_append(kv, k, k, pos)
        with pytest.raises(ValueError):
            int8_kv_decode_attn(q, kv, pos, scale=0.1)
        with pytest.raises(ValueError):
            int8_kv_step(q, k, k, kv, pos, scale=0.1)
    with pytest.raises(ValueError):
        int8_kv_append(kv, k.expand(2, 2, 3, 64), k.expand(2, 2, 3, 64), 126)
    with pytest.raises(ValueError):
        int8_kv_step(q, k[:1], k[:1], kv, 0, scale=0.1)
    with pytest.raises(RuntimeError):
        int8_kv_decode_attn(q, kv, 0, scale=-1.0)


def test_empty_calls():
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn, int8_kv_expand
    kv = _alloc(2, 2, 128, 64)
    e = torch.zeros(0, 2, 1, 64, dtype=BF, device="cuda")
    int8_kv_append(kv, e, e, 0)
    t = torch.zeros(2, 2, 0, 64, dtype=BF, device="cuda")
    int8_kv_append(kv, t, t, 0)
    assert int8_kv_decode_attn(torch.zeros(0, 4, 1, 64, dtype=BF, device="cuda"), kv, 0, scale=0.1).shape == (0, 4, 1, 64)
    k, v = int8_kv_expand(kv, 0)
    assert k.shape == (2, 2, 0, 64) == v.shape


@pytest.mark.parametrize("B,L", [(1, 64), (1, 5000), (5, 640), (40, 1217)])
def test_a_step_right_behind_what_it_reads(B, L):
    """The step's attention starts before its append is done, but not before the
    prompt's append (or the copies of q, k, v) right ahead of it: eager, and
    in a graph whose inputs change between replays."""
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn, int8_kv_step
    S = L + 1
    a, b = _alloc(B, 8, S, 128), _alloc(B, 8, S, 128)
    pos = torch.full((B,), L, dtype=torch.int64, device="cuda")
    pos[B // 2] = L - 1 if B > 1 else L  # (written anew)
    data = []
    for i in range(6):
        k, v = _tokens(B, 8, S, 128, seed=40 + i)
        q = torch.randn(B, 32, 1, 128, device="cuda").to(BF)
        int8_kv_append(b, k[:, :, :L], v[:, :, :L], 0)
        torch.cuda.synchronize()
        int8_kv_append(b, k[:, :, L:], v[:, :, L:], pos)
        torch.cuda.synchronize()
        data.append((q, k, v, int8_kv_decode_attn(q, b, pos, scale=0.09)))
    q, k, v = (torch.zeros_like(x) for x in data[0][:3])

    def run():
        int8_kv_append(a, k[:, :, :L], v[:, :, :L], 0)
        return int8_kv_step(q, k[:, :, L:], v[:, :, L:], a, pos, scale=0.09)

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for graph in (False, True):
        for dq, dk, dv, want in data * 3:
            q.copy_(dq), k.copy_(dk), v.copy_(dv)
            if graph:
                g.replay()
                got = out
            else:
                got = run()
            assert torch.equal(got, want)


def _against(p, part):
    """Signs (T,) that add up what rounding each of p (times 2^14, relative to the largest of its part) to fp16
    leaves, and sum to zero with p as weights: the tokens that leave least are spent on that."""
    u = torch.nn.functional.pad(p, (0, -len(p) % part)).view(-1, part)
    m = u.amax(-1, keepdim=True)
    left = ((u / m * 2.0 ** 14).half().double() * 2.0 ** -14 * m - u).flatten()[:len(p)]
    sign = torch.where(left > 0, 1.0, -1.0).double()
    free = left.abs().argsort()[:len(p) // 2]
    sign[free] = 0
    total = (sign * p).sum().item()
    for i in free[p[free].argsort(descending=True)].tolist():
        sign[i] = 1.0 if total < 0 else -1.0
        total += sign[i].item() * p[i].item()
    return sign


@pytest.mark.parametrize("B,H,KV,D,L,S,part", [(1, 1, 1, 128, 400, 4096, 16), (4, 32, 8, 128, 1000, 1000, 64), (2, 16, 1, 64, 900, 900, 64),
                                               (3, 24, 2, 128, 300, 4096, 16), (4, 40, 8, 64, 1000, 1000, 64)])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_probabilities_are_not_cut_to_16_bits(dtype, B, H, KV, D, L, S, part):
    """Values that follow the sign of what rounding a probability to fp16 would
    leave, for one head of each group.  The bound, relative to the mass
    sum_t p_t |v_t|, twice (the products' sum and the one it is divided by): a
    score is the sum of D / 16 instructions' results, each within 2^-23 of A =
    max_t sum_d |q_d k_d| scale, times factors rounded four times; the
    exponential and the held probability are within 2^-22 each; 8 products of a
    part and the 3 roundings of each join.  Then 2^-39 of every |v| (see the head
    of this file) and half a step of the output."""
    from llms_b200.kernels import int8_kv_append, int8_kv_decode_attn
    kv = _alloc(B, KV, S, D, dtype)
    k = _tokens(B, KV, L, D, dtype, seed=H + L)[0]
    int8_kv_append(kv, k, k, 0)
    q = torch.randn(B, H, 1, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(dtype)
    scale = D ** -0.5
    held = (kv.kq.double() * kv.ks.double().repeat_interleave(64, 2)[..., None])[:, :, :L]
    p = torch.exp((q.double()[:, ::H // KV] @ held.transpose(-1, -2))[:, :, 0] * scale).cpu()
    v = torch.stack([torch.stack([_against(p[b, h], part) for h in range(KV)]) for b in range(B)])
    int8_kv_append(kv, k, v.to("cuda", dtype)[..., None].expand(B, KV, L, D), 0)
    got = int8_kv_decode_attn(q, kv, L - 1, scale=scale)
    want, mass, every = _attend(q, kv, [L] * B, scale)
    A = (q.double().abs() @ held.abs().repeat_interleave(H // KV, 1).transpose(-1, -2)).amax().item() * scale
    rel = 2 * ((D / 16 + 4) * A * 2.0 ** -23 + 2 * 2.0 ** -22 + (8 + 3 * L / part) * 2.0 ** -23)
    assert rel < 2.0 ** -13.8  # (cut probabilities: about 2^-13)
    tol = rel * mass + 2.0 ** -39 * every + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == HF else 0)
    d = (got[:, :, 0].double() - want).abs() - tol
    assert (d <= 0).all(), f"off by {d.max().item():.3e} beyond {tol.flatten()[d.argmax()].item():.3e}"
