"""Projections with 4-bit weights vs their formula in 64 bits.

No product is rounded up to 64 rows.  The sums: K / 16 instructions' sums,
K / group scaled ones, 8 partial ones, each rounded (or cut) within 2^-23 of what
stands there, at most mass = sum_k |x w|; then half a step of the output's type.
Beyond that each weight is rounded too, half a step of its type."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import llms_b200.kernels  # noqa: F401


def _weights(N, K, G, dtype, seed=0):
    """Every 4-bit value, scales of both signs, zero ones, ones far apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(0, 256, (N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    s = torch.randn(N, K // G, device="cuda", generator=g) * 0.01
    s[::7, ::2] = 0
    s[1::5] *= 100
    return w, s.to(dtype)


def _x(M, K, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(100 + seed)
    return torch.randn(M, K, device="cuda", generator=g).to(dtype)


def _dense(w, s):
    u = torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1).double() - 8
    return u * s.double().repeat_interleave(u.shape[1] // s.shape[1], 1)


def _product(x, w, s):
    """(x W^T, its bound) in 64 bits."""
    W, K = _dense(w, s), x.shape[1]
    mass = x.double().abs() @ W.abs().T
    eps = torch.finfo(x.dtype).eps / 2 if x.shape[0] > 64 else 0.0
    return x.double() @ W.T, ((K / 16 + s.shape[1] + 8) * 2.0 ** -23 + eps) * mass


def _check_linear(y, x, w, s):
    want, tol = _product(x, w, s)
    d = (y.double() - want).abs() - tol - torch.finfo(x.dtype).eps / 2 * want.abs()
    assert y.dtype == x.dtype and d.max() <= 0, d.max().item()


def _check_gate(y, x, wg, sg, wu, su):
    (g, tg), (u, tu) = _product(x, wg, sg), _product(x, wu, su)
    want = g * torch.sigmoid(g) * u
    # |silu'| <= 1.1; the exponential, the quotient and the product: 2^-20 of the value
    tol = 1.1 * tg * (u.abs() + tu) + (g * torch.sigmoid(g)).abs() * tu + (2.0 ** -20 + torch.finfo(x.dtype).eps / 2) * want.abs()
    # beyond the type's range the rounding gives infinity, below it steps of the smallest number
    tol = tol + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    want = torch.where(want.abs() > torch.finfo(x.dtype).max, want.sign() * torch.inf, want)
    fin = want.isfinite()
    assert torch.equal(y.isfinite(), fin)
    assert ((y.double() - want).abs() - tol)[fin].max() <= 0


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (1, 6144, 4096), (2, 130, 256), (7, 127, 1152), (8, 128, 1024), (9, 300, 2176),
                                   (16, 512, 896), (17, 65, 384), (33, 257, 1280), (64, 640, 640), (65, 96, 512), (150, 200, 256),
                                   (192, 256, 512), (300, 264, 1024)])
def test_linear(dtype, G, M, N, K):
    from llms_b200.kernels import int4_linear
    x, (w, s) = _x(M, K, dtype), _weights(N, K, G, dtype, seed=M)
    _check_linear(int4_linear(x, w, s), x, w, s)


@pytest.mark.parametrize("K,G", [(32, 32), (64, 32), (96, 32), (160, 32), (64, 64), (192, 64), (320, 64), (1056, 32), (1088, 64),
                                 (65536, 128)])
@pytest.mark.parametrize("M", [1, 12])
def test_columns_that_end_inside_a_chunk(K, G, M):
    from llms_b200.kernels import int4_linear
    x, (w, s) = _x(M, K, BF), _weights(70, K, G, BF, seed=K)
    _check_linear(int4_linear(x, w, s), x, w, s)


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 12288, 4096), (1, 3, 128), (5, 129, 384), (16, 320, 1024), (31, 70, 256), (64, 200, 640),
                                   (100, 128, 256), (200, 136, 512)])
def test_gate_up(dtype, G, M, N, K):
    from llms_b200.kernels import int4_fused_gate_up_silu
    x = _x(M, K, dtype) * 0.1
    wg, sg = _weights(N, K, G, dtype, seed=M)
    wu, su = _weights(N, K, G, dtype, seed=M + 1)
    _check_gate(int4_fused_gate_up_silu(x, wg, sg, wu, su), x, wg, sg, wu, su)


@pytest.mark.parametrize("M", [1, 40])
def test_x_at_the_ends_of_its_range(M):
    """bf16 activations beyond fp16's range, and an infinity and a NaN in one row only."""
    from llms_b200.kernels import int4_linear
    x, (w, s) = _x(M, 512, BF), _weights(64, 512, 64, BF)
    x[:, ::3] *= 2.0 ** 60
    x[:, 1::3] *= 2.0 ** -60
    _check_linear(int4_linear(x, w, s), x, w, s)
    if M > 1:
        x[3, 5], x[7, 9] = torch.inf, torch.nan
        y = int4_linear(x, w, s)
        rows = torch.ones(M, dtype=torch.bool, device="cuda")
        rows[[3, 7]] = False
        _check_linear(y[rows], x[rows], w, s)
        assert not y[3].isfinite().any() and y[7].isnan().all()


def test_strides_views_and_shapes():
    from llms_b200.kernels import int4_fused_gate_up_silu, int4_fused_qkv, int4_linear
    K, N = 256, 96
    w, s = _weights(2 * N, K, 64, BF, seed=2)
    big = torch.randn(6, K + 8, device="cuda").to(BF)
    for x in (big[:, :K], big[:, 8:], big[:, 3:K + 3], big[::2, :K], big[:, :K].reshape(2, 3, K), torch.randn(K, 5, device="cuda").to(BF).t()):
        y = int4_linear(x, w, s)
        assert y.shape == (*x.shape[:-1], 2 * N)
        _check_linear(y.reshape(-1, 2 * N), x.reshape(-1, K), w, s)
    x = big[:, :K]
    # rows of a stacked weight, every second row, scales of a larger table, an unaligned weight
    _check_linear(int4_linear(x, w[N:], s[N:]), x, w[N:], s[N:])
    _check_linear(int4_linear(x, w[::2], s[::2]), x, w[::2], s[::2])
    t = torch.zeros(2 * N, 7, device="cuda", dtype=BF)
    t[:, 2:6] = s
    _check_linear(int4_linear(x, w, t[:, 2:6]), x, w, s)
    u = torch.zeros(2 * N * K // 2 + 1, dtype=torch.uint8, device="cuda")[1:].view(2 * N, K // 2)
    u.copy_(w)
    _check_linear(int4_linear(x, u, s), x, w, s)
    _check_gate(int4_fused_gate_up_silu(x, w[:N], s[:N], u[N:], t[N:, 2:6]), x, w[:N], s[:N], w[N:], s[N:])
    q, k, v = int4_fused_qkv(x, w, s, n_q=N, n_k=N // 2)
    assert torch.equal(torch.cat((q, k, v), -1), int4_linear(x, w, s)) and k.data_ptr() == q.data_ptr() + 2 * N


def test_what_lies_behind_the_output_stays():
    """Rows of y with a stride of their own, through the C entry."""
    from llms_b200 import _capi
    M, N, K, G = 5, 100, 384, 128
    x, (w, s) = _x(M, K, BF), _weights(N, K, G, BF)
    y = torch.full((M + 1, 128), 7.0, dtype=BF, device="cuda")
    st = _capi.lib.b200mm_linear_w4(x.data_ptr(), K, w.data_ptr(), K // 2, s.data_ptr(), K // G, G, y.data_ptr(), 128, M, N, K, 2,
                                    None, 0, _capi.stream_of(x))
    assert st == 0
    _check_linear(y[:M, :N], x, w, s)
    assert (y[:, N:] == 7).all() and (y[M] == 7).all()


@pytest.mark.parametrize("M", [1, 200])
def test_graphs_streams_and_weights_made_just_before(M):
    from llms_b200.kernels import dequantize_grouped, int4_linear, quantize_grouped
    W = (torch.randn(512, 1024, device="cuda") * 0.02).to(BF)
    x = _x(M, 1024, BF)
    for _ in range(3):  # weights and x of the same stream, no wait between
        w, s = quantize_grouped(W, 128)
        y = int4_linear(x, w, s)
        assert torch.equal(y, int4_linear(x, w, s))
        _check_linear(y, x, w, s)
        W = W.flip(0).contiguous()
    assert (dequantize_grouped(w, s).double() - _dense(w, s)).abs().max() == 0
    graphs = []
    for i in range(2):
        xi = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            yi = int4_linear(int4_linear(xi, w, s)[:, :512].repeat(1, 2), w, s)
        graphs.append((g, xi, yi, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for r in range(4):
        for i, (g, xi, yi, st) in enumerate(graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                xi.copy_(x * (1 + i))
                g.replay()
    torch.cuda.synchronize()
    for i, (g, xi, yi, st) in enumerate(graphs):
        assert torch.equal(yi, int4_linear(int4_linear(x * (1 + i), w, s)[:, :512].repeat(1, 2), w, s))


def test_modules():
    from llms_b200.kernels import Int4FFN, Int4Linear, int4_fused_gate_up_silu
    from llms_b200.qwen3 import FFN
    ffn = FFN(256, 384).to("cuda", BF)
    m, lin = Int4FFN.from_eager(ffn, group=64), Int4Linear.from_linear(ffn.down, group=128)
    x, h = _x(3, 256, BF), _x(2, 384, BF)
    with torch.inference_mode():
        y = int4_fused_gate_up_silu(x, m.wg, m.sg, m.wu, m.su)
        _check_gate(y, x, m.wg, m.sg, m.wu, m.su)
        assert torch.equal(m(x), ffn.down(y))
        _check_linear(lin(h), h, lin.qweight, lin.scale)


def _pack(u):
    return (u[:, 0::2] | (u[:, 1::2] << 4)).contiguous()


def _ruled_out(x, w, s, how, big, G):
    """Columns of x at ``big``, each beside a weight or a scale that is zero."""
    w, s, x = w.clone(), s.clone(), x.clone()
    if how == "scales":
        x[:, :G] = big  # a whole group, in every chunk of columns
        s[:, 0] = 0
        x[:, -G:] = -big
        s[:, -1] = 0
    else:
        u = torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1)
        u[:, 5::37] = 8
        x[:, 5::37] = big
        w = _pack(u)
    return x, w, s


@pytest.mark.parametrize("how", ["scales", "weights"])
@pytest.mark.parametrize("big", [2.0 ** 60, 2.0 ** 31 * 1.9921875, 2.0 ** 32, 2.0 ** 100])
@pytest.mark.parametrize("M,K", [(1, 512), (3, 5120), (8, 1024), (8, 5120), (16, 512), (17, 512), (40, 512), (64, 5120)])
def test_large_columns_at_zero_weights_change_nothing(M, K, how, big):
    """Beside columns whose weights are zero the others' products keep every
    bit: the bound counts no mass for them.  (2^31 and a little: the widest
    spread that fp16 still holds for 8-bit values; 2^32: the next one.)"""
    from llms_b200.kernels import int4_fused_gate_up_silu, int4_linear
    G = 64
    x = torch.randint(128, 256, (M, K), device="cuda", generator=torch.Generator(device="cuda").manual_seed(M + K)) / 128
    x[:, 1::2] *= -1
    x = x.to(BF)
    x, w, s = _ruled_out(x, *_weights(70, K, G, BF, seed=K), how, big, G)
    _check_linear(int4_linear(x, w, s), x, w, s)
    s = s * 2.0 ** -8
    _check_gate(int4_fused_gate_up_silu(x, w, s, w.flip(0).contiguous(), s.flip(0).contiguous()), x, w, s, w.flip(0), s.flip(0))


@pytest.mark.parametrize("M,K", [(1, 256), (8, 256), (2, 5120), (12, 256)])
def test_x_below_the_normal_numbers(M, K):
    """All of x subnormal, and subnormal columns beside normal ones whose weights are zero."""
    from llms_b200.kernels import int4_linear
    w, s = _weights(40, K, 32, BF, seed=1)
    s = s * 2.0 ** 40
    x = (torch.randint(-127, 128, (M, K), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 2.0 ** -133).to(BF)
    assert x.abs().max() < 2.0 ** -126 and x.any()
    _check_linear(int4_linear(x, w, s), x, w, s)
    x, w, s = _ruled_out(x, w, s, "weights", 1.0, 32)
    _check_linear(int4_linear(x, w, s), x, w, s)


# K, the most rows of a launch of the stream kernel there (plain, gate-up), and N of a few
# tiles with a ragged end, and of more tiles than SMs
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("K,G", [(4128, 32), (5120, 64), (5120, 128), (8192, 128), (9728, 32), (9728, 128), (12288, 64), (12288, 128)])
@pytest.mark.parametrize("M", [1, 3, 4, 6, 8, 9, 16, 17, 33, 64])
def test_deep_columns(M, K, G, dtype):
    """Beyond 4096 columns x lies in shared memory where it fits and the warps
    take several slices; other rows go to the cluster kernel, deep ones in several launches."""
    from llms_b200.kernels import int4_fused_gate_up_silu, int4_linear
    N = 2500 if M in (3, 8, 33) else 70
    x, (w, s) = _x(M, K, dtype), _weights(N, K, G, dtype, seed=M)
    _check_linear(int4_linear(x, w, s), x, w, s)
    wu, su = _weights(N, K, G, dtype, seed=M + 1)
    x = x * 0.1
    _check_gate(int4_fused_gate_up_silu(x, w, s, wu, su), x, w, s, wu, su)


def test_launches_of_one_call_write_their_own_rows_only():
    """64 rows at 12288 columns take two launches (gate-up four): rows behind the last, and between
    rows of y, stay; a call of the same rows one launch at a time gives the same bits."""
    from llms_b200 import _capi
    from llms_b200.kernels import int4_fused_gate_up_silu, int4_linear
    M, N, K, G = 50, 130, 12288, 128
    x, (w, s), (wu, su) = _x(M, K, BF), _weights(N, K, G, BF), _weights(N, K, G, BF, seed=1)
    y = torch.full((M + 2, 160), 7.0, dtype=BF, device="cuda")
    st = _capi.lib.b200mm_linear_w4(x.data_ptr(), K, w.data_ptr(), K // 2, s.data_ptr(), K // G, G, y.data_ptr(), 160, M, N, K, 2,
                                    None, 0, _capi.stream_of(x))
    assert st == 0 and (y[:, N:] == 7).all() and (y[M:] == 7).all()
    _check_linear(y[:M, :N].contiguous(), x, w, s)
    assert torch.equal(y[:32, :N], int4_linear(x[:32], w, s)) and torch.equal(y[32:M, :N], int4_linear(x[32:], w, s))
    h = x * 0.1
    g = int4_fused_gate_up_silu(h, w, s, wu, su)
    for a in range(0, M - 16, 16):
        assert torch.equal(g[a:a + 16], int4_fused_gate_up_silu(h[a:a + 16], w, s, wu, su))
