"""Projections with 4-bit weights and group scales (the reference has none).

A row's weights come in groups of 32, 64 or 128 columns that share a scale,
``W[n, k] = (u[n, k] - 8) * s[n, k // group]`` with ``u`` in 0..15, two to a byte
(the even column in the low half).  Activations, scales and outputs are in
float16 or bfloat16, sums in fp32, and up to 64 rows of activations no
product is rounded.  Beyond that the weights are expanded to 16 bits (rounded
once more) for the dense GEMM, in memory that the call takes from the caching
allocator: 2 bytes a weight while it runs.  Up to 16 rows 4 bits are the fastest of the
weight types here; from 17 on the 16-bit projections are as fast or faster.
"""

from __future__ import annotations

import torch
from torch import nn

from .. import _capi
from .fused_qkv import TritonAttention

GROUPS = (32, 64, 128)


def quantize_grouped(W: torch.Tensor, group: int = 128, *, dtype: torch.dtype | None = None):
    """Symmetric 4-bit per group: ``s = max|W_group| / 7`` rounded to ``dtype``
    (default: W's, bfloat16 for float32), ``q = clamp(round(W / s), -8, 7)``.

    Returns (uint8 (N, K / 2), scales (N, K / group)).  All-zero groups get
    ``s = 0``."""
    if W.dim() != 2:
        raise ValueError(f"W must be 2D (N, K), got shape {tuple(W.shape)}")
    N, K = W.shape
    if group not in GROUPS or K % group:
        raise ValueError(f"group must be one of {GROUPS} and divide K = {K}, got {group}")
    dtype = dtype or (W.dtype if W.dtype in (torch.float16, torch.bfloat16) else torch.bfloat16)
    g = W.detach().float().view(N, K // group, group)
    s = (g.abs().amax(-1) / 7).to(dtype)
    d = s.float()[..., None]
    q = torch.where(d > 0, torch.round(g / torch.where(d > 0, d, 1.0)), 0.0).clamp_(-8, 7)
    u = (q + 8).to(torch.uint8).view(N, K)
    return (u[:, 0::2] | (u[:, 1::2] << 4)).contiguous(), s.contiguous()


def dequantize_grouped(w: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """The float32 weights (N, K) that ``w``, ``s`` stand for."""
    q = torch.stack((w & 15, w >> 4), dim=-1).view(w.shape[0], -1).float() - 8
    return (q.view(*s.shape, -1) * s.float()[..., None]).view_as(q)


def _check_w4(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, name: str) -> int:
    """The group size of ``w``, ``s``; raises where they do not fit ``x`` or each other."""
    if w.dim() != 2 or w.dtype != torch.uint8:
        raise ValueError(f"{name} must be a 2D uint8 tensor (N, K / 2), got {w.dtype} {tuple(w.shape)}")
    N, K = w.shape
    K *= 2
    if x.shape[-1] != K:
        raise ValueError(f"x last dim {x.shape[-1]} != {name}'s K {K}")
    groups = s.shape[1] if s.dim() == 2 else 0
    if not groups or s.shape[0] != N or K % groups or K // groups not in GROUPS:
        raise ValueError(f"{name} scales must be ({N}, {K} / group) with group one of {GROUPS}, got {tuple(s.shape)}")
    dtype, device = x.dtype, x.device
    if dtype not in (torch.bfloat16, torch.float16) or s.dtype != dtype:
        raise ValueError(f"x ({dtype}) and {name} scales ({s.dtype}) must share a dtype, bfloat16 or float16")
    if device != w.device or device != s.device:
        raise ValueError(f"x ({device}), {name} ({w.device}), scales ({s.device}) must be on the same device")
    return K // groups


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """2-D ``t`` with unit inner stride on 16-byte rows (copied if it is not)."""
    ld, inner = t.stride()
    if inner == 1 and not (t.data_ptr() | ld * t.element_size()) & 15 and ld >= t.shape[1]:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _scales(s: torch.Tensor) -> torch.Tensor:
    ld, inner = s.stride()
    return s if inner == 1 and ld >= s.shape[1] else s.clone(memory_format=torch.contiguous_format)


def _workspace(x: torch.Tensor, M: int, N: int, K: int, gate: int) -> tuple[torch.Tensor | None, int]:
    need = _capi.lib.b200mm_w4_workspace_size(M, N, K, gate) if M > 64 else 0
    return (x.new_empty(need, dtype=torch.uint8) if need else None), need


def int4_linear(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """``x @ W.T`` for the 4-bit weights ``w`` (N, K / 2), ``s`` (N, K / group).

    Args:
        x: (..., K), float16 or bfloat16 on a CUDA device; ``s`` has its dtype.

    Returns:
        (..., N) in ``x``'s dtype.
    """
    group = _check_w4(x, w, s, "W")
    N, K = w.shape[0], x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    y = x.new_empty((*x.shape[:-1], N))
    if M and N:
        _capi.require_cuda(x)
        x2, w, s = _rows16(x2), _rows16(w), _scales(s)
        ws, nb = _workspace(x, M, N, K, 0)
        _capi.launch("b200mm_linear_w4", x, x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), s.data_ptr(),
                     s.stride(0), group, y.data_ptr(), N, M, N, K, _capi.DTYPE_CODES[x.dtype],
                     None if ws is None else ws.data_ptr(), nb)
    return y


def int4_fused_qkv(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, *, n_q: int, n_k: int):
    """``x @ W_qkv.T`` split into q / k / v views of one buffer; as ``int8_fused_qkv``."""
    if n_q + 2 * n_k != w.shape[0]:
        raise ValueError(f"n_q + 2*n_k ({n_q} + 2*{n_k} = {n_q + 2 * n_k}) != W_qkv.shape[0] ({w.shape[0]})")
    return torch.split_with_sizes(int4_linear(x, w, s), (n_q, n_k, n_k), -1)


def int4_fused_gate_up_silu(x: torch.Tensor, wg: torch.Tensor, sg: torch.Tensor, wu: torch.Tensor,
                            su: torch.Tensor) -> torch.Tensor:
    """``silu(x @ Wg.T) * (x @ Wu.T)`` for 4-bit gate and up weights of one shape and group."""
    if wg.shape != wu.shape or sg.shape != su.shape:
        raise ValueError(f"Wg {tuple(wg.shape)}, {tuple(sg.shape)} and Wu {tuple(wu.shape)}, {tuple(su.shape)} must match")
    group = _check_w4(x, wg, sg, "Wg")
    _check_w4(x, wu, su, "Wu")
    N, K = wg.shape[0], x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    y = x.new_empty((*x.shape[:-1], N))
    if M and N:
        _capi.require_cuda(x)
        x2, wg, wu, sg, su = _rows16(x2), _rows16(wg), _rows16(wu), _scales(sg), _scales(su)
        if wg.stride(0) != wu.stride(0):
            wg, wu = wg.contiguous(), wu.contiguous()
        if sg.stride(0) != su.stride(0):
            sg, su = sg.contiguous(), su.contiguous()
        ws, nb = _workspace(x, M, N, K, 1)
        _capi.launch("b200mm_gate_up_silu_w4", x, x2.data_ptr(), x2.stride(0), wg.data_ptr(), wu.data_ptr(),
                     wg.stride(0), sg.data_ptr(), su.data_ptr(), sg.stride(0), group, y.data_ptr(), N, M, N, K,
                     _capi.DTYPE_CODES[x.dtype], None if ws is None else ws.data_ptr(), nb)
    return y


class Int4Linear(nn.Module):
    """Bias-free projection with 4-bit weights (buffers ``qweight`` [N, K / 2]
    uint8 and ``scale`` [N, K / group])."""

    def __init__(self, in_features: int, out_features: int, *, group: int = 128, dtype=torch.bfloat16) -> None:
        super().__init__()
        if group not in GROUPS or in_features % group:
            raise ValueError(f"group must be one of {GROUPS} and divide {in_features}, got {group}")
        self.in_features, self.out_features, self.group = in_features, out_features, group
        self.register_buffer("qweight", torch.full((out_features, in_features // 2), 0x88, dtype=torch.uint8))
        self.register_buffer("scale", torch.ones(out_features, in_features // group, dtype=dtype))

    @classmethod
    def from_linear(cls, lin: nn.Module, *, group: int = 128) -> "Int4Linear":
        if getattr(lin, "bias", None) is not None:
            raise ValueError("Int4Linear serves bias-free projections only")
        W = lin.weight
        w, s = quantize_grouped(W, group)
        out = cls.__new__(cls)
        nn.Module.__init__(out)
        out.in_features, out.out_features, out.group = W.shape[1], W.shape[0], group
        out.register_buffer("qweight", w)
        out.register_buffer("scale", s)
        return out

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int4_linear(x, self.qweight, self.scale)


class Int4FFN(nn.Module):
    """SwiGLU FFN with 4-bit gate / up weights (buffers ``wg, sg, wu, su``) and
    a dense ``down``."""

    def __init__(self, hidden_size: int, intermediate_size: int, *, group: int = 128, dtype=torch.bfloat16) -> None:
        super().__init__()
        for n in ("g", "u"):
            lin = Int4Linear(hidden_size, intermediate_size, group=group, dtype=dtype)
            self.register_buffer("w" + n, lin.qweight)
            self.register_buffer("s" + n, lin.scale)
        self.down = nn.Linear(intermediate_size, hidden_size, bias=False)

    @classmethod
    def from_eager(cls, eager: nn.Module, *, group: int = 128) -> "Int4FFN":
        out = cls.__new__(cls)
        nn.Module.__init__(out)
        for n, lin in (("g", eager.gate), ("u", eager.up)):
            w, s = quantize_grouped(lin.weight, group)
            out.register_buffer("w" + n, w)
            out.register_buffer("s" + n, s)
        out.down = eager.down
        return out

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down(int4_fused_gate_up_silu(x, self.wg, self.sg, self.wu, self.su))


class Int4Attention(TritonAttention):
    """``TritonAttention`` whose fused QKV projection reads 4-bit weights
    (buffers ``w_qkv``, ``s_qkv``) instead of a dense ``W_qkv``."""

    def __init__(self, *, hidden_size: int, num_heads: int, num_kv_heads: int, head_dim: int, rms_eps: float,
                 group: int = 128, dtype=torch.bfloat16) -> None:
        super().__init__(hidden_size=hidden_size, num_heads=num_heads, num_kv_heads=num_kv_heads, head_dim=head_dim,
                         rms_eps=rms_eps)
        del self.W_qkv
        lin = Int4Linear(hidden_size, self.n_q + 2 * self.n_k, group=group, dtype=dtype)
        self.register_buffer("w_qkv", lin.qweight)
        self.register_buffer("s_qkv", lin.scale)

    @classmethod
    def from_eager(cls, eager: nn.Module, *, group: int = 128) -> "Int4Attention":
        """From an engine ``Attention`` (q/k/v Linears) or a ``TritonAttention``."""
        out = cls.__new__(cls)
        nn.Module.__init__(out)
        W = eager.W_qkv if hasattr(eager, "W_qkv") else torch.cat([eager.q.weight, eager.k.weight, eager.v.weight], dim=0)
        out.hidden_size = W.shape[1]
        out.num_heads, out.num_kv_heads, out.head_dim = eager.num_heads, eager.num_kv_heads, eager.head_dim
        out.n_q, out.n_k = eager.num_heads * eager.head_dim, eager.num_kv_heads * eager.head_dim
        w, s = quantize_grouped(W, group)
        out.register_buffer("w_qkv", w)
        out.register_buffer("s_qkv", s)
        out.o, out.q_norm, out.k_norm = eager.o, eager.q_norm, eager.k_norm
        out.decode_attn_op = getattr(eager, "decode_attn_op", None)
        return out

    def project_qkv(self, x: torch.Tensor):
        return int4_fused_qkv(x, self.w_qkv, self.s_qkv, n_q=self.n_q, n_k=self.n_k)
