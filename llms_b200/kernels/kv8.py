"""8-bit KV cache and the decode attention over it.

The engine's cache (``engine/kv_cache.py``) holds K and V in the activation
dtype.  Here each block of 64 tokens of a (row, head) is held in int8 with one
fp32 scale, ``s = max|x| / 127``, ``q = round(x / s)``: half the memory, and
half the bytes of a decode step.

* :class:`Int8KV` -- one layer's storage; :func:`int8_kv_append` puts tokens
  in (prompts, chunks, single tokens), :func:`int8_kv_expand` gives them back
  in the activation dtype;
* :func:`int8_kv_decode_attn` -- GQA attention of one query token per row over
  the storage; :func:`int8_kv_step` -- append of that token and the attention
  in one call;
* :class:`Int8KVCache` -- the layers of a model, in the place of ``KVCache``.

Positions are an int, or an int64 tensor on the device: of one element (every
row) or of one per row.  A row at a negative position is not there: nothing is
stored for it and its attention is zero.  With positions on the device one
captured CUDA graph serves every step and rows of different lengths.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn.functional as F

from .. import _capi

KV8_BLOCK = 64


class Int8KV:
    """One layer's 8-bit K and V for ``rows`` batch rows.

    Args (all on one CUDA device; K and V parts of the same shape and strides):
        kq, vq: int8 (rows, KV, S, D), each head's (S, D) contiguous; S a
            multiple of 64, at most 2**24; D a multiple of 16, at most 256.
        ks, vs: float32 (rows, KV, S / 64), the last dim contiguous.
        kt, vt: activation dtype (rows, KV, 64, D), each head's (64, D)
            contiguous: the tokens, as they came, of the block that the row's
            last append ended in.

    All zero is the empty cache (:meth:`alloc`).  ``length`` is the host's
    count of tokens, kept by :class:`Int8KVCache` only.
    """

    def __init__(self, kq, ks, kt, vq, vs, vt) -> None:
        for name, a, b in (("q", kq, vq), ("s", ks, vs), ("t", kt, vt)):
            if a.shape != b.shape or a.dtype != b.dtype or a.device != b.device or a.stride() != b.stride():
                raise ValueError(f"k{name} and v{name} must share shape, strides, dtype and device")
        if kq.dim() != 4 or kq.dtype != torch.int8:
            raise ValueError(f"kq must be int8 (rows, KV, S, D), got {kq.dtype} {tuple(kq.shape)}")
        rows, KV, S, D = kq.shape
        if S < KV8_BLOCK or S % KV8_BLOCK or S > 1 << 24:
            raise ValueError(f"capacity {S} must be a multiple of {KV8_BLOCK} and at most 2**24")
        if D % 16 or not 16 <= D <= 256:
            raise ValueError(f"head dim {D} must be a multiple of 16 and at most 256")
        if ks.dtype != torch.float32 or ks.shape != (rows, KV, S // KV8_BLOCK):
            raise ValueError(f"ks must be float32 {(rows, KV, S // KV8_BLOCK)}, got {ks.dtype} {tuple(ks.shape)}")
        if kt.shape != (rows, KV, KV8_BLOCK, D):
            raise ValueError(f"kt must be {(rows, KV, KV8_BLOCK, D)}, got {tuple(kt.shape)}")
        if not kq.device == ks.device == kt.device:
            raise ValueError("the parts of the cache must be on the same device")
        if (kq.stride(3), kq.stride(2)) != (1, D) or ks.stride(2) != 1 or (kt.stride(3), kt.stride(2)) != (1, D):
            raise ValueError("each head's tokens, scales and tail must be contiguous")
        code = _capi.dtype_code(kt.dtype)
        self.kq, self.ks, self.kt, self.vq, self.vs, self.vt = kq, ks, kt, vq, vs, vt
        self.rows, self.num_kv_heads, self.capacity, self.head_dim = rows, KV, S, D
        self.dtype, self.device = kt.dtype, kq.device
        self._length, self._tail = 0, -1
        self._c = _capi.Kv8(kq.data_ptr(), ks.data_ptr(), kt.data_ptr(), vq.data_ptr(), vs.data_ptr(), vt.data_ptr(),
                            kq.stride(0), kq.stride(1), ks.stride(0), ks.stride(1), kt.stride(0), kt.stride(1),
                            S, KV, D, code, 0)
        self._ref = ctypes.byref(self._c)
        self._ws: dict[tuple[int, int], int] = {}  # workspace bytes by (B, H)

    @classmethod
    def alloc(cls, *, rows: int, num_kv_heads: int, max_seq_len: int, head_dim: int, dtype, device) -> "Int8KV":
        """An empty cache; the capacity is ``max_seq_len`` rounded up to a multiple of 64."""
        S = max(KV8_BLOCK, -(-max_seq_len // KV8_BLOCK) * KV8_BLOCK)
        q = (rows, num_kv_heads, S, head_dim)
        s = (rows, num_kv_heads, S // KV8_BLOCK)
        t = (rows, num_kv_heads, KV8_BLOCK, head_dim)

        def half():
            return (torch.zeros(q, dtype=torch.int8, device=device), torch.zeros(s, device=device),
                    torch.zeros(t, dtype=dtype, device=device))

        return cls(*half(), *half())

    @property
    def length(self) -> int:
        return self._length

    @length.setter
    def length(self, n: int) -> None:  # by an append that ended at n
        self._length, self._tail = n, (n - 1) // KV8_BLOCK  # (the block that kt, vt hold)

    def _check_rewind(self, n: int) -> None:
        if not 0 <= n <= self._length:
            raise ValueError(f"cannot go to position {n}: the cache holds {self._length} tokens")

    @torch.inference_mode()  # (a cache made in inference mode may be written in no other)
    def rewind(self, n: int) -> None:
        """Forget the tokens from position ``n`` on.  Inside the block that the
        last append ended in the tokens are still there as they came; further
        back the open block's tokens are taken from their 8-bit values."""
        self._check_rewind(n)
        blk, r = divmod(n, KV8_BLOCK)
        if r and blk != self._tail:
            for q, s, t in ((self.kq, self.ks, self.kt), (self.vq, self.vs, self.vt)):
                t[:, :, :r] = (q[:, :, n - r:n].float() * s[:, :, blk, None, None]).to(t.dtype)
            self._tail = blk
        self._length = n


def _pos(pos, B: int, device: torch.device):
    """(host position, device address or None, stride) of a call's positions."""
    if not isinstance(pos, torch.Tensor):
        return int(pos), None, 0
    if pos.dtype != torch.int64 or pos.device != device:
        raise ValueError(f"positions must be int64 on {device}, got {pos.dtype} on {pos.device}")
    n = pos.numel()
    if n == 1:
        return 0, pos.data_ptr(), 0
    if n != B or pos.dim() != 1 or pos.stride(0) != 1:
        raise ValueError(f"positions must be one element or contiguous ({B},), got {tuple(pos.shape)}")
    return 0, pos.data_ptr(), 1


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """4-D ``t`` with a contiguous last dim on 16-byte rows (copied if it is not)."""
    b, h, n, d = t.stride()
    if d == 1 and not ((b | h | n) * t.element_size() | t.data_ptr()) & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_tokens(kv: Int8KV, k: torch.Tensor, v: torch.Tensor) -> None:
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be the same (B, KV, T, D)")
    if k.shape[0] > kv.rows or k.shape[1] != kv.num_kv_heads or k.shape[3] != kv.head_dim:
        raise ValueError(f"k {tuple(k.shape)} does not fit a cache of {tuple(kv.kq.shape)}")
    if k.dtype != kv.dtype or v.dtype != kv.dtype:
        raise ValueError(f"k ({k.dtype}), v ({v.dtype}) must have the cache's dtype {kv.dtype}")
    if k.device != kv.device or v.device != kv.device:
        raise ValueError(f"k ({k.device}), v ({v.device}) must be on the cache's device {kv.device}")


def _check_host_pos(kv: Int8KV, pos, T: int) -> None:
    if not isinstance(pos, torch.Tensor) and not -1 <= pos <= kv.capacity - max(T, 1):
        raise ValueError(f"positions {pos}..{pos + T - 1} are outside the cache (0..{kv.capacity - 1})")


def int8_kv_append(kv: Int8KV, k: torch.Tensor, v: torch.Tensor, pos: int | torch.Tensor) -> None:
    """Store tokens ``k``, ``v`` (B, KV, T, D) in rows 0..B-1 of ``kv`` from
    position ``pos`` on (in place).

    ``pos`` continues the row's last append, or lies in the block of 64 that
    it ended in (its tokens from there on are written anew); 0 begins a row.
    What is stored does not depend on how many tokens come at a time.  Tokens
    past the capacity are refused on the host and dropped for positions on
    the device."""
    _check_tokens(kv, k, v)
    B, _, T, _ = k.shape
    _capi.require_cuda(k)
    _check_host_pos(kv, pos, T)
    host, dev, stride = _pos(pos, B, kv.device)
    if k.numel() == 0:
        return
    k, v = _aligned(k), _aligned(v)
    _capi.launch("b200mm_kv8_append", k, kv._ref, k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], B, T,
                 host, dev, stride)


def int8_kv_expand(kv: Int8KV, length: int, *, batch: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Tokens 0..length-1 of rows 0..batch-1 (default: all) in the cache's
    activation dtype: two (batch, KV, length, D) tensors."""
    B = kv.rows if batch is None else batch
    if not 0 <= length <= kv.capacity or not 0 <= B <= kv.rows:
        raise ValueError(f"length {length}, batch {B} do not fit a cache of {tuple(kv.kq.shape)}")
    _capi.require_cuda(kv.kq)
    shape = (B, kv.num_kv_heads, length, kv.head_dim)
    k = kv.kt.new_empty(shape)
    v = torch.empty_like(k)
    if k.numel():
        _capi.launch("b200mm_kv8_expand", k, kv._ref, k.data_ptr(), v.data_ptr(), *k.stride()[:3], B, length)
    return k, v


def _check_query(kv: Int8KV, q: torch.Tensor) -> None:
    if q.dim() != 4 or q.shape[2] != 1:
        raise ValueError(f"q must be (B, H, 1, D), got {tuple(q.shape)}")
    B, H, _, D = q.shape
    if B > kv.rows or D != kv.head_dim or H < 1 or H % kv.num_kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {tuple(kv.kq.shape)}")
    if q.dtype != kv.dtype or q.device != kv.device:
        raise ValueError(f"q ({q.dtype}, {q.device}) must have the cache's dtype and device ({kv.dtype}, {kv.device})")
    _capi.require_cuda(q)


def _workspace(kv: Int8KV, B: int, H: int) -> tuple[torch.Tensor | None, int]:
    """A call's own workspace, from the caching allocator (so ordered by the
    current stream, and private to the graph that a call is captured into)."""
    need = kv._ws.get((B, H))
    if need is None:
        with _capi.on_device(kv.kq):
            need = kv._ws[(B, H)] = _capi.lib.b200mm_kv8_decode_workspace_size(kv._ref, B, H)
    return (kv.kq.new_empty(need, dtype=torch.uint8) if need else None), need


def int8_kv_decode_attn(q: torch.Tensor, kv: Int8KV, pos: int | torch.Tensor, *, scale: float) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` of one query token per row over tokens
    0..pos of its row (the last token attended to), K / V heads shared by
    groups of H / KV query heads.

    Args:
        q: (B, H, 1, D) in the cache's dtype, B at most the cache's rows.
        pos: int or int64 device tensor (see the module); negative: zeros.

    Returns:
        (B, H, 1, D) in ``q``'s dtype.
    """
    _check_query(kv, q)
    _check_host_pos(kv, pos, 1)
    B, H, _, D = q.shape
    host, dev, stride = _pos(pos, B, kv.device)
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, H, 1, D))
    if B == 0:
        return out
    q = _aligned(q)
    ws, nb = _workspace(kv, B, H)
    _capi.launch("b200mm_kv8_decode", q, kv._ref, q.data_ptr(), *q.stride()[:2], out.data_ptr(), H * D, D, B, H, host, dev,
                 stride, scale, None if ws is None else ws.data_ptr(), nb)
    return out


def int8_kv_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv: Int8KV, pos: int | torch.Tensor, *,
                 scale: float) -> torch.Tensor:
    """One decode step: the new token's ``k``, ``v`` (B, KV, 1, D) enter the
    cache at ``pos``, and ``q`` (B, H, 1, D) attends to tokens 0..pos.  The same
    as :func:`int8_kv_append` followed by :func:`int8_kv_decode_attn`."""
    _check_query(kv, q)
    _check_tokens(kv, k, v)
    B, H, _, D = q.shape
    if k.shape[0] != B or k.shape[2] != 1:
        raise ValueError(f"k {tuple(k.shape)} must hold one token for each of q's {B} rows")
    _check_host_pos(kv, pos, 1)
    host, dev, stride = _pos(pos, B, kv.device)
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, H, 1, D))
    if B == 0:
        return out
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    ws, nb = _workspace(kv, B, H)
    _capi.launch("b200mm_kv8_step", q, kv._ref, q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(),
                 *v.stride()[:2], out.data_ptr(), H * D, D, B, H, host, dev, stride, scale,
                 None if ws is None else ws.data_ptr(), nb)
    return out


class Int8KVCache:
    """The 8-bit caches of a model's layers, in the place of ``KVCache``
    (``engine/kv_cache.py``): ``model.alloc_cache(..., int8=True)``.

    Attention modules call :meth:`attend` instead of writing and slicing
    ``k`` / ``v``.  All rows stand at the same position, ``cur_len``."""

    def __init__(self, layers: list[Int8KV]) -> None:
        self.layers = layers
        self._len = 0

    @classmethod
    def alloc(cls, *, num_layers, max_batch, num_kv_heads, max_seq_len, head_dim, dtype, device) -> "Int8KVCache":
        return cls([Int8KV.alloc(rows=max_batch, num_kv_heads=num_kv_heads, max_seq_len=max_seq_len, head_dim=head_dim,
                                 dtype=dtype, device=device) for _ in range(num_layers)])

    @property
    def capacity(self) -> int:
        return self.layers[0].capacity

    @property
    def cur_len(self) -> int:
        return self._len

    @cur_len.setter
    def cur_len(self, n: int) -> None:
        """Up: tokens that a captured step has put in.  Down: :meth:`seek`."""
        for layer in self.layers:
            layer._check_rewind(min(n, layer.length))
        for layer in self.layers:
            if n > layer.length:
                layer.length = n
            elif n < layer.length:
                layer.rewind(n)
        self._len = n

    def seek(self, pos: int) -> None:
        """Make ``pos`` the next position of every layer: where the tokens end,
        or before (the tokens from there on are forgotten)."""
        for layer in self.layers:  # all or none
            layer._check_rewind(pos)
        for layer in self.layers:
            if pos != layer.length:
                layer.rewind(pos)
        self._len = pos

    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layer_idx: int, start_pos: int) -> torch.Tensor:
        """Cache write and causal GQA attention of ``Attention.forward``
        (engine/attention.py:122-150) for T tokens at ``start_pos``; q (B, H, T,
        D), k and v (B, KV, T, D).  Tokens of earlier calls are read from their
        8-bit values; a prompt's own tokens are seen as they came."""
        layer = self.layers[layer_idx]
        if start_pos != layer.length:
            layer.rewind(start_pos)
        B, H, T, D = q.shape
        end = start_pos + T
        if T == 1:
            out = int8_kv_step(q, k, v, layer, start_pos, scale=D ** -0.5)
            layer.length = end
            return out
        int8_kv_append(layer, k, v, start_pos)
        layer.length = end
        mask = None
        if start_pos:
            fk, fv = int8_kv_expand(layer, end, batch=B)
            fk[:, :, start_pos:], fv[:, :, start_pos:] = k, v
            k, v = fk, fv
            mask = torch.arange(start_pos, end, device=q.device)[:, None] >= torch.arange(end, device=q.device)
        rep = H // layer.num_kv_heads
        if rep > 1:
            k, v = k.repeat_interleave(rep, dim=1), v.repeat_interleave(rep, dim=1)
        return F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=mask is None)
