"""Cases and plain forms of the low-memory decode operators: the 8-bit KV cache with its attention, projections with 4-bit
weights, and log probabilities.

A case's ``op`` names the operator:

* ``prompt``  -- a prompt enters an 8-bit KV cache in one chunk or two and is expanded again, as a chunked prefill does
* ``step``    -- one decode step over the cache: the new token enters it, and each row's query attends to the row's tokens
* ``linear``  -- a projection with 4-bit weights and group scales
* ``gate_up`` -- the fused gate-up-SiLU projection of the same kind
* ``logprobs`` -- log probabilities of given tokens, the entropy and the top alternatives

``own`` false: elementary torch operations; ``own`` true: the framework's calls.
"""

import math

import torch

own = False

BLOCK = 64  # tokens that share a scale in the 8-bit cache
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a 4096-token prompt of one sequence, at once (Qwen3 heads)
        {"name": "prompt 1x4096", "op": "prompt", "B": 1, "KV": 8, "D": 128, "T": 4096, "first": 4096, "dtype": "bf16"},
        # four prompts of an odd length in two chunks, the second one starting inside a block
        {"name": "prompt 4x1537 chunked", "op": "prompt", "B": 4, "KV": 8, "D": 128, "T": 1537, "first": 1000, "dtype": "fp16"},
        # the smallest step: one short conversation, where latency counts
        {"name": "step 1x512", "op": "step", "B": 1, "H": 32, "KV": 8, "D": 128, "L": 512, "ragged": False, "dtype": "bf16"},
        # one long document
        {"name": "step 1x32768", "op": "step", "B": 1, "H": 32, "KV": 8, "D": 128, "L": 32768, "ragged": False, "dtype": "bf16"},
        # a serving batch: rows of every length, some slots of the batch empty
        {"name": "step 32x4096 ragged", "op": "step", "B": 32, "H": 32, "KV": 8, "D": 128, "L": 4096, "ragged": True, "dtype": "bf16"},
        # the largest: a batch of long documents
        {"name": "step 16x32768", "op": "step", "B": 16, "H": 32, "KV": 8, "D": 128, "L": 32768, "ragged": False, "dtype": "bf16"},
        # the fused QKV projection of an 8B model, one token
        {"name": "w4 qkv m1", "op": "linear", "M": 1, "N": 6144, "K": 4096, "G": 128, "dtype": "bf16"},
        # its gate-up projection, one token
        {"name": "w4 gate-up m1", "op": "gate_up", "M": 1, "N": 12288, "K": 4096, "G": 128, "dtype": "bf16"},
        # the gate-up projection for a batch of 16, finer groups
        {"name": "w4 gate-up m16", "op": "gate_up", "M": 16, "N": 12288, "K": 4096, "G": 64, "dtype": "fp16"},
        # one generated token with its five alternatives
        {"name": "logprobs 1", "op": "logprobs", "M": 1, "V": 151936, "top": 5, "masked": False, "dtype": "bf16"},
        # a decode batch
        {"name": "logprobs 64", "op": "logprobs", "M": 64, "V": 151936, "top": 20, "masked": False, "dtype": "bf16"},
        # a prompt scored whole
        {"name": "logprobs 2048", "op": "logprobs", "M": 2048, "V": 151936, "top": 1, "masked": False, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of the range."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["prompt", "step", "step", "linear", "gate_up", "logprobs"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "prompt":
        B = rng.randint(1, 4)
        T = _between(rng, 1, 8192 // B)
        return {"op": op, "B": B, "KV": rng.choice([1, 2, 4, 8]), "D": rng.choice([64, 128]), "T": T, "first": rng.randint(1, T),
                "dtype": dtype}
    if op == "step":
        B, KV = _between(rng, 1, 64), rng.choice([1, 2, 4, 8])
        L = _between(rng, 1, min(32768, 16 * 32768 * 8 // (B * KV)))
        return {"op": op, "B": B, "H": KV * rng.choice([1, 2, 4, 5, 8]), "KV": KV, "D": rng.choice([64, 128]), "L": L,
                "ragged": rng.random() < 0.7, "dtype": dtype}
    if op in ("linear", "gate_up"):
        G = rng.choice([32, 64, 128])
        return {"op": op, "M": _between(rng, 1, 64), "N": _between(rng, 100, 12288), "K": G * _between(rng, 4, 12288 // G), "G": G,
                "dtype": dtype}
    M = _between(rng, 1, 2048)
    return {"op": op, "M": M, "V": _between(rng, 1000, 155000), "top": rng.randint(0, 20), "masked": rng.random() < 0.4,
            "dtype": rng.choice(["bf16", "fp16", "fp32"]) if M <= 1024 else dtype}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------


def _prompt_inputs(c, g, dev):
    """Keys and values as the projections leave them: (B, T, KV, D), seen as (B, KV, T, D)."""
    dt = DTYPES[c["dtype"]]

    def tokens():
        return torch.randn(c["B"], c["T"], c["KV"], c["D"], generator=g, device=dev).to(dt).transpose(1, 2)

    S = -(-c["T"] // BLOCK) * BLOCK
    return {"k": tokens(), "v": tokens(), **_empty_cache(c["B"], c["KV"], S, c["D"], dt, dev)}


def _empty_cache(B, KV, S, D, dt, dev):
    return {
        "kq": torch.zeros(B, KV, S, D, dtype=torch.int8, device=dev), "vq": torch.zeros(B, KV, S, D, dtype=torch.int8, device=dev),
        "ks": torch.zeros(B, KV, S // BLOCK, device=dev), "vs": torch.zeros(B, KV, S // BLOCK, device=dev),
        "kt": torch.zeros(B, KV, BLOCK, D, dtype=dt, device=dev), "vt": torch.zeros(B, KV, BLOCK, D, dtype=dt, device=dev),
    }


def _step_inputs(c, g, dev):
    """A cache whose rows hold pos[b] tokens, and the new token's query, key and value."""
    B, H, KV, D, L, dt = c["B"], c["H"], c["KV"], c["D"], c["L"], DTYPES[c["dtype"]]
    S = -(-L // BLOCK) * BLOCK
    s = _empty_cache(B, KV, S, D, dt, dev)
    if c["ragged"]:
        pos = torch.randint(0, L, (B,), generator=g, device=dev)
        if B > 3:
            pos[B // 2] = -1  # an empty slot of the batch
        pos[-1] = L - 1
    else:
        pos = torch.full((B,), L - 1, device=dev)
    s["pos"] = pos.long()
    # closed blocks: 8-bit values of normally distributed tokens (the largest of 64 x D lies near 4 deviations)
    for n in ("k", "v"):
        for b in range(B):
            s[n + "q"][b].copy_(torch.randn(KV, S, D, generator=g, device=dev).mul_(31).round_().clamp_(-127, 127))
        s[n + "s"].copy_(torch.rand(B, KV, S // BLOCK, generator=g, device=dev) * 0.02 + 0.02)
    # the open block: its tokens in the activations' type, and the 8 bits that they give
    row = torch.arange(BLOCK, device=dev)
    at = pos.clamp(min=0)
    blk, fill = at // BLOCK, at % BLOCK
    here = torch.arange(B, device=dev)
    for n in ("k", "v"):
        tail = torch.randn(B, KV, BLOCK, D, generator=g, device=dev).to(dt)
        s[n + "t"].copy_(tail)
        held = (row[None, :] < fill[:, None])[:, None, :, None]
        q, sc = _quantize(torch.where(held, tail, 0))
        nq = s[n + "q"].view(B, KV, S // BLOCK, BLOCK, D)
        nq[here, :, blk] = q
        s[n + "s"][here, :, blk] = sc

    def token(heads):
        return torch.randn(B, 1, heads, D, generator=g, device=dev).to(dt).transpose(1, 2)

    s.update(q=token(H), k=token(KV), v=token(KV))
    return s


def _pack(W, G, dt):
    """(N, K) -> (N, K / 2) bytes of two 4-bit numbers, the even column low, and the scales (N, K / G)."""
    N, K = W.shape
    g = W.view(N, K // G, G)
    s = (g.abs().amax(-1) / 7).to(dt)
    u = (torch.round(g / s.float()[..., None]).clamp(-8, 7) + 8).to(torch.uint8).view(N, K)
    return (u[:, 0::2] | (u[:, 1::2] << 4)).contiguous(), s.contiguous()


def _weight_inputs(c, g, dev):
    dt = DTYPES[c["dtype"]]
    s = {"x": torch.randn(c["M"], c["K"], generator=g, device=dev).to(dt)}
    for n in ("0", "1") if c["op"] == "gate_up" else ("0",):
        s["w" + n], s["s" + n] = _pack(torch.randn(c["N"], c["K"], generator=g, device=dev) * 0.02, c["G"], dt)
    return s


def _logit_inputs(c, g, dev):
    """Logits with a few strong candidates in each row; ``masked``: all but a tenth of the vocabulary ruled out."""
    M, V = c["M"], c["V"]
    x = torch.randn(M, V, generator=g, device=dev) * 2.5
    strong = torch.randint(0, V, (M, 8), generator=g, device=dev)
    x.scatter_add_(1, strong, torch.rand(M, 8, generator=g, device=dev) * 12)
    if c["masked"]:
        x.masked_fill_(torch.rand(M, V, generator=g, device=dev) > 0.1, -math.inf)
    pick = torch.rand(M, generator=g, device=dev) < 0.5
    tokens = torch.where(pick, strong[:, 0], torch.randint(0, V, (M,), generator=g, device=dev))
    return {"x": x.to(DTYPES[c["dtype"]]), "tokens": tokens}


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    make = {"prompt": _prompt_inputs, "step": _step_inputs, "linear": _weight_inputs, "gate_up": _weight_inputs,
            "logprobs": _logit_inputs}[case["op"]]
    state = make(case, g, dev)
    state["case"] = dict(case)
    if own and "kq" in state:  # the cache object that a program keeps
        from llms_b200.kernels import Int8KV

        state["kv"] = Int8KV(*(state[n] for n in ("kq", "ks", "kt", "vq", "vs", "vt")))
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------------------------


def _quantize(x):
    """(..., 64, D) tokens of a block -> their 8-bit values and the block's scale. The quotient is taken in 64 bits: a rounded one
    falls on the wrong side of a border now and then."""
    s = (x.abs().amax((-2, -1)).double() / 127).float()
    d = s.double()[..., None, None]
    return torch.where(d > 0, torch.round(x.double() / torch.where(d > 0, d, 1.0)), 0.0).to(torch.int8), s


def _plain_prompt(s):
    out = {}
    T = s["case"]["T"]
    for n in ("k", "v"):
        x = s[n]
        B, KV, _, D = x.shape
        q, sc = _quantize(torch.nn.functional.pad(x, (0, 0, 0, -T % BLOCK)).reshape(B, KV, -1, BLOCK, D))
        out[n] = (q.float() * sc[..., None, None]).reshape(B, KV, -1, D)[:, :, :T].to(x.dtype)
        out[n + "s"] = sc
    return out


def _plain_step(s):
    pos, q = s["pos"], s["q"]
    B, KV, S, D = s["kq"].shape
    dev, g = q.device, q.shape[1] // KV
    there = pos >= 0
    at = pos.clamp(min=0)
    blk, fill, here = at // BLOCK, at % BLOCK, torch.arange(B, device=dev)
    row = torch.arange(BLOCK, device=dev)[None, :]

    def enter(n):
        """The new token into the open block; its rows so far get the scale of them all."""
        tail, store, sc = s[n + "t"], s[n + "q"].view(B, KV, S // BLOCK, BLOCK, D), s[n + "s"]
        new = ((row == fill[:, None]) & there[:, None])[:, None, :, None]
        tail.copy_(torch.where(new, s[n], tail))
        held = ((row <= fill[:, None]) & there[:, None])[:, None, :, None]
        bits, scale = _quantize(torch.where(held, tail, 0))
        store[here, :, blk] = torch.where(held, bits, store[here, :, blk])
        sc[here, :, blk] = torch.where(there[:, None], scale, sc[here, :, blk])
        return (store.float() * sc[..., None, None]).view(B, KV, S, D)

    k, v = enter("k"), enter("v")
    scores = (q.float().view(B, KV, g, D) @ k.transpose(-1, -2)) * D**-0.5
    seen = (torch.arange(S, device=dev)[None, :] <= pos[:, None])[:, None, None, :]
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30)).masked_fill(~seen, 0)
    o = (e @ v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return {"out": o.view(B, KV * g, 1, D).to(q.dtype), "ks": s["ks"], "vs": s["vs"], "kt": s["kt"], "vt": s["vt"]}


def _plain_weight(w, sc):
    u = torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1).float() - 8
    return (u.view(*sc.shape, -1) * sc.float()[..., None]).view(u.shape)


def _plain_linear(s):
    return (s["x"].float() @ _plain_weight(s["w0"], s["s0"]).T).to(s["x"].dtype)


def _plain_gate_up(s):
    x = s["x"].float()
    gate, up = x @ _plain_weight(s["w0"], s["s0"]).T, x @ _plain_weight(s["w1"], s["s1"]).T
    return (gate / (1 + torch.exp(-gate)) * up).to(s["x"].dtype)


def _plain_logprobs(s):
    x, top = s["x"], s["case"]["top"]
    f = x.float()
    m = f.amax(-1, keepdim=True)
    d = f - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    entropy = torch.log(z) - torch.where(e > 0, e * d, 0).sum(-1, keepdim=True) / z
    out = {"logprob": (f.gather(1, s["tokens"][:, None]) - lse)[:, 0], "entropy": entropy[:, 0]}
    # value descending, index ascending: one sortable whole number for both (a float's bits sort as a whole number's, mirrored
    # below zero; adding 0 makes -0 and 0 one)
    b = (f + 0.0).view(torch.int32)
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long() << 32
    key -= torch.arange(x.shape[1], device=x.device)
    ids = key.topk(top, -1).indices
    return {**out, "top_ids": ids, "top_logprobs": f.gather(1, ids) - lse}


# ---- one pass -------------------------------------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    op = c["op"]
    if not own:
        return {"prompt": _plain_prompt, "step": _plain_step, "linear": _plain_linear, "gate_up": _plain_gate_up,
                "logprobs": _plain_logprobs}[op](state)
    from llms_b200 import kernels as F

    if op == "prompt":
        kv, k, v, T, first = state["kv"], state["k"], state["v"], c["T"], c["first"]
        F.int8_kv_append(kv, k[:, :, :first], v[:, :, :first], 0)
        if first < T:
            F.int8_kv_append(kv, k[:, :, first:], v[:, :, first:], first)
        ek, ev = F.int8_kv_expand(kv, T)
        return {"k": ek, "v": ev, "ks": kv.ks, "vs": kv.vs}
    if op == "step":
        kv = state["kv"]
        out = F.int8_kv_step(state["q"], state["k"], state["v"], kv, state["pos"], scale=c["D"] ** -0.5)
        return {"out": out, "ks": kv.ks, "vs": kv.vs, "kt": kv.kt, "vt": kv.vt}
    if op == "linear":
        return F.int4_linear(state["x"], state["w0"], state["s0"])
    if op == "gate_up":
        return F.int4_fused_gate_up_silu(state["x"], state["w0"], state["s0"], state["w1"], state["s1"])
    r = F.b200_token_logprobs(state["x"], state["tokens"], top=c["top"])
    return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------


def work(case):
    c, op = case, case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
    if op == "prompt":
        n = 2 * c["B"] * c["KV"] * c["T"] * c["D"]
        # tokens in, 8 bits out; 8 bits in, expanded tokens out; scales
        return {"bytes": n * (size + 1 + 1 + size) + 16 * c["B"] * c["KV"] * (-(-c["T"] // BLOCK)), "flops": 4 * n}
    if op == "step":
        mean = c["L"] / 2 if c["ragged"] else c["L"]
        tokens = c["B"] * c["KV"] * mean
        ends = c["B"] * c["D"] * (2 * c["H"] + 2 * c["KV"]) * size
        return {"bytes": 2 * tokens * (c["D"] + 4 / BLOCK) + ends, "flops": 4 * c["B"] * c["H"] * mean * c["D"]}
    if op in ("linear", "gate_up"):
        n = 2 if op == "gate_up" else 1
        weights = n * c["N"] * (c["K"] // 2 + c["K"] // c["G"] * size)
        return {"bytes": weights + c["M"] * (c["K"] + c["N"]) * size, "flops": 2 * n * c["M"] * c["N"] * c["K"]}
    return {"bytes": c["M"] * (c["V"] * size + 16 + 12 * c["top"]), "flops": 5 * c["M"] * c["V"]}


# ---- 64 bits --------------------------------------------------------------------------------------------------------------------


def _exact_block(x):
    """One block's tokens (n, D) in 64 bits -> the values that its 8 bits stand for, and its scale (held in 32 bits)."""
    largest = x.abs().max()
    if largest == 0:
        return torch.zeros_like(x), torch.zeros((), dtype=torch.float64, device=x.device)
    s = (largest / 127).float().double()
    return torch.round(x / s) * s, s


def _exact_prompt(s):
    c, out = s["case"], {}
    for n in ("k", "v"):
        x = s[n].double()
        blocks = [x[:, :, i:i + BLOCK] for i in range(0, c["T"], BLOCK)]
        pairs = [[[_exact_block(blk[b, h]) for h in range(c["KV"])] for b in range(c["B"])] for blk in blocks]
        out[n] = torch.cat([torch.stack([torch.stack([p[0] for p in row]) for row in blk]) for blk in pairs], 2)
        out[n + "s"] = torch.stack([torch.stack([torch.stack([p[1] for p in row]) for row in blk]) for blk in pairs], 2)
    return out


def _exact_step(s):
    c, q = s["case"], s["q"].double()
    B, H, KV, D = c["B"], c["H"], c["KV"], c["D"]
    out = torch.zeros(B, H, 1, D, dtype=torch.float64, device=q.device)
    scales = {n: s[n].double() for n in ("ks", "vs")}
    tails = {n: s[n].double() for n in ("kt", "vt")}
    for b, p in enumerate(s["pos"].tolist()):
        if p < 0:
            continue
        j, r = p // BLOCK, p % BLOCK
        for n in ("k", "v"):
            tails[n + "t"][b, :, r] = s[n][b, :, 0].double()
        for h in range(KV):
            full = {}
            for n in ("k", "v"):
                open_, sc = _exact_block(tails[n + "t"][b, h, :r + 1])
                closed = s[n + "q"][b, h, :j * BLOCK].double() * scales[n + "s"][b, h, :j].repeat_interleave(BLOCK)[:, None]
                scales[n + "s"][b, h, j] = sc
                full[n] = torch.cat((closed, open_))
            heads = slice(h * (H // KV), (h + 1) * (H // KV))
            out[b, heads, 0] = torch.softmax(q[b, heads, 0] @ full["k"].T / math.sqrt(D), -1) @ full["v"]
    return {"out": out, **scales, **tails}


def _exact_product(x, w, s):
    x, G = x.double(), x.shape[1] // s.shape[1]
    even, odd = (w & 15).double() - 8, (w >> 4).double() - 8
    by = s.double().repeat_interleave(G // 2, 1)
    return x[:, 0::2] @ (even * by).T + x[:, 1::2] @ (odd * by).T


def _exact_logprobs(s):
    top, rows = s["case"]["top"], []
    for x, t in zip(s["x"], s["tokens"].tolist()):
        x = x.double()
        lp = torch.log_softmax(x, 0)
        order = torch.sort(x, descending=True, stable=True).indices[:top]
        rows.append((lp[t], -(lp.exp() * lp.clamp(min=-1e4)).sum(), order, lp[order]))
    return {k: torch.stack([r[i] for r in rows]) for i, k in enumerate(("logprob", "entropy", "top_ids", "top_logprobs"))}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "prompt":
        return _exact_prompt(s)
    if op == "step":
        return _exact_step(s)
    if op == "linear":
        return _exact_product(s["x"], s["w0"], s["s0"])
    if op == "gate_up":
        g, u = _exact_product(s["x"], s["w0"], s["s0"]), _exact_product(s["x"], s["w1"], s["s1"])
        return g * torch.sigmoid(g) * u
    return _exact_logprobs(s)
