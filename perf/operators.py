"""Operators of a block-decode step over a shared affix, each in a plain form and through the package.

``attention``  attention of a whole batch whose requests share one long prefix in the paged cache
``int8``       a projection in 8-bit integers: the activations are quantised per token by the kernel
               that produces them (plain rows, RMSNorm, gated activation), the weights per channel
``rope``       rotary positions in both layouts, on part of the head, with scaled frequencies, the
               rotated keys and the values appended to the paged cache

A case is a dict of plain values, ``prepare`` makes its inputs from a seed, ``run`` is one pass through
the operator and ``exact`` is the operator's definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 256          # cache slots of a page


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # block decode of the served LLaDA shape: 16 requests of 32 masked positions, an 800-token affix of
        # which every request replaces 160 tokens by anchors of its own
        dict(name="attention_block_llada", op="attention", dtype="bf16", batch=16, q_len=32, heads=32, kv_heads=32,
             head_dim=128, prefix=800, suffix_min=416, suffix_max=672, holes=160, spread_pages=False),
        # block decode of the served Dream shape over a long shared document
        dict(name="attention_block_dream", op="attention", dtype="bf16", batch=32, q_len=32, heads=28, kv_heads=4,
             head_dim=128, prefix=8192, suffix_min=300, suffix_max=700, holes=0, spread_pages=False),
        # single tokens of a large batch behind a very long shared prefix
        dict(name="attention_token_long", op="attention", dtype="bf16", batch=64, q_len=1, heads=28, kv_heads=4,
             head_dim=128, prefix=32768, suffix_min=1, suffix_max=1024, holes=0, spread_pages=True),
        # the smallest call: few requests, one token each, where latency counts
        dict(name="attention_token_small", op="attention", dtype="fp16", batch=4, q_len=1, heads=28, kv_heads=4,
             head_dim=128, prefix=600, suffix_min=0, suffix_max=64, holes=0, spread_pages=True),
        # small heads, odd lengths, ragged queries, pages that end inside a tile
        dict(name="attention_odd", op="attention", dtype="fp16", batch=7, q_len=5, heads=6, kv_heads=2, head_dim=64,
             prefix=1001, suffix_min=0, suffix_max=333, holes=77, spread_pages=True),
        # attention output projection of a few rows (the last running requests)
        dict(name="int8_rows_few", op="int8", source="rows", dtype="bf16", rows=33, k=4096, n=4096, bias=False),
        # q/k/v projection of a LLaDA block-decode step behind its norm
        dict(name="int8_norm_qkv", op="int8", source="norm", dtype="bf16", rows=512, k=4096, n=12288, bias=False),
        # feed-forward output projection of the same step behind the gated activation
        dict(name="int8_gate_out", op="int8", source="gate", dtype="bf16", rows=512, k=12288, n=4096, bias=False),
        # Dream q/k/v projection with its bias at refresh size, fp16, an odd number of rows
        dict(name="int8_norm_bias", op="int8", source="norm", dtype="fp16", rows=2305, k=3584, n=4608, bias=True),
        # Dream gate and up projections over a long prompt
        dict(name="int8_norm_wide", op="int8", source="norm", dtype="bf16", rows=4096, k=3584, n=37888, bias=False),
        # one block-decode step of a long context: 16 x 32 rows at far positions, long-context frequencies
        dict(name="rope_decode", op="rope", dtype="bf16", rows=512, heads=32, kv_heads=32, head_dim=128, rotary=128,
             interleaved=False, theta=500000.0, stretch=4.0, factor=1.0, far=131072, skip=0),
        # a long prompt: interleaved pairs on half of the head, an attention factor, rows without a slot
        dict(name="rope_prompt", op="rope", dtype="bf16", rows=16411, heads=28, kv_heads=4, head_dim=128, rotary=64,
             interleaved=True, theta=1000000.0, stretch=1.0, factor=1.2, far=1000000, skip=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "int8", "rope"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attention":
        heads, kv_heads = rng.choice([(32, 32), (28, 4), (32, 8), (6, 2), (8, 1)])
        head_dim = rng.choice([128, 128, 64])
        q_len = _log(rng, 1, 40)
        batch = _log(rng, 1, 64)
        prefix = _log(rng, 1, 32768)
        while batch * q_len * heads * prefix > 32 * 32 * 28 * 8192:
            prefix = max(prefix // 2, 1)
        suffix_max = _log(rng, 1, 1024)
        return dict(op=op, dtype=dtype, batch=batch, q_len=q_len, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    prefix=prefix, suffix_min=rng.randint(0, suffix_max), suffix_max=suffix_max,
                    holes=rng.choice([0, rng.randint(0, prefix)]), spread_pages=rng.random() < 0.5)
    if op == "int8":
        k, n = 16 * _log(rng, 8, 1184), 16 * _log(rng, 4, 2368)
        rows = _log(rng, 1, 4096)
        while rows * k * n > 4096 * 3584 * 37888:
            rows = max(rows // 2, 1)
        return dict(op=op, source=rng.choice(["rows", "norm", "gate"]), dtype=dtype, rows=rows, k=k, n=n,
                    bias=rng.random() < 0.5)
    heads, kv_heads = rng.choice([(32, 32), (28, 4), (32, 8), (5, 1)])
    head_dim = rng.choice([128, 64])
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, 8000), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                rotary=rng.choice([head_dim, head_dim // 2, head_dim // 4]), interleaved=rng.random() < 0.5,
                theta=rng.choice([10000.0, 500000.0, 1000000.0]), stretch=rng.choice([1.0, 4.0, 8.0]),
                factor=rng.choice([1.0, 1.2]), far=_log(rng, 4096, 1000000), skip=rng.choice([0, 5]))


# ------------------------------------------------------------------------------------ inputs
def _dtype(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]


def _randn(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and state.get("keep") is not None:
        from acache_b200.model.acache_attention import pack_keep_mask
        state["keep_words"] = pack_keep_mask(state["keep"])   # a batch's holes stay the same over all layers of a step
    return state


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": _prepare_attention, "int8": _prepare_int8, "rope": _prepare_rope}[case["op"]](case, seed, gen)


def _prepare_attention(case, seed, gen):
    """The shared prefix in the cache's first slots, every request's own tokens in pages of its own; queries and
    keys of a size at which the softmax is neither flat nor a single key."""
    rng = np.random.default_rng(seed)
    batch, prefix, dt = case["batch"], case["prefix"], _dtype(case)
    q_lens = rng.integers((case["q_len"] + 1) // 2, case["q_len"] + 1, batch) if case["spread_pages"] else np.full(batch, case["q_len"])
    k_lens = rng.integers(case["suffix_min"], case["suffix_max"] + 1, batch)
    n_prefix_pages = -(-prefix // PAGE)
    pages = -(-k_lens // PAGE)
    order = n_prefix_pages + rng.permutation(int(pages.sum()))       # a request's pages lie anywhere
    slots, at = [], 0
    for n, p in zip(k_lens, pages):
        own_pages = order[at:at + p]
        at += p
        slots.append((own_pages[:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:n])
    prefix_slots = np.arange(prefix)
    if case["spread_pages"]:
        prefix_slots = (rng.permutation(n_prefix_pages)[:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:prefix]
    n_pages = n_prefix_pages + int(pages.sum())
    shape = (max(n_pages, 1), PAGE, case["kv_heads"], case["head_dim"])

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()

    keep = None
    if case["holes"]:
        keep = torch.ones(batch, prefix, dtype=torch.bool)
        for b in range(batch):
            keep[b, torch.from_numpy(rng.permutation(prefix)[:case["holes"]])] = False
        keep = keep.cuda()
    return dict(
        case=case, q=_randn(gen, int(q_lens.sum()), case["heads"], case["head_dim"]).to(dt),
        k_cache=_randn(gen, *shape, scale=1.3).to(dt), v_cache=_randn(gen, *shape).to(dt), prefix_slots=dev(prefix_slots),
        cu_q=dev(np.concatenate([[0], np.cumsum(q_lens)])), cu_k=dev(np.concatenate([[0], np.cumsum(k_lens)])),
        slots=dev(np.concatenate(slots)), keep=keep, q_lens=q_lens.tolist(), k_lens=k_lens.tolist(),
        scale=case["head_dim"] ** -0.5, keep_words=None)


def _prepare_int8(case, seed, gen):
    """Activations with a few large channels, as language models have them; weights that were quantised before."""
    rows, k, n, dt = case["rows"], case["k"], case["n"], _dtype(case)
    channel = torch.exp(0.5 * _randn(gen, k))
    wq = torch.randint(-127, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
    state = dict(case=case, wq=wq, w_scale=(0.5 + torch.rand(n, generator=gen, device="cuda")) * (0.04 / 127),
                 bias=_randn(gen, n).to(dt) if case["bias"] else None, eps=1e-5, norm_w=None)
    if case["source"] == "gate":
        state["x"] = torch.cat([_randn(gen, rows, k), _randn(gen, rows, k) * channel], dim=1).to(dt)
    else:
        state["x"] = (_randn(gen, rows, k) * channel).to(dt)
    if case["source"] == "norm":
        state["norm_w"] = (1.0 + 0.2 * _randn(gen, k)).to(dt)
    return state


def _inv_freq(case):
    return case["theta"] ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"]) / case["stretch"]


def _prepare_rope(case, seed, gen):
    rows, d, dt = case["rows"], case["head_dim"], _dtype(case)
    pages = -(-rows // PAGE) + 2
    perm = torch.randperm(pages, generator=gen, device="cuda")
    slots = (perm[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:rows].to(torch.int32)
    if case["skip"]:
        slots[::case["skip"]] = -1
    start = torch.randint(0, max(case["far"] - rows, 1), (1,), generator=gen, device="cuda")
    qkv = _randn(gen, rows, (case["heads"] + 2 * case["kv_heads"]) * d).to(dt)       # one projection's output
    nq, nk = case["heads"] * d, case["kv_heads"] * d
    cache = (pages, PAGE, case["kv_heads"], d)
    return dict(case=case, q=qkv[:, :nq].unflatten(1, (-1, d)), k=qkv[:, nq:nq + nk].unflatten(1, (-1, d)),
                v=qkv[:, nq + nk:].unflatten(1, (-1, d)), positions=start + torch.arange(rows, device="cuda"), slots=slots,
                inv_freq=_inv_freq(case).cuda(), k_cache=_randn(gen, *cache).to(dt), v_cache=_randn(gen, *cache).to(dt))


# -------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "int8": _own_int8, "rope": _own_rope}[op](state)
    return {"attention": _plain_attention, "int8": _plain_int8, "rope": _plain_rope}[op](state)


def _own_attention(s):
    from acache_b200.model.acache_attention import shared_prefix_attention
    return shared_prefix_attention(
        s["q"], s["k_cache"], s["v_cache"], s["prefix_slots"], s["cu_q"], s["cu_k"], s["slots"], s["scale"],
        prefix_keep=s["keep_words"] if s["keep_words"] is not None else s["keep"],
        max_seqlen_q=max(s["q_lens"]), max_seqlen_k=max(s["k_lens"]))


def _own_int8(s):
    from acache_b200 import ops
    if s["case"]["source"] == "rows":
        xq, xs = ops.quantize_rows(s["x"])
    elif s["case"]["source"] == "norm":
        xq, xs = ops.rmsnorm_int8(s["x"], s["norm_w"], s["eps"])
    else:
        xq, xs = ops.act_mul_halves_int8(s["x"], "silu")
    return ops.linear_int8(xq, xs, s["wq"], s["w_scale"], s["bias"], out_dtype=s["x"].dtype)


def _own_rope(s):
    from acache_b200 import ops
    c = s["case"]
    q = ops.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"], s["slots"],
                        interleaved=c["interleaved"], attention_factor=c["factor"])
    return q, s["k_cache"], s["v_cache"]


def _plain_attention(s):
    c = s["case"]
    hkv, d = c["kv_heads"], c["head_dim"]
    group = c["heads"] // hkv
    k_rows, v_rows = s["k_cache"].view(-1, hkv, d), s["v_cache"].view(-1, hkv, d)
    prefix = s["prefix_slots"].long()
    kp, vp = k_rows[prefix].float(), v_rows[prefix].float()
    out = torch.zeros_like(s["q"])
    q0 = k0 = 0
    for b, (nq, nk) in enumerate(zip(s["q_lens"], s["k_lens"])):
        mine = s["slots"][k0:k0 + nk].long()
        k = torch.cat([kp, k_rows[mine].float()]).permute(1, 2, 0)                    # [hkv, d, keys]
        v = torch.cat([vp, v_rows[mine].float()]).transpose(0, 1)                     # [hkv, keys, d]
        q = s["q"][q0:q0 + nq].float().view(nq, hkv, group * d).transpose(0, 1).reshape(hkv, nq * group, d)
        w = (q @ k) * s["scale"]
        if s["keep"] is not None:
            w[:, :, :prefix.numel()].masked_fill_(~s["keep"][b], float("-inf"))
        top = w.amax(-1, keepdim=True) if w.shape[-1] else w.new_zeros(*w.shape[:-1], 1)
        w = torch.exp(w - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = w.sum(-1, keepdim=True)
        o = torch.where(total > 0, (w @ v) / total, torch.zeros((), device=w.device))
        out[q0:q0 + nq] = o.view(hkv, nq, group, d).transpose(0, 1).reshape(nq, hkv * group, d).to(out.dtype)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _plain_int8(s):
    source, x = s["case"]["source"], s["x"].float()
    if source == "norm":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * s["norm_w"].float()
    elif source == "gate":
        gate, up = x.chunk(2, dim=1)
        x = gate / (1 + torch.exp(-gate)) * up
    top = x.abs().amax(-1, keepdim=True)
    xq = torch.where(top > 0, torch.round(x * 127 / top), torch.zeros_like(x))
    out = (xq @ s["wq"].float().t()) * (top / 127) * s["w_scale"]
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(s["x"].dtype)


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]           # far positions lose their angle in 32 bits
    cos = (torch.cos(angle) * c["factor"]).float()[:, None]
    sin = (torch.sin(angle) * c["factor"]).float()[:, None]

    def rotate(x):
        r, rest = x[..., :c["rotary"]].float(), x[..., c["rotary"]:].float()
        a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else r.chunk(2, dim=-1)
        lo, hi = a * cos - b * sin, b * cos + a * sin
        r = torch.stack([lo, hi], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([lo, hi], dim=-1)
        return torch.cat([r, rest], dim=-1).to(x.dtype)

    live = (s["slots"] >= 0).nonzero().squeeze(1)
    at = s["slots"][live].long()
    s["k_cache"].view(-1, c["kv_heads"], c["head_dim"])[at] = rotate(s["k"])[live]
    s["v_cache"].view(-1, c["kv_heads"], c["head_dim"])[at] = s["v"][live]
    return rotate(s["q"]), s["k_cache"], s["v_cache"]


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    return {"attention": _exact_attention, "int8": _exact_int8, "rope": _exact_rope}[case["op"]](case, s)


def _exact_attention(case, s):
    """softmax over the kept prefix keys and the request's own keys, one KV head at a time."""
    hkv, d = case["kv_heads"], case["head_dim"]
    group = case["heads"] // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for h in range(hkv):
        keys, values = s["k_cache"][:, :, h].reshape(-1, d), s["v_cache"][:, :, h].reshape(-1, d)
        for b in range(case["batch"]):
            names = s["prefix_slots"] if s["keep"] is None else s["prefix_slots"][s["keep"][b]]
            names = torch.cat([names, s["slots"][cu_k[b]:cu_k[b + 1]]]).long()
            if names.numel() == 0 or cu_q[b] == cu_q[b + 1]:
                continue
            q = s["q"][cu_q[b]:cu_q[b + 1], h * group:(h + 1) * group].double()
            score = torch.einsum("qgd,kd->qgk", q, keys[names].double()) * s["scale"]
            weight = torch.exp(score - torch.logsumexp(score, dim=-1, keepdim=True))
            out[cu_q[b]:cu_q[b + 1], h * group:(h + 1) * group] = torch.einsum("qgk,kd->qgd", weight, values[names].double())
    return out


def _exact_int8(case, s):
    """The quantised row is round(127 x / max|x|), ties to even; its scale is max|x| / 127."""
    k = case["k"]
    out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
    w = s["wq"].double().t().contiguous()
    for at in range(0, case["rows"], 1024):
        x = s["x"][at:at + 1024].double()
        if case["source"] == "norm":
            x = x / torch.sqrt(x.square().sum(1, keepdim=True) / k + s["eps"]) * s["norm_w"].double()
        if case["source"] == "gate":
            x = x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:]
        top = x.abs().max(dim=1, keepdim=True).values
        part = torch.round(127 * x / top.clamp_min(1e-300)) @ w * (top / 127)
        part *= s["w_scale"].double()
        out[at:at + 1024] = part if s["bias"] is None else part + s["bias"].double()
    return out


def _exact_rope(case, s):
    """Pair (x_i, x_j) is the complex number x_i + i x_j, turned by position x frequency."""
    half = case["rotary"] // 2
    idx = torch.arange(half, device="cuda")
    first, second = (2 * idx, 2 * idx + 1) if case["interleaved"] else (idx, idx + half)
    turn = torch.polar(torch.full((case["rows"], half), float(case["factor"]), dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * s["inv_freq"][None])

    def rotate(x):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    k_cache, v_cache = s["k_cache"].double().flatten(0, 1), s["v_cache"].double().flatten(0, 1)
    live = s["slots"] >= 0
    k_cache[s["slots"][live].long()] = rotate(s["k"])[live]
    v_cache[s["slots"][live].long()] = s["v"][live].double()
    return rotate(s["q"]), k_cache.view(s["k_cache"].shape), v_cache.view(s["v_cache"].shape)


# ------------------------------------------------------------------------------------- work
def work(case):
    """What one pass has to read, write and compute (suffixes at their mean length)."""
    if case["op"] == "attention":
        hkv, d, batch = case["kv_heads"], case["head_dim"], case["batch"]
        q_len = case["q_len"] if not case["spread_pages"] else (case["q_len"] + (case["q_len"] + 1) // 2) / 2
        suffix = (case["suffix_min"] + case["suffix_max"]) / 2
        rows = batch * q_len
        nbytes = 4 * (case["prefix"] + batch * suffix) * hkv * d + 4 * rows * case["heads"] * d + 4 * (case["prefix"] + batch * suffix)
        nbytes += batch * case["prefix"] / 8 if case["holes"] else 0
        return {"bytes": int(nbytes), "flops": int(4 * rows * (case["prefix"] - case["holes"] + suffix) * case["heads"] * d)}
    if case["op"] == "int8":
        rows, k, n = case["rows"], case["k"], case["n"]
        source = 2 if case["source"] == "gate" else 1
        return {"bytes": 2 * rows * k * source + n * k + 4 * n + 2 * rows * n + (2 * k if case["source"] == "norm" else 0),
                "flops": 2 * rows * k * n}
    rows, h, hkv, d = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
    live = 1 - (1 / case["skip"] if case["skip"] else 0)
    return {"bytes": int(rows * (4 * h * d + 8 * hkv * d * live + 12)),
            "flops": int(3 * rows * (h + hkv * live) * case["rotary"])}
