"""Pieces shared by the two served architectures: RoPE tables, the fused
projection + RoPE + K/V scatter step, and the block-level kernels."""
from __future__ import annotations

import torch
from torch import nn

from .. import ops


def build_rope_table(length: int, head_dim: int, theta: float, dtype: torch.dtype, device,
                     scaling: dict | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(cos, sin)`` tables ``[length, head_dim]`` in the half-split layout
    ``cat(freqs, freqs)`` (reference: nano-vdllm/model/modeling_llada.py:392-402).
    Built once on the host in fp32 so that every device holds identical bits.  With ``scaling`` (a
    model's ``rope_scaling``, see ``ops.rope_frequencies``; "default" is none) the angles are formed in 64 bits from the
    stretched frequencies; an attention factor is not in the tables (``rope_score_factor``), so that
    they stay pure rotations and cached keys can be relocated by further ones."""
    if stretches(scaling):
        inv_freq, _ = model_rope_frequencies(head_dim, theta, scaling)
        freqs = torch.outer(torch.arange(length, dtype=torch.float64), inv_freq)
        emb = torch.cat((freqs, freqs), dim=-1)
        return emb.cos().to(dtype).to(device), emb.sin().to(dtype).to(device)
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim))
    freqs = torch.outer(torch.arange(length, dtype=torch.float32), inv_freq)
    emb = torch.cat((freqs, freqs), dim=-1)
    return emb.cos().to(dtype).to(device), emb.sin().to(dtype).to(device)


def stretches(scaling: dict | None) -> bool:
    """Whether a configuration's ``rope_scaling`` asks for other frequencies than the plain ones: configuration objects
    of the transformers package answer ``{"rope_type": "default", ...}`` where none was given."""
    return scaling is not None and scaling.get("rope_type", scaling.get("type", "default")) != "default"


def model_rope_frequencies(head_dim: int, theta: float, scaling: dict):
    """``ops.rope_frequencies`` of a served model: its tables hold for every length, so a scaling that
    depends on the current one is refused."""
    if scaling.get("rope_type", scaling.get("type")) == "dynamic":
        raise ValueError("rope_type 'dynamic' changes the frequencies with the sequence length: cached keys would not fit")
    return ops.rope_frequencies(head_dim, theta, scaling)


def rope_score_factor(head_dim: int, theta: float, scaling: dict | None) -> float:
    """What a scaling's attention factor (on sine and cosine of queries and keys alike) does to the scores."""
    return model_rope_frequencies(head_dim, theta, scaling)[1] ** 2 if stretches(scaling) else 1.0


# Which projections of the model blocks run on this package's CTA-pair tcgen05 GEMMs
# (``ops.linear*``) instead of the library GEMM, for 16-bit models whose shapes the kernels take:
#   OWN_QKV      q/k/v projection with bias, RoPE and the cache scatter in its epilogue
#   OWN_GATE_UP  gate and up projections as one GEMM with the gated activation in its epilogue
#   OWN_DENSE    the plain projections (attention output, feed-forward output): "sliced" = where
#                the K range is cut into slices (few rows: block decode), True = always
#   OWN_HEAD     the output head; for greedy unmasking it returns arg-max and confidence and
#                never writes the logits
# Without a TMA multicast of operand tiles every SM pulls its own tiles from L2, which bounds a
# CTA-pair GEMM at 55-70 GB/s of operand bytes per SM: 0.82-0.93 of the library GEMM at these
# shapes.  With the work fused into their epilogues the QKV, gate/up and output-head projections
# come out level with or ahead of the library GEMM plus the separate kernels, so they are on.  The
# two plain projections have 4096 output columns: at block-decode row counts that is 16-32 whole
# tiles for 74 CTA pairs, so there the K range can be cut into slices that run as tiles of their
# own, and the normalisation kernel that follows adds the fp32 slices (``dense_pending``).  A
# sliced launch costs 6-9 us more than the library GEMM whatever K, so the launch plan
# (``ops.linear_partials_splits``) only slices long K ranges: the feed-forward output projection
# (K = 12288: 46 against 41 us) runs here, the attention output projection (K = 4096: 22 against
# 15 us) stays with the library.
OWN_QKV = True
OWN_GATE_UP = True
OWN_DENSE = "sliced"
OWN_HEAD = True

# The older single-CTA form of the fused QKV projection (128 x 128 tiles); kept for comparison,
# slower than both the CTA-pair kernel and the library GEMM + RoPE/scatter kernel.
FUSED_QKV = False


def set_own_gemm(on: bool):
    """Switches every projection to this package's kernels (True) or to the library GEMM (False)."""
    global OWN_QKV, OWN_GATE_UP, OWN_DENSE, OWN_HEAD
    OWN_QKV = OWN_GATE_UP = OWN_DENSE = OWN_HEAD = bool(on)


def dense(x, weight, bias=None):
    """An ``nn.Linear`` of the model blocks on 2-D activations."""
    if OWN_DENSE is True and ops._gemm_ok(x, weight):
        return ops.linear(x, weight, bias)
    return torch.nn.functional.linear(x, weight, bias)


def dense_pending(x, weight, bias=None):
    """A projection whose output is only ever added to the residual stream by the next
    ``RMSNorm.forward(x, delta)``: returns either the output itself or, where slicing the K range
    pays (``ops.linear_partials_splits``), its float32 slices ``[n_splits, n, out]``."""
    if OWN_DENSE and bias is None and ops._gemm_ok(x, weight):
        if ops.linear_partials_splits(x.shape[0], x.shape[1], weight.shape[0]) > 1:
            return ops.linear_partials(x, weight)
        if OWN_DENSE is True:
            return ops.linear(x, weight)
        return torch.nn.functional.linear(x, weight)
    if OWN_DENSE is True and ops._gemm_ok(x, weight):
        return ops.linear(x, weight, bias)
    return torch.nn.functional.linear(x, weight, bias)


def select_pending(delta, rows):
    """``delta`` restricted to the given rows, for either form ``dense_pending`` returns."""
    if delta is None:
        return None
    return delta.index_select(1 if delta.dim() == 3 else 0, rows)


class FusedProjections:
    """Weights of one block in the layouts the fused projection kernels read: q/k/v rows
    interleaved inside every head (``ops.interleave_heads``), gate and up rows interleaved with
    each other (``ops.interleave_rows``).  These are copies (the parameters keep their natural
    layout for state dicts), made on first use by the kernel that needs them; ``stale()`` tells
    when the parameters were replaced since."""

    def __init__(self):
        self.qkv_w = self.qkv_b = self.gate_up_w = None
        self._stamp = None

    @staticmethod
    def _stamp_of(params):
        return tuple((p.data_ptr(), p._version) for p in params if p is not None)

    def stale(self, params):
        return self._stamp != self._stamp_of(params)

    def reset(self, params):
        self.qkv_w = self.qkv_b = self.gate_up_w = None
        self._stamp = self._stamp_of(params)

    def qkv(self, w_qkv, b_qkv, head_dim):
        if self.qkv_w is None and head_dim == 128 and w_qkv.is_cuda and w_qkv.dtype in (torch.bfloat16, torch.float16):
            self.qkv_w = ops.interleave_heads(w_qkv)
            self.qkv_b = ops.interleave_heads(b_qkv) if b_qkv is not None else None
        return self.qkv_w, self.qkv_b

    def gate_up(self, gate, up):
        if (self.gate_up_w is None and gate.shape[0] % 8 == 0 and gate.is_cuda
                and gate.dtype in (torch.bfloat16, torch.float16)):
            self.gate_up_w = ops.interleave_rows(gate, up)
        return self.gate_up_w


class Int8Projections:
    """The projections of one block in 8-bit integers (``ops.linear_int8``): copies of the weights quantised per
    output channel when the object is made; the activations are quantised per token by the kernel that produces them
    (norm, gated activation, or ``ops.quantize_rows`` after attention).  A projection whose parameters were replaced or
    written in place since is quantised again at its next call, into the same buffers, so that captured graphs read the new
    values too.  A write through ``.data`` leaves no trace on a parameter: call ``refresh()`` (a model's ``quantize_int8()``)
    after it."""

    def __init__(self, **projections):
        self.projections = projections              # name -> the nn.Linear modules whose outputs lie side by side
        for name, mods in projections.items():
            w = mods[0].weight
            if w.dtype not in (torch.bfloat16, torch.float16) or not w.is_cuda:
                raise ValueError(f"8-bit projections need a 16-bit model on the GPU, not {w.dtype} on {w.device}")
            if w.shape[1] % 16 or sum(m.weight.shape[0] for m in mods) % 16:
                raise ValueError(f"{name}: the sizes of an 8-bit projection are multiples of 16")
        self._made, self._stamps = {}, {}
        self.refresh()

    def _stamp_of(self, name):
        return FusedProjections._stamp_of([p for m in self.projections[name] for p in (m.weight, m.bias)])

    def refresh(self):
        """Quantises every projection's present parameters."""
        for name in self.projections:
            self._make(name)

    # buffers that can be written again outside of inference mode, whatever mode the first call ran in
    @torch.inference_mode(False)
    @torch.no_grad()
    def _make(self, name):
        mods = self.projections[name]
        w = mods[0].weight
        rows, cols = sum(m.weight.shape[0] for m in mods), w.shape[1]
        q, scale, bias = self._made.get(name, (None, None, None))
        if q is None or q.device != w.device:
            q = torch.empty(rows, cols, dtype=torch.int8, device=w.device)
            scale = torch.empty(rows, dtype=torch.float32, device=w.device)
            bias = torch.empty(rows, dtype=w.dtype, device=w.device) if mods[0].bias is not None else None
            self._made[name] = (q, scale, bias)
        at = 0
        for m in mods:
            part = slice(at, at + m.weight.shape[0])
            at = part.stop
            q_part, scale_part = ops.quantize_rows(m.weight.data)
            q[part].copy_(q_part)
            scale[part].copy_(scale_part)
            if bias is not None:
                bias[part].copy_(m.bias.data)
        self._stamps[name] = self._stamp_of(name)

    def _weights(self):
        for name in self.projections:
            if self._stamps[name] != self._stamp_of(name):
                self._make(name)
        return self._made

    def __call__(self, name, quantised, dtype):
        if self._stamps[name] != self._stamp_of(name):
            self._make(name)
        w, scale, bias = self._made[name]
        return ops.linear_int8(quantised[0], quantised[1], w, scale, bias, out_dtype=dtype)


def concat_gate_up(gate_proj, up_proj):
    """One buffer ``[2F, in]`` holding the gate rows then the up rows; the two parameters become
    views of it (state-dict names and values unchanged), so one library GEMM computes both."""
    w = torch.cat([gate_proj.weight.data, up_proj.weight.data], dim=0)
    f = gate_proj.out_features
    gate_proj.weight.data, up_proj.weight.data = w[:f], w[f:]
    return w


def gated_mlp_input(h, fused: FusedProjections, gate_proj, up_proj, act: str, gate_up_cat=None):
    """``act(gate_proj(h)) * up_proj(h)``: one GEMM of this package with the activation in its
    epilogue (``OWN_GATE_UP``), else one library GEMM over the concatenated weights followed by the
    activation kernel on its two halves, else two projections and the activation kernel."""
    if OWN_GATE_UP and gate_proj.bias is None and h.dtype in (torch.bfloat16, torch.float16) and h.is_cuda:
        w = fused.gate_up(gate_proj.weight.data, up_proj.weight.data)
        if w is not None and ops._gemm_ok(h, w):
            return ops.linear_swiglu(h, w, act)
    if (gate_up_cat is not None and gate_proj.bias is None
            and gate_up_cat.data_ptr() == gate_proj.weight.data_ptr() and h.shape[1] % 8 == 0):
        return ops.act_mul_halves(dense(h, gate_up_cat), act)
    return ops.act_mul(dense(h, gate_proj.weight, gate_proj.bias), dense(h, up_proj.weight, up_proj.bias), act)


def project_qkv(h, w_qkv, b_qkv, n_heads, n_kv_heads, head_dim, position_ids, cos, sin, attn, ctx, fused=None):
    """Returns ``(q, k, v)`` views for the attention call; with the fused path ``k``/``v`` are
    ``None`` because they only exist in the paged cache."""
    n = h.shape[0]
    D, nh, hkv = head_dim, n_heads, n_kv_heads
    caching = attn.k_cache.numel() > 0 and ctx.slot_mapping is not None
    if OWN_QKV and caching and fused is not None and cos.stride(0) * cos.element_size() % 16 == 0:
        wi, bi = fused.qkv(w_qkv, b_qkv, D)
        if wi is not None and ops._gemm_ok(h, wi):
            q = ops.linear_qkv_rope_scatter(h, wi, bi, nh, hkv, D, position_ids, cos, sin, attn.k_cache, attn.v_cache,
                                            ctx.slot_mapping)
            attn.kv_already_stored = True
            return q, None, None
    if (FUSED_QKV and caching and D == 128 and h.dtype in (torch.bfloat16, torch.float16) and h.shape[1] % 64 == 0
            and h.stride(0) % 8 == 0):
        q = ops.qkv_rope_scatter(h, w_qkv, b_qkv, nh, hkv, D, position_ids, cos, sin, attn.k_cache, attn.v_cache,
                                 ctx.slot_mapping)
        attn.kv_already_stored = True
        return q, None, None
    return rotate_and_store(dense(h, w_qkv, b_qkv), n_heads, n_kv_heads, head_dim, position_ids, cos, sin, attn, ctx)


def rotate_and_store(qkv, n_heads, n_kv_heads, head_dim, position_ids, cos, sin, attn, ctx):
    """Splits a q/k/v projection's output, rotates q and k in place and, in a caching step, scatters k and v."""
    n, D, nh, hkv = qkv.shape[0], head_dim, n_heads, n_kv_heads
    caching = attn.k_cache.numel() > 0 and ctx.slot_mapping is not None
    q, k, v = qkv[:, : nh * D], qkv[:, nh * D: (nh + hkv) * D], qkv[:, (nh + hkv) * D:]
    q, k, v = q.view(n, nh, D), k.view(n, hkv, D), v.view(n, hkv, D)
    if caching:
        ops.rope_store(q, k, v, position_ids, cos, sin, attn.k_cache, attn.v_cache, ctx.slot_mapping)
        attn.kv_already_stored = True
    else:
        ops.rope_store(q, k, None, position_ids, cos, sin)
        attn.kv_already_stored = False
    return q, k, v


class RopeCache:
    """Grows on demand (reference: nano-vdllm/model/modeling_llada.py:373-402)."""

    def __init__(self, head_dim: int, theta: float, table_dtype: torch.dtype, scaling: dict | None = None):
        self.head_dim, self.theta, self.table_dtype, self.scaling = head_dim, theta, table_dtype, scaling
        self.cos = self.sin = None

    def get(self, length: int, device):
        if self.cos is None or self.cos.shape[0] < length or self.cos.device != torch.device(device):
            n = max(int(length), 1)
            n = 1 << (n - 1).bit_length()  # power of two: few rebuilds
            self.cos, self.sin = build_rope_table(n, self.head_dim, self.theta, self.table_dtype, device, self.scaling)
        return self.cos, self.sin


class RMSNorm(nn.Module):
    def __init__(self, size: int, eps: float, device=None, dtype=None):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(size, device=device, dtype=dtype))
        self.eps = eps

    def forward(self, x, delta=None):
        """``delta`` (optional): a residual update that is added to ``x`` IN PLACE before the
        normalisation (one fused kernel); either form that ``dense_pending`` returns."""
        if delta is None:
            return ops.rmsnorm(x, self.weight, self.eps)
        if x.shape[-1] % (16 // x.element_size()) != 0 or x.shape[-1] > 1024 * (16 // x.element_size()):
            if delta.dim() == 3:    # float32 slices of the projection (``dense_pending``)
                delta = delta.sum(0).to(x.dtype)
            x.add_(delta)  # row shapes the fused kernel does not take
            return ops.rmsnorm(x, self.weight, self.eps)
        return ops.add_rmsnorm(x, delta, self.weight, self.eps)
