"""The operators of a block-decode step over a shared affix used together: one layer stage by stage against 64
bits, and the engine with its switches for them."""
import itertools
import random

import pytest
import torch

from test_engine_gpu import _dream, _llada, _random_requests, _serve_config

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _quantise64(y):
    top = y.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * y / top), torch.zeros_like(y)), top / 127


def test_one_layer_stage_by_stage():
    """norm -> 8-bit q/k/v -> rotate (long-context frequencies) and append -> attention over the shared affix and the own
    keys -> 8-bit output projection, captured in a graph and replayed; the 64-bit form of every stage starts from what
    the stage before it left."""
    from acache_b200 import _lib, ops
    from acache_b200.model.acache_attention import pack_keep_mask, shared_prefix_attention

    g = torch.Generator().manual_seed(3)
    nh, hkv, D, hid, A, T = 8, 2, 128, 1024, 300, 9
    own = [40, 0, 131]                                # earlier keys of every request
    n, page = 3 * T, 256
    x = torch.randn(n, hid, generator=g).to(BF).to(DEV)
    norm_w = (1 + 0.1 * torch.randn(hid, generator=g)).to(BF).to(DEV)
    wq, ws = ops.quantize_rows((torch.randn((nh + 2 * hkv) * D, hid, generator=g) * hid ** -0.5).to(BF).to(DEV))
    oq, osc = ops.quantize_rows((torch.randn(hid, nh * D, generator=g) * (nh * D) ** -0.5).to(BF).to(DEV))
    kc, vc = (torch.randn(8, page, hkv, D, generator=g).to(BF).to(DEV) for _ in range(2))
    inv, factor = ops.rope_frequencies(D, 500000.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096))
    inv = inv.to(DEV)
    free = torch.arange(A, 8 * page)[torch.randperm(8 * page - A, generator=g)].to(torch.int32)
    slots, at, new = [], 0, []
    for k in own:
        s = free[at:at + k + T]
        at += k + T
        slots.append(s)
        new.append(s[k:])
    cu_q = torch.arange(0, n + 1, T, dtype=torch.int32, device=DEV)
    cu_k = torch.tensor([0, *itertools.accumulate(len(s) for s in slots)], dtype=torch.int32, device=DEV)
    read, write = torch.cat(slots).to(DEV), torch.cat(new).to(DEV)
    keep = torch.rand(3, A, generator=g) > 0.2
    words, prefix = pack_keep_mask(keep.to(DEV)), torch.arange(A, dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(30000 + 7 * i, 30000 + 7 * i + T) for i in range(3)]).to(DEV)

    def layer():
        h = ops.rmsnorm_int8(x, norm_w, 1e-5)
        qkv = ops.linear_int8(*h, wq, ws)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([nh * D, hkv * D, hkv * D], dim=1))
        qr = ops.rope_append(q, k, v, pos, inv, kc, vc, write, attention_factor=factor)
        att = shared_prefix_attention(qr, kc, vc, prefix, cu_q, cu_k, read, prefix_keep=words, max_seqlen_q=T, max_seqlen_k=max(own) + T)
        a = ops.quantize_rows(att.reshape(n, -1))
        return h, qkv, qr, att, a, ops.linear_int8(*a, oq, osc)

    eager = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    kc.view(-1, hkv, D)[write.long()] = 0
    vc.view(-1, hkv, D)[write.long()] = 0
    graph.replay()
    torch.cuda.synchronize()
    _lib.check_device_errors()
    flat = lambda t: [v for u in t for v in (u if isinstance(u, tuple) else (u,))]
    for e, r in zip(flat(eager), flat(out)):
        assert torch.equal(e, r)
    (hq, hs), qkv, qr, att, (aq, as_), y = out
    eps = torch.finfo(BF).eps      # 2^-7: a rounding to bf16 (8 significant bits) is off by at most eps / 2 of the value
    y64 = x.double()
    y64 = y64 * torch.rsqrt(y64.square().mean(1, keepdim=True) + 1e-5) * norm_w.double()
    want, scale = _quantise64(y64)
    assert ((hq.double() - want).abs() <= 1).all() and (hq.double() != want).double().mean() < 1e-3     # near ties only
    ref = (hq.double() @ wq.double().T) * hs.double()[:, None] * ws.double()
    assert ((qkv.double() - ref).abs() <= ref.abs() * (eps / 2 + 2.0 ** -21)).all()
    angle = pos.double()[:, None] * inv
    c, s = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]

    def rotate(t):
        a, b = t.double().unflatten(1, (-1, D)).chunk(2, dim=-1)
        return torch.cat([a * c - b * s, b * c + a * s], dim=-1)

    def close(got, want, size):
        assert ((got.double() - want).abs() <= want.abs() * eps / 2 + size * 2.0 ** -20).all()

    close(qr, rotate(qkv[:, :nh * D]), qkv.double().abs().max() * factor)
    close(kc.view(-1, hkv, D)[write.long()], rotate(qkv[:, nh * D:(nh + hkv) * D]), qkv.double().abs().max() * factor)
    assert torch.equal(vc.view(-1, hkv, D)[write.long()], qkv[:, (nh + hkv) * D:].unflatten(1, (-1, D)))
    K, V = kc.double().view(-1, hkv, D), vc.double().view(-1, hkv, D)
    for b in range(3):
        names = torch.cat([prefix[keep[b].to(DEV)], read[cu_k[b]:cu_k[b + 1]]]).long()
        for h in range(nh):
            w = torch.softmax((qr[b * T:(b + 1) * T, h].double() @ K[names, h * hkv // nh].T) * D ** -0.5, -1)
            o, size = w @ V[names, h * hkv // nh], w @ V[names, h * hkv // nh].abs()
            # weights rounded to bf16, fp32 scores and sums, one rounding of the result
            assert ((att[b * T:(b + 1) * T, h].double() - o).abs() <= o.abs() * eps / 2 + size * (eps / 2 + 2.0 ** -15)).all()
    want, scale = _quantise64(att.double().reshape(n, -1))
    assert torch.equal(aq.double(), want)
    ref = (aq.double() @ oq.double().T) * as_.double()[:, None] * osc.double()
    assert ((y.double() - ref).abs() <= ref.abs() * (eps / 2 + 2.0 ** -21)).all()


def _arch(kind, **kw):
    from oracle.models import ArchSpec

    base = dict(n_layers=2, d_model=256, n_heads=4, n_kv_heads=4 if kind == "llada" else 2, ffn=192, vocab=180, rope_theta=10000.0,
                rms_eps=1e-5 if kind == "llada" else 1e-6, act="silu", mask_id=179)
    base.update(kw)
    return ArchSpec(kind, **base)


def _serve(model, hf_cfg, arch, kind, reqs, G, T, **switches):
    from acache_b200 import _lib
    from acache_b200.model_runner import ModelRunner
    from acache_b200.sequence import Sequence

    cfg = _serve_config(hf_cfg, arch, kind, BF, threshold=0.6, anchor_ratio=0.2, max_num_seqs=4, num_kvcache_blocks=40,
                        cache_block_size=64, block_length=T, gen_length=G, **switches)
    runner = ModelRunner(model, cfg)
    seqs = [Sequence(r["prompt"], block_length=T, gen_length=G, cache_block_size=64, mask_id=arch.mask_id,
                     prompt_affix_start=r["affix_start"], prompt_affix_end=r["affix_end"],
                     generation_start=r["generation_start"]) for r in reqs]
    outs, _ = runner.generate_with_acache(seqs)
    _lib.check_device_errors()
    return outs


@pytest.mark.parametrize("kind", ["llada", "dream"])
def test_engine_multiplies_the_shared_span_once(kind):
    """``share_span_once``: the tokens of the per-request layout, up to choices that a rounding decides (the two orders of
    the sums differ by bf16 roundings; the models' greedy choices agree in 80 % as in the engine's other layouts),
    replayed from graphs exactly as run eagerly, and the operator really runs."""
    from acache_b200.model import acache_attention as aa
    from acache_b200.model import attention as at
    from oracle.models import random_state_dict

    arch = _arch(kind)
    weights = random_state_dict(arch, seed=11, std=0.2)
    A, G, T = 70, 16, 8
    rng = random.Random(4)
    affix = [rng.randint(1, 170) for _ in range(A)]
    reqs = _random_requests(rng, arch, 6, A, G, ["prefix"], affix)
    hf_cfg, model = (_llada if kind == "llada" else _dream)(arch, weights, BF)
    plain = _serve(model, hf_cfg, arch, kind, reqs, G, T, group_shared_span=False)
    calls = []

    def counted(*a, **k):
        calls.append(1)
        return aa.shared_prefix_attention(*a, **k)

    old, at.shared_prefix_attention = at.shared_prefix_attention, counted
    try:
        once = _serve(model, hf_cfg, arch, kind, reqs, G, T, share_span_once=True, use_cuda_graphs=False)
        assert calls
        graphs = _serve(model, hf_cfg, arch, kind, reqs, G, T, share_span_once=True, use_cuda_graphs=True)
    finally:
        at.shared_prefix_attention = old
    total = sum(len(o) for o in plain)
    same = sum(a == b for p, o in zip(plain, once) for a, b in zip(p, o))
    print(f"agreement: tokens {same}/{total}")
    assert same >= 0.8 * total
    assert [len(o) for o in graphs] == [len(o) for o in plain] and all(arch.mask_id not in o for o in graphs)
    # a graph is captured with room for longer reads than the step has, which may split the keys in other places
    assert sum(a == b for p, o in zip(once, graphs) for a, b in zip(p, o)) >= 0.8 * total


@pytest.mark.parametrize("kind", ["llada", "dream"])
def test_models_run_their_projections_in_8_bits(kind):
    """Logits of the 8-bit model against the 16-bit one: every quantised operand is off by at most half of 1/127 of its
    row's maximum (about 1 % of its size at random inputs), eight projections deep: some per cent of the logits' size,
    and not none.  Replaced parameters are quantised again; a 32-bit model is refused."""
    from oracle.models import random_state_dict

    arch = _arch(kind)
    weights = random_state_dict(arch, seed=5, std=0.05)
    make = _llada if kind == "llada" else _dream
    _, m16 = make(arch, weights, BF)
    _, m8 = make(arch, weights, BF)
    m8.quantize_int8()
    rng = random.Random(1)
    reqs = _random_requests(rng, arch, 3, 40, 8, ["prefix"], [rng.randint(1, 170) for _ in range(40)])
    hf_cfg = m16.config
    seen = {}

    def logits_of(model, name):
        from acache_b200.model_runner import ModelRunner
        from acache_b200.sequence import Sequence

        cfg = _serve_config(hf_cfg, arch, kind, BF, threshold=0.6, anchor_ratio=0.2, max_num_seqs=4, num_kvcache_blocks=40,
                            cache_block_size=64, block_length=8, gen_length=8)
        runner = ModelRunner(model, cfg)
        real = runner._forward_model

        def spy(*a, **k):
            k["greedy_stats"] = False
            out = real(*a, **k)
            if out.logits is not None:
                seen.setdefault(name, out.logits.float())
            return out

        runner._forward_model = spy
        seqs = [Sequence(r["prompt"], block_length=8, gen_length=8, cache_block_size=64, mask_id=arch.mask_id,
                         prompt_affix_start=r["affix_start"], prompt_affix_end=r["affix_end"],
                         generation_start=r["generation_start"]) for r in reqs]
        outs, _ = runner.generate_with_acache(seqs)
        assert all(arch.mask_id not in o for o in outs)

    logits_of(m16, "16")
    logits_of(m8, "8")
    rel = (seen["8"] - seen["16"]).norm() / seen["16"].norm()
    assert 1e-4 < rel < 0.15, rel
    blocks = m8.model.transformer["blocks"] if kind == "llada" else m8.model.layers
    before = blocks[0].int8._weights()["gate_up"][1].clone()
    p = (blocks[0].ff_proj if kind == "llada" else blocks[0].mlp.gate_proj).weight
    p.data = p.data * 2
    after = blocks[0].int8._weights()["gate_up"][1]
    assert torch.equal(after[: p.shape[0]], before[: p.shape[0]] * 2) and torch.equal(after[p.shape[0]:], before[p.shape[0]:])
    with pytest.raises(ValueError):
        make(arch, weights, torch.float32)[1].quantize_int8()


def test_engine_with_everything_on():
    """Long-context frequencies, 8-bit projections and the shared span multiplied once, through the engine's switches."""
    from oracle.models import random_state_dict

    arch = _arch("llada")
    weights = random_state_dict(arch, seed=21, std=0.2)
    A, G, T = 70, 16, 8
    rng = random.Random(9)
    affix = [rng.randint(1, 170) for _ in range(A)]
    reqs = _random_requests(rng, arch, 5, A, G, ["prefix", "infix"], affix)
    hf_cfg, model = _llada(arch, weights, BF)
    outs = _serve(model, hf_cfg, arch, "llada", reqs, G, T, share_span_once=True, int8_projections=True)
    assert all(len(o) for o in outs) and all(arch.mask_id not in o for o in outs)
    assert model.model.transformer["blocks"][0].int8 is not None


def test_rope_scaling_of_a_model_reaches_tables_and_scores():
    from acache_b200 import ops
    from acache_b200.model.configuration import LLaDAConfig
    from acache_b200.model.modeling_common import build_rope_table
    from acache_b200.model.modeling_llada import LLaDALlamaBlock, RopeCache

    scaling = dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096)
    cfg = LLaDAConfig(d_model=256, n_heads=2, n_kv_heads=2, n_layers=1, mlp_hidden_size=64, rope_scaling=scaling)
    block = LLaDALlamaBlock(0, cfg, RopeCache(128, cfg.rope_theta, torch.float32, scaling), device=DEV, dtype=BF)
    inv, factor = ops.rope_frequencies(128, cfg.rope_theta, scaling)
    assert abs(block.attn.scale - factor ** 2 * 128 ** -0.5) < 1e-12
    cos, sin = block.rotary_emb.get(5000, DEV)
    angle = torch.arange(cos.shape[0], dtype=torch.float64)[:, None] * inv
    torch.testing.assert_close(cos[:, :64].double().cpu(), angle.cos(), rtol=0, atol=2.0 ** -24)
    torch.testing.assert_close(sin[:, 64:].double().cpu(), angle.sin(), rtol=0, atol=2.0 ** -24)
    # without a scaling the tables are what they were
    a, b = build_rope_table(300, 128, 500000.0, torch.float32, "cpu"), RopeCache(128, 500000.0, torch.float32).get(300, "cpu")
    assert torch.equal(a[0], b[0][:300])
    with pytest.raises(ValueError):
        LLaDALlamaBlock(0, LLaDAConfig(d_model=256, n_heads=2, n_kv_heads=2, mlp_hidden_size=64,
                                       rope_scaling=dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=4096)),
                        None, device=DEV, dtype=BF)


@pytest.mark.parametrize("kind", ["llada", "dream"])
def test_8_bit_weights_are_made_at_start_and_again_when_asked(kind):
    """The copies exist when ``quantize_int8`` returns (an engine sizes its cache right after); the first forward makes
    none.  Weights written through ``.data`` are quantised by the next ``quantize_int8``, weights written in place by
    the next call, both into the buffers that captured graphs read."""
    from acache_b200 import ops
    from oracle.models import random_state_dict

    arch = _arch(kind, d_model=1024, n_heads=8, n_kv_heads=8 if kind == "llada" else 2, ffn=4096)
    _, model = (_llada if kind == "llada" else _dream)(arch, random_state_dict(arch, seed=5, std=0.05), BF)
    blocks = model.model.transformer["blocks"] if kind == "llada" else model.model.layers
    linears = [m for b in blocks for m in b.modules() if isinstance(m, torch.nn.Linear)]
    copies = sum(m.weight.numel() + 4 * m.weight.shape[0] for m in linears)
    assert copies > 16 << 20
    # bytes asked for: the allocator does not split a remainder below 1 MB off a block, which memory_allocated() counts
    held = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]
    base = held()
    model.quantize_int8()
    assert copies <= held() - base < 1.02 * copies + (1 << 20)

    # what the first use of a projection allocates: its result and scratch
    before = held()
    block = blocks[0]
    x = torch.randn(5, 1024, device=DEV).to(BF)
    block.int8("gate_up", ops.quantize_rows(x), BF)
    assert held() - before < copies / 16

    buffers = {n: t[0].data_ptr() for n, t in block.int8._made.items()}
    w = (block.ff_out if kind == "llada" else block.mlp.down_proj).weight
    name = "ff_out" if kind == "llada" else "down"
    h = ops.quantize_rows(torch.randn(5, 4096, device=DEV).to(BF))
    was = block.int8(name, h, BF)
    w.data.mul_(2.0)                                   # no trace on the parameter
    model.quantize_int8()
    assert torch.equal(block.int8(name, h, BF), was * 2)
    with torch.no_grad():
        w.mul_(0.5)
    with torch.inference_mode():
        assert torch.equal(block.int8(name, h, BF), was)
    w.data.mul_(2.0)
    model.quantize_int8()                              # outside of inference mode again
    assert torch.equal(block.int8(name, h, BF), was * 2)
    assert {n: t[0].data_ptr() for n, t in block.int8._made.items()} == buffers


@pytest.mark.parametrize("kind,A,G", [("llada", 300, 16), ("dream", 700, 24), ("llada", 70, 600)])
def test_the_shared_span_s_layout_and_plan_in_eager_steps_and_graphs(kind, A, G):
    """``share_span_once``, every decode step: the kept span keys and the own keys of a request are exactly the slots of its
    read map; the operator's result is the per-request operator's on those slots (both round weights and result to the
    type); the bound it plans for is that of the own keys, within 256, eager or captured; replayed tokens equal eager ones."""
    from acache_b200 import _lib
    from acache_b200.model import acache_attention as aa
    from acache_b200.model import attention as at
    from acache_b200.model_runner import ModelRunner
    from acache_b200.sequence import Sequence
    from acache_b200.utils import get_context
    from oracle.models import random_state_dict

    arch = _arch(kind)
    weights = random_state_dict(arch, seed=11, std=0.2)
    T = 8
    rng = random.Random(A)
    affix = [rng.randint(1, 170) for _ in range(A)]
    reqs = _random_requests(rng, arch, 6, A, G, ["prefix"], affix)
    hf_cfg, model = (_llada if kind == "llada" else _dream)(arch, weights, BF)
    eps, state, bounds = torch.finfo(BF).eps, {}, {False: set(), True: set()}

    def spied(q, kc, vc, prefix, cu_q, cu_k, read, scale, *, prefix_keep, max_seqlen_q, max_seqlen_k):
        out = aa.shared_prefix_attention(q, kc, vc, prefix, cu_q, cu_k, read, scale, prefix_keep=prefix_keep,
                                         max_seqlen_q=max_seqlen_q, max_seqlen_k=max_seqlen_k)
        bounds[state["graphs"]].add(max_seqlen_k)
        if not state["graphs"]:
            longest = max(state["lens"])
            assert longest <= max_seqlen_k < longest + 256
            cu = torch.tensor([0, *itertools.accumulate(len(m) for m in state["maps"])], dtype=torch.int32, device=DEV)
            slots = torch.tensor([x for m in state["maps"] for x in m], dtype=torch.int32, device=DEV)
            other = aa.acache_attention(q, kc, vc, cu_q, cu, slots, scale).double()
            size = aa.acache_attention(q, kc, vc.abs(), cu_q, cu, slots, scale).double() * (1 + eps)
            tol = 2 * (other.abs() * eps / 2 + size * (eps / 2 + 2.0 ** -15)) + other.abs() * eps ** 2
            assert ((out.double() - other).abs() <= tol).all()
            state["checked"] = state.get("checked", 0) + 1
        return out

    def serve(graphs):
        state["graphs"] = graphs
        cfg = _serve_config(hf_cfg, arch, kind, BF, threshold=0.6, anchor_ratio=0.2, max_num_seqs=4, num_kvcache_blocks=120,
                            cache_block_size=64, block_length=T, gen_length=G, share_span_once=True, use_cuda_graphs=graphs)
        runner = ModelRunner(model, cfg)
        real = runner.prepare_decoding_acache

        def prepare(seqs, active_indices=None, graphs=None):
            positions = real(seqs, active_indices, graphs=graphs)
            ctx, ps = get_context(), runner._pick(seqs, active_indices)
            if ctx.shared_prefix is not None:
                prefix, words = (t.cpu() for t in ctx.shared_prefix)
                bits = (words[:, :, None] >> torch.arange(32)) & 1
                keep = bits.flatten(1)[:, :prefix.numel()].bool()
                cu, read = ctx.cu_seqlens_k.tolist(), ctx.read_slot_mapping.cpu()
                state["maps"] = [[int(x) for x in s.read_slot_map] for s in ps]
                state["lens"] = [b - a for a, b in zip(cu, cu[1:])]
                for i, s in enumerate(ps):
                    assert len(state["maps"][i]) == len(s)
                    assert sorted(prefix[keep[i]].tolist() + read[cu[i]:cu[i + 1]].tolist()) == sorted(state["maps"][i])
            return positions

        runner.prepare_decoding_acache = prepare
        seqs = [Sequence(r["prompt"], block_length=T, gen_length=G, cache_block_size=64, mask_id=arch.mask_id,
                         prompt_affix_start=r["affix_start"], prompt_affix_end=r["affix_end"],
                         generation_start=r["generation_start"]) for r in reqs]
        outs, _ = runner.generate_with_acache(seqs)
        _lib.check_device_errors()
        return outs

    old, at.shared_prefix_attention = at.shared_prefix_attention, spied
    try:
        eager = serve(False)
        assert state["checked"] > 0
        replayed = serve(True)
    finally:
        at.shared_prefix_attention = old
    assert bounds[True] <= bounds[False] and bounds[True]
    assert replayed == eager


@pytest.mark.parametrize("kind,nh,hkv", [("llada", 4, 4), ("dream", 4, 2)])
@pytest.mark.parametrize("max_num_seqs", [1, 4])
@pytest.mark.parametrize("scaling", [dict(rope_type="linear", factor=4.0),
                                     dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=64)])
def test_engine_with_rope_scaling_equals_the_oracle(kind, nh, hkv, max_num_seqs, scaling, monkeypatch):
    """A model with stretched frequencies in fp32, affixes at the start, inside and at the end (cached keys are relocated, by
    query or into copies): greedy tokens and anchors of the CPU restatement with the same frequencies, whose queries carry
    the attention factor of queries and keys."""
    import functools

    import oracle.engine
    import oracle.models
    from acache_b200 import _lib, ops
    from acache_b200.model import configuration
    from acache_b200.model_runner import ModelRunner
    from acache_b200.sequence import Sequence
    from oracle.models import ArchSpec, OracleModel, random_state_dict
    from oracle.rope import apply_rope

    rng = random.Random(5)
    arch = ArchSpec(kind, n_layers=2, d_model=64, n_heads=nh, n_kv_heads=hkv, ffn=96, vocab=160, rope_theta=10000.0,
                    rms_eps=1e-5 if kind == "llada" else 1e-6, act="silu", mask_id=159)
    inv, factor = ops.rope_frequencies(16, 10000.0, scaling)

    def table(length, head_dim, theta, dtype=torch.float32):
        assert head_dim == 16 and theta == 10000.0
        angle = torch.arange(length, dtype=torch.float64)[:, None] * torch.cat([inv, inv])
        return angle.cos().to(dtype), angle.sin().to(dtype)

    def rope_qk(q, k, positions, theta):
        cos, sin = table(int(positions.max()) + 1, q.shape[-1], theta)
        return apply_rope(q, cos[positions], sin[positions]) * factor ** 2, apply_rope(k, cos[positions], sin[positions])

    monkeypatch.setattr(oracle.engine, "rope_table", table)
    monkeypatch.setattr(oracle.models, "llada_rope_qk", rope_qk)
    monkeypatch.setattr(oracle.models, "dream_rope_qk", rope_qk)
    for name in ("LLaDAConfig", "DreamConfig"):
        monkeypatch.setattr(configuration, name, functools.partial(getattr(configuration, name), rope_scaling=scaling))
    weights = random_state_dict(arch, seed=11, std=0.3)
    A, G, T = 13, 8, 4
    affix = [rng.randint(1, 150) for _ in range(A)]
    reqs = _random_requests(rng, arch, 6, A, G, ["infix", "prefix", "suffix"], affix)

    def expected():
        o_req = []
        for r in reqs:
            toks = list(r["prompt"]) + ([arch.mask_id] * G if r["generation_start"] is None else [])
            o_req.append(dict(tokens=toks, affix_start=r["affix_start"], affix_end=r["affix_end"],
                              generation_start=len(r["prompt"]) if r["generation_start"] is None else r["generation_start"],
                              gen_length=G))
        return oracle.engine.generate_with_acache(OracleModel(arch, weights, torch.float32), o_req, anchor_ratio=0.3,
                                                  threshold=0.6, block_length=T)

    want, want_nfe, want_anchors = expected()
    hf_cfg, model = (_llada if kind == "llada" else _dream)(arch, weights, torch.float32)
    cfg = _serve_config(hf_cfg, arch, kind, torch.float32, threshold=0.6, anchor_ratio=0.3, max_num_seqs=max_num_seqs,
                        num_kvcache_blocks=32, block_length=T, gen_length=G)
    runner = ModelRunner(model, cfg)
    seqs = [Sequence(r["prompt"], block_length=T, gen_length=G, cache_block_size=8, mask_id=arch.mask_id,
                     prompt_affix_start=r["affix_start"], prompt_affix_end=r["affix_end"],
                     generation_start=r["generation_start"]) for r in reqs]
    outs, nfe = runner.generate_with_acache(seqs)
    _lib.check_device_errors()
    assert [s.anchor_positions for s in seqs] == want_anchors
    assert outs == want and nfe == want_nfe
    # the frequencies matter: the plain ones give other tokens
    monkeypatch.undo()
    assert expected()[0] != want


@pytest.mark.parametrize("kind", ["llada", "dream"])
def test_engine_with_stretched_frequencies_8_bits_and_the_shared_span_once(kind, monkeypatch):
    """All three in one engine: replayed tokens equal eager ones, and the switches act (blocks in 8 bits, scaled scores)."""
    import functools

    from acache_b200 import ops
    from acache_b200.model import configuration
    from oracle.models import random_state_dict

    scaling = dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=64)
    for name in ("LLaDAConfig", "DreamConfig"):
        monkeypatch.setattr(configuration, name, functools.partial(getattr(configuration, name), rope_scaling=scaling))
    arch = _arch(kind)
    A, G, T = 150, 16, 8
    rng = random.Random(12)
    affix = [rng.randint(1, 170) for _ in range(A)]
    reqs = _random_requests(rng, arch, 5, A, G, ["prefix"], affix)
    hf_cfg, model = (_llada if kind == "llada" else _dream)(arch, random_state_dict(arch, seed=21, std=0.2), BF)
    eager, graphs = (_serve(model, hf_cfg, arch, kind, reqs, G, T, share_span_once=True, int8_projections=True, use_cuda_graphs=on)
                     for on in (False, True))
    assert graphs == eager and all(arch.mask_id not in o for o in eager)
    blocks = model.model.transformer["blocks"] if kind == "llada" else model.model.layers
    attn = blocks[0].attn if kind == "llada" else blocks[0].self_attn.attn
    factor = ops.rope_frequencies(64, arch.rope_theta, scaling)[1]
    assert blocks[0].int8 is not None and abs(attn.scale - factor ** 2 * 64 ** -0.5) < 1e-12
