"""Attention of a batch over one shared prefix against a plain 64-bit form."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _fn():
    from acache_b200 import _lib
    from acache_b200.model import acache_attention as m

    _lib.load()
    return _lib, m


def _reference(q, kc, vc, prefix, cu_q, cu_k, slots, scale, keep=None):
    """One request and one KV head at a time in 64 bits; also the sum of the weights' absolute values times |v|,
    the size that rounding errors are relative to."""
    total, nh, D = q.shape
    hkv = kc.shape[-2]
    K, V = kc.double().reshape(-1, hkv, D), vc.double().reshape(-1, hkv, D)
    out, size = torch.zeros(total, nh, D, dtype=torch.float64), torch.zeros(total, nh, D, dtype=torch.float64)
    for b in range(len(cu_q) - 1):
        p = prefix if keep is None else prefix[keep[b]]
        names = torch.cat([p, slots[cu_k[b]:cu_k[b + 1]]]).long()
        names = names[names >= 0]
        if names.numel() == 0:
            continue
        for h in range(nh):
            k, v = K[names, h * hkv // nh], V[names, h * hkv // nh]
            s = (q[cu_q[b]:cu_q[b + 1], h].double() @ k.T) * scale
            w = torch.softmax(s, -1)
            out[cu_q[b]:cu_q[b + 1], h] = w @ v
            size[cu_q[b]:cu_q[b + 1], h] = w @ v.abs()
    return out, size


def _tolerance(ref, size, dtype):
    """The weights are rounded to the type before the product with V (half a step of every term) while their sum is
    not; the result is rounded once; scores and sums in fp32 add 2^-16 of the terms at these sizes (scores up to
    about 30: an absolute error of 30 * 2^-22 in the exponent)."""
    eps = torch.finfo(dtype).eps
    return ref.abs() * eps / 2 + size * (eps / 2 + 2.0 ** -15) + torch.finfo(dtype).smallest_normal * eps


def _inputs(q_lens, k_lens, prefix, nh, hkv, D, dtype, seed=0, holes=0.0, drop=0.0, page=16):
    g = torch.Generator().manual_seed(seed)
    n_slots = prefix + sum(k_lens) + 3 * page
    n_slots = -(-n_slots // page) * page
    kc, vc = (torch.randn(n_slots // page, page, hkv, D, generator=g).to(dtype) for _ in range(2))
    perm = torch.randperm(n_slots, generator=g).to(torch.int32)
    pre, slots = perm[:prefix].clone(), perm[prefix:prefix + sum(k_lens)].clone()
    if holes:
        pre[torch.rand(prefix, generator=g) < holes] = -1
        slots[torch.rand(slots.numel(), generator=g) < holes] = -1
    keep = torch.rand(len(q_lens), prefix, generator=g) >= drop if drop else None
    q = torch.randn(sum(q_lens), nh, D, generator=g).to(dtype) * 2
    cu_q = torch.tensor([0, *itertools.accumulate(q_lens)], dtype=torch.int32)
    cu_k = torch.tensor([0, *itertools.accumulate(k_lens)], dtype=torch.int32)
    return q, kc, vc, pre, cu_q, cu_k, slots, keep


def _run(m, q, kc, vc, pre, cu_q, cu_k, slots, keep, scale=None, packed=False, **kw):
    d = [t.to(DEV) for t in (q, kc, vc, pre, cu_q, cu_k, slots)]
    keep = None if keep is None else keep.to(DEV)
    if packed:
        keep = m.pack_keep_mask(keep)
    return m.shared_prefix_attention(*d, scale, prefix_keep=keep, **kw)


def _check(m, case, scale=None, **kw):
    q, kc, vc, pre, cu_q, cu_k, slots, keep = case
    got = _run(m, *case, scale=scale, **kw).cpu().double()
    ref, size = _reference(q, kc, vc, pre, cu_q.tolist(), cu_k.tolist(), slots, scale or q.shape[-1] ** -0.5, keep)
    bad = (got - ref).abs() > _tolerance(ref, size, q.dtype)
    assert not bad.any(), ((got - ref).abs().max(), bad.nonzero()[:4])
    return got


HEADS = [(4, 4, 128), (28, 4, 128), (6, 2, 64), (5, 1, 64)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nh,hkv,D", HEADS)
@pytest.mark.parametrize("q_lens,k_lens,prefix", [
    ([1], [0], 1), ([1], [1], 0), ([1, 1, 1], [5, 0, 17], 63), ([1] * 9, [33] * 9, 257), ([2, 0, 5], [0, 64, 700], 1000),
    ([32, 32], [300, 16], 129), ([7] * 5, [1, 2, 3, 64, 65], 640), ([40, 3], [129, 1], 2049)])
def test_lengths_heads_and_types(q_lens, k_lens, prefix, nh, hkv, D, dtype):
    _lib, m = _fn()
    _check(m, _inputs(q_lens, k_lens, prefix, nh, hkv, D, dtype, seed=prefix + nh))
    _lib.check_device_errors()


@pytest.mark.parametrize("nh,hkv,D", [(4, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("q_lens,k_lens,prefix", [([1, 1], [40, 0], 300), ([16] * 4, [100, 3, 0, 260], 513), ([33, 60, 1], [5, 0, 130], 65)])
def test_holes_and_dropped_keys(q_lens, k_lens, prefix, nh, hkv, D):
    _lib, m = _fn()
    case = _inputs(q_lens, k_lens, prefix, nh, hkv, D, BF, seed=3, holes=0.3, drop=0.4)
    a = _check(m, case)
    assert torch.equal(a, _run(m, *case, packed=True).cpu().double())
    keep = case[-1]
    keep[0] = False                                    # a request that drops the whole prefix
    keep[-1, ::2] = False
    _check(m, case)
    _lib.check_device_errors()


def test_rows_without_any_key_are_zero_and_rows_behind_the_batch_stay():
    _lib, m = _fn()
    for q_lens in ([1, 2, 1], [40, 2, 30]):
        q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs(q_lens, [10, 0, 0], 100, 4, 2, 64, BF, drop=0.5)
        keep[1] = False                                # nothing kept and nothing of its own
        got = _check(m, (q, kc, vc, pre, cu_q, cu_k, slots, keep))
        assert (got[q_lens[0]:q_lens[0] + q_lens[1]] == 0).all()
        pre[:] = -1
        slots[:] = -1
        assert (_run(m, q, kc, vc, pre, cu_q, cu_k, slots, None) == 0).all()
        # through the C ABI with a caller's output: two rows behind the last request
        lib = _lib.load()
        pad = torch.cat([q, q[:2]]).to(DEV)
        out = torch.full_like(pad, 7.0)
        d = [t.to(DEV) for t in (kc, vc, cu_q, cu_k)]
        n = pad.shape[0]
        nbytes = lib.acache_shared_prefix_attention_scratch_bytes(n, 4, 2, 64, 3, max(q_lens), 10, 0)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        mine = torch.arange(10, dtype=torch.int32, device=DEV)
        assert lib.acache_shared_prefix_attention(
            pad.data_ptr(), pad.stride(0), out.data_ptr(), out.stride(0), d[0].data_ptr(), d[1].data_ptr(), kc.numel() // 128, n,
            4, 2, 64, 2, None, 0, None, 0, d[2].data_ptr(), d[3].data_ptr(), 3, max(q_lens), 10, mine.data_ptr(), 10, 0.125,
            scratch.data_ptr(), nbytes, None, torch.cuda.current_stream().cuda_stream) == 0
        assert (out[-2:] == 7).all() and (out[q_lens[0]:-2] == 0).all() and not (out[:q_lens[0]] == 0).all()


def test_strided_queries_large_scores_and_scale():
    _lib, m = _fn()
    q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs([5, 32], [70, 200], 400, 8, 2, 128, BF, seed=8)
    wide = torch.randn(37, 8 * 128 + 64).to(BF)
    wide[:, 64:] = q.view(37, -1)
    qs = wide.to(DEV)[:, 64:].unflatten(1, (8, 128))   # a slice of a wider projection output
    d = [t.to(DEV) for t in (kc, vc, pre, cu_q, cu_k, slots)]
    assert torch.equal(m.shared_prefix_attention(qs, *d), m.shared_prefix_attention(q.to(DEV), *d))
    # a maximum that keeps growing along the keys: rescaling in every tile
    order = torch.argsort(kc.view(-1, 2, 128)[pre.long(), 0, 0].float())
    pre = pre[order]
    q[:, :, 0] = 40
    _check(m, (q, kc, vc, pre, cu_q, cu_k, slots, keep), scale=0.25)


def test_nan_and_infinities():
    """A dropped key's K and V do not reach the rows that drop it, whatever they hold; a kept one's do."""
    _lib, m = _fn()
    for q_lens in ([1, 1], [1, 40]):
        q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs(q_lens, [20, 20], 300, 2, 2, 128, BF, seed=5, drop=0.2)
        keep[0, 7], keep[1, 7] = False, True
        clean = _check(m, (q, kc, vc, pre, cu_q, cu_k, slots, keep))
        for cache, value in ((vc, float("nan")), (vc, float("inf")), (kc, float("nan")), (kc, float("inf"))):
            page = cache.clone()
            page.view(-1, 2, 128)[pre[7].long(), 0, 3] = value
            k2, v2 = (page, vc) if cache is kc else (kc, page)
            got = _run(m, q, k2, v2, pre, cu_q, cu_k, slots, keep).cpu().double()
            ref, size = _reference(q, kc, vc, pre, cu_q.tolist(), cu_k.tolist(), slots, 128 ** -0.5, keep)
            n0 = q_lens[0]
            assert ((got - ref).abs() <= _tolerance(ref, size, BF))[:n0].all()          # request 0 drops the key
            assert torch.equal(got[n0:, 1], clean[n0:, 1])                              # the other KV head
            if cache is vc:
                assert not torch.isfinite(got[n0:, 0, 3]).any()                         # request 1 reads it
                assert torch.equal(got[n0:, 0, 4:], clean[n0:, 0, 4:])
            elif value != value:
                assert torch.isnan(got[n0:, 0]).all()
        holes = pre.clone()                            # a hole for everyone: its row is never read
        holes[7] = -1
        page = vc.clone()
        page.view(-1, 2, 128)[pre[7].long()] = float("nan")
        got = _run(m, q, kc, page, holes, cu_q, cu_k, slots, None).cpu()
        assert torch.isfinite(got).all()
        q[0, 0, 5] = float("nan")
        got = _run(m, q, kc, vc, pre, cu_q, cu_k, slots, keep).cpu()
        assert torch.isnan(got[0, 0]).all() and torch.isfinite(got[0, 1]).all() and torch.isfinite(got[1:]).all()


def test_agrees_with_the_per_request_operator():
    """The same keys through ``acache_attention``: both round the weights and the result to the type."""
    _lib, m = _fn()
    q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs([32] * 4, [100, 300, 64, 1], 800, 4, 4, 128, BF, seed=1, drop=0.2)
    got = _check(m, (q, kc, vc, pre, cu_q, cu_k, slots, keep))
    runs = [torch.cat([torch.where(keep[b], pre, -1), slots[cu_k[b]:cu_k[b + 1]]]) for b in range(4)]
    cu = torch.tensor([0, *itertools.accumulate(r.numel() for r in runs)], dtype=torch.int32)
    d = [t.to(DEV) for t in (q, kc, vc, cu_q, cu, torch.cat(runs))]
    other = m.acache_attention(*d).cpu().double()
    ref, size = _reference(q, kc, vc, pre, cu_q.tolist(), cu_k.tolist(), slots, 128 ** -0.5, keep)
    assert ((got - other).abs() <= 2 * _tolerance(ref, size, BF)).all()


def test_graphs_streams_and_repeats():
    """Two captured graphs replayed on two streams at once, a side stream, and bit-equal repeats."""
    _lib, m = _fn()
    cases = [_inputs([1] * 6, [900] * 6, 4000, 8, 2, 128, BF, seed=s, drop=0.1) for s in (1, 2)]
    dev = [[t.to(DEV) for t in c] for c in cases]

    def call(c):
        return m.shared_prefix_attention(*c[:7], prefix_keep=c[7], max_seqlen_q=1, max_seqlen_k=900)

    want = [call(c).clone() for c in dev]
    for w, c in zip(want, dev):
        assert torch.equal(w, call(c))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for c in dev:
        with torch.cuda.stream(side):
            call(c)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w, o)
    _lib.check_device_errors()


def test_bad_slots_are_reported_and_refusals():
    _lib, m = _fn()
    q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs([1, 2], [5, 6], 70, 4, 2, 64, BF)
    n = kc.numel() // 128
    for name, at in (("prefix", pre), ("own", slots)):
        old = int(at[1])
        at[1] = n
        got = _run(m, q, kc, vc, pre, cu_q, cu_k, slots, None)
        with pytest.raises(_lib.AcacheError):
            _lib.check_device_errors()
        assert torch.isfinite(got).all()
        at[1] = old
    case = (q, kc, vc, pre, cu_q, cu_k, slots, keep)
    assert _run(m, q[:0], kc, vc, pre, cu_q * 0, cu_k, slots, None).shape == (0, 4, 64)
    assert _run(m, q[:0], kc, vc, pre, cu_q[:1], cu_k[:1], slots[:0], None).shape == (0, 4, 64)
    with pytest.raises(NotImplementedError):
        _run(m, q.float(), kc.float(), vc.float(), pre, cu_q, cu_k, slots, None)
    with pytest.raises(NotImplementedError):
        _run(m, q[..., :32].contiguous(), kc[..., :32].contiguous(), vc[..., :32].contiguous(), pre, cu_q, cu_k, slots, None)
    for i, bad in ((3, pre.long()), (5, cu_k[:2]), (0, q.to(HF))):
        args = list(case)
        args[i] = bad
        with pytest.raises(AssertionError):
            _run(m, *args)
    with pytest.raises(AssertionError):
        _run(m, *case[:7], torch.ones(2, 69, dtype=torch.bool))


@pytest.mark.parametrize("q_lens,nh,hkv,D,prefix,drop", [([100] * 13, 4, 2, 128, 12800, 0.0), ([700, 1, 659, 80], 6, 2, 64, 16000, 0.3),
                                                        ([40] * 128, 8, 1, 128, 3000, 0.1)])
def test_prefix_tiles_shared_out_over_all_sms(q_lens, nh, hkv, D, prefix, drop):
    """Row blocks that do not divide the SMs evenly: a CTA's share ends inside one row block's keys and goes on in the
    next (20, 17 x 2 and 160 blocks of 256 rows over 100, 125 and 24 key tiles)."""
    _lib, m = _fn()
    k_lens = [3 + i % 5 for i in range(len(q_lens))]
    q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs(q_lens, k_lens, prefix, nh, hkv, D, BF, seed=2, drop=drop)
    got = _run(m, q, kc, vc, pre, cu_q, cu_k, slots, keep).cpu().double()
    again = _run(m, q, kc, vc, pre, cu_q, cu_k, slots, keep).cpu().double()
    assert torch.equal(got, again)
    g = torch.Generator().manual_seed(1)
    K, V = kc.to(DEV).view(-1, hkv, D), vc.to(DEV).view(-1, hkv, D)
    for b in sorted({0, 1, len(q_lens) - 1, len(q_lens) // 2}):
        p = pre if keep is None else pre[keep[b]]
        names = torch.cat([p, slots[cu_k[b]:cu_k[b + 1]]]).long().to(DEV)
        for h in range(nh):
            k, v = K[names, h * hkv // nh].double(), V[names, h * hkv // nh].double()
            w = torch.softmax((q[cu_q[b]:cu_q[b + 1], h].to(DEV).double() @ k.T) * D ** -0.5, -1)
            ref, size = (w @ v).cpu(), (w @ v.abs()).cpu()
            assert ((got[cu_q[b]:cu_q[b + 1], h] - ref).abs() <= _tolerance(ref, size, BF)).all()
    _lib.check_device_errors()


def test_slots_beyond_32_bit_offsets_and_the_largest_batch():
    """Cache rows whose element offsets pass 2^31, and 2047 requests in one call (one more is refused)."""
    _lib, m = _fn()
    nh = hkv = 32
    D, page = 128, 256
    pages = 2 ** 31 // (page * hkv * D) + 8             # 2048 pages and a few: offsets above 2^31 elements
    kc = torch.empty(pages, page, hkv, D, dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    g = torch.Generator().manual_seed(0)
    last = (pages - 4) * page
    k_new, v_new = torch.randn(4 * page, hkv, D, generator=g).to(BF), torch.randn(4 * page, hkv, D, generator=g).to(BF)
    kc.view(-1, hkv, D)[last:], vc.view(-1, hkv, D)[last:] = k_new.to(DEV), v_new.to(DEV)
    for q_lens in ([1, 1], [1, 40], [5, 130]):
        q = torch.randn(sum(q_lens), nh, D, generator=g).to(BF)
        pre = torch.arange(300, dtype=torch.int32)
        own = torch.arange(400, 640, dtype=torch.int32)
        cu_q = torch.tensor([0, q_lens[0], sum(q_lens)], dtype=torch.int32)
        cu_k = torch.tensor([0, 100, 240], dtype=torch.int32)
        got = m.shared_prefix_attention(q.to(DEV), kc, vc, (pre + last).to(DEV), cu_q.to(DEV), cu_k.to(DEV), (own + last).to(DEV)).cpu().double()
        ref, size = _reference(q, k_new.view(4, page, hkv, D), v_new.view(4, page, hkv, D), pre, cu_q.tolist(), cu_k.tolist(), own, D ** -0.5)
        assert ((got - ref).abs() <= _tolerance(ref, size, BF)).all()
    del kc, vc
    n = 2047
    q, kc, vc, pre, cu_q, cu_k, slots, keep = _inputs([1] * n, [i % 3 for i in range(n)], 70, 2, 1, 64, BF, drop=0.5)
    _check(m, (q, kc, vc, pre, cu_q, cu_k, slots, keep))
    with pytest.raises(OverflowError):
        _run(m, torch.cat([q, q[:1]]), kc, vc, pre, torch.arange(n + 2, dtype=torch.int32), torch.cat([cu_k, cu_k[-1:]]), slots, None)
    _lib.check_device_errors()


def test_bad_offsets_stay_inside_the_arrays():
    """Offsets that run backwards or past the arrays: nothing outside is read or written, the other rows are right."""
    _lib, m = _fn()
    for q_lens in ([2, 3, 2], [40, 60, 70]):
        q, kc, vc, pre, cu_q, cu_k, slots, _ = _inputs(q_lens, [10, 20, 30], 150, 4, 2, 64, BF)
        want = _run(m, q, kc, vc, pre, cu_q, cu_k, slots, None, max_seqlen_q=max(q_lens), max_seqlen_k=30)
        bad_q, bad_k = cu_q.clone(), cu_k.clone()
        bad_q[-1] = 10 ** 6
        bad_k[-1] = 10 ** 6
        got = _run(m, q, kc, vc, pre, bad_q, bad_k, slots, None, max_seqlen_q=max(q_lens), max_seqlen_k=30)
        assert torch.equal(got, want)
        bad_k[1] = -5
        got = _run(m, q, kc, vc, pre, cu_q, bad_k, slots, None, max_seqlen_q=max(q_lens), max_seqlen_k=30)
        assert torch.isfinite(got).all() and torch.equal(got[cu_q[2]:], want[cu_q[2]:])


@pytest.mark.parametrize("n,batch,prefix", [(4, 2, 10), (300, 8, 2000)])
def test_a_padded_batch_without_queries(n, batch, prefix):
    """Rows of q behind requests that have none (offsets all zero): the call returns, and nothing of its output is written."""
    _lib, m = _fn()
    q, kc, vc, pre, _, cu_k, slots, keep = _inputs([0] * batch, [5] * batch, prefix, 4, 2, 64, BF, drop=0.3)
    q, cu_q = torch.randn(n, 4, 64).to(BF), torch.zeros(batch + 1, dtype=torch.int32)
    for kw in ({}, {"max_seqlen_q": 0}, {"max_seqlen_q": 3}):
        assert _run(m, q, kc, vc, pre, cu_q, cu_k, slots, keep, **kw).shape == q.shape
    lib = _lib.load()
    out = torch.full((n, 4, 64), 7.0, dtype=BF, device=DEV)
    d = [t.to(DEV) for t in (q, kc, vc, pre, cu_q, cu_k, slots)]
    for max_q in (0, 3):
        nbytes = lib.acache_shared_prefix_attention_scratch_bytes(n, 4, 2, 64, batch, max_q, 5, prefix)
        scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=DEV)
        assert lib.acache_shared_prefix_attention(
            d[0].data_ptr(), 256, out.data_ptr(), 256, d[1].data_ptr(), d[2].data_ptr(), kc.numel() // 128, n, 4, 2, 64, 2,
            d[3].data_ptr(), prefix, None, 0, d[4].data_ptr(), d[5].data_ptr(), batch, max_q, 5, d[6].data_ptr(), slots.numel(), 0.125,
            scratch.data_ptr(), nbytes, None, torch.cuda.current_stream().cuda_stream) == 0
        assert (out == 7).all()
    _lib.check_device_errors()


@pytest.mark.parametrize("q_lens,k_lens,prefix,kernels", [([1, 1], [20, 3], 0, 1), ([1, 1], [20, 3], 300, 2), ([40, 60], [20, 300], 300, 3)])
def test_launches_are_counted_as_they_are_made(q_lens, k_lens, prefix, kernels):
    """The binding's count against the kernels that the profiler sees."""
    _lib, m = _fn()
    case = [t.to(DEV) for t in _inputs(q_lens, k_lens, prefix, 14, 2, 64, BF)[:7]]
    kw = dict(max_seqlen_q=max(q_lens), max_seqlen_k=max(k_lens))
    m.shared_prefix_attention(*case, **kw)
    torch.cuda.synchronize()
    before = _lib.LAUNCHES
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        m.shared_prefix_attention(*case, **kw)
        torch.cuda.synchronize()
    assert _lib.LAUNCHES - before == kernels
    seen = [e.name for e in prof.events() if "rows_kernel" in e.name or "wide_parts_kernel" in e.name or "merge_kernel" in e.name]
    assert len(seen) in (0, kernels), seen             # 0: no profiler on this machine


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_lens", [[1], [20], [120]])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_a_long_flat_tail_behind_large_weights(q_lens, where, dtype):
    """Every 32nd key has the weight 1 and a value of 0, the others share the rest with one tiny weight: each weight is rounded by no
    more than half a step of its own, also where fp16 numbers of its size are subnormal.  (Weights of 700.49, 100.49 and 20.49
    steps of 2^-24: rounded on that grid they would all be off by half of one.)"""
    _lib, m = _fn()
    n, D = 32768, 64
    for steps in (700.49, 100.49, 20.49):
        low = torch.tensor(steps / 2 ** 24, dtype=torch.float64).log()
        high = low.to(dtype).double()
        q = torch.zeros(sum(q_lens), 2, D, dtype=dtype)
        q[..., :2] = 8.0
        kc, vc = torch.zeros(n // 256, 256, 1, D, dtype=dtype), torch.ones(n // 256, 256, 1, D, dtype=dtype)
        keys, values = kc.view(-1, D), vc.view(-1, D)
        keys[:, 0], keys[:, 1] = high, low - high      # scores (8 x + 8 y) / 8
        keys[::32], values[::32] = 0, 0
        slots, none = torch.arange(n, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
        pre, own = (slots, none) if where == "prefix" else (none, slots)
        cu_q = torch.tensor([0, sum(q_lens)], dtype=torch.int32)
        _check(m, (q, kc, vc, pre, cu_q, torch.tensor([0, own.numel()], dtype=torch.int32), own, None))
