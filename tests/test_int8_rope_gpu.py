"""Projections in 8-bit integers with their quantising producers, and rotary positions from frequencies,
against plain 64-bit forms of the same definitions."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _ops():
    from acache_b200 import _lib, ops

    _lib.load()
    return _lib, ops


def _quantise64(y):
    """(q, scale) of every row in 64 bits."""
    top = y.abs().amax(1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * y / top), torch.zeros_like(y)), (top / 127).squeeze(1)


def _act64(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    return g.clamp_min(0) if act == "relu" else 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))


# widths: a register row of every variant, one no vector divides, one beyond the register rows
@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("n,cols", [(1, 16), (5, 64), (33, 1000), (7, 2056), (3, 4096), (9, 4104), (2, 12288), (3, 18944), (4, 1003), (2, 33000)])
def test_quantize_rows_is_exact_for_16_bit_rows(n, cols, dtype):
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(n * cols)
    x = (torch.randn(n, cols, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 4)).to(dtype)
    x[0, : cols // 2] = x[0, : cols // 2].abs().max() / 2          # 63.5: a tie, which goes to the even 64
    q, scale = ops.quantize_rows(x.to(DEV))
    want_q, want_s = _quantise64(x.double())
    if dtype == torch.float32:
        # the product by 127 / a instead of a division (2 units of the last place) and the rounding to 21 bits (4 units)
        # move a value of at most 127 by at most 6 * 2^-17: only entries within 2^-13 of a tie may differ, by one
        near = ((127 * x.double() / x.double().abs().amax(1, keepdim=True)) % 1 - 0.5).abs() <= 2.0 ** -13
        diff = (q.cpu().double() - want_q).abs()
        assert (diff[~near] == 0).all() and diff.max() <= 1
    else:
        assert torch.equal(q.cpu().double(), want_q)
    torch.testing.assert_close(scale.cpu().double(), want_s, rtol=2.0 ** -24, atol=0)


def test_quantize_rows_strides_zeros_and_non_finite_rows():
    _lib, ops = _ops()
    base = torch.randn(12, 200, device=DEV).to(BF)
    x = base[::2, 8:136]                              # rows 400 elements apart, 16-byte aligned
    q, s = ops.quantize_rows(x)
    wq, ws = _quantise64(x.double())
    assert torch.equal(q.double(), wq)
    x = base[:, 3:131]                                # rows that no 16-byte vector fits
    assert torch.equal(ops.quantize_rows(x)[0].double(), _quantise64(x.double())[0])
    bad = base[:, :128].clone()
    bad[0] = 0
    bad[1, 5] = float("inf")
    bad[2, 127] = float("nan")
    bad[3, 0] = float("-inf")
    bad[4] = torch.finfo(BF).smallest_normal * 2.0 ** -5      # below the normal range: kept in proportion
    bad[4, 7] *= 2
    for rows in (bad, torch.nn.functional.pad(bad, (3, 0))[:, 3:]):     # both kernels
        q, s = ops.quantize_rows(rows)
        assert s[0] == 0 and (q[0] == 0).all()
        assert torch.isnan(s[1:4]).all() and (q[1:4] == 0).all()
        assert torch.equal(q[4].double(), _quantise64(bad.double())[0][4])
        assert torch.isfinite(s[5:]).all() and torch.equal(q[5:].double(), _quantise64(bad.double())[0][5:])


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("n,cols,with_delta", [(1, 64, False), (33, 4096, True), (5, 3584, False), (3, 1003, True), (2, 33000, True)])
def test_rmsnorm_int8(n, cols, with_delta, dtype):
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(cols + n)
    x, w = torch.randn(n, cols, generator=g).to(dtype), (1 + 0.2 * torch.randn(cols, generator=g)).to(dtype)
    d = torch.randn(n, cols, generator=g).to(dtype) if with_delta else None
    xd = x.to(DEV).clone()
    q, s = ops.rmsnorm_int8(xd, w.to(DEV), 1e-5, None if d is None else d.to(DEV))
    if d is not None:
        x = (x.float() + d.float()).to(dtype)
    assert torch.equal(xd.cpu(), x)
    y = x.double()
    y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + 1e-5) * w.double()
    _check_quantised(q, s, y, rel=cols ** 0.5 * 2.0 ** -23)


def _check_quantised(q, s, y, rel):
    """``rel``: relative error of the fp32 row values and of their maximum; entries further than that from a tie
    are equal (2^-12 more for the rounding to 21 bits), the others differ by at most one."""
    wq, ws = _quantise64(y)
    exact = 127 * y / y.abs().amax(1, keepdim=True)
    near = (exact.abs() % 1 - 0.5).abs() <= 127 * 2 * rel + 2.0 ** -12
    diff = (q.cpu().double() - wq).abs()
    assert (diff[~near] == 0).all() and diff.max() <= 1
    torch.testing.assert_close(s.cpu().double(), ws, rtol=rel + 2.0 ** -23, atol=0)


@pytest.mark.parametrize("act", ["silu", "relu", "gelu"])
@pytest.mark.parametrize("n,ffn,dtype", [(1, 16, BF), (17, 12288, BF), (5, 18944, HF), (3, 1001, BF), (4, 512, torch.float32)])
def test_act_mul_halves_int8(n, ffn, dtype, act):
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(ffn)
    x = torch.randn(n, 2 * ffn, generator=g).to(dtype)
    q, s = ops.act_mul_halves_int8(x.to(DEV), act)
    # exp / erf within a few fp32 steps; gelu loses the steps of 1 + erf where that cancels: absolute, of the largest value
    y = _act64(x[:, :ffn].double(), act) * x[:, ffn:].double()
    _check_quantised(q, s, y, rel=2.0 ** -20)


INT8_SHAPES = [(1, 16, 16), (1, 64, 64), (33, 4096, 4096), (77, 448, 272), (300, 512, 384), (513, 144, 2048), (64, 12288, 4096), (700, 272, 1040)]


@pytest.mark.parametrize("tile", [(0, 0), (1, 64), (1, 256), (2, 128), (2, 224), (1, 96)])
@pytest.mark.parametrize("n,k,out", INT8_SHAPES)
def test_linear_int8_matches_64_bits(n, k, out, tile):
    """The sums are exact integers (odd sizes, full-range entries); then an int -> fp32 rounding, two products and an
    addition in fp32 (4 x 2^-24 of the terms) and one rounding to the output type."""
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(n + k + out)
    x = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (out, k), generator=g, dtype=torch.int8)
    xs, ws = torch.rand(n, generator=g) * 0.02, torch.rand(out, generator=g) * 0.001
    dtype = HF if n % 2 == 0 else BF
    b = torch.randn(out, generator=g).to(dtype) if k % 32 else None
    acc = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    ref = acc if b is None else acc + b.double()
    ops.GEMM_TILE = tile
    try:
        got = ops.linear_int8(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), None if b is None else b.to(DEV), out_dtype=dtype)
    finally:
        ops.GEMM_TILE = (0, 0)
    _lib.check_device_errors()
    terms = acc.abs() + (0 if b is None else b.double().abs())
    tol = ref.abs() * torch.finfo(dtype).eps / 2 + 2 * terms * 2.0 ** -22 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((got.cpu().double() - ref).abs() <= tol).all(), (got.cpu().double() - ref).abs().max()


def test_linear_int8_largest_sums_and_poisoned_rows():
    _lib, ops = _ops()
    k = 131056                                        # -128 * -128 * k = 2.147e9, just below 2^31
    x = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((32, k), -128, dtype=torch.int8, device=DEV)
    xs = torch.tensor([1.0, 0.0, float("nan")], device=DEV) * 2.0 ** -31
    got = ops.linear_int8(x, xs, w, torch.ones(32, device=DEV), out_dtype=HF)
    want = torch.tensor(128 * 128 * k * 2.0 ** -31).to(HF)
    assert (got[0].cpu() == want).all() and (got[1] == 0).all() and torch.isnan(got[2]).all()
    _lib.check_device_errors()


def test_linear_int8_refusals():
    _lib, ops = _ops()
    x = torch.zeros(4, 64, dtype=torch.int8, device=DEV)
    w = torch.zeros(32, 64, dtype=torch.int8, device=DEV)
    xs, ws = torch.zeros(4, device=DEV), torch.zeros(32, device=DEV)
    assert ops.linear_int8(x[:0], xs[:0], w, ws).shape == (0, 32)
    with pytest.raises(AssertionError):
        ops.linear_int8(x, xs[:3], w, ws)
    with pytest.raises(AssertionError):
        ops.linear_int8(x.to(torch.uint8), xs, w, ws)
    with pytest.raises(NotImplementedError):
        ops.linear_int8(x, xs, w, ws, out_dtype=torch.float32)
    with pytest.raises(NotImplementedError):           # in_features not a multiple of 16
        ops.linear_int8(x[:, :24].contiguous(), xs, w[:, :24].contiguous(), ws)
    with pytest.raises(NotImplementedError):           # out_features not a multiple of 16
        ops.linear_int8(x, xs, w[:24], ws[:24])
    with pytest.raises(OverflowError):
        z = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
        ops.linear_int8(z, xs[:1], torch.zeros(16, 131072, dtype=torch.int8, device=DEV), ws[:16])


# ------------------------------------------------------------------------------------ rotary
def _rotate64(x, positions, inv_freq, interleaved, factor):
    half = inv_freq.numel()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = positions.double()[:, None] * inv_freq.cpu()
    c, s = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
    y = x.double().clone()
    y[..., a] = x.double()[..., a] * c - x.double()[..., b] * s
    y[..., b] = x.double()[..., b] * c + x.double()[..., a] * s
    return y


def _close_rotated(got, want, x):
    """one rounding to the type, and sine, cosine and two products in fp32 (2^-21 of the pair's size)."""
    got, want = got.cpu().double(), want.cpu()
    size = x.abs().double().cpu().amax(-1, keepdim=True)
    tol = want.abs() * torch.finfo(x.dtype).eps / 2 + size * 2.0 ** -20 + 2.0 ** -25
    assert ((got - want).abs() <= tol).all(), (got - want).abs().max()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,nh,hkv,D,rot,dtype", [(1, 1, 1, 64, 64, BF), (33, 28, 4, 128, 128, BF), (7, 5, 1, 64, 16, HF), (300, 8, 8, 128, 64, HF),
                                                  (5, 3, 3, 80, 20, BF), (9, 4, 2, 128, 6, torch.float32), (4, 2, 2, 40, 0, BF)])
def test_rope_append(n, nh, hkv, D, rot, dtype, interleaved):
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(n + D)
    width = (nh + 2 * hkv) * D
    qkv = torch.randn(n, width + 8, generator=g).to(dtype).to(DEV)[:, :width]
    q, k, v = qkv[:, : nh * D].unflatten(1, (nh, D)), qkv[:, nh * D: (nh + hkv) * D].unflatten(1, (hkv, D)), qkv[:, (nh + hkv) * D:].unflatten(1, (hkv, D))
    before = qkv.clone()
    inv = (500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).to(DEV)
    pos = torch.randint(-5, 1_000_000, (n,), generator=g).to(DEV)
    kc, vc = torch.randn(3, 256, hkv, D, generator=g).to(dtype).to(DEV), torch.randn(3, 256, hkv, D, generator=g).to(dtype).to(DEV)
    slots = torch.randperm(768, generator=g)[:n].to(torch.int32)
    slots[n // 2] = -1
    want_k, want_v = kc.double().cpu().view(-1, hkv, D), vc.double().cpu().view(-1, hkv, D)
    rk = _rotate64(k.cpu(), pos.cpu(), inv, interleaved, 1.25)
    live = slots >= 0
    want_k[slots[live].long()], want_v[slots[live].long()] = rk[live], v.cpu().double()[live]
    out = ops.rope_append(q, k, v, pos, inv, kc, vc, slots.to(DEV), interleaved=interleaved, attention_factor=1.25)
    _close_rotated(out, _rotate64(q.cpu(), pos.cpu(), inv, interleaved, 1.25), q)
    _close_rotated(kc.view(-1, hkv, D), want_k, kc.view(-1, hkv, D).abs().amax().expand(1, 1, 1).to(dtype))
    assert torch.equal(vc.view(-1, hkv, D).cpu().double(), want_v) and torch.equal(qkv, before)
    q2, k2 = ops.rope_append(q, k, v, pos, inv, interleaved=interleaved, attention_factor=1.25)
    assert torch.equal(q2, out)
    _close_rotated(k2, rk, k)
    _lib.check_device_errors()


def test_rope_append_agrees_with_the_table_form():
    """Half layout over the whole head at near positions: the fp32 tables of ``rope_store`` hold the same angles."""
    _lib, ops = _ops()
    from acache_b200.model.modeling_common import build_rope_table

    q, k = torch.randn(64, 4, 128, device=DEV).to(BF), torch.randn(64, 4, 128, device=DEV).to(BF)
    pos = torch.arange(64, device=DEV)
    cos, sin = build_rope_table(64, 128, 10000.0, torch.float32, DEV)
    inv, factor = ops.rope_frequencies(128, 10000.0)
    oq, ok = ops.rope_append(q, k, None, pos, inv.to(DEV), attention_factor=factor)
    ops.rope_store(q, k, None, pos, cos, sin)
    # angles up to 64 differ by 64 * 2^-23: far below one bf16 step, so the two differ in rare last bits
    torch.testing.assert_close(oq.float(), q.float(), rtol=2 ** -7, atol=2 ** -14)
    torch.testing.assert_close(ok.float(), k.float(), rtol=2 ** -7, atol=2 ** -14)


def test_rope_append_reports_slots_outside_the_cache():
    _lib, ops = _ops()
    q, k = torch.randn(3, 2, 64, device=DEV).to(BF), torch.randn(3, 2, 64, device=DEV).to(BF)
    kc = torch.zeros(1, 256, 2, 64, dtype=BF, device=DEV)
    vc = torch.zeros_like(kc)
    inv = ops.rope_frequencies(64, 10000.0)[0].to(DEV)
    slots = torch.tensor([3, 256, -2], dtype=torch.int32, device=DEV)
    ops.rope_append(q, k, k, torch.arange(3, device=DEV), inv, kc, vc, slots)
    with pytest.raises(_lib.AcacheError):
        _lib.check_device_errors()
    written = (vc.view(256, -1).abs().sum(1) > 0).nonzero().flatten().tolist()
    assert written == [3]


def test_offsets_beyond_32_bits():
    """Outputs, weights and cache rows whose element offsets pass 2^31."""
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(0)
    n, out, k = 17000, 126464, 16                     # 2.15e9 outputs
    x = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(DEV)
    w = torch.randint(-128, 128, (out, k), generator=g, dtype=torch.int8).to(DEV)
    xs, ws = torch.rand(n, generator=g).to(DEV), torch.rand(out, generator=g).to(DEV)
    y = ops.linear_int8(x, xs, w, ws)
    for rows in (slice(0, 3), slice(n - 300, n)):
        ref = (x[rows].double() @ w.double().T) * xs[rows].double()[:, None] * ws.double()
        assert ((y[rows].double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -21)).all()
    del y
    w = torch.randint(-128, 128, (131056, 16512), dtype=torch.int8, device=DEV)      # 2.16e9 weights
    ws = torch.rand(131056, device=DEV)
    x = torch.randint(-128, 128, (40, 16512), dtype=torch.int8, device=DEV)
    y = ops.linear_int8(x, xs[:40], w, ws)
    ref = (x.double() @ w[-64:].double().T) * xs[:40].double()[:, None] * ws[-64:].double()
    assert ((y[:, -64:].double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -21)).all()
    del w, y
    big = torch.zeros(2, 2 ** 30 + 64, dtype=torch.float16, device=DEV)[:, :4096]    # rows 2^30 elements apart
    big[1] = torch.randn(4096, device=DEV).half()
    q, _ = ops.quantize_rows(big)
    assert torch.equal(q.double(), _quantise64(big.double())[0])
    del big
    pages = 2 ** 31 // (256 * 32 * 128) + 2
    kc = torch.empty(pages, 256, 32, 128, dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    t = torch.randn(6, 32, 128, device=DEV).to(BF)
    slots = torch.arange(pages * 256 - 6, pages * 256, dtype=torch.int32, device=DEV)
    inv = ops.rope_frequencies(128, 500000.0)[0].to(DEV)
    ops.rope_append(t, t, t, torch.arange(6, device=DEV), inv, kc, vc, slots)
    assert torch.equal(vc.view(-1, 32, 128)[-6:], t)
    _close_rotated(kc.view(-1, 32, 128)[-6:], _rotate64(t.cpu(), torch.arange(6), inv, False, 1.0), t)
    _lib.check_device_errors()


def test_rmsnorm_int8_refuses_rows_that_overlap_when_it_writes_them():
    _lib, ops = _ops()
    x = torch.randn(1, 64, device=DEV).to(BF)
    w = torch.ones(64, dtype=BF, device=DEV)
    q, s = ops.rmsnorm_int8(x.expand(4, 64), w, 1e-5)            # read only: fine
    assert torch.equal(q[0], q[3])
    with pytest.raises(AssertionError):
        ops.rmsnorm_int8(x.expand(4, 64), w, 1e-5, torch.zeros(4, 64, dtype=BF, device=DEV))


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 48, 49, 64, 65, 255, 256, 257])
@pytest.mark.parametrize("k,out", [(16, 32), (80, 48), (1040, 4112), (4096, 1008)])
def test_linear_int8_at_the_edges_of_its_forms(n, k, out):
    """Row counts around the few-row kernel's tiles and the 256-row ones, K ranges that end inside a step of 64 or a
    k block of 128, column counts that end inside a tile; rows of a wider tensor; integers, so every sum is exact."""
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(n * k)
    wide = torch.randint(-128, 128, (n, k + 32), generator=g, dtype=torch.int8).to(DEV)
    x = wide[:, 16:16 + k]
    w = torch.randint(-128, 128, (out, k), generator=g, dtype=torch.int8).to(DEV)
    xs, ws = torch.rand(n, generator=g).to(DEV), torch.rand(out, generator=g).to(DEV)
    y = ops.linear_int8(x, xs, w, ws)
    ref = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    assert ((y.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -21)).all()
    _lib.check_device_errors()


@pytest.mark.parametrize("cols", [64, 2048, 3584, 12288, 40000, 50])
def test_norm_whose_weighted_values_leave_the_range(cols):
    """x * weight beyond fp32 where the norm is not: the factor has to come first."""
    from acache_b200 import ops

    g = torch.Generator().manual_seed(cols)
    x = torch.randn(5, cols, generator=g) * 2.0 ** 60
    x[1] *= 2.0 ** -60
    x[2, 0] = float("nan")
    x[3] = 0
    w = torch.randn(cols, generator=g) * 2.0 ** 90
    x, w = x.to(torch.bfloat16), w.to(torch.bfloat16)
    q, scale = ops.rmsnorm_int8(x.to(DEV), w.to(DEV), 1e-6)
    q, scale = q.cpu(), scale.cpu().double()
    assert torch.isnan(scale[2]) and (q[2:4] == 0).all() and scale[3] == 0
    rows = [0, 1, 4]
    y = x.double()[rows]
    y = y / (y.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    top = y.abs().amax(1)
    # scale: the square root of a sum of `cols` squares, a few roundings of 2^-24 each, the sum's in a tree of at most
    # 128 in line; q: half a step and the same relative error of at most 127 steps
    rel = 2.0 ** -24 * (128 / 2 + 8)
    assert ((scale[rows] - top / 127).abs() <= top / 127 * rel).all()
    assert ((q[rows].double() - 127 * y / top[:, None]).abs() <= 0.5 + 127 * 2 * rel).all()


@pytest.mark.parametrize("bn", [64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("n,k,out", [(600, 1168, 9472), (300, 4240, 1232), (2000, 128, 9472)])
def test_linear_int8_rings_that_wrap_inside_tiles(n, k, out, bn):
    """Several tiles a pair, k blocks that are no multiple of the ring's stages, slices of the K range: every width of the
    tiles; exact integer sums, two roundings of 2^-24 and one to the output type."""
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(n + k)
    x = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(DEV)
    w = torch.randint(-128, 128, (out, k), generator=g, dtype=torch.int8).to(DEV)
    xs, ws = torch.rand(n, generator=g).to(DEV), torch.rand(out, generator=g).to(DEV)
    ops.GEMM_TILE = (0, bn)
    try:
        y = [ops.linear_int8(x, xs, w, ws) for _ in range(3)]
    finally:
        ops.GEMM_TILE = (0, 0)
    ref = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    assert ((y[0].double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -21)).all()
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
    _lib.check_device_errors()


@pytest.mark.parametrize("cols", [64, 2048, 12288, 50, 40000])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_far_below_zero_that_make_a_row_s_largest_value(act, cols):
    """Large up values behind gates where the activation is tiny.  silu: a power of two (2^-22), a reciprocal or division
    (2 steps), four products and a sum, and for -88, where e^x is below the normal range, two steps of 2^-149 of its 2^-127:
    below 2^-19.  gelu: down to -3 two steps of erff (2^-23) over
    1 + erf (2^-8.5): 2^-14; below, the rounded argument t = x / sqrt 2 (two roundings of 2^-24) changes erfc by 2 t^2 = x^2
    times that, erfcf is off by 4 steps, three products."""
    _lib, ops = _ops()
    gates = [-20.0, -33.5, -50.0, -64.0, -80.0, -87.0, -88.0] if act == "silu" else [-3.0, -4.0, -5.0, -6.5, -8.0]
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(len(gates), 2 * cols, generator=g)
    for i, v in enumerate(gates):
        at = torch.randperm(cols, generator=g)[: cols // 2]
        x[i, at] = v * (1 - torch.rand(len(at), generator=g) * 2.0 ** -6)
        x[i, at[0]] = v
        tiny = float(_act64(torch.tensor([v], dtype=torch.float64), act).abs())
        x[i, cols + at] = (torch.randn(len(at), generator=g) * 100 / tiny).clamp(-3e38, 3e38)
    x = x.to(BF)
    q, s = ops.act_mul_halves_int8(x.to(DEV), act)
    y = _act64(x[:, :cols].double(), act) if act == "silu" else _gelu64(x[:, :cols].double())
    y = y * x[:, cols:].double()
    assert (y.abs().amax(1) > 20).all()                # the gates above decide the scale
    for i, v in enumerate(gates):
        rel = 2.0 ** -19 if act == "silu" else (2.0 ** -14 if v >= -3 else (v * v + 8) * 2.0 ** -23)
        _check_quantised(q[i:i + 1], s[i:i + 1], y[i:i + 1], rel)


@pytest.mark.parametrize("cols", [64, 4096, 50, 40000])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gates_at_the_ends_of_the_range(act, cols):
    """Finite gates up to the largest number, of either sign: the activation is the gate or zero, nothing overflows on the way."""
    _lib, ops = _ops()
    top = torch.finfo(BF).max
    x = torch.randn(8, 2 * cols, generator=torch.Generator().manual_seed(cols))
    for i, v in enumerate([top, 2.5e38, 1e30, 129.0, -129.0, -1e30, -2.5e38, -top]):
        x[i, 3], x[i, cols + 3] = v, 0.5
    x = x.to(BF)
    q, s = ops.act_mul_halves_int8(x.to(DEV), act)
    y = (_act64(x[:, :cols].double(), act) if act != "gelu" else _gelu64(x[:, :cols].double())) * x[:, cols:].double()
    assert torch.isfinite(s).all()
    for i in range(8):
        # silu and gelu of gates around 0 as in their own tests; of a gate beyond 128 exact, in all rows that it decides
        _check_quantised(q[i:i + 1], s[i:i + 1], y[i:i + 1], 2.0 ** -14 if act == "gelu" else 2.0 ** -19)


def _gelu64(x):
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))      # 1 + erf(x / sqrt 2) without its cancellation


@pytest.mark.parametrize("n,cols", [(3, 4096), (2, 1003), (2, 33000), (40, 256)])
def test_quantize_rows_is_exact_for_fp32_rows(n, cols):
    """Values next to ties k + 1/2, one to many steps of fp32 above and below, and exact ties: 127 x and (k + 1/2) a are exact in 64
    bits (31 and 32 significant bits), so the expected integer is too."""
    _lib, ops = _ops()
    g = torch.Generator().manual_seed(cols)
    top = (1 + torch.rand(n, 1, generator=g)) * torch.exp2(torch.randint(-120, 120, (n, 1), generator=g).float())
    if n > 9:
        top[9] *= 2.0 ** -30                           # subnormal for the smallest exponents
        top[8] = 2.0 ** -140
    top[0] = 127.0                                     # exact ties exist: x = k + 1/2
    k = torch.randint(0, 127, (n, cols), generator=g).double()
    x = ((k + 0.5) * top.double() / 127).float()
    steps = torch.randint(-3, 4, (n, cols), generator=g)
    far = torch.rand(n, cols, generator=g) < 0.3
    steps = torch.where(far, steps * 37, steps)
    x = (x.view(torch.int32) + steps.to(torch.int32)).clamp_min(0).view(torch.float32)
    x[0, ::3] = (k[0, ::3] + 0.5).float()
    x = torch.minimum(x, top) * (1 - 2 * (torch.rand(n, cols, generator=g) < 0.5).float())
    x[:, cols // 2] = top[:, 0]
    t = 127 * x.double().abs()
    m = (t / top.double()).floor()
    tie = (m + 0.5) * top.double()
    want = (m + ((t > tie) | ((t == tie) & (m % 2 == 1)))) * x.double().sign()
    assert (t == tie).any() and ((t / top.double()) % 1 - 0.5).abs().median() < 2.0 ** -13
    for rows in (x.to(DEV), torch.nn.functional.pad(x.to(DEV), (1, 0))[:, 1:]):       # both kernels
        q, _ = ops.quantize_rows(rows)
        assert torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("tile", [(1, 80), (2, 16), (0, 48)])
def test_a_tile_width_of_the_16_bit_projections_leaves_linear_int8_alone(tile):
    """``GEMM_TILE`` serves both families; widths that only the 16-bit kernels have mean the automatic choice here."""
    _lib, ops = _ops()
    x = torch.randint(-128, 128, (300, 256), dtype=torch.int8, device=DEV)
    w = torch.randint(-128, 128, (512, 256), dtype=torch.int8, device=DEV)
    xs, ws = torch.rand(300, device=DEV), torch.rand(512, device=DEV)
    want = ops.linear_int8(x, xs, w, ws)
    ops.GEMM_TILE = tile
    try:
        assert torch.equal(ops.linear_int8(x, xs, w, ws), want)
    finally:
        ops.GEMM_TILE = (0, 0)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,nh,hkv,D,rot", [(1, 2, 1, 128, 128), (33, 4, 2, 64, 32), (6, 3, 1, 40, 24), (4, 2, 2, 128, 0), (7, 1, 1, 12, 8),
                                           (5, 2, 1, 256, 64)])
def test_rope_append_vectors_of_fp32(n, nh, hkv, D, rot, interleaved):
    """Rows that whole 16-byte vectors of four values fit, on which the vector kernel runs (heads beyond 128: the other one)."""
    test_rope_append(n, nh, hkv, D, rot, torch.float32, interleaved)
