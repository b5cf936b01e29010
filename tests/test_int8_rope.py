"""Host side of the 8-bit projections and the rotary frequencies: no GPU needed."""
import math

import pytest
import torch


def test_entry_points_validate_without_a_gpu():
    from acache_b200 import _lib

    lib = _lib.load()
    assert lib.acache_quantize_rows(None, 0, 4, 64, 9, None, None, None) == -1            # dtype
    assert lib.acache_quantize_rows(None, 0, 0, 64, 2, None, None, None) == 0             # no rows
    assert lib.acache_quantize_rows(None, 0, 1, 64, 2, None, None, None) == -1            # null pointers
    assert lib.acache_rmsnorm_int8(None, 0, None, 0, None, 1, 0, 1e-5, 2, None, None, None) == -1
    assert lib.acache_act_mul_halves_int8(None, 0, 1, 64, 3, 2, None, None, None) == -1   # activation
    assert lib.acache_linear_int8(None, 0, None, 0, 64, None, None, 64, None, 2, None, 0, 0, None, 0, None, None) == 0
    assert lib.acache_linear_int8(None, 0, None, 1, 64, None, None, 64, None, 0, None, 0, 0, None, 0, None, None) == -2  # fp32 out
    assert lib.acache_linear_int8(None, 0, None, 1, 64, None, None, 64, None, 2, None, 0, 0, None, 0, None, None) == -1
    bad = 1 << 20                                                                         # never dereferenced
    assert lib.acache_linear_int8(bad, 64, bad, 1, 72, bad, bad, 64, None, 2, bad, 64, 0, None, 0, None, None) == -2
    assert lib.acache_linear_int8(bad, 64, bad, 1, 131072, bad, bad, 64, None, 2, bad, 64, 0, None, 0, None, None) == -4
    rope = [None, 0, None, 0, None, 0, 1, 2, 1, 64, 2, None, None, 64, 0, 1.0, None, 0, None, None, None, 0, None, None]
    assert lib.acache_rope_append(*rope) == -1
    rope[6] = 0
    assert lib.acache_rope_append(*rope) == 0
    rope[13] = 66
    assert lib.acache_rope_append(*rope) == -1            # more rotary dimensions than the head has
    rope[13] = 63
    assert lib.acache_rope_append(*rope) == -1            # odd


def test_rope_frequencies():
    from acache_b200.ops import rope_frequencies

    base, one = rope_frequencies(128, 500000.0)
    assert base.dtype == torch.float64 and base.shape == (64,) and one == 1.0
    assert base[0] == 1.0 and math.isclose(base[1].item(), 500000.0 ** (-2 / 128))
    lin, _ = rope_frequencies(128, 500000.0, dict(rope_type="linear", factor=4.0))
    torch.testing.assert_close(lin * 4, base)
    ntk, _ = rope_frequencies(128, 500000.0, dict(rope_type="ntk", factor=4.0))
    assert ntk[0] == 1.0 and math.isclose((base[-1] / ntk[-1]).item(), 4.0, rel_tol=1e-12)     # the slowest pair turns 4x slower
    dyn = dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=4096)
    torch.testing.assert_close(rope_frequencies(128, 500000.0, dyn, seq_len=4096)[0], base)
    assert math.isclose((base[-1] / rope_frequencies(128, 500000.0, dyn, seq_len=8192)[0][-1]).item(), 3.0, rel_tol=1e-12)
    yarn, factor = rope_frequencies(128, 10000.0, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096))
    plain = rope_frequencies(128, 10000.0)[0]
    ratio = plain / yarn
    assert math.isclose(factor, 0.1 * math.log(8.0) + 1) and ratio[0] == 1 and math.isclose(ratio[-1].item(), 8.0, rel_tol=1e-12)
    assert (ratio[1:] >= ratio[:-1] - 1e-12).all()
    turns = 4096 * plain / (2 * math.pi)
    torch.testing.assert_close(ratio[turns > 40], torch.ones_like(ratio[turns > 40]))
    l3, _ = rope_frequencies(128, 500000.0, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                  original_max_position_embeddings=8192))
    wave = 2 * math.pi / base
    torch.testing.assert_close(l3[wave < 8192 / 4], base[wave < 8192 / 4])
    torch.testing.assert_close(l3[wave > 8192] * 8, base[wave > 8192])
    for bad in (dict(rope_type="linear", factor=0.5), dict(rope_type="spiral", factor=2.0, original_max_position_embeddings=1)):
        with pytest.raises(ValueError):
            rope_frequencies(128, 10000.0, bad)
    with pytest.raises(ValueError):
        rope_frequencies(63, 10000.0)


def test_a_default_rope_type_leaves_a_model_as_it_is():
    """What configuration objects answer where no scaling was given: tables and scores are those without one."""
    from acache_b200.model.modeling_common import RopeCache, build_rope_table, rope_score_factor

    want = build_rope_table(5000, 128, 500000.0, torch.float32, "cpu")
    for scaling in (dict(rope_type="default", rope_theta=500000.0), dict(type="default"), {}):
        got = build_rope_table(5000, 128, 500000.0, torch.float32, "cpu", scaling)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert rope_score_factor(128, 500000.0, scaling) == 1.0
        cached = RopeCache(128, 500000.0, torch.float32, scaling).get(5000, "cpu")
        assert torch.equal(cached[1][:5000], want[1])


def test_few_rows_of_a_narrow_projection_with_a_long_k_range_are_sliced():
    """One CTA per 32 columns would stream the whole weight matrix through a few SMs: the K range goes to the tiles that cut
    it into slices, whose sums need scratch."""
    from acache_b200 import _lib

    need = _lib.load().acache_linear_int8_scratch_bytes
    for rows, k, out in ((1, 131056, 64), (3, 131056, 32), (16, 32768, 256), (32, 16384, 1024), (64, 12288, 4096)):
        assert need(rows, k, out, 0) >= 2 * rows * out * 4, (rows, k, out)
    for rows, k, out in ((1, 4096, 4096), (16, 12288, 4096), (33, 4096, 4096), (32, 18944, 3584)):
        assert need(rows, k, out, 0) == 0, (rows, k, out)
