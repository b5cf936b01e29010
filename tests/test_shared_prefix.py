"""Host side of shared-prefix attention: no GPU needed."""
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


def _args(**changed):
    at = 1 << 20                                       # aligned, never dereferenced: every call here is refused or empty
    args = dict(q=at, q_stride=256, out=at, o_stride=256, k=at, v=at, num_slots=64, total_q=4, n_heads=4, n_kv_heads=2, head_dim=64,
                dtype=2, prefix_slots=at, prefix_len=10, keep=None, keep_stride=2, cu_q=at, cu_k=at, batch=2, max_q=2, max_k=4,
                read=at, n_slots=8, scale=0.125, scratch=at, scratch_bytes=0, err=None, stream=None)
    assert not set(changed) - set(args)
    return list({**args, **changed}.values())


EINVAL, EUNSUPPORTED, ELIMIT = -1, -2, -4


@pytest.mark.parametrize("changed,code", [
    ({}, EINVAL),                                      # no scratch
    ({"scale": 0.0}, EINVAL), ({"scale": -0.125}, EINVAL), ({"scale": float("nan")}, EINVAL), ({"scale": float("inf")}, EINVAL),
    ({"scale": 3e38}, EINVAL),                         # infinite in the kernels' base 2
    ({"n_heads": 3}, EINVAL), ({"q": None}, EINVAL), ({"read": None}, EINVAL), ({"prefix_slots": None}, EINVAL), ({"dtype": 9}, EINVAL),
    ({"keep": 1 << 20, "keep_stride": 1}, EINVAL), ({"keep": (1 << 20) + 4}, EINVAL), ({"keep": 1 << 20, "prefix_len": 65}, EINVAL),
    ({"head_dim": 96}, EUNSUPPORTED), ({"dtype": 0}, EUNSUPPORTED), ({"q_stride": 260}, EUNSUPPORTED), ({"q": (1 << 20) + 2}, EUNSUPPORTED),
    ({"batch": 2048}, ELIMIT), ({"total_q": (1 << 22) + 1}, ELIMIT),
    ({"total_q": 0}, 0), ({"batch": 0}, 0), ({"max_q": 0}, 0)])
def test_calls_that_are_refused_or_empty(changed, code):
    from acache_b200 import _lib

    lib = _lib.load()
    big = 1 << 60 if changed.get("scale") is not None else 0      # enough scratch: the scale alone is at fault
    assert lib.acache_shared_prefix_attention(*_args(**{"scratch_bytes": big, **changed})) == code


def test_scratch_bytes():
    from acache_b200 import _lib

    need = _lib.load().acache_shared_prefix_attention_scratch_bytes
    assert need(0, 4, 2, 64, 1, 1, 1, 1) == 0 and need(4, 3, 2, 64, 1, 1, 1, 1) == 0
    for sizes in ((1, 1, 1, 64, 1, 1, 0, 0), (1024, 32, 32, 128, 32, 32, 800, 8192), (64, 28, 4, 128, 64, 1, 100, 32768)):
        total_q, nh, _, D = sizes[:4]
        row = total_q * nh * (D + 1) * 4
        assert need(*sizes) % row == 0 and need(*sizes) >= 2 * row
        assert need(*sizes[:5], 1 << 30, *sizes[6:]) == need(*sizes[:5], total_q, *sizes[6:])   # a request has at most all queries


@pytest.mark.parametrize("sizes", [(4, 4, 2, 64, 2, 0, 4, 10), (4, 4, 2, 64, 2, 0, 0, 0), (300, 28, 4, 128, 8, 0, 1024, 32768)])
def test_requests_without_queries_need_no_scratch(sizes):
    """A padded batch: rows of q, but no request has one.  In a process of its own: an integer division by zero ends it."""
    import subprocess
    import sys

    code = f"from acache_b200 import _lib; assert _lib.load().acache_shared_prefix_attention_scratch_bytes(*{sizes}) == 0"
    assert subprocess.run([sys.executable, "-c", code], cwd=REPO).returncode == 0


@pytest.mark.parametrize("sizes,kernels", [
    ((4, 4, 2, 64, 2, 0, 4, 10), 0),                   # nothing to compute
    ((4, 4, 2, 64, 4, 1, 100, 0), 1),                  # no prefix, the own part writes the output
    ((64, 28, 4, 128, 64, 1, 1024, 32768), 2),         # the own part merges in place
    ((4, 4, 2, 64, 4, 1, 100000, 0), 2),               # few long ranges and their merge
    ((1024, 28, 4, 128, 32, 32, 700, 8192), 3)])       # own rows that fill the wide tiles
def test_the_number_of_kernels_that_a_call_launches(sizes, kernels):
    import ctypes

    from acache_b200 import _lib

    lib, n = _lib.load(), ctypes.c_int32(-1)
    nbytes = lib.acache_shared_prefix_attention_plan(*sizes, ctypes.byref(n))
    assert n.value == kernels
    assert nbytes == lib.acache_shared_prefix_attention_scratch_bytes(*sizes) == lib.acache_shared_prefix_attention_plan(*sizes, None)
