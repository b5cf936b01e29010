"""Capturing the block-decode forward when the host gets in its way."""
import gc
import random
import warnings

import pytest
import torch

from test_decode_layer_gpu import BF, DEV, _arch
from test_engine_gpu import _llada, _random_requests, _serve_config

pytestmark = pytest.mark.gpu


def _setup():
    from oracle.models import random_state_dict

    arch = _arch("llada")
    rng = random.Random(3)
    affix = [rng.randint(1, 170) for _ in range(40)]
    reqs = _random_requests(rng, arch, 4, 40, 16, ["prefix"], affix)
    hf_cfg, model = _llada(arch, random_state_dict(arch, seed=2, std=0.2), BF)
    return arch, reqs, hf_cfg, model


def _serve(arch, reqs, hf_cfg, model, graphs, in_capture=None):
    from acache_b200 import _lib
    from acache_b200.model_runner import ModelRunner
    from acache_b200.sequence import Sequence

    cfg = _serve_config(hf_cfg, arch, "llada", BF, threshold=0.6, max_num_seqs=4, num_kvcache_blocks=40, cache_block_size=64,
                        block_length=8, gen_length=16, use_cuda_graphs=graphs)
    runner = ModelRunner(model, cfg)
    real = runner._decode_forward

    def forward(*a, **k):
        out = real(*a, **k)
        if in_capture is not None and torch.cuda.is_current_stream_capturing():
            in_capture()
        return out

    runner._decode_forward = forward
    seqs = [Sequence(r["prompt"], block_length=8, gen_length=16, cache_block_size=64, mask_id=arch.mask_id,
                     prompt_affix_start=r["affix_start"], prompt_affix_end=r["affix_end"],
                     generation_start=r["generation_start"]) for r in reqs]
    outs, _ = runner.generate_with_acache(seqs)
    _lib.check_device_errors()
    return outs, cfg


def test_a_cyclic_collection_falls_into_a_capture():
    """Garbage that holds another graph, and enough allocations inside the capture for an automatic collection: the other graph
    may not be destroyed before the capture has ended."""
    setup = _setup()
    want, _ = _serve(*setup, graphs=False)
    calls = []

    class Holder:
        pass

    def garbage():
        calls.append(1)
        for _ in range(50):
            [[] for _ in range(100)]

    old = gc.get_threshold()
    gc.collect()
    gc.set_threshold(10 ** 6)                          # the holder stays in the youngest generation until the capture
    holder = Holder()
    holder.me = holder
    holder.graph = torch.cuda.CUDAGraph()
    x = torch.zeros(8, device=DEV)
    with torch.cuda.graph(holder.graph):
        x.add_(1)
    del holder                                         # garbage from here on

    def in_capture():
        gc.set_threshold(20, 1, 1)
        garbage()

    try:
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            got, cfg = _serve(*setup, graphs=True, in_capture=in_capture)
    finally:
        gc.set_threshold(*old)
    assert calls and cfg.use_cuda_graphs and got == want


def test_serving_goes_on_eagerly_when_a_capture_is_refused():
    """A host call that no capture allows ends the capture with an error: one warning, and the tokens of eager serving."""
    setup = _setup()
    want, _ = _serve(*setup, graphs=False)

    def refused():
        with pytest.raises(RuntimeError):
            torch.cuda.synchronize()

    before = torch.cuda.current_stream()
    with pytest.warns(UserWarning, match="capture of the decode forward failed"):
        got, cfg = _serve(*setup, graphs=True, in_capture=refused)
    assert not cfg.use_cuda_graphs and got == want
    assert torch.cuda.current_stream() == before
