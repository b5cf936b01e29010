"""Runner -> attention side channel and small helpers.

The engine publishes the ragged-batch metadata of the step it is about to run
through one process-global ``Context``; every attention layer reads it.  Field
names and order follow the reference (reference: nano-vdllm/utils.py:7-59).
"""
from __future__ import annotations

import random
from dataclasses import dataclass

import numpy as np
import torch


@dataclass
class Context:
    is_caching: bool = False
    cu_seqlens_q: torch.Tensor | None = None
    cu_seqlens_k: torch.Tensor | None = None
    seqlens: torch.Tensor | None = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: torch.Tensor | None = None
    block_tables: torch.Tensor | None = None
    use_acache: bool = False
    read_slot_mapping: torch.Tensor | None = None
    shared_kv_lens: torch.Tensor | None = None
    affix_shifts: torch.Tensor | None = None
    # not in the reference: the engine guarantees that all requests of this step name the shared
    # span the same way (see model_runner.attention_read_runs), attention may stage it per group
    group_shared_span: bool = False
    # not in the reference: (slots of the span that all requests of this step share, keep-mask words); the read map
    # then names each request's other keys only and attention multiplies the span once for all requests
    shared_prefix: tuple | None = None


_CONTEXT = Context()


def get_context() -> Context:
    return _CONTEXT


def set_context(
    is_caching,
    cu_seqlens_q=None,
    cu_seqlens_k=None,
    seqlens=None,
    max_seqlen_q=0,
    max_seqlen_k=0,
    slot_mapping=None,
    block_tables=None,
    use_acache=False,
    read_slot_mapping=None,
    shared_kv_lens=None,
    affix_shifts=None,
):
    global _CONTEXT
    _CONTEXT = Context(
        is_caching=is_caching,
        cu_seqlens_q=cu_seqlens_q,
        cu_seqlens_k=cu_seqlens_k,
        seqlens=seqlens,
        max_seqlen_q=max_seqlen_q,
        max_seqlen_k=max_seqlen_k,
        slot_mapping=slot_mapping,
        block_tables=block_tables,
        use_acache=use_acache,
        read_slot_mapping=read_slot_mapping,
        shared_kv_lens=shared_kv_lens,
        affix_shifts=affix_shifts,
    )


def reset_context():
    global _CONTEXT
    _CONTEXT = Context()


def add_gumbel_noise(logits, temperature):
    """Gumbel-max perturbation used for temperature sampling; identity at
    temperature 0 (reference: nano-vdllm/utils.py:61-72)."""
    if temperature == 0:
        return logits
    u = torch.rand_like(logits, dtype=logits.dtype)
    return logits.exp() / (-torch.log(u)) ** temperature


def set_seed(seed):
    torch.manual_seed(seed)
    random.seed(seed)
    np.random.seed(seed)
    torch.backends.cudnn.deterministic = True
    torch.backends.cudnn.benchmark = False
