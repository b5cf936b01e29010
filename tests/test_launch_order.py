"""Kernels that may become resident while the one before them in the stream still runs: read as text, no GPU needed."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "acache_b200" / "csrc"


def _kernels():
    """(file, name, body without comments) of every kernel."""
    out = []
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for at in re.finditer(r"__global__", text):
            rest = text[at.start():]
            begin = rest.index("{")
            name = next(n for n in re.findall(r"(\w+)\s*\(", rest[:begin])
                        if n not in ("__launch_bounds__", "__cluster_dims__", "resident"))
            depth = 0
            for i, c in enumerate(rest[begin:]):
                depth += (c == "{") - (c == "}")
                if depth == 0:
                    break
            out.append((path.name, name, rest[begin + 1:begin + i]))
    return out


CHAINED = [k for k in _kernels() if "chain_release" in k[2]]


def test_kernels_are_found():
    names = {name for _, name, _ in CHAINED}
    assert {"rows_kernel", "wide_parts_kernel", "merge_kernel", "linear_tc_kernel", "quantise_kernel", "rope_append_kernel"} <= names


@pytest.mark.parametrize("file,name,body", CHAINED, ids=[k[1] for k in CHAINED])
def test_every_released_kernel_waits_unconditionally_before_it_reads(file, name, body):
    """The writes of earlier kernels are only promised to a thread that has waited: the wait is a statement of the
    kernel's own block under no condition, and nothing before it reads what a tensor holds."""
    top, depth, found = "", 0, None
    for i, c in enumerate(body):
        depth += (c == "{") - (c == "}")
        if depth == 0:
            top += c
            if top.endswith("chain_wait();"):
                found = i
                break
    assert found is not None, f"{file}: {name} has no wait in its own block"
    before = top[:-len("chain_wait();")].rstrip()
    assert before == "" or before[-1] in ";}", f"{file}: {name} waits under a condition"
    reads = re.findall(r"cp_async16|ld_global_nc|ldg|request_range|slots\[|cu_q\[|tma_load", body[:found])
    assert not reads, f"{file}: {name} reads before it waits: {reads}"
