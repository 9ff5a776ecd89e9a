"""Kernels that may be launched while the previous kernel of the stream still runs: each has to wait for it before it
touches global memory.  Read from the sources, since a missing wait is a race that a run need not show."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transarch_b200", "csrc")


def _strip(text):
    return re.sub(r"/\*.*?\*/", " ", re.sub(r"//[^\n]*", " ", text), flags=re.S)


def _body(text, name):
    """Body of the __global__ function `name`."""
    at = re.search(r"__global__[^;{]*?\b" + name + r"\s*\(", text)
    assert at, f"{name} is not defined beside its launch"
    start = i = text.index("{", at.end())
    depth = 0
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]
        i += 1


def _chained():
    """(file, kernel) of every kernel that launch_chained, or a launch with the attribute written out, may start."""
    out = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = _strip(open(path).read())
        for name in sorted(set(re.findall(r"__global__[^;{]*?\b(\w+_kernel)\s*\(", text))):
            if "cudaLaunchKernelEx" in text or re.search(r"launch_chained\s*\([^;]*\b" + name + r"\b", text):
                out.append((os.path.basename(path), name))
    return out


def test_there_are_kernels_to_look_at():
    names = {n for _, n in _chained()}
    assert {"draft_tree_masks_kernel", "latent_write_kernel", "sparse_mla_cached_few_kernel", "mla_merge_kernel",
            "fp8_block_gemm_wide_kernel", "fp8_quantise_rows_kernel", "topk_select_kernel"} <= names


@pytest.mark.parametrize("path,name", _chained())
def test_waits_before_it_touches_global_memory(path, name):
    body = _body(_strip(open(os.path.join(CSRC, path)).read()), name)
    assert "pdl_wait_prior()" in body
    before = body[:body.index("pdl_wait_prior()")]
    assert "__ldg" not in before and "return" not in before and "atomic" not in before
