"""CPU tests of the serving-step operators' edges: rules their sources keep, and
refusals of the C entry points (placeholder addresses are compared and never read)."""

import ctypes
import os
import re

import pytest

from hcp_vllm_plugin_b200 import _capi as C
from hcp_vllm_plugin_b200 import build as B


def test_chained_kernels_read_nothing_as_constant():
    """A kernel launched as a programmatic dependent may be resident while the one before it writes, so
    its loads of global memory have to be ordinary ones: no read-only path, asked for or implied."""
    chained = []
    for name in sorted(os.listdir(B.CSRC)):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(B.CSRC, name)).read())
        if name.endswith(".cuh") and "chain_wait()" in text and name != "sm100_ptx.cuh":
            chained.append(name)
            for word in ("__ldg", "ld.global.nc", "__restrict__", "tex1Dfetch"):
                assert word not in text, (name, word)
    assert chained == ["decode_q4.cuh", "norm_rope.cuh", "q4_cache.cuh", "step_plan.cuh"]
