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


def _addr(i):
    return 0x7F0000000000 + i * 0x10000000


def _args(cls, base, over):
    a = cls()
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return a


PLAN = dict(context_lens=_addr(1), new_lens=_addr(2), pos_base=_addr(14), block_table=_addr(3), block_table_stride=24,
            block_table_width=8, free_blocks=_addr(4), num_free=9, free_head=_addr(5), query_start=_addr(6),
            seq_lens=_addr(7), positions=_addr(8), slot_mapping=_addr(9), token_req=_addr(10), kv_lens=_addr(11),
            free_head_out=_addr(12), missing_out=_addr(13), num_reqs=4, block_size=16, num_tokens=6)


@pytest.mark.parametrize("over", [
    dict(seq_lens=_addr(1)), dict(seq_lens=_addr(2)), dict(seq_lens=_addr(14) + 12), dict(query_start=_addr(1) - 16),
    dict(query_start=_addr(2) + 12), dict(token_req=_addr(1)), dict(kv_lens=_addr(1) - 20), dict(positions=_addr(4)),
    dict(slot_mapping=_addr(4) - 40), dict(missing_out=_addr(5)), dict(missing_out=_addr(4) + 32), dict(free_head_out=_addr(1)),
    dict(missing_out=_addr(12)), dict(seq_lens=_addr(6) + 16), dict(kv_lens=_addr(10) + 20), dict(slot_mapping=_addr(8) + 40),
    dict(seq_lens=_addr(3)), dict(context_lens=_addr(3) + 4 * (24 + 7)), dict(free_blocks=_addr(3) + 4 * (3 * 24 - 8)),
    dict(positions=_addr(3) - 44), dict(free_head_out=_addr(3) + 4 * (3 * 24 + 7))])
def test_plan_outputs_may_not_overlap(over):
    """Blocks sum the lengths while others write the results: an output in the place of an input (or of
    another output) is refused; advancing the lengths in place is the obvious one."""
    a = _args(C.HcpStepPlanArgs, PLAN, over)
    assert C.load().hcp_kv_plan_step(ctypes.byref(a), None) == 1



# q, k and v of one projection: 8 query heads, 2 KV heads of 128 dims, rows of 12 heads
QKV = _addr(1)
ROPE = dict(dtype=C.HCP_BF16, num_heads=8, num_kv_heads=2, head_dim=128, q=QKV, q_row_stride=1536, k=QKV + 2048,
            k_row_stride=1536, v=QKV + 2560, v_row_stride=1536, q_out=_addr(4), q_out_row_stride=1024, k_out=_addr(5),
            k_out_row_stride=256, positions=_addr(6), num_tokens=4, cos_sin=_addr(7), table_rows=100, table_stride=128,
            table_dtype=C.HCP_F32, rotary=128, interleaved=0, eps=1e-6, q_weight=_addr(8), k_weight=_addr(9),
            kv_cache=_addr(10), slot_mapping=_addr(11), num_blocks=9, block_size=16, cache_kind=C.HCP_ROPE_CACHE_SAME)


@pytest.mark.parametrize("over", [
    dict(v=QKV + 2048, k_out=QKV + 2048, k_out_row_stride=1536),        # values in the place of the keys' results
    dict(k_out=QKV + 2560, k_out_row_stride=1536),                      # the keys' results in the place of the values
    dict(k_out=QKV + 2560, k_out_row_stride=1536, cache_kind=C.HCP_ROPE_CACHE_Q4),
    dict(k_out=QKV + 2304, k_out_row_stride=1536), dict(k_out=QKV, k_out_row_stride=1536),
    dict(q_out=QKV + 256, q_out_row_stride=1536), dict(q_out=QKV, q_out_row_stride=1024),
    dict(q_out=QKV + 1024, q_out_row_stride=1536), dict(k_out=QKV + 2048, k_out_row_stride=256),
    dict(k_out=_addr(4) + 512, k_out_row_stride=1024), dict(q_out=_addr(5) - 2048, q_out_row_stride=1024)])
def test_norm_rope_outputs_may_not_overlap_other_rows(over):
    """Results may stand in the place of their own inputs; anywhere else in q, k or v, or in each other,
    what is read depends on what was written before."""
    assert C.load().hcp_qk_norm_rope(ctypes.byref(_args(C.HcpNormRopeArgs, ROPE, over)), None) == 1


DECODE = dict(dtype=C.HCP_BF16, num_heads=28, num_kv_heads=4, head_dim=128, scale=0.1, block_size=16, q=_addr(1), q_rows=3,
              q_row_stride=28 * 128, kv_cache=_addr(2), num_blocks=9, block_table=_addr(3), block_table_rows=3,
              block_table_stride=8, block_table_width=8, kv_lens=_addr(4), token_req=None, out=_addr(5),
              out_row_stride=28 * 128, out_dtype=C.HCP_BF16, lse=_addr(6), lse_stride=3, workspace=_addr(7),
              workspace_bytes=1 << 40)


@pytest.mark.parametrize("scale,taken", [(1e-44, True), (2e38, True), (2.4e38, False), (3.4e38, False)])
def test_decode_q4_scale_range(scale, taken):
    """Scores are kept in powers of two: a scale times log2(e) has to be finite in 32 bits."""
    a = _args(C.HcpDecodeQ4Args, DECODE, dict(scale=scale))
    assert (C.load().hcp_decode_q4_workspace_bytes(ctypes.byref(a)) > 0) == taken
    if not taken:
        assert C.load().hcp_decode_q4_splitkv(ctypes.byref(a), None) == 1


@pytest.mark.parametrize("over", [
    dict(out=_addr(1) + 256), dict(out=_addr(1), out_dtype=C.HCP_F32), dict(out=_addr(1), out_row_stride=2 * 28 * 128),
    dict(out=_addr(1) + 28 * 256 - 16), dict(lse=_addr(1)), dict(lse=_addr(5) + 1024), dict(out=_addr(1), lse=_addr(1))])
def test_decode_q4_results_may_not_overlap(over):
    """Pieces of a row end at different times: a result may replace its own query row, and nothing else that is read."""
    assert C.load().hcp_decode_q4_splitkv(ctypes.byref(_args(C.HcpDecodeQ4Args, DECODE, over)), None) == 1


@pytest.mark.parametrize("value", [0, 256, -16, 3 * 1024 + 1008])
def test_gather_q4_results_may_not_overlap(value):
    key = _addr(1)
    assert C.load().hcp_kv_cache_gather_q4(_addr(4), 9, 16, 4, 128, _addr(3), 4, key, key + value, 512, 512, C.HCP_BF16, None) == 1
