"""Argument refusals of the serving-step entry points, on the CPU: placeholder
addresses are compared and never read, and every case is refused before the
first CUDA call (or has nothing to do).  Host tensors are refused by the torch
front end."""

import ctypes

import pytest
import torch

from hcp_vllm_plugin_b200 import _capi as C
from hcp_vllm_plugin_b200 import ops

OK, INVALID, UNSUPPORTED = 0, 1, 2
BASE = 0x7F0000000000


def _addr(i):
    return BASE + i * 0x10000000


@pytest.fixture(scope="module")
def lib():
    return C.load()


def _args(cls, base, over):
    a = cls()
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return a


PLAN = dict(context_lens=_addr(1), new_lens=_addr(2), pos_base=None, block_table=_addr(3), block_table_stride=8,
            block_table_width=8, free_blocks=_addr(4), num_free=9, free_head=_addr(5), query_start=_addr(6),
            seq_lens=_addr(7), positions=_addr(8), slot_mapping=_addr(9), token_req=_addr(10), kv_lens=_addr(11),
            free_head_out=_addr(12), missing_out=_addr(13), num_reqs=4, block_size=16, num_tokens=4)


@pytest.mark.parametrize("over,want", [
    (dict(num_reqs=-1), INVALID), (dict(num_tokens=-1), INVALID), (dict(block_size=0), INVALID),
    (dict(block_table_width=-1), INVALID), (dict(block_table_stride=7), INVALID), (dict(num_free=-1), INVALID),
    (dict(free_head=None), INVALID), (dict(query_start=None), INVALID), (dict(missing_out=None), INVALID),
    (dict(free_head_out=None), INVALID), (dict(free_head_out=_addr(5)), INVALID), (dict(context_lens=None), INVALID),
    (dict(new_lens=None), INVALID), (dict(seq_lens=None), INVALID), (dict(block_table=None), INVALID),
    (dict(free_blocks=None), INVALID), (dict(positions=None), INVALID), (dict(slot_mapping=None), INVALID),
    (dict(token_req=None), INVALID), (dict(kv_lens=None), INVALID), (dict(num_tokens=1 << 31), UNSUPPORTED),
    (dict(num_free=1 << 31), UNSUPPORTED), (dict(block_table_width=1 << 31, block_table_stride=1 << 31), UNSUPPORTED)])
def test_plan_refusals(lib, over, want):
    assert lib.hcp_kv_plan_step(ctypes.byref(_args(C.HcpStepPlanArgs, PLAN, over)), None) == want
    assert lib.hcp_kv_plan_step(None, None) == INVALID


ROPE = dict(dtype=C.HCP_BF16, num_heads=28, num_kv_heads=4, head_dim=128, q=_addr(1), q_row_stride=28 * 128, k=_addr(2),
            k_row_stride=512, v=_addr(3), v_row_stride=512, q_out=_addr(4), q_out_row_stride=28 * 128, k_out=_addr(5),
            k_out_row_stride=512, positions=_addr(6), num_tokens=4, cos_sin=_addr(7), table_rows=100, table_stride=128,
            table_dtype=C.HCP_F32, rotary=128, interleaved=0, eps=1e-6, q_weight=_addr(8), k_weight=_addr(9),
            kv_cache=_addr(10), slot_mapping=_addr(11), num_blocks=9, block_size=16, cache_kind=C.HCP_ROPE_CACHE_Q4)


@pytest.mark.parametrize("over,want", [
    (dict(num_tokens=0), OK), (dict(num_tokens=-1), INVALID), (dict(num_tokens=1 << 31), UNSUPPORTED),
    (dict(dtype=C.HCP_F32), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(num_heads=0), INVALID),
    (dict(num_kv_heads=-4), INVALID), (dict(num_heads=5000), UNSUPPORTED), (dict(table_dtype=C.HCP_F16), UNSUPPORTED),
    (dict(rotary=0), UNSUPPORTED), (dict(rotary=136), UNSUPPORTED), (dict(rotary=20), UNSUPPORTED),
    (dict(table_stride=120), INVALID), (dict(table_stride=130), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("inf")), INVALID), (dict(eps=float("nan")), INVALID), (dict(table_rows=-1), INVALID),
    (dict(cache_kind=3), INVALID), (dict(block_size=24), UNSUPPORTED), (dict(block_size=0), INVALID),
    (dict(num_blocks=0), INVALID), (dict(kv_cache=None), INVALID), (dict(kv_cache=_addr(10) + 8), INVALID),
    (dict(slot_mapping=None), INVALID), (dict(v=None), INVALID), (dict(v_row_stride=504), INVALID),
    (dict(q=None), INVALID), (dict(q=_addr(1) + 2), INVALID), (dict(q_row_stride=28 * 128 + 4), INVALID),
    (dict(q_row_stride=0), INVALID), (dict(q_out=None), INVALID), (dict(q_out_row_stride=8), INVALID), (dict(k=None), INVALID),
    (dict(k_out=None), INVALID), (dict(k_out=_addr(5) + 8), INVALID), (dict(positions=None), INVALID),
    (dict(cos_sin=None), INVALID), (dict(cos_sin=_addr(7) + 4), INVALID), (dict(q_weight=_addr(8) + 2), INVALID),
    (dict(k_weight=_addr(9) + 4), INVALID)])
def test_norm_rope_refusals(lib, over, want):
    assert lib.hcp_qk_norm_rope(ctypes.byref(_args(C.HcpNormRopeArgs, ROPE, over)), None) == want
    assert lib.hcp_qk_norm_rope(None, None) == INVALID


ROWS = dict(key=_addr(1), value=_addr(2), n=4, ks=512, vs=512, slots=_addr(3), cache=_addr(4), nb=9, bs=16, hkv=4, d=128, dt=C.HCP_BF16)


@pytest.mark.parametrize("over,want", [
    (dict(n=0), OK), (dict(n=-1), INVALID), (dict(n=1 << 31), UNSUPPORTED), (dict(dt=C.HCP_F32), UNSUPPORTED),
    (dict(d=96), UNSUPPORTED), (dict(bs=24), UNSUPPORTED), (dict(bs=256), UNSUPPORTED), (dict(hkv=0), INVALID),
    (dict(hkv=70000), UNSUPPORTED), (dict(nb=0), INVALID), (dict(key=None), INVALID), (dict(value=None), INVALID),
    (dict(slots=None), INVALID), (dict(cache=None), INVALID), (dict(key=_addr(1) + 8), INVALID),
    (dict(cache=_addr(4) + 4), INVALID), (dict(ks=508), INVALID), (dict(vs=516), INVALID)])
def test_q4_rows_refusals(lib, over, want):
    a = {**ROWS, **over}
    assert lib.hcp_kv_cache_update_q4(a["key"], a["value"], a["n"], a["ks"], a["vs"], a["slots"], a["cache"], a["nb"], a["bs"],
                                      a["hkv"], a["d"], a["dt"], None) == want
    assert lib.hcp_kv_cache_gather_q4(a["cache"], a["nb"], a["bs"], a["hkv"], a["d"], a["slots"], a["n"], a["key"], a["value"],
                                      a["ks"], a["vs"], a["dt"], None) == want


DECODE = dict(dtype=C.HCP_BF16, num_heads=28, num_kv_heads=4, head_dim=128, scale=0.1, block_size=16, q=_addr(1), q_rows=3,
              q_row_stride=28 * 128, kv_cache=_addr(2), num_blocks=9, block_table=_addr(3), block_table_rows=3,
              block_table_stride=8, block_table_width=8, kv_lens=_addr(4), token_req=None, out=_addr(5),
              out_row_stride=28 * 128, out_dtype=C.HCP_BF16, lse=_addr(6), lse_stride=3, workspace=_addr(7),
              workspace_bytes=1 << 40)


@pytest.mark.parametrize("over,want", [
    (dict(q_rows=0), OK), (dict(q_rows=-1), INVALID), (dict(q_rows=1 << 31), UNSUPPORTED), (dict(dtype=C.HCP_F32), UNSUPPORTED),
    (dict(head_dim=96), UNSUPPORTED), (dict(num_heads=30), INVALID), (dict(num_heads=68), UNSUPPORTED), (dict(num_kv_heads=0), INVALID),
    (dict(block_size=24), UNSUPPORTED), (dict(out_dtype=C.HCP_F16), UNSUPPORTED), (dict(scale=0.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(q=None), INVALID), (dict(q=_addr(1) + 4), INVALID),
    (dict(q_row_stride=28 * 128 - 8), INVALID), (dict(q_row_stride=28 * 128 + 4), INVALID), (dict(out=None), INVALID),
    (dict(out_row_stride=8), INVALID), (dict(kv_lens=None), INVALID), (dict(kv_cache=None), INVALID),
    (dict(kv_cache=_addr(2) + 8), INVALID), (dict(num_blocks=0), INVALID), (dict(num_blocks=1 << 31), INVALID),
    (dict(block_table=None), INVALID), (dict(block_table_rows=0), INVALID), (dict(block_table_rows=2), INVALID),
    (dict(block_table_width=0), INVALID), (dict(block_table_stride=7), INVALID),
    (dict(block_table_width=1 << 28, block_table_stride=1 << 28), UNSUPPORTED), (dict(lse_stride=2), INVALID)])
def test_decode_q4_refusals(lib, over, want):
    a = _args(C.HcpDecodeQ4Args, DECODE, over)
    assert lib.hcp_decode_q4_splitkv(ctypes.byref(a), None) == want
    need = lib.hcp_decode_q4_workspace_bytes(ctypes.byref(a))
    assert need == -1 if want != OK else need > 0
    assert lib.hcp_decode_q4_splitkv(None, None) == INVALID and lib.hcp_decode_q4_workspace_bytes(None) == -1


def test_decode_q4_workspace(lib):
    """The workspace's size depends on rows and heads, on no length; one that is missing, short or misaligned is refused."""
    need = lib.hcp_decode_q4_workspace_bytes(ctypes.byref(_args(C.HcpDecodeQ4Args, DECODE, {})))
    for over in (dict(num_blocks=10000), dict(block_table_width=5000, block_table_stride=5000)):
        assert lib.hcp_decode_q4_workspace_bytes(ctypes.byref(_args(C.HcpDecodeQ4Args, DECODE, over))) == need
    for over in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(workspace=_addr(7) + 8)):
        assert lib.hcp_decode_q4_splitkv(ctypes.byref(_args(C.HcpDecodeQ4Args, DECODE, over)), None) == INVALID


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    checks = {"hcp_step_plan_args": C.HcpStepPlanArgs, "hcp_norm_rope_args": C.HcpNormRopeArgs, "hcp_decode_q4_args": C.HcpDecodeQ4Args}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "hcp_ring.h"', "int main(void) {"]
    for st, cls in checks.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{f} %zu\\n", offsetof({st}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run([cc, "-I", include, str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for st, cls in checks.items():
        assert int(got[st]) == ctypes.sizeof(cls), st
        for f, _ in cls._fields_:
            assert int(got[f"{st}.{f}"]) == getattr(cls, f).offset, f"{st}.{f}"


def test_host_tensors_are_refused():
    q, k = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    i32, i64 = torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    table, cache = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(ops.kv_cache_q4_shape(3, 2, 16, 64), dtype=torch.uint8)
    calls = [
        lambda: ops.kv_plan_step(i32, i32, table, i32, i32, block_size=16, num_tokens=4),
        lambda: ops.qk_norm_rope(q, k, i64, torch.zeros(9, 64)),
        lambda: ops.kv_cache_update_q4(k, k, cache, i64),
        lambda: ops.kv_cache_gather_q4(cache, i64, torch.bfloat16),
        lambda: ops.decode_splitkv_q4(q, cache, table, i32, scale=1.0, out=q),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="CPU path"):
            call()


def test_q4_cache_shape():
    assert ops.kv_cache_q4_shape(5, 4, 16, 128) == (5, 4, 16, 144) and ops.kv_cache_q4_shape(1, 2, 128, 64) == (1, 2, 128, 72)
    for bad in ((5, 4, 8, 128), (5, 4, 16, 96), (5, 4, 48, 64)):
        with pytest.raises(ValueError):
            ops.kv_cache_q4_shape(*bad)


def test_q4_reference_round_trip():
    """The restatement that the GPU tests compare with: what is written reads back within half a step, bytes of other slots stay."""
    import numpy as np
    import serving_ref as R
    rng = np.random.default_rng(0)
    for dtype, d, bs in ((torch.bfloat16, 128, 32), (torch.float16, 64, 16)):
        x = R.round16(rng.standard_normal((9, 2, d)), dtype)
        cache = rng.integers(0, 256, (2, 2, bs, 9 * d // 8)).astype(np.uint8)
        slots = rng.permutation(2 * bs)[:9]
        before = cache.copy()
        R.write_q4(cache, x, x[::-1], slots, dtype)
        assert np.count_nonzero(cache != before) <= 9 * 2 * 9 * d // 8
        k, v = R.read_q4(cache, slots, dtype)
        for got, ref in ((k, x), (v, x[::-1])):
            g, r = got.reshape(-1, 64), ref.reshape(-1, 64)
            rng_ = (r.max(-1) - r.min(-1))[:, None]
            assert (np.abs(g - r) <= rng_ / 30 * (1 + 2.0 ** -8) + rng_ * 2.0 ** -8).all()
        again = cache.copy()
        R.write_q4(again, x, x[::-1], slots, dtype)
        assert (again == cache).all()
