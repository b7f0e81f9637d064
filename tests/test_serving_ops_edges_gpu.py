"""GPU tests of the serving-step operators where single calls went wrong or could:
values of very different sizes, neighbours in a stream, calls that fail, captures."""

import numpy as np
import pytest
import torch

import serving_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from hcp_vllm_plugin_b200 import _capi, ops
    _capi.load()
    yield ops
    assert _capi.device_status() == 0


def _i32(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


# ------------------------------------------------------------------ values of very different sizes

def _check_by_weight(got, lse, q, k, v, scale, dtype, what, rounded=1.08 * 2.0 ** -11):
    """One row against 64 bits, each key's share of the bar in proportion to its own weight.

    With p_j the softmax weights and top_j the largest |v| of key j's 64 dims: a score is off by at most
    dx = 2^-17 scale sum_d |q_d| max_j |k_jd| (64 products summed in 32 bits per group, then the groups),
    which moves the result by at most (e^(2 dx) - 1) sum p_j top_j; ex2 by 2^-21, and 2^-15 covers it and the
    normalisation.  p_j s_j is rounded to 11 bits, off by 2^-11 p_j s_j |n_j - 8|, where 8 s_j <= 1.08 top_j
    (15 s_j is the range, at most 2 top_j, rounded by 2^-8); below fp16's normal numbers it is off by 2^-25 of
    a unit that is at most 2^-8 of the largest p s, so by 8 n 2^-33 max p_j s_j <= n 2^-32 sum p_j top_j in all.
    Each of a tile's sums rounds by 2^-23 of what is summed, n / 16 tiles of them twice."""
    n, group = k.shape[0], q.shape[0] // k.shape[1]
    for i in range(q.shape[0]):
        kh, vh = k[:, i // group], v[:, i // group]
        x = kh @ q[i] * scale
        m = x.max()
        p = np.exp(x - m)
        total = p.sum()
        o = p @ vh / total
        top = np.repeat(np.abs(vh).reshape(n, -1, 64).max(-1), 64, axis=1)
        held = p @ top / total
        dx = 2.0 ** -17 * scale * (np.abs(q[i]) * np.abs(kh).max(0)).sum()
        slack = held * (np.expm1(2 * dx) + rounded + 2.0 ** -15 + n / 8 * 2.0 ** -23 + n * 2.0 ** -32)
        eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        bar = slack + eps * (np.abs(o) + slack) + (2.0 ** -25 if dtype == F16 else 0.0)
        assert (np.abs(got[i] - o) <= bar).all(), (what, i, np.max(np.abs(got[i] - o) / bar))
        ref = m + np.log(total)
        assert abs(lse[i] - ref) <= dx + 2.0 ** -20 * (abs(ref) + 1) + n / 16 * 2.0 ** -24, (what, i)


@pytest.mark.parametrize("h,hkv,d,dtype", [(28, 4, 128, BF16), (14, 2, 64, F16), (32, 2, 128, BF16), (12, 1, 64, BF16)])
@pytest.mark.parametrize("case", ["first", "inside", "no weight", "falling"])
def test_decode_q4_large_values_without_weight(ops, case, h, hkv, d, dtype):
    """A value far larger than the others whose key has next to no weight, or had one until a better key came,
    costs the others nothing.  Rows are many, so that one warp passes over many tiles of a row."""
    gen = torch.Generator().manual_seed(h + d)
    rows, bs, nb = 48, 16, 60
    n = nb * bs - 5
    small, large = (2.0 ** -14, 2.0 ** 14) if dtype == F16 else (1.0, 2.0 ** 34)
    k, v = torch.randn(n, hkv, d, generator=gen), torch.randn(n, hkv, d, generator=gen)
    q = 1 + 0.25 * torch.randn(rows, h, d, generator=gen)
    if case == "falling":   # scores rise from -40 to 0 while values fall
        line = torch.linspace(0, 1, n)[:, None, None]
        k = 0.25 * k - (1 - line) * 40 / d ** 0.5
        v = v * small * (large / small) ** (1 - line)
    else:
        at = [0] if case == "first" else [5, 400, 401, n - 1]
        v *= small
        for j in at:
            k[j] = -(200.0 if case == "no weight" else 45.0) / d ** 0.5
            v[j] *= large / small
    k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k.cuda(), v.cuda(), cache, torch.arange(n, device="cuda"))
    kq, vq = R.read_q4(cache.cpu().numpy(), np.arange(n), dtype)
    table, lens, req = torch.arange(nb, dtype=torch.int32, device="cuda").view(1, nb), _i32([n] * rows), _i32([0] * rows)
    for kind in (dtype, torch.float32):
        out, lse = torch.zeros(rows, h, d, dtype=kind, device="cuda"), torch.zeros(h, rows, device="cuda")
        ops.decode_splitkv_q4(q.cuda(), cache, table, lens, scale=d ** -0.5, out=out, lse=lse, token_req=req)
        o, l = R.f64(out), R.f64(lse)
        for r in range(0, rows, 7):
            _check_by_weight(o[r], l[:, r], R.f64(q[r]), kq, vq, d ** -0.5, kind, (case, r))


# ------------------------------------------------------------------ neighbours in a stream

def test_decode_right_after_the_plan_sees_its_pages(ops):
    """Attention as the kernel right behind the plan, over a table whose new entries stand beside old ones."""
    gen = torch.Generator().manual_seed(30)
    reqs, width, h, hkv, d, bs = 200, 24, 28, 4, 128, 16
    nb = reqs * width
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    rows = torch.randn(4096, hkv, d, generator=gen).to(BF16).cuda()
    for at in range(0, nb * bs, 4096):
        n = min(4096, nb * bs - at)
        ops.kv_cache_update_q4(rows[:n], rows[:n].flip(0), cache, torch.arange(at, at + n, device="cuda"))
    q, free = torch.randn(reqs, h, d, generator=gen).to(BF16).cuda(), torch.randperm(nb, generator=gen).int().cuda()
    head = torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.full((reqs, width), -1, dtype=torch.int32, device="cuda")
    held, outs, wants = np.zeros(reqs, np.int64), [], []
    for step in range(12):
        new = torch.randint(0, 33, (reqs,), generator=gen).numpy()
        ctx, add = _i32(held), _i32(new)
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        plan = ops.kv_plan_step(ctx, add, table, free, head, block_size=bs, num_tokens=reqs)
        ops.decode_splitkv_q4(q, cache, table, plan.seq_lens, scale=d ** -0.5, out=out)
        torch.cuda.synchronize()
        want = torch.zeros_like(q)
        ops.decode_splitkv_q4(q, cache, table.clone(), plan.seq_lens.clone(), scale=d ** -0.5, out=want)
        outs.append(out), wants.append(want)
        held, head = held + new, plan.free_head.clone()
        assert plan.missing.item() == 0
    for a, b in zip(outs, wants):
        assert torch.equal(a, b)


def test_plan_takes_vectors_between_the_rows_of_a_table(ops):
    """Rows of a wider buffer may hold the step's other vectors behind their table entries: nothing is shared."""
    reqs, width, wide, bs = 5, 6, 20, 16
    buf = torch.full((reqs, wide), -1, dtype=torch.int32, device="cuda")
    context, new = np.array([0, 20, 33, 7, 64]), np.array([5, 1, 20, 0, 9])
    buf[0, 8:13], buf[2, 10:15], buf[4, 7:8] = _i32(context), _i32(new), 2
    table = np.full((reqs, width), -1, np.int32)
    for i, c in enumerate(context):
        table[i, : -(-c // bs)] = 100 + 10 * i + np.arange(-(-c // bs))
    buf[:, :width] = _i32(table)
    free = np.arange(40, 60)
    want = R.plan(context, new, table, free, 2, bs, 40)
    got = ops.kv_plan_step(buf[0, 8:13], buf[2, 10:15], buf[:, :width], _i32(free), buf[4, 7:8], block_size=bs, num_tokens=40)
    for name, t in got._asdict().items():
        np.testing.assert_array_equal(t.cpu().numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(buf[:, :width].cpu().numpy(), want["block_table"])


# ------------------------------------------------------------------ calls that fail on the host

class _Driver:
    """The few driver calls that make a launch fail without reaching the GPU."""

    def __init__(self):
        import ctypes
        self.lib, self.byref, self.ptr = ctypes.CDLL("libcuda.so.1"), ctypes.byref, ctypes.c_void_p
        torch.zeros(1, device="cuda")  # torch's context is the current one

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = self.ptr()
        self("cuStreamCreate", self.byref(s), 0)
        return s


def _plan_args(keep):
    """Arguments of a small plan, and the tensors behind them."""
    from hcp_vllm_plugin_b200 import _capi as C
    i32 = lambda *x: keep.append(torch.tensor(x, dtype=torch.int32, device="cuda")) or keep[-1].data_ptr()  # noqa: E731
    i64 = lambda n: keep.append(torch.zeros(n, dtype=torch.int64, device="cuda")) or keep[-1].data_ptr()  # noqa: E731
    return C.HcpStepPlanArgs(context_lens=i32(3, 4), new_lens=i32(1, 1), block_table=i32(7, 8), block_table_stride=1,
                             block_table_width=1, free_blocks=i32(9), num_free=1, free_head=i32(0), query_start=i32(0, 0, 0),
                             seq_lens=i32(0, 0), positions=i64(2), slot_mapping=i64(2), token_req=i32(0, 0), kv_lens=i32(0, 0),
                             free_head_out=i32(0), missing_out=i32(0), num_reqs=2, block_size=16, num_tokens=2)


def test_a_failed_launch_is_reported_once(ops):
    """A launch that the runtime refuses is that call's error, and no later call's."""
    import ctypes

    from hcp_vllm_plugin_b200 import _capi as C
    lib, cu, keep = C.load(), _Driver(), []
    a = _plan_args(keep)
    k = torch.ones(2, 2, 64, dtype=BF16, device="cuda")
    cache = torch.zeros(1, 2, 16, 128, dtype=BF16, device="cuda")
    slots = torch.arange(2, device="cuda")
    torch.cuda.synchronize()
    # a stream that waits for the legacy one is being captured: nothing can be launched into the legacy stream
    s, graph = cu.stream(), cu.ptr()
    cu("cuStreamBeginCapture_v2", s, 0)
    rc = lib.hcp_kv_plan_step(ctypes.byref(a), None)
    cu.lib.cuStreamEndCapture(s, cu.byref(graph))
    cu("cuStreamDestroy_v2", s)
    assert rc not in (0, 1, 2), rc
    ops.kv_cache_update(k, k, cache, slots)
    torch.cuda.synchronize()
    assert bool((cache[0, :, :2] == 1).all())
    assert lib.hcp_kv_plan_step(ctypes.byref(a), None) == 0


def test_a_captured_stream_of_another_context_takes_nothing(ops):
    """Kernels go to the current context alone: a captured stream of another one gets no launch, and the
    calls after it are not affected."""
    import ctypes

    from hcp_vllm_plugin_b200 import _capi as C
    lib, cu, keep = C.load(), _Driver(), []
    a = _plan_args(keep)
    torch.cuda.synchronize()
    other, popped, graph = cu.ptr(), cu.ptr(), cu.ptr()
    cu("cuCtxCreate_v2", cu.byref(other), 0, 0)   # current now
    s = cu.stream()
    cu("cuStreamBeginCapture_v2", s, 2)
    cu("cuCtxPopCurrent_v2", cu.byref(popped))
    rc = lib.hcp_kv_plan_step(ctypes.byref(a), s)
    cu("cuCtxPushCurrent_v2", other)
    cu.lib.cuStreamEndCapture(s, cu.byref(graph))
    cu("cuStreamDestroy_v2", s)
    cu("cuCtxPopCurrent_v2", cu.byref(popped))
    cu("cuCtxDestroy_v2", other)
    assert rc != 0
    assert lib.hcp_kv_plan_step(ctypes.byref(a), None) == 0
    torch.cuda.synchronize()


def test_a_captured_stream_of_another_device_is_refused(ops):
    """As outside of captures (HCP_ERR_INVALID), before anything is launched: the capture goes on."""
    import ctypes

    from hcp_vllm_plugin_b200 import _capi as C
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    lib, keep = C.load(), []
    a = _plan_args(keep)
    torch.cuda.synchronize()
    x, graph = torch.zeros(4, device="cuda:1"), torch.cuda.CUDAGraph()
    with torch.cuda.device(1):
        with torch.cuda.graph(graph):
            stream = torch.cuda.current_stream().cuda_stream
            with torch.cuda.device(0):
                rc = lib.hcp_kv_plan_step(ctypes.byref(a), stream)
            x += 1
        graph.replay()
        torch.cuda.synchronize()
    assert rc == 1 and x.tolist() == [1.0] * 4


def test_every_entry_point_can_be_captured(ops):
    """The attention, merge and 16-bit cache calls in one graph, replayed on new inputs: as eager, bit for bit."""
    from hcp_vllm_plugin_b200 import _capi as C
    gen = torch.Generator().manual_seed(31)
    t, keys, h, hkv, d, bs = 300, 400, 28, 4, 128, 16
    fresh = lambda *shape: torch.randn(*shape, generator=gen).to(BF16).cuda()  # noqa: E731
    q, k, v, kc, vc = fresh(t, h, d), fresh(keys, hkv, d), fresh(keys, hkv, d), fresh(t, hkv, d), fresh(t, hkv, d)
    cache, slots = torch.zeros(40, hkv, bs, 2 * d, dtype=BF16, device="cuda"), torch.randperm(640, generator=gen)[:t].cuda()
    oa, ob, out = (torch.zeros(t, h, d, dtype=BF16, device="cuda") for _ in range(3))
    la, lb, lse = (torch.zeros(h, t, device="cuda") for _ in range(3))
    many, many_lse = torch.zeros(2, t, h, d, device="cuda"), torch.zeros(2, h, t, device="cuda")
    joined = torch.zeros(t, h, d, dtype=BF16, device="cuda")

    def run():
        ops.kv_cache_update(kc, vc, cache, slots)
        kg, vg = ops.kv_cache_gather(cache, slots)
        ops.ring_attn_fwd(q, ops.make_work([(0, t, 0, 0, (C.HCP_SRC_A, 0, keys, -1), None)]), scale=0.1, num_kv_heads=hkv,
                          out=oa, lse=la, k_a=k, v_a=v)
        ops.ring_attn_fwd(q, ops.make_work([(0, t, 0, 0, (C.HCP_SRC_A, 0, t, 0), None)]), scale=0.1, num_kv_heads=hkv,
                          out=ob, lse=lb, k_a=kg, v_a=vg)
        ops.merge_attn_states(out, oa, la, ob, lb, output_lse=lse)
        many[0].copy_(oa), many[1].copy_(ob), many_lse[0].copy_(la), many_lse[1].copy_(lb)
        ops.merge_attn_states_n(joined, many, many_lse)
        return [x.clone() for x in (cache, kg, vg, oa, ob, out, lse, joined)]

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(2):
        for x in (q, k, v, kc, vc):
            x.copy_(torch.randn(x.shape, generator=gen))
        slots.copy_(torch.randperm(640, generator=gen)[:t])
        cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        held = [x.clone() for x in got]
        cache.zero_()
        for a, b in zip(held, run()):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ results in the place of inputs

@pytest.mark.parametrize("kind", ["same", "q4"])
@pytest.mark.parametrize("t", [1, 45, 700])
def test_norm_rope_in_place_beside_the_values(ops, kind, t):
    """q and k of one projection's output turned where they stand, with the values behind them going into the
    cache: as with results of their own.  One tensor as keys and values will do where the results stand elsewhere."""
    gen = torch.Generator().manual_seed(t)
    h, hkv, d, bs = 8, 2, 128, 16
    qkv = torch.randn(t, (h + 2 * hkv) * d, generator=gen).to(BF16).cuda()
    nb = t // bs + 2
    shape = (nb, hkv, bs, 2 * d) if kind == "same" else ops.kv_cache_q4_shape(nb, hkv, bs, d)
    dtype = BF16 if kind == "same" else torch.uint8
    pos, slots = torch.randint(0, 90, (t,), generator=gen).cuda(), torch.randperm(nb * bs, generator=gen)[:t].cuda()
    angle = torch.rand(90, d // 2, generator=gen, dtype=torch.float64) * 6
    table = torch.cat([angle.cos(), angle.sin()], -1).float().cuda()
    w = (1 + 0.2 * torch.randn(d, generator=gen)).to(BF16).cuda()

    def run(buf, in_place, shared=False):
        q, k, v = (x.view(t, -1, d) for x in buf.split([h * d, hkv * d, hkv * d], -1))
        cache = torch.zeros(shape, dtype=dtype, device="cuda")
        out = dict(q_out=q, k_out=k) if in_place else {}
        a, b = ops.qk_norm_rope(q, k, pos, table, q_weight=w, k_weight=w, value=k if shared else v, kv_cache=cache,
                                slot_mapping=slots, **out)
        return a.clone(), b.clone(), v.clone(), cache

    for x, y in zip(run(qkv.clone(), False), run(qkv.clone(), True)):
        assert torch.equal(x, y)
    _, k_out, _, cache = run(qkv.clone(), False, shared=True)
    want = torch.zeros_like(cache)
    raw = qkv[:, h * d: (h + hkv) * d].view(t, hkv, d)
    (ops.kv_cache_update if kind == "same" else ops.kv_cache_update_q4)(k_out, raw, want, slots)
    assert torch.equal(cache.view(torch.uint8), want.view(torch.uint8))


# ------------------------------------------------------------------ the smallest scales

@pytest.mark.parametrize("h,hkv,d,dtype", [(28, 4, 128, BF16), (12, 1, 64, F16)])
@pytest.mark.parametrize("scale,size", [(1e-44, 1.0), (1e-30, 1.0), (1e-12, 1e-38)])
def test_decode_q4_scales_that_vanish(ops, scale, size, h, hkv, d, dtype):
    """A scale (or a query) so small that their product leaves 32 bits: every key weighs the same, and keys that
    are not there still weigh nothing."""
    if dtype == F16 and size != 1.0:
        size = 2.0 ** -24
    gen = torch.Generator().manual_seed(33)
    bs, nb, lens = 16, 30, [1, 7, 16, 33, 470]
    n = nb * bs
    cache = torch.full(ops.kv_cache_q4_shape(nb, hkv, bs, d), 0xFF, dtype=torch.uint8, device="cuda")
    k, v = (torch.randn(480, hkv, d, generator=gen).to(dtype) for _ in range(2))
    ops.kv_cache_update_q4(k[:470].cuda(), v[:470].cuda(), cache, torch.arange(470, device="cuda"))
    kq, vq = R.read_q4(cache.cpu().numpy(), np.arange(470), dtype)
    q = (torch.randn(len(lens), h, d, generator=gen).double() * size).to(dtype)
    table = torch.arange(nb, dtype=torch.int32, device="cuda").view(1, nb)
    out, lse = torch.zeros(len(lens), h, d, device="cuda"), torch.zeros(h, len(lens), device="cuda")
    ops.decode_splitkv_q4(q.cuda(), cache, table, _i32(lens), scale=scale, out=out, lse=lse, token_req=_i32([0] * len(lens)))
    o, l = R.f64(out), R.f64(lse)
    for r, n in enumerate(lens):
        _check_by_weight(o[r], l[:, r], R.f64(q[r]), kq[:n], vq[:n], scale, torch.float32, (scale, n))


# ------------------------------------------------------------------ joins

@pytest.mark.parametrize("h,hkv,d,dtype,rows,longest", [
    (28, 4, 128, BF16, 24, 60000), (4, 4, 64, BF16, 32, 900), (4, 4, 128, F16, 36, 700), (32, 32, 64, F16, 4, 3000)])
def test_decode_q4_joins_of_unequal_rows(ops, h, hkv, d, dtype, rows, longest):
    """One row of very many parts among short ones, and 127 to 147 pairs of one head each (the join's form goes by
    the mean number of parts)."""
    gen = torch.Generator().manual_seed(rows)
    bs, nb = 16, 120
    k, v = (torch.randn(nb * bs, hkv, d, generator=gen).to(dtype) for _ in range(2))
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k.cuda(), v.cuda(), cache, torch.arange(nb * bs, device="cuda"))
    kq, vq = R.read_q4(cache.cpu().numpy(), np.arange(nb * bs), dtype)
    lens = torch.randint(1, 300, (rows,), generator=gen).numpy() if h != hkv else torch.randint(300, longest, (rows,), generator=gen).numpy()
    lens[rows // 3] = longest
    table = torch.randint(0, nb, (rows, -(-longest // bs)), generator=gen, dtype=torch.int32)
    q = torch.randn(rows, h, d, generator=gen).to(dtype)
    out, lse = torch.zeros(rows, h, d, dtype=dtype, device="cuda"), torch.zeros(h, rows, device="cuda")
    ops.decode_splitkv_q4(q.cuda(), cache, table.cuda(), _i32(lens), scale=d ** -0.5, out=out, lse=lse)
    o, l, t = R.f64(out), R.f64(lse), table.numpy()
    for r in sorted({0, 1, rows // 3, rows - 1}):
        p = np.arange(lens[r])
        at = t[r, p // bs].astype(np.int64) * bs + p % bs
        _check_by_weight(o[r], l[:, r], R.f64(q[r]), kq[at], vq[at], d ** -0.5, dtype, (r, int(lens[r])))


# ------------------------------------------------------------------ results of more than 8 bits

@pytest.mark.parametrize("h,hkv,d,dtype,kind", [(28, 4, 128, BF16, torch.float32), (32, 2, 128, BF16, torch.float32),
                                                (14, 2, 64, F16, F16), (14, 2, 64, F16, torch.float32), (12, 1, 128, F16, F16)])
@pytest.mark.parametrize("n", [2, 5, 40, 700])
def test_decode_q4_weights_of_22_bits(ops, n, h, hkv, d, dtype, kind):
    """Where the result is not rounded to bf16, a weight's second 11 bits are multiplied too: off by 1.08 * 2^-22 of
    each term and not by 2^-11.  Small queries, so that the scores' own share of the bar is small."""
    gen = torch.Generator().manual_seed(n + h)
    rows, bs, nb = 6, 16, 44
    k, v = (torch.randn(nb * bs, hkv, d, generator=gen).to(dtype) for _ in range(2))
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k.cuda(), v.cuda(), cache, torch.arange(nb * bs, device="cuda"))
    kq, vq = R.read_q4(cache.cpu().numpy(), np.arange(n), dtype)
    q = (torch.randn(rows, h, d, generator=gen) * 2.0 ** -6).to(dtype)
    out, lse = torch.zeros(rows, h, d, dtype=kind, device="cuda"), torch.zeros(h, rows, device="cuda")
    ops.decode_splitkv_q4(q.cuda(), cache, torch.arange(nb, dtype=torch.int32, device="cuda").view(1, nb), _i32([n] * rows),
                          scale=d ** -0.5, out=out, lse=lse, token_req=_i32([0] * rows))
    o, l = R.f64(out), R.f64(lse)
    for r in range(rows):
        _check_by_weight(o[r], l[:, r], R.f64(q[r]), kq, vq, d ** -0.5, kind, (n, r), rounded=1.08 * 2.0 ** -22)


def test_decode_q4_in_place(ops):
    """The result in the place of the queries: as with a result of its own, rows that are cut and joined among them."""
    gen = torch.Generator().manual_seed(40)
    rows, h, hkv, d, bs, nb = 7, 28, 4, 128, 16, 100
    k, v = (torch.randn(nb * bs, hkv, d, generator=gen).to(BF16).cuda() for _ in range(2))
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k, v, cache, torch.arange(nb * bs, device="cuda"))
    table = torch.randint(0, nb, (rows, 1200), generator=gen, dtype=torch.int32).cuda()
    lens, qkv = _i32([19000, 1, 0, 700, 5000, 33, 16]), torch.randn(rows, (h + 2 * hkv) * d, generator=gen).to(BF16).cuda()
    q = qkv[:, : h * d].view(rows, h, d)
    out, lse = torch.zeros(rows, h, d, dtype=BF16, device="cuda"), torch.zeros(h, rows, device="cuda")
    ops.decode_splitkv_q4(q, cache, table, lens, scale=0.1, out=out, lse=lse)
    for _ in range(5):
        buf, again = qkv.clone(), torch.zeros_like(lse)
        mine = buf[:, : h * d].view(rows, h, d)
        ops.decode_splitkv_q4(mine, cache, table, lens, scale=0.1, out=mine, lse=again)
        assert torch.equal(mine, out) and torch.equal(again, lse) and torch.equal(buf[:, h * d:], qkv[:, h * d:])


def test_blocks_given_back_are_taken_again(ops):
    """A finished request's blocks, written over the last taken entries of the list with the head lowered, go to the
    next requests; no block is ever held twice."""
    gen = torch.Generator().manual_seed(41)
    reqs, width, bs = 6, 5, 16
    free = torch.randperm(18, generator=gen).int().cuda()
    head = torch.zeros(1, dtype=torch.int32, device="cuda")
    table, held = torch.full((reqs, width), -1, dtype=torch.int32, device="cuda"), np.zeros(reqs, np.int64)
    for step in range(30):
        new = np.minimum(torch.randint(0, 30, (reqs,), generator=gen).numpy(), 45 - held)
        plan = ops.kv_plan_step(_i32(held), _i32(new), table, free, head, block_size=bs, num_tokens=200)
        assert plan.missing.item() == 0
        held, head = held + new, plan.free_head.clone()
        mine = [table[i, : -(-int(c) // bs)].tolist() for i, c in enumerate(held)]
        flat = sum(mine, [])
        assert len(set(flat)) == len(flat) == int(head) and sorted(flat + free[int(head):].tolist()) == list(range(18))
        for i in np.flatnonzero(held >= 40):
            n = len(mine[i])
            free[int(head) - n: int(head)] = _i32(mine[i])
            head -= n
            held[i] = 0
