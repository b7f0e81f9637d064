"""GPU tests of the serving-step operators (step plan, norm and rotation, the
4-bit cache and attention over it) against plain restatements in 64 bits, at
the lengths, masks, strides and sizes where they can go wrong, and in a run
together as a serving step uses them, eager and captured."""

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


def _randn(gen, *shape, dtype=BF16):
    return torch.randn(*shape, generator=gen).to(dtype)


# ------------------------------------------------------------------ step plan

def _check_plan(ops, context, new, width, free, head, bs, tokens, base=None, wide=0):
    rng = np.random.default_rng(len(context) * 7 + bs)
    reqs = len(context)
    table = rng.permutation(reqs * width + 1)[: reqs * width].reshape(reqs, width).astype(np.int32) + 1000
    want = R.plan(context, new, table, free, head, bs, tokens, base)
    buf = torch.full((reqs, width + wide), 77, dtype=torch.int32, device="cuda")
    bt = buf[:, :width]
    bt.copy_(torch.from_numpy(table))
    for _ in range(2):  # a repeated call writes the same
        got = ops.kv_plan_step(_i32(context), _i32(new), bt, _i32(free), _i32([head]), block_size=bs, num_tokens=tokens,
                               pos_base=None if base is None else _i32(base))
        for name, t in got._asdict().items():
            np.testing.assert_array_equal(t.cpu().numpy(), want[name], err_msg=name)
        np.testing.assert_array_equal(bt.cpu().numpy(), want["block_table"])
    assert bool((buf[:, width:] == 77).all())
    return want


def test_plan_decode_step(ops):
    context = [0, 1, 15, 16, 17, 31, 32, 100]
    w = _check_plan(ops, context, [1] * 8, 9, np.arange(500, 540), 3, 16, 8)
    assert w["missing"] == [0] and w["free_head"] == [3 + 3]


@pytest.mark.parametrize("bs", [16, 32, 48, 128])
@pytest.mark.parametrize("reqs,seed", [(1, 0), (7, 1), (256, 2), (257, 3), (700, 4)])
def test_plan_mixed_batches(ops, bs, reqs, seed):
    rng = np.random.default_rng(seed)
    context = rng.integers(0, 300, reqs)
    new = np.where(rng.random(reqs) < 0.4, 0, rng.integers(0, 90, reqs))
    total = int(new.sum())
    _check_plan(ops, context, new, 400 // bs + 2, rng.permutation(reqs * 40).astype(np.int32), 5, bs, total + 33,
                base=rng.integers(0, 100000, reqs), wide=3)


def test_plan_long_request_and_empty_ones(ops):
    _check_plan(ops, [0, 40000, 0, 5], [0, 9001, 0, 0], 3300, np.arange(2000), 0, 16, 9001)
    _check_plan(ops, [5, 6], [0, 0], 4, np.arange(9), 0, 16, 0)       # nothing new, no rows
    _check_plan(ops, [5, 6], [0, 0], 4, np.arange(9), 0, 16, 300)     # padding only
    _check_plan(ops, [], [], 4, np.arange(9), 2, 16, 5)               # no requests


def test_plan_refuses_nothing_but_tells_what_is_missing(ops):
    w = _check_plan(ops, [10, 20, 0], [40, 50, 16], 8, np.arange(4), 1, 16, 106)   # the free list ends
    assert w["missing"][0] == 4 and w["free_head"] == [4]
    w = _check_plan(ops, [30, 0], [40, 10], 2, np.arange(9), 0, 16, 50)            # the row ends
    assert w["missing"][0] == 3
    _check_plan(ops, [3, 4], [5, 6], 4, np.arange(0), 0, 16, 11)                   # an empty free list
    _check_plan(ops, [3, 4], [20, 20], 4, np.arange(6), 9, 16, 40)                 # a head past the list
    _check_plan(ops, [3, -4, 7], [20, -2, 4], 4, np.arange(6), 0, 16, 30)          # negative lengths count as 0
    _check_plan(ops, [3, 4], [20, 20], 4, np.arange(6), 0, 16, 25)                 # fewer rows than tokens


# ------------------------------------------------------------------ 4-bit cache

def _rows_q4(gen, n, hkv, d, dtype):
    """Rows with the groups that are special: constant, tiny and large ranges, an outlier, infinities and NaN."""
    x = torch.randn(n, hkv, d, generator=gen)
    if n > 8:
        x[1, 0, :64] = 0.75
        x[2] *= 1e-7
        x[3] *= 3e4 if dtype == F16 else 1e30
        x[4, :, 5] = 40.0
        x[5, 0, 3] = float("inf")
        x[6, -1, d - 1] = float("nan")
        x[7, 0, 0] = -float("inf")
        x[8] = x[8].abs() + 100
    return x.to(dtype)


@pytest.mark.parametrize("dtype,hkv,d,bs", [(BF16, 4, 128, 16), (F16, 2, 64, 32), (BF16, 1, 64, 128), (F16, 3, 128, 64)])
@pytest.mark.parametrize("n", [1, 5, 16, 83])
def test_update_and_gather_q4(ops, dtype, hkv, d, bs, n):
    gen = torch.Generator().manual_seed(n * 100 + d + bs)
    nb = 7 + n // bs
    key, value = _rows_q4(gen, n, hkv, d, dtype), _rows_q4(gen, n, hkv, d, dtype).flip(0)
    slots = torch.randperm(nb * bs, generator=gen)[:n]
    if n > 8:
        slots[0], slots[n // 2], slots[-1] = -1, nb * bs, -(1 << 40)
    start = torch.randint(0, 256, ops.kv_cache_q4_shape(nb, hkv, bs, d), generator=gen, dtype=torch.uint8)
    want = start.numpy().copy()
    R.write_q4(want, key.float().numpy(), value.float().numpy(), slots.numpy(), dtype)
    cache = start.cuda()
    wide = torch.randn(n, 3, hkv, d, generator=gen).to(dtype).cuda()  # strided rows
    wide[:, 0], wide[:, 2] = key.cuda(), value.cuda()
    ops.kv_cache_update_q4(wide[:, 0], wide[:, 2], cache, slots.cuda())
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    ek, ev = R.read_q4(want, slots.numpy(), dtype)
    got = torch.full((n + 2, 2, hkv, d), 7.0, dtype=dtype, device="cuda")
    ops.kv_cache_gather_q4(cache, slots.cuda(), dtype, key=got[:, 0], value=got[:, 1])
    for side, ref in ((0, ek), (1, ev)):
        np.testing.assert_array_equal(got[:n, side].float().cpu().numpy(), R.round16(ref, dtype))
    assert bool((got[n:] == 7.0).all())
    k2, v2 = ops.kv_cache_gather_q4(cache, slots.cuda(), dtype)
    assert torch.equal(k2.view(torch.int16), got[:n, 0].contiguous().view(torch.int16))
    assert torch.equal(v2.view(torch.int16), got[:n, 1].contiguous().view(torch.int16))


@pytest.mark.parametrize("first", [0, 3, 16, 21])
@pytest.mark.parametrize("dtype,d,bs", [(BF16, 128, 16), (F16, 64, 64)])
def test_update_and_gather_of_consecutive_slots(ops, first, dtype, d, bs):
    """A request's chunk through its pages: whole tiles, partial first and last tiles."""
    gen = torch.Generator().manual_seed(first + d)
    n, hkv, nb = 150, 2, 14
    pages = torch.randperm(nb, generator=gen)
    pos = torch.arange(first, first + n)
    slots = pages[pos // bs] * bs + pos % bs
    key, value = _rows_q4(gen, n, hkv, d, dtype), _rows_q4(gen, n, hkv, d, dtype)
    start = torch.randint(0, 256, ops.kv_cache_q4_shape(nb, hkv, bs, d), generator=gen, dtype=torch.uint8)
    want = start.numpy().copy()
    R.write_q4(want, key.float().numpy(), value.float().numpy(), slots.numpy(), dtype)
    cache = start.cuda()
    ops.kv_cache_update_q4(key.cuda(), value.cuda(), cache, slots.cuda())
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    k, v = ops.kv_cache_gather_q4(cache, slots.cuda(), dtype)
    ek, ev = R.read_q4(want, slots.numpy(), dtype)
    np.testing.assert_array_equal(k.float().cpu().numpy(), R.round16(ek, dtype))
    np.testing.assert_array_equal(v.float().cpu().numpy(), R.round16(ev, dtype))


def test_q4_nothing_to_do(ops):
    cache = torch.full(ops.kv_cache_q4_shape(2, 2, 16, 64), 3, dtype=torch.uint8, device="cuda")
    none = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    slots = torch.zeros(0, dtype=torch.int64, device="cuda")
    ops.kv_cache_update_q4(none, none, cache, slots)
    k, v = ops.kv_cache_gather_q4(cache, slots, BF16)
    assert k.shape == (0, 2, 64) and v.shape == (0, 2, 64) and bool((cache == 3).all())


def test_q4_error_is_half_a_step(ops):
    """Every element reads back within half a step of its group, the step's and the result's own rounding on top:
    |x' - x| <= s/2 + 15 |s - range/15| + eps/2 |x'| (clamping only ever pulls n back towards x)."""
    gen = torch.Generator().manual_seed(8)
    x = (torch.randn(64, 2, 128, generator=gen) * 3).to(BF16)
    cache = torch.zeros(ops.kv_cache_q4_shape(4, 2, 16, 128), dtype=torch.uint8, device="cuda")
    slots = torch.randperm(64, generator=gen).cuda()
    ops.kv_cache_update_q4(x.cuda(), x.flip(0).cuda(), cache, slots)
    k, v = ops.kv_cache_gather_q4(cache, slots, BF16)
    for got, ref in ((k, x), (v, x.flip(0))):
        g, r = (R.f64(t).reshape(-1, 64) for t in (got, ref))
        rng = (r.max(-1) - r.min(-1))[:, None]
        step = rng / 15 * (1 + 2.0 ** -8)
        assert (np.abs(g - r) <= step / 2 + rng * 2.0 ** -8 + np.abs(g) * 2.0 ** -8).all()


# ------------------------------------------------------------------ norm and rotation

def _angles(rows, rotary, dtype):
    half = rotary // 2
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([a.cos(), a.sin()], -1).to(dtype)


def _check_rows(got, x, want, dtype):
    """Half a step of rounding, and 32-bit arithmetic before it: the sum of up to 128 squares is off by at most
    2^-17 relative (2^-18 in its root), each product by 2^-24, so 2^-17 of |a| + |b| <= 2 * the row's largest."""
    g = R.f64(got)
    nan = np.isnan(want)
    assert (np.isnan(g) == nan).all()
    eps = torch.finfo(dtype).eps / 2
    top = np.abs(np.where(nan, 0, want)).max(-1, keepdims=True)
    slack = 2.0 ** -15 * top
    bar = eps * (np.abs(want) + slack) + slack + 2.0 ** -25
    assert (np.abs(g - want)[~nan] <= np.broadcast_to(bar, want.shape)[~nan]).all(), np.nanmax(np.abs(g - want) - bar)


@pytest.mark.parametrize("t", [1, 3, 64, 331])
@pytest.mark.parametrize("h,hkv,d,dtype,rotary,interleaved,tab,weights", [
    (28, 4, 128, BF16, 128, False, "f32", True),
    (28, 4, 128, BF16, 128, True, "same", False),
    (14, 2, 64, F16, 32, True, "same", True),
    (5, 1, 64, BF16, 64, False, "f32", True),
    (1, 1, 128, F16, 8, False, "f32", True),
    (3, 3, 128, F16, 64, False, "same", True),
    (16, 8, 64, BF16, 24, True, "f32", False),
])
def test_norm_rope(ops, t, h, hkv, d, dtype, rotary, interleaved, tab, weights):
    gen = torch.Generator().manual_seed(t * 31 + h + rotary)
    qkv = torch.randn(t, (h + 2 * hkv) * d, generator=gen).to(dtype)
    qkv[0] *= 30
    if t > 2:
        qkv[1] = 0                      # a row without anything: rsqrt(eps) * 0
        qkv[2] *= 1e-3
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen)).to(dtype) for _ in range(2))
    wq, wk = (wq, wk) if weights else (None, None)
    rows = 500
    pos = torch.randint(0, rows, (t,), generator=gen)
    table = _angles(rows, rotary, torch.float32 if tab == "f32" else dtype)
    q, k = qkv[:, : h * d].view(t, h, d), qkv[:, h * d: (h + hkv) * d].view(t, hkv, d)
    dev = qkv.cuda()
    qd, kd = dev[:, : h * d].view(t, h, d), dev[:, h * d: (h + hkv) * d].view(t, hkv, d)
    cu = lambda x: None if x is None else x.cuda()  # noqa: E731
    kw = dict(q_weight=cu(wq), k_weight=cu(wk), eps=1e-6, interleaved=interleaved)
    gq, gk = ops.qk_norm_rope(qd, kd, pos.cuda(), table.cuda(), **kw)
    for got, x, w in ((gq, q, wq), (gk, k, wk)):
        _check_rows(got, x, R.norm_rope(R.f64(x), None if w is None else R.f64(w), pos.numpy(), R.f64(table), 1e-6,
                                        interleaved), dtype)
    # in place, in the projection's own buffer: the same values, the values' part untouched
    v0 = dev[:, (h + hkv) * d:].clone()
    ops.qk_norm_rope(qd, kd, pos.cuda(), table.cuda(), q_out=qd, k_out=kd, **kw)
    assert torch.equal(qd, gq) and torch.equal(kd, gk) and torch.equal(dev[:, (h + hkv) * d:], v0)


@pytest.mark.parametrize("kind", ["same", "q4"])
@pytest.mark.parametrize("h,hkv,d,dtype,rotary,interleaved,bs", [
    (28, 4, 128, BF16, 128, False, 16), (14, 2, 64, F16, 32, True, 32), (3, 3, 128, F16, 64, False, 64),
    (4, 1, 64, BF16, 64, False, 128), (6, 2, 128, BF16, 40, True, 16)])
@pytest.mark.parametrize("t", [1, 70, 1700])
def test_norm_rope_writes_the_cache(ops, kind, h, hkv, d, dtype, rotary, interleaved, bs, t):
    """The cache write of the same pass equals the scatter of the rotated keys and the values, byte for byte."""
    gen = torch.Generator().manual_seed(t + d + rotary)
    q, k, v = (_randn(gen, t, n, d, dtype=dtype).cuda() for n in (h, hkv, hkv))
    if t > 20:
        v[3, 0, 2] = float("inf")
        k[4, 0, 1] = float("nan")
    w = (1 + 0.3 * torch.randn(d, generator=gen)).to(dtype).cuda()
    pos = torch.randint(0, 600, (t,), generator=gen)
    nb = t // bs + 3
    slots = torch.randperm(nb * bs, generator=gen)[:t]
    if t > 20:
        pos[5], pos[6] = -1, 600        # padding, and a position past the table
        slots[7], slots[8] = -1, nb * bs
    table = _angles(600, rotary, torch.float32).cuda()
    shape = (nb, hkv, bs, 2 * d) if kind == "same" else ops.kv_cache_q4_shape(nb, hkv, bs, d)
    start = (torch.randn(shape, generator=gen).to(dtype) if kind == "same"
             else torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8)).cuda()
    cache, want = start.clone(), start.clone()
    kw = dict(q_weight=w, k_weight=w, interleaved=interleaved)
    q_out, k_out = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    ops.qk_norm_rope(q, k, pos.cuda(), table, q_out=q_out, k_out=k_out, value=v, kv_cache=cache, slot_mapping=slots.cuda(), **kw)
    pq, pk = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    ops.qk_norm_rope(q, k, pos.cuda(), table, q_out=pq, k_out=pk, **kw)
    bits = lambda x: x.view(torch.int16)  # noqa: E731
    assert torch.equal(bits(q_out), bits(pq)) and torch.equal(bits(k_out), bits(pk))
    if t > 20:
        assert bool((q_out[5] == 9.0).all()) and bool((k_out[5] == 9.0).all())
        assert bool(q_out[6].isnan().all()) and bool(k_out[6].isnan().all())
        slots[5] = slots[6] = -1
    (ops.kv_cache_update if kind == "same" else ops.kv_cache_update_q4)(k_out, v, want, slots.cuda())
    assert torch.equal(cache.view(torch.uint8), want.view(torch.uint8))


def test_norm_rope_without_rows(ops):
    q, k = torch.zeros(0, 4, 64, dtype=BF16, device="cuda"), torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    pos, table = torch.zeros(0, dtype=torch.int64, device="cuda"), _angles(8, 64, torch.float32).cuda()
    gq, gk = ops.qk_norm_rope(q, k, pos, table)
    assert gq.shape == q.shape and gk.shape == k.shape


# ------------------------------------------------------------------ attention over the 4-bit cache

def _filled(ops, gen, nb, hkv, bs, d, dtype, scale=1.0):
    """A cache whose every slot is written, on the GPU."""
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    n = nb * bs
    ops.kv_cache_update_q4((_randn(gen, n, hkv, d) * scale).to(dtype).cuda(), _randn(gen, n, hkv, d, dtype=dtype).cuda(), cache,
                           torch.arange(n, device="cuda"))
    return cache


def _check_attention(got, lse, q, k, v, scale, dtype, what):
    """One row against 64 bits.  With a_i = scale * sum_d |q_d| max_j |k_jd| (i a head): a score is off by at most
    2^-17 a_i (64 products summed in 32 bits per group, then the groups), so each weight by that and 2^-21 of ex2.
    The products p_j s_j are rounded to fp16, half a step of 2^-10 off: 2^-11 p_j s_j |n_j - 8| of a result whose p_j
    sum to 1.  |n - 8| <= 8, and 15 s <= 2 top (1 + 2^-8, s being rounded), so 8 s <= 1.08 top: 1.08 * 2^-11 top.
    Each of a tile's sums rounds by 2^-23, n / 16 tiles of them twice."""
    n = k.shape[0]
    o, l = R.attention(q, k, v, scale)
    if n == 0:
        assert (got == 0).all() and (lse == -np.inf).all()
        return
    g = q.shape[0] // k.shape[1]
    a = np.array([scale * (np.abs(q[i]) * np.abs(k[:, i // g]).max(0)).sum() for i in range(q.shape[0])])
    top = np.array([np.abs(v[:, i // g]).max() for i in range(q.shape[0])])
    dx = 2.0 ** -17 * a
    slack = top * (2 * dx + 1.08 * 2.0 ** -11 + 2.0 ** -15 + n / 8 * 2.0 ** -23)
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    bar = slack[:, None] + eps * (np.abs(o) + slack[:, None]) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert (np.abs(got - o) <= bar).all(), (what, np.max(np.abs(got - o) / bar))
    assert (np.abs(lse - l) <= dx + 2.0 ** -20 * (np.abs(l) + 1) + n / 16 * 2.0 ** -24).all(), what


def _run_decode(ops, cache, q, lens, table, dtype, req=None, out_dtype=None, **kw):
    rows, h, d = q.shape
    out = torch.full((rows + 1, h, d), 5.0, dtype=out_dtype or dtype, device="cuda")
    lse = torch.full((h, rows + 2), 5.0, device="cuda")
    scale = d ** -0.5
    ops.decode_splitkv_q4(q.cuda(), cache, table.cuda(), _i32(lens), scale=scale, out=out, lse=lse,
                          token_req=None if req is None else _i32(req), **kw)
    torch.cuda.synchronize()
    o, l = R.f64(out), R.f64(lse)
    assert (o[rows:] == 5).all() and (l[:, rows:] == 5).all()   # rows behind the last stay
    host = cache.cpu().numpy()
    nb, hkv, bs, _ = host.shape
    kmem, vmem = R.read_q4(host, np.arange(nb * bs), dtype) if nb * bs <= 40000 else (None, None)
    t = table.numpy()
    for r in range(rows):
        i = r if req is None else int(req[r])
        if i < 0 or i >= t.shape[0]:
            assert (o[r] == 5).all() and (l[:, r] == 5).all()
            continue
        n = min(max(0, int(lens[r])), t.shape[1] * bs)
        p = np.arange(n)
        page = t[i, p // bs]
        p, page = p[(page >= 0) & (page < nb)], page[(page >= 0) & (page < nb)]
        slots = page.astype(np.int64) * bs + p % bs
        _check_attention(o[r], l[:, r], R.f64(q[r]), kmem[slots], vmem[slots], scale, out_dtype or dtype, (r, n))
    return out, lse


GEOMETRIES = [(28, 4, 128, BF16, 16), (14, 2, 64, F16, 32), (16, 1, 128, BF16, 64), (9, 1, 64, BF16, 16),
              (4, 4, 128, F16, 128), (1, 1, 64, F16, 16), (24, 2, 128, F16, 32), (8, 1, 64, BF16, 16)]


@pytest.mark.parametrize("h,hkv,d,dtype,bs", GEOMETRIES)
def test_decode_q4_lengths(ops, h, hkv, d, dtype, bs):
    """Lengths around tiles and pages, an empty row, one that crosses several blocks' pieces; unequal rows together."""
    gen = torch.Generator().manual_seed(h + d)
    lens = [0, 1, 15, 16, 17, 2, 500, 0, 33, 64, 777, 1300, 31, 3]
    width = -(-max(lens) // bs)
    nb = len(lens) * width + 1
    nb = min(nb, 3000 // bs)   # pages are shared between rows
    cache = _filled(ops, gen, nb, hkv, bs, d, dtype)
    table = torch.randint(0, nb, (len(lens), width), generator=gen, dtype=torch.int32)
    q = _randn(gen, len(lens), h, d, dtype=dtype)
    _run_decode(ops, cache, q, lens, table, dtype)
    _run_decode(ops, cache, q, lens, table, dtype, out_dtype=torch.float32)


@pytest.mark.parametrize("h,hkv,d,dtype,bs,n", [(28, 4, 128, BF16, 16, 20011), (14, 2, 64, F16, 64, 9999), (12, 1, 128, BF16, 32, 30000)])
def test_decode_q4_one_long_row(ops, h, hkv, d, dtype, bs, n):
    gen = torch.Generator().manual_seed(n)
    nb = 64
    cache = _filled(ops, gen, nb, hkv, bs, d, dtype, scale=2.0)
    table = torch.randint(0, nb, (1, -(-n // bs)), generator=gen, dtype=torch.int32)
    _run_decode(ops, cache, _randn(gen, 1, h, d, dtype=dtype) * 2, [n], table, dtype)


def test_decode_q4_many_short_rows(ops):
    """More rows than threads that sum the lengths, empty and padding rows among them."""
    gen = torch.Generator().manual_seed(3)
    rows, h, hkv, d, bs, nb = 301, 7, 1, 128, 16, 50
    cache = _filled(ops, gen, nb, hkv, bs, d, BF16)
    lens = torch.randint(0, 90, (rows,), generator=gen).numpy()
    lens[::17] = 0
    req = torch.randint(0, 40, (rows,), generator=gen).numpy()
    req[5::23] = -1
    req[300] = 40   # past the table
    table = torch.randint(0, nb, (40, 6), generator=gen, dtype=torch.int32)
    _run_decode(ops, cache, _randn(gen, rows, h, d), lens, table, BF16, req=req)


def test_decode_q4_nothing_visible(ops):
    gen = torch.Generator().manual_seed(4)
    cache = _filled(ops, gen, 4, 2, 16, 64, BF16)
    table = torch.zeros(3, 2, dtype=torch.int32)
    _run_decode(ops, cache, _randn(gen, 3, 4, 64), [0, -5, 0], table, BF16)
    _run_decode(ops, cache, _randn(gen, 3, 4, 64), [20, 20, 20], table, BF16, req=[-1, -1, 7])
    out = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    ops.decode_splitkv_q4(out, cache, table.cuda(), _i32([]), scale=1.0, out=out)


def test_decode_q4_pages_outside_the_cache_hold_no_keys(ops):
    gen = torch.Generator().manual_seed(5)
    h, hkv, d, bs, nb = 28, 4, 128, 16, 30
    cache = _filled(ops, gen, nb, hkv, bs, d, BF16)
    table = torch.randint(0, nb, (4, 20), generator=gen, dtype=torch.int32)
    table[0, 3], table[0, 4], table[1, 0] = -1, nb, 2 ** 31 - 1
    table[2, :] = -1
    _run_decode(ops, cache, _randn(gen, 4, h, d), [300, 100, 200, 5000], table, BF16)  # the last length is cut to the row


def test_decode_q4_unwritten_bytes_behind_the_last_key(ops):
    """The tail of a row's last tile is whatever memory held: infinities and NaN there change nothing."""
    gen = torch.Generator().manual_seed(6)
    h, hkv, d, bs, nb = 14, 2, 64, 16, 12
    for dtype in (BF16, F16):
        cache = torch.full(ops.kv_cache_q4_shape(nb, hkv, bs, d), 0xFF, dtype=torch.uint8, device="cuda")
        clean = torch.zeros_like(cache)
        lens = [5, 17, 40]
        table = torch.arange(9, dtype=torch.int32).view(3, 3)
        slots = torch.cat([table[r].long()[torch.arange(n) // bs] * bs + torch.arange(n) % bs for r, n in enumerate(lens)]).cuda()
        k, v = _randn(gen, len(slots), hkv, d, dtype=dtype).cuda(), _randn(gen, len(slots), hkv, d, dtype=dtype).cuda()
        q = _randn(gen, 3, h, d, dtype=dtype)
        for c in (cache, clean):
            ops.kv_cache_update_q4(k, v, c, slots)
        a, b = _run_decode(ops, cache, q, lens, table, dtype), _run_decode(ops, clean, q, lens, table, dtype)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_q4_nan_keys_show(ops):
    """A key or value that was not finite gives NaN to its head's rows and to no other."""
    gen = torch.Generator().manual_seed(7)
    h, hkv, d, bs, nb = 8, 2, 128, 16, 400
    n = nb * bs
    k, v = _randn(gen, n, hkv, d), _randn(gen, n, hkv, d)
    k[3000, 0, 5] = float("inf")
    v[4000, 1, 70] = float("nan")
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k.cuda(), v.cuda(), cache, torch.arange(n, device="cuda"))
    table = torch.arange(nb, dtype=torch.int32, device="cuda").view(1, nb).repeat(2, 1)
    q = _randn(gen, 2, h, d).cuda()
    out, lse = torch.empty_like(q), torch.empty(h, 2, device="cuda")
    ops.decode_splitkv_q4(q, cache, table, _i32([n, 2990]), scale=d ** -0.5, out=out, lse=lse)
    assert bool(out[0, :4].isnan().all()) and bool(lse[:4, 0].isnan().all())
    assert bool(out[0, 4:, 64:].isnan().all()) and bool(out[0, 4:, :64].isfinite().all()) and bool(lse[4:, 0].isfinite().all())
    assert bool(out[1].isfinite().all()) and bool(lse[:, 1].isfinite().all())


def test_decode_q4_extreme_scores(ops):
    """Scores far apart (a running maximum that keeps rising) and queries of zero."""
    gen = torch.Generator().manual_seed(9)
    h, hkv, d, bs, nb = 7, 1, 128, 16, 40
    n = nb * bs
    k = _randn(gen, n, hkv, d)
    k *= torch.linspace(0.1, 30, n)[:, None, None]
    k = k.to(BF16)
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k.cuda(), _randn(gen, n, hkv, d).cuda(), cache, torch.arange(n, device="cuda"))
    q = _randn(gen, 2, h, d) * 4
    q[1] = 0
    _run_decode(ops, cache, q, [n, n - 3], torch.arange(nb, dtype=torch.int32).view(1, nb).repeat(2, 1), BF16)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_q4_scales_far_apart(ops, dtype):
    """Values and queries whose size changes by powers of ten from token to token and head to head."""
    gen = torch.Generator().manual_seed(14)
    h, hkv, d, bs, nb = 14, 2, 128, 16, 30
    n = nb * bs
    v = torch.randn(n, hkv, d, generator=gen) * 10.0 ** torch.linspace(-4, 3, n)[:, None, None]
    v[:, 1] = v[:, 1].flip(0)
    v[40:60, :, :64] = 0.25     # groups without a range
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(_randn(gen, n, hkv, d, dtype=dtype).cuda(), v.to(dtype).cuda(), cache, torch.arange(n, device="cuda"))
    q = (torch.randn(3, h, d, generator=gen) * 10.0 ** torch.linspace(-4, 1, h)[:, None]).to(dtype)
    table = torch.arange(nb, dtype=torch.int32).view(1, nb).repeat(3, 1)
    _run_decode(ops, cache, q, [n, 200, 45], table, dtype)
    # scores up to 10^6: the largest key takes all, and everything stays finite
    ops.kv_cache_update_q4((torch.randn(n, hkv, d, generator=gen) * 300).to(dtype).cuda(), v.to(dtype).cuda(), cache,
                           torch.arange(n, device="cuda"))
    _run_decode(ops, cache, (torch.randn(3, h, d, generator=gen) * 300).to(dtype), [n, 200, 45], table, dtype)
    # far past fp16's range either way, in bf16 (64 bits do not pass 10^38 either)
    if dtype == BF16:
        for size in (1e-30, 1e30):
            ops.kv_cache_update_q4(_randn(gen, n, hkv, d).cuda(), (torch.randn(n, hkv, d, generator=gen) * size).to(dtype).cuda(), cache,
                                   torch.arange(n, device="cuda"))
            _run_decode(ops, cache, _randn(gen, 3, h, d), [n, 200, 45], table, dtype)
            _run_decode(ops, cache, (torch.randn(3, h, d, generator=gen) * 1e-20).to(dtype), [n, 200, 45], table, dtype)
            ops.kv_cache_update_q4((torch.randn(n, hkv, d, generator=gen) * size).to(dtype).cuda(), v.to(dtype).cuda(), cache,
                                   torch.arange(n, device="cuda"))
            _run_decode(ops, cache, (torch.randn(3, h, d, generator=gen) / size).to(dtype), [n, 200, 45], table, dtype)


def test_decode_q4_strided_rows_and_own_workspace(ops):
    gen = torch.Generator().manual_seed(10)
    rows, h, hkv, d, bs, nb = 5, 28, 4, 128, 16, 40
    cache = _filled(ops, gen, nb, hkv, bs, d, BF16)
    lens, wide = _i32([100, 600, 3, 0, 250]), torch.randint(0, nb, (rows, 50), generator=gen, dtype=torch.int32).cuda()
    big = _randn(gen, rows, 2 * h, d).cuda()
    obig = torch.full((rows, 3 * h, d), 4.0, dtype=BF16, device="cuda")
    ref = torch.empty(rows, h, d, dtype=BF16, device="cuda")
    ops.decode_splitkv_q4(big[:, h:].contiguous(), cache, wide[:, :40].contiguous(), lens, scale=0.1, out=ref)
    ws = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
    ops.decode_splitkv_q4(big[:, h:], cache, wide[:, :40], lens, scale=0.1, out=obig[:, h: 2 * h], workspace=ws)
    assert torch.equal(obig[:, h: 2 * h], ref) and bool((obig[:, :h] == 4).all()) and bool((obig[:, 2 * h:] == 4).all())


def test_decode_q4_is_the_same_every_time(ops):
    gen = torch.Generator().manual_seed(11)
    cache = _filled(ops, gen, 64, 4, 16, 128, BF16)
    table = torch.randint(0, 64, (6, 700), generator=gen, dtype=torch.int32).cuda()
    q, lens = _randn(gen, 6, 28, 128).cuda(), _i32([11000, 10, 5000, 0, 9999, 128])
    first = None
    for _ in range(5):
        out, lse = torch.empty_like(q), torch.empty(28, 6, device="cuda")
        ops.decode_splitkv_q4(q, cache, table, lens, scale=0.1, out=out, lse=lse)
        first = first or (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_decode_q4_on_two_streams(ops):
    gen = torch.Generator().manual_seed(12)
    probs = []
    for i in range(2):
        cache = _filled(ops, gen, 64, 4, 16, 128, BF16)
        probs.append((_randn(gen, 3, 28, 128).cuda(), cache, torch.randint(0, 64, (3, 600), generator=gen, dtype=torch.int32).cuda(),
                      _i32([9000, 77 + i, 5000])))
    run = lambda q, c, t, n: (out := torch.empty_like(q), ops.decode_splitkv_q4(q, c, t, n, scale=0.1, out=out))[0]  # noqa: E731
    serial = [run(*p) for p in probs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        res = []
        for s, p in zip(streams, probs):
            with torch.cuda.stream(s):
                res.append(run(*p))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, serial))


def test_q4_cache_past_32_bit_offsets(ops):
    """Pages whose bytes lie past 4 GB: write, read back and attend."""
    gen = torch.Generator().manual_seed(13)
    h, hkv, d, bs = 28, 4, 128, 16
    nb = 5_000_000_000 // (hkv * bs * 144)
    cache = torch.zeros(ops.kv_cache_q4_shape(nb, hkv, bs, d), dtype=torch.uint8, device="cuda")
    n = 200
    pages = torch.tensor([nb - 1 - 3 * i for i in range(-(-n // bs))])
    pos = torch.arange(n)
    slots = pages[pos // bs] * bs + pos % bs
    k, v = _randn(gen, n, hkv, d), _randn(gen, n, hkv, d)
    ops.kv_cache_update_q4(k.cuda(), v.cuda(), cache, slots.cuda())
    gk, gv = ops.kv_cache_gather_q4(cache, slots.cuda(), BF16)
    small = torch.zeros(ops.kv_cache_q4_shape(13, hkv, bs, d), dtype=torch.uint8, device="cuda")
    ops.kv_cache_update_q4(k.cuda(), v.cuda(), small, pos.cuda())
    sk, sv = ops.kv_cache_gather_q4(small, pos.cuda(), BF16)
    assert torch.equal(gk, sk) and torch.equal(gv, sv)
    q = _randn(gen, 1, h, d).cuda()
    a, b = torch.empty_like(q), torch.empty_like(q)
    ops.decode_splitkv_q4(q, cache, pages.int().view(1, -1).cuda(), _i32([n]), scale=0.1, out=a)
    ops.decode_splitkv_q4(q, small, torch.arange(13, dtype=torch.int32, device="cuda").view(1, -1), _i32([n]), scale=0.1, out=b)
    assert torch.equal(a, b)


# ------------------------------------------------------------------ together

class _Step:
    """A model layer's serving step over the 4-bit cache: plan, norm + rotation + cache write, attention."""

    def __init__(self, ops, gen, reqs, rows, width, h=28, hkv=4, d=128, bs=16):
        self.ops, self.h, self.hkv, self.d, self.bs, self.rows = ops, h, hkv, d, bs, rows
        self.nb = reqs * width
        self.cache = torch.full(ops.kv_cache_q4_shape(self.nb, hkv, bs, d), 0xFF, dtype=torch.uint8, device="cuda")
        self.table = torch.full((reqs, width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(self.nb, generator=gen).int().cuda()
        self.head = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.context = torch.zeros(reqs, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(reqs, dtype=torch.int32, device="cuda")
        self.qkv = torch.zeros(rows, (h + 2 * hkv) * d, dtype=BF16, device="cuda")
        self.w = (1 + 0.2 * torch.randn(d, generator=gen)).to(BF16).cuda()
        self.angles = _angles(2000, d, torch.float32).cuda()
        self.out = torch.zeros(rows, h, d, dtype=BF16, device="cuda")
        self.lse = torch.zeros(h, rows, device="cuda")
        self.q = torch.zeros(rows, h, d, dtype=BF16, device="cuda")
        self.k = torch.zeros(rows, hkv, d, dtype=BF16, device="cuda")

    def run(self):
        h, hkv, d = self.h, self.hkv, self.d
        q, k, v = (x.view(self.rows, -1, d) for x in self.qkv.split([h * d, hkv * d, hkv * d], -1))
        plan = self.ops.kv_plan_step(self.context, self.new, self.table, self.free, self.head, block_size=self.bs, num_tokens=self.rows)
        self.ops.qk_norm_rope(q, k, plan.positions, self.angles, q_weight=self.w, k_weight=self.w, q_out=self.q, k_out=self.k,
                              value=v, kv_cache=self.cache, slot_mapping=plan.slot_mapping)
        self.ops.decode_splitkv_q4(self.q, self.cache, self.table, plan.kv_lens, scale=d ** -0.5, out=self.out, lse=self.lse,
                                   token_req=plan.token_req)
        self.context.copy_(plan.seq_lens)
        self.head.copy_(plan.free_head)


def _feed(step, gen, new):
    step.qkv.copy_(torch.randn(step.qkv.shape, generator=gen).to(BF16))
    step.new.copy_(_i32(new))


def _check_step(step, held, new):
    """The step's rows against attention over everything written so far, read back from the cache one slot at a time."""
    host, table = step.cache.cpu().numpy(), step.table.cpu().numpy()
    q, out, lse = R.f64(step.q), R.f64(step.out), R.f64(step.lse)
    row = 0
    for i, n in enumerate(new):
        p = np.arange(held[i] + n)
        k, v = R.read_q4(host, table[i, p // step.bs].astype(np.int64) * step.bs + p % step.bs, BF16)
        for u in range(n):
            seen = held[i] + u + 1
            _check_attention(out[row], lse[:, row], q[row], k[:seen], v[:seen], step.d ** -0.5, BF16, (i, seen))
            row += 1
    assert (out[row:] == 0).all() and (lse[:, row:] == 0).all()  # padding rows: never written


def test_steps_together(ops):
    """A prefill step, a mixed step and decodes, eager."""
    gen = torch.Generator().manual_seed(20)
    step = _Step(ops, gen, 4, 80, 12)
    held = [0] * 4
    for new in ([30, 0, 17, 1], [1, 40, 16, 0], [1, 1, 1, 1], [1, 1, 0, 1]):
        step.out.zero_(), step.lse.zero_()
        _feed(step, gen, new)
        step.run()
        torch.cuda.synchronize()
        _check_step(step, held, new)
        held = [a + b for a, b in zip(held, new)]
        assert step.context.tolist() == held
    pages = step.table[step.table >= 0].tolist()
    assert len(pages) == len(set(pages)) == int(step.head)


def test_captured_step_follows_the_lengths(ops):
    """One captured step, replayed with other lengths and rows: equal to the eager run bit for bit."""
    news = [[9, 0, 20], [1, 33, 1], [1, 1, 1], [0, 1, 1], [1, 1, 1], [17, 0, 30]]
    eager, graph_step = (_Step(ops, torch.Generator().manual_seed(21), 3, 48, 12) for _ in range(2))
    _feed(graph_step, torch.Generator().manual_seed(1), [0, 0, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph_step.run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graph_step.run()
    gens = [torch.Generator().manual_seed(22) for _ in range(2)]
    held = [0] * 3
    for new in news:
        for s, g in zip((eager, graph_step), gens):
            s.out.zero_(), s.lse.zero_()
            _feed(s, g, new)
        eager.run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.out, graph_step.out) and torch.equal(eager.lse, graph_step.lse)
        assert torch.equal(eager.table, graph_step.table) and torch.equal(eager.cache, graph_step.cache)
        _check_step(graph_step, held, new)
        held = [a + b for a, b in zip(held, new)]


def test_calls_wait_for_what_comes_before_them(ops):
    """The calls may be scheduled while the kernel before them runs out: inputs written just before, by a
    slow kernel of the same stream or of another one behind an event, are the ones they see."""
    gen = torch.Generator().manual_seed(28)
    cache = _filled(ops, gen, 64, 4, 16, 128, BF16)
    table = torch.randint(0, 64, (3, 300), generator=gen, dtype=torch.int32).cuda()
    q, lens = _randn(gen, 3, 28, 128).cuda(), _i32([4000, 17, 2500])
    key, value = _randn(gen, 40, 4, 128).cuda(), _randn(gen, 40, 4, 128).cuda()
    slots, pos, tab = torch.randperm(1024, generator=gen)[:40].cuda(), torch.arange(3).cuda() + 5, _angles(64, 128, torch.float32).cuda()
    kq = _randn(gen, 3, 4, 128).cuda()

    def chain(c, q_in, n, t):
        out, lse = torch.empty_like(q), torch.empty(28, 3, device="cuda")
        plan = ops.kv_plan_step(n, n.sign(), t, n, n[:1] * 0, block_size=16, num_tokens=3)
        qr, _ = ops.qk_norm_rope(q_in, kq, pos, tab)
        ops.kv_cache_update_q4(key, value, c, slots)
        ops.decode_splitkv_q4(qr, c, t, n, scale=0.1, out=out, lse=lse)
        k, v = ops.kv_cache_gather_q4(c, slots, BF16)
        return out, lse, k, v, plan.kv_lens, plan.positions, t.clone()

    want = chain(cache.clone(), q, lens, table.clone())
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    for other in (False, True):
        for _ in range(3):
            c, q_in, n, t = torch.zeros_like(cache), torch.zeros_like(q), torch.zeros_like(lens), torch.zeros_like(table)
            torch.cuda.synchronize()
            with torch.cuda.stream(side if other else torch.cuda.current_stream()):
                for _ in range(4):
                    busy = (busy @ busy).clamp(-1, 1)
                c.copy_(cache), q_in.copy_(q), n.copy_(lens), t.copy_(table)
            torch.cuda.current_stream().wait_stream(side)
            got = chain(c, q_in, n, t)
            c.zero_(), q_in.zero_(), n.zero_(), t.zero_()   # and what follows waits for them
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_two_captured_decodes_do_not_share_partials(ops):
    """Two graphs replayed at once on two streams, each with its own partial sums."""
    gen = torch.Generator().manual_seed(23)
    probs, graphs, refs = [], [], []
    for i in range(2):
        cache = _filled(ops, gen, 64, 4, 16, 128, BF16)
        q, table = _randn(gen, 2, 28, 128).cuda(), torch.randint(0, 64, (2, 700), generator=gen, dtype=torch.int32).cuda()
        lens, out = _i32([11000, 9000 - i]), torch.zeros(2, 28, 128, dtype=BF16, device="cuda")
        ref = torch.empty_like(out)
        ops.decode_splitkv_q4(q, cache, table, lens, scale=0.1, out=ref)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.decode_splitkv_q4(q, cache, table, lens, scale=0.1, out=out)
        probs.append((q, cache, table, lens, out))
        graphs.append(g)
        refs.append(ref)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for p, ref in zip(probs, refs):
            assert torch.equal(p[4], ref)
            p[4].zero_()
        torch.cuda.synchronize()


def test_a_captured_16_bit_decode_keeps_its_partials(ops):
    """Streams can be captured by every entry point; a captured split-KV decode keeps the buffer of
    its partials when a later call needs a larger one, and a graph's buffer serves no other call."""
    gen = torch.Generator().manual_seed(27)
    h, hkv, d, keys = 28, 4, 128, 6000

    def problem(n):
        q = _randn(gen, n, h, d).cuda()
        k, v = _randn(gen, n * keys, hkv, d).cuda(), _randn(gen, n * keys, hkv, d).cuda()
        return q, k, v, np.array([(i, i * keys, keys, -1, 0, 0) for i in range(n)], np.int32), torch.zeros_like(q)

    run = lambda q, k, v, s, out: ops.decode_splitkv(q, s, scale=0.1, num_kv_heads=hkv, out=out, peer_k=k, peer_v=v)  # noqa: E731
    small, large = problem(2), problem(40)
    run(*small)
    want = small[4].clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(*small)
        graphs.append(g)
    run(*large)
    ref = large[4].clone()
    junk = [torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(64)]
    for g in graphs:
        small[4].zero_()
        g.replay()
        run(*large)
        torch.cuda.synchronize()
        assert torch.equal(small[4], want) and torch.equal(large[4], ref)
    del junk


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured ones: nothing has to be warmed up."""
    import subprocess
    import sys
    code = """
import torch
from hcp_vllm_plugin_b200 import ops
cache = torch.zeros(ops.kv_cache_q4_shape(4, 2, 16, 128), dtype=torch.uint8, device="cuda")
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
table, free, head, ctx, new = i32(*([-1] * 4)).view(2, 2), i32(0, 1, 2, 3), i32(0), i32(0, 0), i32(5, 3)
q, k, v = (torch.randn(8, n, 128, device="cuda").bfloat16() for n in (4, 2, 2))
tab = torch.cat([torch.ones(9, 64, device="cuda"), torch.zeros(9, 64, device="cuda")], -1)
out = torch.zeros_like(q)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    plan = ops.kv_plan_step(ctx, new, table, free, head, block_size=16, num_tokens=8)
    qr, kr = ops.qk_norm_rope(q, k, plan.positions, tab, value=v, kv_cache=cache, slot_mapping=plan.slot_mapping)
    ops.decode_splitkv_q4(qr, cache, table, plan.kv_lens, scale=0.1, out=out, token_req=plan.token_req)
    kc, vc = ops.kv_cache_gather_q4(cache, plan.slot_mapping, torch.bfloat16)
g.replay()
torch.cuda.synchronize()
assert table[:, 0].tolist() == [0, 1] and (vc - v).abs().max() < 0.6
assert (out[0].view(2, 2, 128) - vc[0][:, None]).abs().max() < 0.05   # the first row sees one key
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_q4_decode_joins_a_peer_partial(ops):
    """Local keys in 4 bits, peer keys in 16: each with its LSE, joined by merge_attn_states."""
    gen = torch.Generator().manual_seed(24)
    rows, h, hkv, d, bs, nb, peer = 3, 28, 4, 128, 16, 60, 200
    cache = _filled(ops, gen, nb, hkv, bs, d, BF16)
    table, lens = torch.randint(0, nb, (rows, 30), generator=gen, dtype=torch.int32), [300, 0, 17]
    q, pk, pv = _randn(gen, rows, h, d), _randn(gen, rows * peer, hkv, d), _randn(gen, rows * peer, hkv, d)
    scale = d ** -0.5
    lo, ll = torch.empty(rows, h, d, device="cuda"), torch.empty(h, rows, device="cuda")
    po, pl = torch.empty(rows, h, d, device="cuda"), torch.empty(h, rows, device="cuda")
    ops.decode_splitkv_q4(q.cuda(), cache, table.cuda(), _i32(lens), scale=scale, out=lo, lse=ll)
    seqs = np.array([(r, r * peer, peer, -1, 0, 0) for r in range(rows)], np.int32)
    ops.decode_splitkv(q.cuda(), seqs, scale=scale, num_kv_heads=hkv, out=po, lse=pl, peer_k=pk.cuda(), peer_v=pv.cuda())
    out, lse = torch.empty(rows, h, d, device="cuda"), torch.empty(h, rows, device="cuda")
    ops.merge_attn_states(out, po, pl, lo, ll, output_lse=lse)
    kmem, vmem = R.read_q4(cache.cpu().numpy(), np.arange(nb * bs), BF16)
    for r in range(rows):
        p = np.arange(lens[r])
        slots = table.numpy()[r, p // bs].astype(np.int64) * bs + p % bs
        k = np.concatenate([R.f64(pk)[r * peer: (r + 1) * peer], kmem[slots]])
        v = np.concatenate([R.f64(pv)[r * peer: (r + 1) * peer], vmem[slots]])
        # the merge's own weights: expf and its sums, 2^-20 of each term
        o, l = R.attention(R.f64(q[r]), k, v, scale)
        assert np.abs(R.f64(out[r]) - o).max() <= 1e-3 and np.abs(R.f64(lse[:, r]) - l).max() <= 1e-3


def test_gathered_prefix_feeds_the_prefill_kernel(ops):
    """A chunk attends its 4-bit prefix as the rows the gather gives back."""
    from hcp_vllm_plugin_b200 import _capi as C
    gen = torch.Generator().manual_seed(25)
    h, hkv, d, bs, prefix, chunk = 8, 2, 128, 16, 100, 40
    cache = _filled(ops, gen, 10, hkv, bs, d, BF16)
    slots = torch.arange(prefix)
    kp, vp = ops.kv_cache_gather_q4(cache, slots.cuda(), BF16)
    q, kl, vl = _randn(gen, chunk, h, d).cuda(), _randn(gen, chunk, hkv, d).cuda(), _randn(gen, chunk, hkv, d).cuda()
    out, lse = torch.empty_like(q), torch.empty(h, chunk, device="cuda")
    ops.ring_attn_fwd(q, ops.make_work([(0, chunk, 0, 0, (C.HCP_SRC_A, 0, prefix, -1), (C.HCP_SRC_B, 0, chunk, 0))]),
                      scale=d ** -0.5, num_kv_heads=hkv, out=out, lse=lse, k_a=kp, v_a=vp, k_b=kl, v_b=vl)
    for i in range(chunk):
        k = np.concatenate([R.f64(kp), R.f64(kl)[: i + 1]])
        v = np.concatenate([R.f64(vp), R.f64(vl)[: i + 1]])
        o, l = R.attention(R.f64(q[i]), k, v, d ** -0.5)
        # the prefill kernel's bar: 2e-3, and half a step of its 16-bit output
        assert (np.abs(R.f64(out[i]) - o) <= 2e-3 + 2.0 ** -8 * np.abs(o)).all()
        assert np.abs(R.f64(lse[:, i]) - l).max() <= 1e-3


def test_shapes_that_do_not_fit_are_refused(ops):
    """Every refusal comes before a launch: outputs and caches stay."""
    t = lambda *shape, dtype=BF16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    i32, i64, u8 = torch.int32, torch.int64, torch.uint8
    q, k, v, pos, tab = t(4, 8, 128), t(4, 2, 128), t(4, 2, 128), t(4, dtype=i64), t(9, 128, dtype=torch.float32)
    slots, cache = t(4, dtype=i64), t(3, 2, 16, 144, dtype=u8)
    rope = lambda q=q, k=k, pos=pos, tab=tab, **kw: ops.qk_norm_rope(q, k, pos, tab, **kw)  # noqa: E731
    wrote = dict(value=v, kv_cache=cache, slot_mapping=slots)
    dec = lambda q=q, cache=cache, bt=t(4, 3, dtype=i32), lens=t(4, dtype=i32), out=q.clone(), **kw: ops.decode_splitkv_q4(  # noqa: E731
        q, cache, bt, lens, **{"scale": 0.1, "out": out, **kw})
    plan = lambda c=t(3, dtype=i32), n=t(3, dtype=i32), bt=t(3, 5, dtype=i32), f=t(9, dtype=i32), h=t(1, dtype=i32), **kw: (  # noqa: E731
        ops.kv_plan_step(c, n, bt, f, h, **{"block_size": 16, "num_tokens": 3, **kw}))
    refused = [
        lambda: rope(q=t(4, 8, 128, dtype=torch.float32)), lambda: rope(k=t(3, 2, 128)), lambda: rope(k=t(4, 2, 64)),
        lambda: rope(pos=t(3, dtype=i64)), lambda: rope(pos=t(4, dtype=i32)), lambda: rope(tab=t(9, 128, dtype=F16)),
        lambda: rope(tab=t(9, 256, dtype=torch.float32)[:, ::2]), lambda: rope(tab=t(9, 20, dtype=torch.float32)),
        lambda: rope(tab=t(9, 130, dtype=torch.float32)), lambda: rope(q_weight=t(64)), lambda: rope(k_weight=t(128, dtype=F16)),
        lambda: rope(q_out=t(4, 8, 64)), lambda: rope(k_out=t(4, 2, 128, dtype=F16)), lambda: rope(q=t(4, 128, 8).transpose(1, 2)),
        lambda: rope(value=v), lambda: rope(kv_cache=cache), lambda: rope(**{**wrote, "value": t(4, 1, 128)}),
        lambda: rope(**{**wrote, "slot_mapping": t(3, dtype=i64)}), lambda: rope(**{**wrote, "kv_cache": t(3, 2, 16, 72, dtype=u8)}),
        lambda: rope(**{**wrote, "kv_cache": t(3, 1, 16, 144, dtype=u8)}), lambda: rope(**{**wrote, "kv_cache": t(3, 2, 24, 144, dtype=u8)}),
        lambda: rope(**{**wrote, "kv_cache": t(3, 2, 16, 256, dtype=F16)}), lambda: rope(**{**wrote, "kv_cache": t(3, 2, 16, 128)}),
        lambda: rope(eps=-1.0), lambda: rope(q=t(4, 8, 96), k=t(4, 2, 96), tab=t(9, 96, dtype=torch.float32)),
        lambda: ops.kv_cache_update_q4(k, t(4, 2, 128, dtype=F16), cache, slots), lambda: ops.kv_cache_update_q4(k, t(3, 2, 128), cache, slots),
        lambda: ops.kv_cache_update_q4(t(4, 3, 128), t(4, 3, 128), cache, slots), lambda: ops.kv_cache_update_q4(k, v, cache, t(4, dtype=i32)),
        lambda: ops.kv_cache_update_q4(k, v, t(3, 2, 16, 256), slots), lambda: ops.kv_cache_update_q4(k, v, cache[:, :, ::2], slots),
        lambda: ops.kv_cache_update_q4(t(4, 2, 136)[:, :, 8:], v, cache, slots),
        lambda: ops.kv_cache_gather_q4(cache, slots, torch.float32), lambda: ops.kv_cache_gather_q4(cache, slots, BF16, key=t(3, 2, 128)),
        lambda: ops.kv_cache_gather_q4(cache, slots, BF16, value=t(4, 2, 128, dtype=F16)), lambda: ops.kv_cache_gather_q4(cache, slots, BF16, key=t(4, 1, 128)),
        lambda: dec(q=t(4, 8, 64)), lambda: dec(q=t(4, 7, 128), out=t(4, 7, 128)), lambda: dec(q=t(4, 34, 128), out=t(4, 34, 128)),
        lambda: dec(lens=t(3, dtype=i32)), lambda: dec(lens=t(4, dtype=i64)), lambda: dec(bt=t(3, 3, dtype=i32)),
        lambda: dec(bt=t(4, 3, dtype=i64)), lambda: dec(bt=t(4, 6, dtype=i32)[:, ::2]), lambda: dec(out=t(3, 8, 128)),
        lambda: dec(out=t(4, 8, 128, dtype=F16)), lambda: dec(lse=t(8, 3, dtype=torch.float32)), lambda: dec(lse=t(7, 4, dtype=torch.float32)),
        lambda: dec(scale=0.0), lambda: dec(scale=float("nan")), lambda: dec(token_req=t(3, dtype=i32)), lambda: dec(workspace=t(64, dtype=u8)),
        lambda: dec(cache=t(3, 2, 24, 144, dtype=u8)), lambda: dec(cache=t(0, 2, 16, 144, dtype=u8)),
        lambda: plan(n=t(2, dtype=i32)), lambda: plan(c=t(3, dtype=i64)), lambda: plan(bt=t(2, 5, dtype=i32)), lambda: plan(bt=t(3, 5, dtype=i64)),
        lambda: plan(f=t(9, dtype=i64)), lambda: plan(h=t(0, dtype=i32)), lambda: plan(pos_base=t(2, dtype=i32)), lambda: plan(block_size=0),
        lambda: plan(num_tokens=-1), lambda: plan(bt=t(3, 10, dtype=i32)[:, ::2]), lambda: plan(f=t(18, dtype=i32)[::2]),
    ]
    from hcp_vllm_plugin_b200._capi import HcpError
    for n, call in enumerate(refused):
        with pytest.raises((ValueError, HcpError)):
            call()
            raise AssertionError(f"call {n} was taken")
    torch.cuda.synchronize()
    assert bool((cache == 0).all())


def test_on_the_tensors_device_not_the_current_one(ops):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    gen = torch.Generator().manual_seed(26)
    with torch.cuda.device(1):
        step = _Step(ops, gen, 2, 8, 4)
        _feed(step, gen, [3, 4])
    step.run()
    torch.cuda.synchronize(1)
    _check_step(step, [0, 0], [3, 4])
