"""What the serving-step operators are measured on: planning a step's cache
slots on the GPU, norm and rotation of queries and keys, the 4-bit paged cache
and single-token attention over it.

Four kinds of case:

``plan``    ``ops.kv_plan_step``: block tables, slots, positions and lengths of
            one engine step from the requests' lengths;
``rope``    ``ops.qk_norm_rope``: per-head RMS norm and rotation of q and k, and
            the cache write of k and v in the same pass;
``chunk``   ``ops.kv_cache_update_q4`` then ``ops.kv_cache_gather_q4``: one
            chunk of a chunked prefill goes into the 4-bit cache and the whole
            context comes back as 16-bit rows for the prefill kernel;
``decode``  ``ops.decode_splitkv_q4``: one query row per sequence over its
            4-bit paged keys.

The 4-bit cache is uint8 [num_blocks, Hkv, block_size, 9 * D / 8].  A group is
64 dims of one token, head and side (K or V): it has a scale s and a lowest
value m in the 16-bit type of the rows, and each element is m + s * n with a
whole number n in 0..15.  One (block, head) is block_size / 16 tiles of 16
tokens, 18 * D bytes each:

  [0, 8D)     K: token j at j * D/2; 32-bit words of 8 dims, block b of 8 dims at
              word (b%8)/2 * 2*D/64 + b/8*2 + b%2; dim 8b+i in bits 4i..4i+3
  [8D, 16D)   V: block b of 8 dims at 64b; token 4t+i, dims 8b+2m and 8b+2m+1 in
              the low and high half of byte 16t + 4m + i
  [16D, 18D)  token j at j * D/8: (s, m) of each K group, then of each V group
"""

import math
import random

import torch

own = False

#: Query heads, KV heads, head size: the geometry of the benchmark's model, and the small one of the decode tests.
LARGE, SMALL = (28, 4, 128), (14, 2, 64)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX_POSITION = 131072
EPS = 1e-6


def _plan(name, requests, newest, longest, block_size, padded):
    return {"name": name, "kind": "plan", "requests": requests, "newest": newest, "longest": longest, "block_size": block_size, "padded": padded}


def _rope(name, tokens, heads, dtype, rotary, interleaved, table, cache, block_size):
    h, hkv, d = heads
    return {"name": name, "kind": "rope", "tokens": tokens, "heads": h, "kv_heads": hkv, "dim": d, "dtype": dtype, "rotary": rotary,
            "interleaved": interleaved, "table": table, "cache": cache, "block_size": block_size}


def _chunk(name, tokens, context, heads, dtype, block_size):
    _, hkv, d = heads
    return {"name": name, "kind": "chunk", "tokens": tokens, "context": context, "kv_heads": hkv, "dim": d, "dtype": dtype, "block_size": block_size}


def _decode(name, rows, shortest, longest, heads, dtype, block_size):
    h, hkv, d = heads
    return {"name": name, "kind": "decode", "rows": rows, "shortest": shortest, "longest": longest, "heads": h, "kv_heads": hkv, "dim": d,
            "dtype": dtype, "block_size": block_size}


def listed():
    return [
        # a handful of requests that each decode one token: the smallest step, where only latency counts
        _plan("plan_decode_8", 8, 1, 2048, 16, 8),
        # a full serving batch of decodes with long contexts
        _plan("plan_decode_1024", 1024, 1, 32768, 16, 1024),
        # a continuous batch: prefill chunks beside decodes and idle requests, in a buffer padded to its captured size
        _plan("plan_mixed_257", 257, 128, 8192, 32, 20000),
        # the decode step of the benchmark's batch of 64, keys and values into the 16-bit cache
        _rope("rope_decode_64", 64, LARGE, "bf16", 128, False, "f32", "same", 16),
        # one 16k-token prefill chunk straight into the 4-bit cache
        _rope("rope_prefill_16384_q4", 16384, LARGE, "bf16", 128, False, "f32", "q4", 16),
        # an odd chunk in fp16: small heads, half of each rotated in neighbouring pairs, no cache
        _rope("rope_f16_4099", 4099, SMALL, "f16", 32, True, "same", "none", 16),
        # the tail of a short prompt joins its cached prefix
        _chunk("chunk_33_of_500", 33, 500, LARGE, "bf16", 16),
        # one chunk of a long chunked prefill: 4096 tokens written, 64k read back
        _chunk("chunk_4096_of_65536", 4096, 65536, LARGE, "bf16", 16),
        # an interactive batch with short contexts
        _decode("decode_16_short", 16, 1, 300, LARGE, "bf16", 16),
        # one request with a 128k-token context: the long axis alone has to fill the card
        _decode("decode_1_131072", 1, 131072, 131072, LARGE, "bf16", 16),
        # ragged lengths, empty rows among them, small heads in fp16, larger pages
        _decode("decode_33_ragged_f16", 33, 0, 9001, SMALL, "f16", 32),
        # the benchmark's long-context decode batch: 64 sequences of 32768 cached tokens
        _decode("decode_64_32768", 64, 32768, 32768, LARGE, "bf16", 16),
    ]


def _between(rng, low, high):
    """A whole number between two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "chunk", "decode"])
    heads, dtype, bs = rng.choice([LARGE, SMALL]), rng.choice(["bf16", "f16"]), rng.choice([16, 32, 64])
    if kind == "plan":
        requests = _between(rng, 1, 1024)
        newest = rng.choice([1, _between(rng, 2, max(2, 20000 // requests))])
        c = _plan("", requests, newest, _between(rng, 16, 32768), bs, requests * newest + rng.choice([0, rng.randrange(100)]))
    elif kind == "rope":
        rotary = rng.choice([heads[2], heads[2] // 2])
        c = _rope("", _between(rng, 1, 16384), heads, dtype, rotary, rng.random() < 0.5, rng.choice(["f32", "same"]), rng.choice(["none", "same", "q4"]), bs)
    elif kind == "chunk":
        context = _between(rng, 16, 65536)
        c = _chunk("", _between(rng, 1, min(context, 4096)), context, heads, dtype, bs)
    else:
        rows = _between(rng, 1, 64)
        longest = _between(rng, 16, min(131072, 64 * 32768 // rows))
        c = _decode("", rows, rng.choice([0, 1, longest // 2, longest]), longest, heads, dtype, bs)
    del c["name"]
    return c


def _lengths(case):
    """A decode case's lengths: they belong to the case, so that its work is known; the first row is the longest."""
    r = random.Random("%(rows)d %(shortest)d %(longest)d" % case)
    return [case["longest"]] + [r.randint(case["shortest"], case["longest"]) for _ in range(case["rows"] - 1)]


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _quantised(x):
    """Whole numbers, scales and lowest values of x [..., D] in groups of 64: (n uint8 [..., D], s, m [..., D/64] in x's type)."""
    g = x.float().unflatten(-1, (-1, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((high - low) / 15.0).to(x.dtype).float()
    n = torch.where(s > 0, torch.round((g - low) / torch.where(s > 0, s, 1.0)).clamp(0, 15), 0.0)
    return n.to(torch.uint8).flatten(-2), s.to(x.dtype).squeeze(-1), low.to(x.dtype).squeeze(-1)


def _pairs(n):
    """Two whole numbers to a byte, the even one in the low half."""
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _tiles(k, v):
    """Tiles uint8 [n, 18 * D] of k and v [n, 16, D]."""
    n, _, d = k.shape
    (kn, ks, km), (vn, vs, vm) = _quantised(k), _quantised(v)
    kb = _pairs(kn).view(n, 16, d // 64, 4, 2, 4).permute(0, 1, 3, 2, 4, 5).reshape(n, 8 * d)
    vb = _pairs(vn).view(n, 4, 4, d // 8, 4).permute(0, 3, 1, 4, 2).reshape(n, 8 * d)
    side = [torch.stack([s, m], -1).flatten(-2) for s, m in ((ks, km), (vs, vm))]
    return torch.cat([kb, vb, torch.cat(side, -1).contiguous().view(torch.uint8).reshape(n, 2 * d)], -1)


def _cache_q4(blocks, hkv, bs, d, dtype, g):
    """A filled 4-bit cache.  A few thousand tiles of quantised normal rows stand at random places of it."""
    tiles = blocks * hkv * (bs // 16)
    some = min(tiles, 4096)
    pool = _tiles(_normal((some, 16, d), dtype, g), _normal((some, 16, d), dtype, g))
    return pool[torch.randint(some, (tiles,), generator=g, device="cuda")].view(blocks, hkv, bs, 9 * d // 8)


def _slots(positions, table, bs):
    """Cache slots of one request's positions through its row of block ids."""
    return table[positions // bs].long() * bs + positions % bs


def _prepare_plan(case, g):
    r, bs = case["requests"], case["block_size"]
    context = torch.randint(0, case["longest"] + 1, (r,), generator=g, device="cuda", dtype=torch.int32)
    if case["newest"] == 1:
        new = torch.ones(r, device="cuda", dtype=torch.int32)
    else:  # chunks, decodes and requests that wait
        new = torch.randint(0, case["newest"] + 1, (r,), generator=g, device="cuda", dtype=torch.int32)
        new = torch.where(torch.rand(r, generator=g, device="cuda") < 0.5, new.clamp(max=1), new)
    width = -(-(case["longest"] + case["newest"]) // bs)
    blocks = r * width + 7
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    table = ids[: r * width].view(r, width).clone()
    table[torch.arange(width, device="cuda") >= (-(-context // bs))[:, None]] = -1
    base = torch.randint(0, 4, (r,), generator=g, device="cuda", dtype=torch.int32) * 16384  # the chunk of a split sequence that this GPU holds
    spare = r * (-(-case["newest"] // bs) + 1) + 16
    return {"context": context, "new": new, "table": table, "free": torch.randperm(spare, generator=g, device="cuda").to(torch.int32) + blocks,
            "head": torch.tensor([5], device="cuda", dtype=torch.int32), "base": base}


def _prepare_rope(case, g):
    t, h, hkv, d, bs, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["block_size"], TYPES[case["dtype"]]
    qkv = _normal((t, (h + 2 * hkv) * d), dtype, g)  # as the projection leaves it
    q, k, v = (x.view(t, -1, d) for x in qkv.split([h * d, hkv * d, hkv * d], -1))
    s = {"q": q, "k": k, "v": v, "qw": (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype),
         "kw": (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)}
    start = int(torch.randint(0, MAX_POSITION - t + 1, (1,), generator=g, device="cuda"))
    s["positions"] = torch.arange(start, start + t, device="cuda") if t > 64 else torch.randint(0, MAX_POSITION, (t,), generator=g, device="cuda")
    half = case["rotary"] // 2
    angle = torch.arange(MAX_POSITION, device="cuda", dtype=torch.float64)[:, None] * (1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
    s["table"] = torch.cat([angle.cos(), angle.sin()], -1).to(torch.float32 if case["table"] == "f32" else dtype)
    blocks = -(-t // bs) + 3
    pages = torch.randperm(blocks, generator=g, device="cuda")
    s["slots"] = _slots(torch.arange(t, device="cuda"), pages, bs)
    if case["cache"] == "same":
        s["cache"] = torch.zeros(blocks, hkv, bs, 2 * d, device="cuda", dtype=dtype)
    elif case["cache"] == "q4":
        s["cache"] = torch.zeros(blocks, hkv, bs, 9 * d // 8, device="cuda", dtype=torch.uint8)
    return s


def _prepare_chunk(case, g):
    t, n, hkv, d, bs, dtype = case["tokens"], case["context"], case["kv_heads"], case["dim"], case["block_size"], TYPES[case["dtype"]]
    blocks = -(-n // bs) + 3
    pages = torch.randperm(blocks, generator=g, device="cuda")
    slots = _slots(torch.arange(n, device="cuda"), pages, bs)
    return {"cache": _cache_q4(blocks, hkv, bs, d, dtype, g), "key": _normal((t, hkv, d), dtype, g), "value": _normal((t, hkv, d), dtype, g),
            "slots": slots, "new": slots[n - t:].clone()}


def _prepare_decode(case, g):
    h, hkv, d, bs, dtype = case["heads"], case["kv_heads"], case["dim"], case["block_size"], TYPES[case["dtype"]]
    lens = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    width = -(-case["longest"] // bs)
    blocks = case["rows"] * width + 3
    table = torch.randperm(blocks, generator=g, device="cuda")[: case["rows"] * width].to(torch.int32).view(case["rows"], width).clone()
    table[torch.arange(width, device="cuda") >= (-(-lens // bs))[:, None]] = -1
    return {"cache": _cache_q4(blocks, hkv, bs, d, dtype, g), "q": _normal((case["rows"], h, d), dtype, g), "table": table, "lens": lens}


def prepare(case, seed):
    state = globals()["_prepare_" + case["kind"]](case, _generator(seed))
    return {"case": case, **state}


# ---------------------------------------------------------------- plain forms

def _plan_plain(s):
    case, table, free = s["case"], s["table"], s["free"]
    bs, tokens, width, spare = case["block_size"], case["padded"], table.shape[1], free.shape[0]
    context, new = s["context"].clamp(min=0).long(), s["new"].clamp(min=0).long()
    lens = context + new
    have, wanted = (context + bs - 1) // bs, (lens + bs - 1) // bs
    need = (wanted.clamp(max=width) - have).clamp(min=0)
    first = s["head"].long() + need.cumsum(0) - need
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    col = torch.arange(width, device="cuda")
    nth = col - have[:, None]
    at = first[:, None] + nth
    taken = torch.where(at < spare, free[at.clamp(0, spare - 1)], -1)
    table.copy_(torch.where((nth >= 0) & (nth < need[:, None]), taken, table))
    row = torch.arange(tokens, device="cuda")
    req = torch.searchsorted(starts[1:], row, right=True)
    real = req < new.shape[0]
    r = req.clamp(max=new.shape[0] - 1)
    pos = context[r] + row - starts[r]
    page = torch.where(pos // bs < width, table[r, (pos // bs).clamp(0, width - 1)], -1)
    end = s["head"].long() + need.sum()
    missing = (wanted - have).clamp(min=0).sum() - (end.clamp(max=spare) - s["head"].long())
    return {"query_start": starts.int(), "seq_lens": lens.int(), "positions": torch.where(real, pos + s["base"].long()[r], -1),
            "slot_mapping": torch.where(real & (page >= 0), page.long() * bs + pos % bs, -1), "token_req": torch.where(real, r, -1).int(),
            "kv_lens": torch.where(real, pos + 1, 0).int(), "free_head": end.clamp(max=spare).int(), "missing": missing.int(), "block_table": table}


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, table, positions, interleaved):
    cos, sin = table[positions].float()[:, None].chunk(2, -1)
    rot, rest = x[..., : 2 * cos.shape[-1]], x[..., 2 * cos.shape[-1]:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = rot.chunk(2, -1)
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([rot, rest], -1)


def _places(slots, hkv, bs, d):
    """Where the bytes of each slot and head stand in the cache, [n, Hkv, 9 * D / 8]: K's and V's by pairs of dims, then the scales and lowest values."""
    tile = (slots // bs)[:, None] * (hkv * (bs // 16)) + torch.arange(hkv, device="cuda") * (bs // 16) + (slots % bs // 16)[:, None]
    j = (slots % 16)[:, None]
    c = torch.arange(d // 2, device="cuda")
    b, e = c // 4, c % 4
    key = j * (d // 2) + ((b % 8 // 2) * (2 * (d // 64)) + b // 8 * 2 + b % 2) * 4 + e
    value = 8 * d + b * 64 + j // 4 * 16 + e * 4 + j % 4
    more = 16 * d + j * (d // 8) + torch.arange(d // 8, device="cuda")
    return tile[:, :, None] * (18 * d) + torch.cat([key, value, more], -1)[:, None]


def _write_q4(cache, slots, k, v):
    d = k.shape[-1]
    (kn, ks, km), (vn, vs, vm) = _quantised(k), _quantised(v)
    more = torch.cat([torch.stack([ks, km], -1).flatten(-2), torch.stack([vs, vm], -1).flatten(-2)], -1).contiguous().view(torch.uint8)
    cache.view(-1)[_places(slots, cache.shape[1], cache.shape[2], d)] = torch.cat([_pairs(kn), _pairs(vn), more], -1)


def _read_q4(cache, slots, dtype):
    d = cache.shape[-1] * 8 // 9
    raw = cache.view(-1)[_places(slots, cache.shape[1], cache.shape[2], d)]
    n = torch.stack([raw[..., :d] & 15, raw[..., :d] >> 4], -1).flatten(-2).float().unflatten(-1, (2, d // 64, 64))
    more = raw[..., d:].contiguous().view(dtype).float().unflatten(-1, (2, d // 64, 2))
    x = (n * more[..., 0, None] + more[..., 1, None]).flatten(-2).to(dtype)
    return x[..., 0, :], x[..., 1, :]


def _rope_plain(s):
    case = s["case"]
    dtype = TYPES[case["dtype"]]
    q = _rotated(_normed(s["q"], s["qw"]), s["table"], s["positions"], case["interleaved"]).to(dtype)
    k = _rotated(_normed(s["k"], s["kw"]), s["table"], s["positions"], case["interleaved"]).to(dtype)
    if case["cache"] == "none":
        return {"q": q, "k": k}
    if case["cache"] == "same":
        s["cache"][s["slots"] // case["block_size"], :, s["slots"] % case["block_size"]] = torch.cat([k, s["v"]], -1)
        return {"q": q, "k": k, "cache": s["cache"]}
    _write_q4(s["cache"], s["slots"], k, s["v"])
    kc, vc = _read_q4(s["cache"], s["slots"], dtype)
    return {"q": q, "k": k, "cached_k": kc, "cached_v": vc}


def _chunk_plain(s):
    _write_q4(s["cache"], s["new"], s["key"], s["value"])
    k, v = _read_q4(s["cache"], s["slots"], TYPES[s["case"]["dtype"]])
    return {"k": k, "v": v}


def _opened(cache, table, dtype):
    """K and V fp32 [rows, Hkv, positions, D] of the pages in the table's rows."""
    hkv, bs, d = cache.shape[1], cache.shape[2], cache.shape[3] * 8 // 9
    rows, width = table.shape
    tiles = cache[table.clamp(min=0).long()].transpose(1, 2).reshape(rows, hkv, width * (bs // 16), 18 * d)
    kb = tiles[..., : 8 * d].unflatten(-1, (16, 4, d // 64, 2, 4)).permute(0, 1, 2, 3, 5, 4, 6, 7).flatten(4)
    vb = tiles[..., 8 * d: 16 * d].unflatten(-1, (d // 8, 4, 4, 4)).permute(0, 1, 2, 4, 6, 3, 5).flatten(3, 4).flatten(4)
    more = tiles[..., 16 * d:].contiguous().view(dtype).float().unflatten(-1, (16, 2, d // 64, 2))
    sides = []
    for side, raw in enumerate((kb, vb)):
        n = torch.stack([raw & 15, raw >> 4], -1).flatten(-2).float().unflatten(-1, (d // 64, 64))
        sides.append((n * more[..., side, :, 0, None] + more[..., side, :, 1, None]).flatten(-2).flatten(2, 3))
    return sides


def _decode_plain(s):
    case, q = s["case"], s["q"]
    rows, h, d = q.shape
    hkv = case["kv_heads"]
    k, v = _opened(s["cache"], s["table"], q.dtype)
    score = torch.matmul(q.float().view(rows, hkv, h // hkv, d), k.transpose(-1, -2)) * d ** -0.5
    score = score.masked_fill(torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).view(rows, h).t()
    return {"out": out.view(rows, h, d).to(q.dtype), "lse": lse.contiguous()}


# ---------------------------------------------------------------- the framework's calls

def _plan_own(s):
    from hcp_vllm_plugin_b200 import ops

    plan = ops.kv_plan_step(s["context"], s["new"], s["table"], s["free"], s["head"], block_size=s["case"]["block_size"],
                            num_tokens=s["case"]["padded"], pos_base=s["base"])
    return {"query_start": plan.query_start, "seq_lens": plan.seq_lens, "positions": plan.positions, "slot_mapping": plan.slot_mapping,
            "token_req": plan.token_req, "kv_lens": plan.kv_lens, "free_head": plan.free_head, "missing": plan.missing, "block_table": s["table"]}


def _rope_own(s):
    from hcp_vllm_plugin_b200 import ops

    more = {} if s["case"]["cache"] == "none" else {"value": s["v"], "kv_cache": s["cache"], "slot_mapping": s["slots"]}
    q, k = ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                            interleaved=s["case"]["interleaved"], **more)
    if s["case"]["cache"] == "none":
        return {"q": q, "k": k}
    if s["case"]["cache"] == "same":
        return {"q": q, "k": k, "cache": s["cache"]}
    kc, vc = ops.kv_cache_gather_q4(s["cache"], s["slots"], q.dtype)
    return {"q": q, "k": k, "cached_k": kc, "cached_v": vc}


def _chunk_own(s):
    from hcp_vllm_plugin_b200 import ops

    ops.kv_cache_update_q4(s["key"], s["value"], s["cache"], s["new"])
    k, v = ops.kv_cache_gather_q4(s["cache"], s["slots"], s["key"].dtype)
    return {"k": k, "v": v}


def _decode_own(s):
    from hcp_vllm_plugin_b200 import ops

    q = s["q"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[1], q.shape[0], device=q.device, dtype=torch.float32)
    ops.decode_splitkv_q4(q, s["cache"], s["table"], s["lens"], scale=q.shape[2] ** -0.5, out=out, lse=lse)
    return {"out": out, "lse": lse}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _plan_own, "rope": _rope_own, "chunk": _chunk_own, "decode": _decode_own}[kind](state)
    return {"plan": _plan_plain, "rope": _rope_plain, "chunk": _chunk_plain, "decode": _decode_plain}[kind](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "plan":
        r, t, bs = case["requests"], case["padded"], case["block_size"]
        mean = 1.0 if case["newest"] == 1 else 0.25 * case["newest"] + 0.5
        taken = r * mean / bs
        # lengths and bases in, lengths and starts out, each token's four values, the ids taken and those of the pages written to
        return {"bytes": r * 20 + t * 24 + taken * 8 + min(t, r * (mean / bs + 1)) * 4, "flops": 0}
    if case["kind"] == "rope":
        t, h, hkv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        n = t * (h + hkv) * d * 4 + t * 8 + t * case["rotary"] * (4 if case["table"] == "f32" else 2)
        if case["cache"] != "none":
            n += t * hkv * d * 2 + t * 8
        if case["cache"] == "same":
            n += t * hkv * d * 4
        if case["cache"] == "q4":  # written, read again by the call that gives the values, which writes 16 bits each
            n += 2 * t * hkv * d * 9 // 8 + t * hkv * d * 4
        return {"bytes": n, "flops": t * (h + hkv) * (4 * d + 3 * case["rotary"])}
    if case["kind"] == "chunk":
        t, n, hkv, d = case["tokens"], case["context"], case["kv_heads"], case["dim"]
        return {"bytes": t * hkv * d * (4 + 9 / 8) + n * hkv * d * (4 + 9 / 8) + 8 * (t + n), "flops": 4 * (t + n) * hkv * d}
    total, h, hkv, d = sum(_lengths(case)), case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": total * hkv * d * 9 / 8 + case["rows"] * h * (4 * d + 4) + total / case["block_size"] * 4, "flops": 4 * total * h * d}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_quantised(x, dtype):
    """The values, in 64 bits, that rows of the type hold in the cache."""
    out = torch.empty_like(x)
    for first in range(0, x.shape[-1], 64):
        g = x[..., first: first + 64]
        low = g.min(-1, keepdim=True).values
        s = ((g.max(-1, keepdim=True).values - low) / 15).to(dtype).double()
        n = torch.round((g - low) / s).clamp(0, 15)
        out[..., first: first + 64] = low + s * torch.where(s == 0, torch.zeros_like(n), n)
    return out


def _exact_rows(cache, table_row, head, count, dtype):
    """K and V in 64 bits, [count, D], of one request's first tokens and one head: each element is fetched by its own place."""
    bs, d = cache.shape[2], cache.shape[3] * 8 // 9
    p = torch.arange(count, device="cuda")
    flat = cache.reshape(-1)
    start = (table_row.long()[p // bs] * cache.shape[1] + head) * (bs * 9 * d // 8) + p % bs // 16 * (18 * d)
    side = []
    word, shift, vbyte = [], [], []
    for i in range(d):
        b = i // 8
        word.append(4 * (b % 8 // 2 * 2 * (d // 64) + b // 8 * 2 + b % 2) + i % 8 // 2)
        shift.append(4 * (i % 2))
        vbyte.append(8 * d + 64 * b + 4 * (i % 8 // 2))
    word, shift, vbyte = (torch.tensor(x, device="cuda") for x in (word, shift, vbyte))
    j = p % 16
    for k, at in enumerate((j[:, None] * (d // 2) + word, vbyte + (j // 4 * 16 + j % 4)[:, None])):
        n = (flat[start[:, None] + at].long() >> shift) & 15
        x = torch.empty(count, d, dtype=torch.float64, device="cuda")
        for grp in range(d // 64):
            a = start + 16 * d + j * (d // 8) + (k * (d // 64) + grp) * 4
            pair = flat[a[:, None] + torch.arange(4, device="cuda")].contiguous().view(dtype).double()
            x[:, 64 * grp: 64 * grp + 64] = n[:, 64 * grp: 64 * grp + 64].double() * pair[:, :1] + pair[:, 1:]
        side.append(x)
    return side


def _exact_rope(s, case):
    table, pos, w = s["table"].double(), s["positions"], {"q": s["qw"].double(), "k": s["kw"].double()}
    half = case["rotary"] // 2
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w[name]
        y = x.clone()
        for i in range(half):
            c, n = table[pos, i][:, None], table[pos, half + i][:, None]
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            y[..., a] = x[..., a] * c - x[..., b] * n
            y[..., b] = x[..., a] * n + x[..., b] * c
        out[name] = y
    if case["cache"] == "same":
        bs = case["block_size"]
        cache = torch.zeros(s["cache"].shape, dtype=torch.float64, device="cuda")
        both = torch.cat([out["k"], s["v"].double()], -1)
        for head in range(case["kv_heads"]):
            cache[s["slots"] // bs, head, s["slots"] % bs] = both[:, head]
        out["cache"] = cache
    if case["cache"] == "q4":
        dtype = TYPES[case["dtype"]]
        out["cached_k"] = _exact_quantised(out["k"].to(dtype).double(), dtype)
        out["cached_v"] = _exact_quantised(s["v"].double(), dtype)
    return out


def _exact_chunk(s, case):
    n, t, bs, dtype = case["context"], case["tokens"], case["block_size"], TYPES[case["dtype"]]
    pages = s["slots"][::bs] // bs
    heads = [_exact_rows(s["cache"], pages, h, n, dtype) for h in range(case["kv_heads"])]
    k, v = (torch.stack([x[i] for x in heads], 1) for i in (0, 1))
    k[n - t:], v[n - t:] = _exact_quantised(s["key"].double(), dtype), _exact_quantised(s["value"].double(), dtype)
    return {"k": k, "v": v}


def _exact_decode(s, case):
    q = s["q"].double()
    rows, h, d = q.shape
    group = h // case["kv_heads"]
    out = torch.zeros(rows, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((h, rows), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lengths(case)):
        for head in range(case["kv_heads"] if n else 0):
            k, v = _exact_rows(s["cache"], s["table"][r], head, n, s["q"].dtype)
            mine = slice(head * group, head * group + group)
            score = q[r, mine] @ k.t() / math.sqrt(d)
            lse[mine, r] = torch.logsumexp(score, -1)
            out[r, mine] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers: they have to be equal
    s = prepare(case, seed)
    return {"rope": _exact_rope, "chunk": _exact_chunk, "decode": _exact_decode}[case["kind"]](s, case)
