"""Plain restatements (numpy, 64 bits, loops) of the serving-step operators:
step plan, norm and rotation, the 4-bit cache and attention over it.  They are
written from the definitions in ``include/hcp_ring.h`` and the byte layout in
``q4_cache.cuh``, one token at a time."""

from __future__ import annotations

import numpy as np
import torch

TILE = 16


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().to("cpu", torch.float64).numpy()


def round16(x: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    """Nearest value of the 16-bit type (ties to even), in 32 bits."""
    with np.errstate(over="ignore"):
        return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dtype).float().numpy()


def bits16(x: np.ndarray, dtype: torch.dtype) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dtype).view(torch.int16).numpy().view(np.uint16)


# ------------------------------------------------------------------ the plan

def plan(context, new, table, free, head, block_size, num_tokens, base=None):
    table = table.copy()
    reqs, width = len(context), table.shape[1]
    out = {"query_start": [0], "seq_lens": [], "positions": np.full(num_tokens, -1, np.int64),
           "slot_mapping": np.full(num_tokens, -1, np.int64), "token_req": np.full(num_tokens, -1, np.int32),
           "kv_lens": np.zeros(num_tokens, np.int32)}
    head = min(max(head, 0), len(free))
    missing, t = 0, 0
    for i in range(reqs):
        c, n = max(0, int(context[i])), max(0, int(new[i]))
        have, want = -(-c // block_size), -(-(c + n) // block_size)
        for k in range(have, want):
            if k < width and head < len(free):
                table[i, k] = free[head]
                head += 1
            else:
                missing += 1
                if k < width:
                    table[i, k] = -1
        for p in range(c, c + n):
            if t < num_tokens:
                page = table[i, p // block_size] if p // block_size < width else -1
                out["positions"][t] = p + (0 if base is None else int(base[i]))
                out["slot_mapping"][t] = page * block_size + p % block_size if page >= 0 else -1
                out["token_req"][t] = i
                out["kv_lens"][t] = p + 1
            t += 1
        out["seq_lens"].append(c + n)
        out["query_start"].append(t)
    return {**out, "free_head": [head], "missing": [missing], "block_table": table}


# ------------------------------------------------------------------ norm and rotation

def norm_rope(x, weight, positions, table, eps, interleaved):
    """x [T, H, D] and table in 64 bits -> [T, H, D]; rows of positions past the table are NaN."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * weight
    half = table.shape[1] // 2
    out = y.copy()
    for t, p in enumerate(positions):
        if p < 0:
            continue
        if p >= table.shape[0]:
            out[t] = np.nan
            continue
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = table[p, i], table[p, half + i]
            out[t, :, a] = y[t, :, a] * c - y[t, :, b] * s
            out[t, :, b] = y[t, :, b] * c + y[t, :, a] * s
    return out


# ------------------------------------------------------------------ the 4-bit cache

def group(x: np.ndarray, dtype: torch.dtype):
    """Whole numbers, scale and lowest value of one group of 64 (in 32 bits, as defined)."""
    x = np.asarray(x, np.float32)
    nan = np.float32(np.nan)
    if not np.isfinite(x).all():
        return np.zeros(64, np.uint8), nan, nan
    lo, hi = x.min(), x.max()
    with np.errstate(over="ignore"):
        s = round16(np.array([(hi - lo) / np.float32(15)]), dtype)[0]
    if not np.isfinite(s):
        return np.zeros(64, np.uint8), nan, nan
    if s == 0:
        return np.zeros(64, np.uint8), s, lo
    return np.clip(np.rint((x - lo) / s), 0, 15).astype(np.uint8), s, lo


def write_q4(cache: np.ndarray, key, value, slots, dtype) -> None:
    """key/value [n, Hkv, D] fp32 into uint8 [num_blocks, Hkv, block_size, 9 * D / 8], one element at a time."""
    nb, hkv, bs, last = cache.shape
    d = last * 8 // 9
    groups = d // 64
    flat = cache.reshape(-1)
    for i, slot in enumerate(slots):
        if slot < 0 or slot >= nb * bs:
            continue
        blk, off = divmod(int(slot), bs)
        sub, j = divmod(off, TILE)
        for h in range(hkv):
            tile = ((blk * hkv + h) * (bs // TILE) + sub) * 18 * d
            for side, rows in enumerate((key, value)):
                for g in range(groups):
                    n, s, lo = group(rows[i, h, 64 * g: 64 * g + 64], dtype)
                    at = tile + 16 * d + j * (d // 8) + 4 * (side * groups + g)
                    pair = bits16(np.array([s, lo]), dtype)
                    if np.isnan(s):
                        pair[:] = NAN16[dtype]
                    flat[at: at + 4] = pair.view(np.uint8)
                    for e in range(64):
                        dim = 64 * g + e
                        b = dim // 8
                        if side == 0:
                            word = (b % 8) // 2 * 2 * groups + b // 8 * 2 + b % 2
                            byte = tile + j * (d // 2) + 4 * word + dim % 8 // 2
                        else:
                            byte = tile + 8 * d + 64 * b + j // 4 * 16 + dim % 8 // 2 * 4 + j % 4
                        keep = flat[byte] & (0xF0 if dim % 2 == 0 else 0x0F)
                        flat[byte] = keep | (n[e] << (0 if dim % 2 == 0 else 4))


#: What a NaN of 32 bits becomes in 16 (the quiet NaN with a positive sign).
NAN16 = {torch.bfloat16: np.uint16(0x7FFF), torch.float16: np.uint16(0x7FFF)}


def read_q4(cache: np.ndarray, slots, dtype):
    """K and V [n, Hkv, D] in 64 bits, unrounded; zeros for slots outside the cache."""
    nb, hkv, bs, last = cache.shape
    d = last * 8 // 9
    groups = d // 64
    flat = cache.reshape(-1)
    slots = np.asarray(slots, np.int64)
    out = np.zeros((2, len(slots), hkv, d))
    dims = np.arange(d)
    b = dims // 8
    word = (b % 8) // 2 * 2 * groups + b // 8 * 2 + b % 2
    shift = 4 * (dims % 2)
    for i, slot in enumerate(slots):
        if slot < 0 or slot >= nb * bs:
            continue
        blk, off = divmod(int(slot), bs)
        sub, j = divmod(off, TILE)
        for h in range(hkv):
            tile = ((blk * hkv + h) * (bs // TILE) + sub) * 18 * d
            kn = (flat[tile + j * (d // 2) + 4 * word + dims % 8 // 2] >> shift) & 15
            vn = (flat[tile + 8 * d + 64 * b + j // 4 * 16 + dims % 8 // 2 * 4 + j % 4] >> shift) & 15
            at = tile + 16 * d + j * (d // 8)
            prm = torch.from_numpy(flat[at: at + d // 8].copy()).view(dtype).double().numpy().reshape(2, groups, 2)
            for side, n in enumerate((kn, vn)):
                out[side, i, h] = n * np.repeat(prm[side, :, 0], 64) + np.repeat(prm[side, :, 1], 64)
    return out[0], out[1]


def attention(q, k, v, scale):
    """One row: q [H, D], k/v [n, Hkv, D] in 64 bits -> out [H, D], lse [H]."""
    h, d = q.shape
    if k.shape[0] == 0:
        return np.zeros((h, d)), np.full(h, -np.inf)
    group_size = h // k.shape[1]
    out, lse = np.zeros((h, d)), np.zeros(h)
    for i in range(h):
        s = k[:, i // group_size] @ q[i] * scale
        m = s.max()
        p = np.exp(s - m)
        lse[i] = m + np.log(p.sum())
        out[i] = p @ v[:, i // group_size] / p.sum()
    return out, lse
