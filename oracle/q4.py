"""CPU oracle of the 4-bit KV pool, its attention and the GPU-built step tables, in
numpy and plain Python, from the definitions in include/serving_engine_b200.h.

Quantisation is stated in fp32 operation by operation (its codes are compared bit for
bit); reading back and attention are in float64.
"""
from __future__ import annotations

import numpy as np

GROUP = 64
BLOCK = 16


def k_nibble(d: int, r: int, i: int) -> int:
    """Place, in nibbles, of K's code of token r, dim i in its row."""
    w = min(d, 128)
    g = w // GROUP
    panel, grp, c = i // w, i % w // GROUP, i % GROUP
    word = panel * 8 * w + r * (w // 2) + (c // 16) * 8 * g + grp * 8 + (c // 8 % 2) * 4
    return 2 * word + (c % 2) * 4 + (c % 8) // 2


def v_nibble(d: int, r: int, i: int) -> int:
    w = min(d, 128)
    g = w // GROUP
    panel, grp, c, pair = i // w, i % w // GROUP, i % GROUP, r // 2
    turn = 2 * (pair % 4) if g == 2 else 4 * (pair // 2 % 2)
    word = panel * 8 * w + pair * w + ((c // 8) ^ turn) * 8 * g + grp * 8 + (c // 4 % 2) * 4
    return 2 * word + (r % 2) * 4 + c % 4


def pair_byte(d: int, r: int, grp: int) -> int:
    w = min(d, 128)
    g = w // GROUP
    return 8 * d + (grp // g) * 64 * g + (r * g + grp % g) * 4


def quantise(x: np.ndarray):
    """x [..., D] (values of the element type) -> codes uint8, scale fp16, low fp16 [..., D / 64]."""
    x = np.asarray(x, np.float32)
    x = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = x.min(-1), x.max(-1)  # NaN propagates
    bad = ~(np.isfinite(lo) & np.isfinite(hi))
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        scale = np.minimum((hi - lo) * np.float32(1 / 15), np.float32(65504)).astype(np.float16)
        low = np.clip(lo, np.float32(-65504), np.float32(65504)).astype(np.float16)
        s32, l32 = scale.astype(np.float32), low.astype(np.float32)
        inv = np.where(s32 > 0, np.float32(1) / s32, np.float32(0)).astype(np.float32)
        y = (x - l32[..., None]) * inv[..., None]
        n = np.where(bad[..., None], 0, np.rint(np.clip(np.nan_to_num(y), 0, 15))).astype(np.uint8)
    nan = np.array(0x7FFF, np.uint16).view(np.float16)
    scale, low = np.where(bad, nan, scale), np.where(bad, nan, low)
    return n.reshape(*n.shape[:-2], -1), scale, low


def write(plane: np.ndarray, x: np.ndarray, slots) -> None:
    """plane uint8 [blocks, H, 9 * D]; x [n, H, D] into its slots (those out of range skipped)."""
    d = x.shape[-1]
    where = k_nibble if write.kind == "k" else v_nibble
    n, scale, low = quantise(x)
    pairs = np.stack((scale, low), -1).view(np.uint8)  # [n, H, G * 4] grouped per (scale, low)
    pairs = pairs.reshape(*scale.shape, 4)
    table = np.array([[where(d, r, i) for i in range(d)] for r in range(BLOCK)])
    for t, s in enumerate(np.asarray(slots)):
        if not 0 <= s < plane.shape[0] * BLOCK:
            continue
        b, r = divmod(int(s), BLOCK)
        for h in range(x.shape[1]):
            row = plane[b, h]
            for i in range(d):
                at = table[r, i]
                keep = 0xF0 if at % 2 == 0 else 0x0F
                row[at // 2] = (row[at // 2] & keep) | (int(n[t, h, i]) << (4 * (at % 2)))
            for g in range(d // GROUP):
                at = pair_byte(d, r, g)
                row[at:at + 4] = pairs[t, h, g]


def write_kv(k_plane, v_plane, k, v, slots) -> None:
    for kind, plane, x in (("k", k_plane, k), ("v", v_plane, v)):
        write.kind = kind
        write(plane, x, slots)


def read(plane: np.ndarray, kind: str, d: int) -> np.ndarray:
    """uint8 [blocks, H, 9 * D] -> the values, float64 [blocks, 16, H, D]."""
    where = k_nibble if kind == "k" else v_nibble
    at = np.array([[where(d, r, i) for i in range(d)] for r in range(BLOCK)])
    n = (plane[..., at // 2] >> (4 * (at % 2)).astype(np.uint8)) & 15  # [blocks, H, 16, D]
    pb = np.array([[[pair_byte(d, r, g) + b for b in range(4)] for g in range(d // GROUP)] for r in range(BLOCK)])
    pairs = np.ascontiguousarray(plane[..., pb]).view(np.float16).astype(np.float64)  # [blocks, H, 16, G, 2]
    with np.errstate(invalid="ignore"):
        x = n.reshape(*n.shape[:-1], -1, GROUP) * pairs[..., 0:1] + pairs[..., 1:2]
    return x.reshape(*n.shape).transpose(0, 2, 1, 3)


def attention(q, k_plane, v_plane, block_table, q_starts, q_lens, k_lens, q_pos, scale, causal=True):
    """q float64 [T, HQ, D] -> (O, LSE, bound): O = 0 and LSE = -inf where nothing is seen, NaN
    rows left out of every sum; bound [T, HQ] is the largest |v| that the query sees."""
    t, hq, d = q.shape
    hkv = k_plane.shape[1]
    o, lse, top = np.zeros((t, hq, d)), np.full((t, hq), -np.inf), np.zeros((t, hq))
    for r in range(len(q_lens)):
        nk = max(int(k_lens[r]), 0)
        if nk == 0:
            continue
        ids = np.asarray(block_table[r][:-(-nk // BLOCK)])
        ok = (ids >= 0) & (ids < k_plane.shape[0])
        safe = np.where(ok, ids, 0)
        k = read(k_plane[safe], "k", d).reshape(-1, hkv, d)[:nk]
        v = read(v_plane[safe], "v", d).reshape(-1, hkv, d)[:nk]
        ok = np.repeat(ok, BLOCK)[:nk]
        for i in range(int(q_lens[r])):
            tok = int(q_starts[r]) + i
            seen = ok & (np.arange(nk) <= int(q_pos[r]) + i if causal else True)
            if not seen.any():
                continue
            for h in range(hq):
                kv = h // (hq // hkv)
                s = (k[seen, kv] @ q[tok, h]) * scale
                m = s.max()
                p = np.exp(s - m)
                o[tok, h] = p @ v[seen, kv] / p.sum()
                lse[tok, h] = m + np.log(p.sum())
                top[tok, h] = np.abs(v[seen, kv]).max()
    return o, lse, top


def step_tables(q_lens, context_lens, block_table, free_ids, head, count, total):
    """The metadata of seb_step_tables by a loop over rows; block_table is a copy that it extends."""
    table = np.array(block_table)
    rows, width = table.shape
    starts, k_lens, q_pos = [], [], []
    item, pos, slot = [-1] * total, [0] * total, [-1] * total
    t = taken = 0
    for r in range(rows):
        q, ctx = max(int(q_lens[r]), 0), max(int(context_lens[r]), 0)
        starts.append(t)
        k_lens.append(ctx + q)
        q_pos.append(ctx)
        for col in range(-(-ctx // BLOCK), min(-(-(ctx + q) // BLOCK), width)):
            table[r, col] = free_ids[(head + taken) % len(free_ids)] if taken < count else -1
            taken += 1
        for i in range(q):
            if t < total:
                p = ctx + i
                item[t], pos[t] = r, p
                if p // BLOCK < width and table[r, p // BLOCK] >= 0:
                    slot[t] = int(table[r, p // BLOCK]) * BLOCK + p % BLOCK
            t += 1
    used = min(taken, count)
    return starts, k_lens, q_pos, item, pos, slot, table, ((head + used) % len(free_ids), count - used)
