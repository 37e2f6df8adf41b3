"""The operators of serving from a KV pool held in 4 bits, as workloads: their cases,
their plain form in elementary torch operations, and the calls a user makes.

Three operators make up one step of a model over such a pool:

* ``tables`` -- from each request's context length and new tokens: the per-row
  metadata, the block-table entries and the per-token slots, with new blocks taken
  from a free list that is on the GPU;
* ``append`` -- RMSNorm of every query and key head and the rotary embedding of both,
  with K and V written to their slots of the pool; what a 4-bit pool holds is read
  back as the values it stands for;
* ``attention`` -- paged causal attention over the pool.

The 4-bit pool. One layer is two uint8 planes (K and V) of shape [num_blocks,
kv heads, 9 * head_dim]: a row holds one kv head of one 16-token block. Each token's
head is cut in groups of 64 values, x ~ scale * n + low with n in 0..15 and scale and
low in fp16. Bytes [0, 8 * head_dim) are the codes and bytes [8 * head_dim, 9 *
head_dim) the (scale, low) pairs. Both are cut in panels of at most 128 dims; a
panel's pairs are ordered by token, then group. ``_nibbles_k`` and ``_nibbles_v`` say
where in a row each code is; no byte holds codes of two tokens.
"""
import math
import random

import torch

own = False  # True: run() calls the framework's operators instead of the plain forms

BLOCK = 16
GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------ cases
def listed():
    return [
        # A single chat request just after a short prompt: launch latency.
        attention("attend-1-request", rows=1, k_min=75, k_max=75, hq=32, hkv=8, d=128, dtype="bf16"),
        # The decode benchmark's batch: 64 requests, contexts uniform in [1024, 8192].
        attention("attend-decode-64", rows=64, k_min=1024, k_max=8192, hq=32, hkv=8, d=128, dtype="bf16"),
        # The end-to-end configuration's batch: 256 requests with lognormal contexts, head_dim 64.
        attention("attend-decode-256-d64", rows=256, k_min=32, k_max=4352, spread="lognormal", hq=32, hkv=8, d=64,
                  dtype="fp16"),
        # Two long documents, of which each call reads all: few rows, a long axis.
        attention("attend-long-2", rows=2, k_min=120001, k_max=131072, hq=32, hkv=8, d=128, dtype="fp16"),
        # Drafted tokens being checked: 1 to 8 new tokens a request, the 64/8-head shape, and
        # two rows of a fixed-shape batch that hold no request.
        attention("attend-drafts-48", rows=48, k_min=200, k_max=6000, q_min=1, q_max=8, pad_rows=2, hq=64, hkv=8,
                  d=128, dtype="bf16"),
        # The chunked-prefill benchmark's batch: 512 new tokens behind a context of 2048, 16 requests.
        attention("attend-chunk-16x512", rows=16, k_min=2560, k_max=2560, q_min=512, q_max=512, hq=32, hkv=8, d=128,
                  dtype="bf16"),
        # A decode step's tokens, one per request.
        append("append-decode-64", tokens=64, hq=32, hkv=8, d=128, dtype="bf16", pool="4bit", norm=True),
        # A prefill step's token budget; no norms, as in a model that only rotates.
        append("append-prefill-8192", tokens=8192, hq=32, hkv=8, d=128, dtype="bf16", pool="4bit", norm=False),
        # The same pass into the 16-bit pool, an odd number of tokens, head_dim 64.
        append("append-16bit-2047-d64", tokens=2047, hq=32, hkv=8, d=64, dtype="fp16", pool="16bit", norm=True),
        # One decode step of the 256-request batch.
        tables("tables-decode-256", rows=256, q_min=1, q_max=1, ctx_max=4352, width=272),
        # A mixed step: prefill chunks of odd sizes next to single tokens.
        tables("tables-mixed-64", rows=64, q_min=1, q_max=300, ctx_max=8000, width=520),
        # A large deployment's step, many rows and many tokens.
        tables("tables-4096", rows=4096, q_min=1, q_max=12, ctx_max=16000, width=1024),
    ]


def attention(name, rows, k_min, k_max, hq, hkv, d, dtype, q_min=1, q_max=1, spread="uniform", pad_rows=0):
    """k_min..k_max: keys of a row, its own new tokens among them; pad_rows: rows more, of one token and no keys."""
    return dict(name=name, op="attention", rows=rows, k_min=k_min, k_max=k_max, q_min=q_min, q_max=q_max,
                spread=spread, pad_rows=pad_rows, hq=hq, hkv=hkv, d=d, dtype=dtype)


def append(name, tokens, hq, hkv, d, dtype, pool, norm):
    return dict(name=name, op="append", tokens=tokens, hq=hq, hkv=hkv, d=d, dtype=dtype, pool=pool, norm=norm)


def tables(name, rows, q_min, q_max, ctx_max, width):
    return dict(name=name, op="tables", rows=rows, q_min=q_min, q_max=q_max, ctx_max=ctx_max, width=width)


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "tables"])
    dtype = rng.choice(["bf16", "fp16"])
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    d = rng.choice([64, 128])
    if op == "attention":
        kind = rng.choice(["decode", "drafts", "chunk"])
        k_max = _log(rng, 17, 131072 if kind == "decode" else 8192)
        cells = 64 * 8192 * 8 * 128  # the decode batch's, padded
        fit = max(1, cells // (k_max * hkv * d))
        q_min, q_max = {"decode": (1, 1), "drafts": (1, rng.randint(2, 9)), "chunk": (1, _log(rng, 16, 640))}[kind]
        q_max = min(q_max, k_max)
        if kind == "chunk":  # at most the chunked-prefill batch's scores
            fit = min(fit, max(1, 16 * 512 * 32 * 2560 // (q_max * hkv * group * k_max)))
        rows = min(_log(rng, 1, 256), fit)
        c = attention("", rows, rng.randint(1, k_max), k_max, hkv * group, hkv, d, dtype, q_min, q_max,
                      rng.choice(["uniform", "lognormal"]), rng.choice([0, 0, 1]))
    elif op == "append":
        c = append("", min(8192, _log(rng, 1, 9000)), hkv * group, hkv, d, dtype, rng.choice(["4bit", "4bit", "16bit"]),
                   rng.random() < 0.8)
    else:
        ctx_max = _log(rng, 16, 16000)
        q_max = rng.choice([1, rng.randint(2, 12), _log(rng, 16, 500)])
        rows = min(_log(rng, 1, 4096), 50000 // q_max)
        c = tables("", rows, 1, q_max, ctx_max, (ctx_max + q_max + BLOCK - 1) // BLOCK + rng.randint(0, 9))
    del c["name"]
    return c


# --------------------------------------------------- where the pool keeps its codes
def _nibbles_k(d, device):
    """[16, d]: the position of K's code (token r, dim i) in its row, in nibbles (2 * byte + 1 for a byte's upper half)."""
    width, groups = min(d, 128), min(d, 128) // GROUP
    r = torch.arange(BLOCK, device=device)[:, None]
    i = torch.arange(d, device=device)[None, :]
    panel, grp, c = i // width, i % width // GROUP, i % GROUP
    byte = (panel * 8 * width + r * (width // 2) + c // 16 * (8 * groups) + grp * 8 + c % 16 // 8 * 4
            + c % 2 * 2 + c % 8 // 4)
    return 2 * byte + c % 4 // 2


def _nibbles_v(d, device):
    """The same for V: two tokens' codes of the same dims are neighbours, 16 bits of one and 16 of the other."""
    width, groups = min(d, 128), min(d, 128) // GROUP
    r = torch.arange(BLOCK, device=device)[:, None]
    i = torch.arange(d, device=device)[None, :]
    panel, grp, c, pair = i // width, i % width // GROUP, i % GROUP, r // 2
    turn = 2 * (pair % 4) if groups == 2 else 4 * (pair // 2 % 2)
    byte = (panel * 8 * width + pair * width + (c // 8 ^ turn) * (8 * groups) + grp * 8 + c % 8 // 4 * 4
            + r % 2 * 2 + c % 4 // 2)
    return 2 * byte + c % 2


def _layout(d, device):
    lay = {}
    for plane, where in (("k", _nibbles_k(d, device)), ("v", _nibbles_v(d, device))):
        order = where.argsort(1)  # dims in the order of their codes: neighbours share a byte
        lay[plane] = {"at": where, "low": order[:, 0::2], "high": order[:, 1::2],
                      "byte": where.gather(1, order)[:, 0::2] // 2}
    groups = min(d, 128) // GROUP
    r = torch.arange(BLOCK, device=device)[:, None, None]
    g = torch.arange(d // GROUP, device=device)[None, :, None]
    b = torch.arange(4, device=device)[None, None, :]
    lay["pairs"] = 8 * d + g // groups * (64 * groups) + r * (4 * groups) + g % groups * 4 + b  # [16, d / 64, 4] bytes
    return lay


# ------------------------------------------------------------------ the plain forms
def _quantise(x):
    """x [..., d] fp32 -> (codes uint8 [..., d], scale and low fp16 [..., d / 64])."""
    x = x.unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) * (1.0 / 15.0)).clamp(max=65504.0).half()
    low = low.clamp(-65504.0, 65504.0).half()
    inverse = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(scale, dtype=torch.float32))
    n = ((x - low.float()[..., None]) * inverse[..., None]).round().clamp(0.0, 15.0)
    return n.to(torch.uint8).flatten(-2), scale, low


def _dequantise(n, scale, low):
    return (n.float().unflatten(-1, (-1, GROUP)) * scale.float()[..., None] + low.float()[..., None]).flatten(-2)


def _pack_blocks(x, lay, plane):
    """x [blocks, 16, heads, d] -> the plane's rows, uint8 [blocks, heads, 9 * d]."""
    n, scale, low = _quantise(x.float())
    d = x.shape[-1]
    rows = torch.empty(x.shape[0], x.shape[2], 9 * d, dtype=torch.uint8, device=x.device)
    n = n.transpose(1, 2)
    l = lay[plane]
    index = lambda dims: dims.expand(*n.shape[:2], BLOCK, d // 2)  # noqa: E731
    rows[..., l["byte"].flatten()] = (n.gather(-1, index(l["low"])) | n.gather(-1, index(l["high"])) << 4).flatten(-2)
    pairs = torch.stack((scale, low), -1).transpose(1, 2).contiguous().view(torch.uint8)
    rows[..., lay["pairs"].flatten()] = pairs.flatten(-3)
    return rows


def _unpack_blocks(rows, lay, plane, d):
    """The plane's rows [..., 9 * d] -> the values they stand for, fp32 [..., 16, d]."""
    codes = rows[..., :8 * d]
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).index_select(-1, lay[plane]["at"].flatten())
    pairs = rows.index_select(-1, lay["pairs"].flatten()).view(torch.float16).unflatten(-1, (BLOCK, d // GROUP, 2))
    return _dequantise(n.unflatten(-1, (BLOCK, d)), pairs[..., 0], pairs[..., 1])


def _plain_attention(s):
    c, lay, d = s["case"], s["layout"], s["case"]["d"]
    hkv, group, total = c["hkv"], c["hq"] // c["hkv"], s["q"].shape[0]
    table = s["metadata"]["block_table"].long()
    k = _unpack_blocks(s["k_cache"][table], lay, "k", d).transpose(2, 3).flatten(1, 2)  # [rows, keys, hkv, d]
    v = _unpack_blocks(s["v_cache"][table], lay, "v", d).transpose(2, 3).flatten(1, 2)
    md = s["metadata"]
    q_lens, q_starts = md["q_lens"].long(), md["q_starts"].long()
    step = torch.arange(s["q_max"], device=k.device)
    token = (q_starts[:, None] + step).clamp(max=total - 1)
    q = s["q"][token].float().unflatten(2, (hkv, group))  # [rows, q_max, hkv, group, d]
    score = (q.permute(0, 2, 3, 1, 4).flatten(2, 3) @ k.permute(0, 2, 3, 1)).unflatten(2, (group, -1)) * s["scale"]
    j = torch.arange(k.shape[1], device=k.device)
    seen = (j < md["k_lens"].long()[:, None, None]) & (j <= md["q_pos_offsets"].long()[:, None, None] + step[:, None])
    score = torch.where(seen[:, None, None], score, torch.full_like(score[:1, :1, :1, :1, :1], -math.inf))
    top = score.amax(-1, keepdim=True)
    shift = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (score - shift).exp()
    mass = p.sum(-1, keepdim=True)
    some = mass > 0
    o = (p.flatten(2, 3) @ v.transpose(1, 2)).unflatten(2, (group, -1)) / torch.where(some, mass, torch.ones_like(mass))
    lse = torch.where(some, shift + mass.log(), torch.full_like(mass, -math.inf))[..., 0]
    row = torch.searchsorted(q_starts + q_lens, torch.arange(total, device=k.device), right=True)
    at = torch.arange(total, device=k.device) - q_starts[row]
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[row, at]
    return [o.to(s["q"].dtype), lse.permute(0, 3, 1, 2).flatten(2, 3)[row, at]]


def _norm_rotate(x, weight, eps, cos, sin):
    """x [tokens, heads, d] fp32; the sum of squares is taken over halves, then over neighbours."""
    half = x.shape[-1] // 2
    if weight is not None:
        sq = x * x
        sq = sq[..., :half] + sq[..., half:]
        while sq.shape[-1] > 1:
            sq = sq[..., 0::2] + sq[..., 1::2]
        x = x * (1.0 / (sq * (1.0 / x.shape[-1]) + eps).sqrt()) * weight.float()
    a, b = x[..., :half], x[..., half:]
    cos, sin = cos.float()[:, None], sin.float()[:, None]
    return torch.cat((a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]), -1)


def _write_slots(pool, x, slots, lay, plane):
    """x [tokens, heads, d] to the pool's slots, in its format."""
    n, scale, low = _quantise(x.float())
    heads, d = x.shape[1:]
    r, l = slots % BLOCK, lay[plane]
    row = (slots // BLOCK * heads)[:, None] + torch.arange(heads, device=x.device)  # [tokens, heads]
    index = lambda dims: dims[r][:, None].expand(-1, heads, -1)  # noqa: E731
    code = n.gather(-1, index(l["low"])) | n.gather(-1, index(l["high"])) << 4
    flat = pool.view(-1)
    flat[row[..., None] * (9 * d) + l["byte"][r][:, None]] = code
    pairs = torch.stack((scale, low), -1).view(torch.uint8).flatten(-2)
    flat[row[..., None] * (9 * d) + lay["pairs"][r].flatten(1)[:, None]] = pairs


def _read_slots(pool, slots, lay, plane, d):
    rows, r = pool[slots // BLOCK], slots % BLOCK
    at = lay[plane]["at"][r][:, None].expand(-1, rows.shape[1], -1)
    n = rows.gather(-1, at // 2) >> (at % 2 * 4).to(torch.uint8) & 15
    pairs = rows.gather(-1, lay["pairs"][r].flatten(1)[:, None].expand(-1, rows.shape[1], -1)).view(torch.float16)
    pairs = pairs.unflatten(-1, (-1, 2))
    return _dequantise(n, pairs[..., 0], pairs[..., 1])


def _plain_append(s):
    c, lay, slots = s["case"], s["layout"], s["slots"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    x = s["qkv"].float().unflatten(1, (hq + 2 * hkv, d))
    dtype = s["qkv"].dtype
    q = _norm_rotate(x[:, :hq], s["q_weight"], s["eps"], s["cos"], s["sin"]).to(dtype)
    k = _norm_rotate(x[:, hq:hq + hkv], s["k_weight"], s["eps"], s["cos"], s["sin"]).to(dtype)
    v = s["qkv"].unflatten(1, (hq + 2 * hkv, d))[:, hq + hkv:]
    if c["pool"] == "16bit":
        s["k_cache"].view(-1, hkv, d)[slots] = k
        s["v_cache"].view(-1, hkv, d)[slots] = v
        return [q, s["k_cache"], s["v_cache"]]
    _write_slots(s["k_cache"], k, slots, lay, "k")
    _write_slots(s["v_cache"], v, slots, lay, "v")
    return [q, _read_slots(s["k_cache"], slots, lay, "k", d).to(dtype),
            _read_slots(s["v_cache"], slots, lay, "v", d).to(dtype)]


def _plain_tables(s):
    q, ctx, table, free = s["q_lens"].long(), s["context_lens"].long(), s["block_table"], s["free_ids"]
    total, rows = s["total_query"], s["q_lens"].shape[0]
    head, count = s["free_state"][0].long(), s["free_state"][1].long()
    k = ctx + q
    ends = q.cumsum(0)
    starts = ends - q
    old, new = (ctx + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK
    first = (new - old).cumsum(0) - (new - old)
    col = torch.arange(table.shape[1], device=q.device)
    index = first[:, None] + col - old[:, None]
    fresh = (col >= old[:, None]) & (col < new[:, None])
    ids = torch.where(index < count, free[(head + index) % free.shape[0]], torch.full_like(free[:1], -1))
    table.copy_(torch.where(fresh, ids, table))
    t = torch.arange(total, device=q.device)
    row = torch.searchsorted(ends, t, right=True)
    real = row < rows
    at = row.clamp(max=rows - 1)
    pos = torch.where(real, ctx[at] + t - starts[at], torch.zeros_like(t))
    block = table[at, (pos // BLOCK).clamp(max=table.shape[1] - 1)].long()
    slot = torch.where(real & (block >= 0), block * BLOCK + pos % BLOCK, torch.full_like(t, -1))
    taken = torch.minimum((new - old).sum(), count)
    i32 = torch.int32
    return [starts.to(i32), k.to(i32), ctx.to(i32), torch.where(real, row, torch.full_like(row, -1)).to(i32), pos, slot,
            table, torch.stack(((head + taken) % free.shape[0], count - taken)).to(i32)]


# --------------------------------------------------------------------------- inputs
def _normal(shape, g, dtype):
    """Standard normal values; the last axis keeps some channels that are larger and off zero, as keys have."""
    x = torch.randn(shape, generator=g, device="cuda")
    d = shape[-1]
    gain = torch.ones(d, device="cuda")
    gain[5::29] = 3.0
    shift = torch.zeros(d, device="cuda")
    shift[5::29] = 2.0
    return (x * gain + shift).to(dtype)


def _pool(blocks, c, lay, g):
    """K and V planes full of quantised data: slots that no row reaches hold what an earlier request left."""
    k = torch.empty(blocks, c["hkv"], 9 * c["d"], dtype=torch.uint8, device="cuda")
    v = torch.empty_like(k)
    step = max(1, (1 << 25) // (BLOCK * c["hkv"] * c["d"]))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        shape = (n, BLOCK, c["hkv"], c["d"])
        k[i:i + n] = _pack_blocks(_normal(shape, g, DTYPES[c["dtype"]]), lay, "k")
        v[i:i + n] = _pack_blocks(torch.randn(shape, generator=g, device="cuda").to(DTYPES[c["dtype"]]), lay, "v")
    return k, v


def _new_tokens(c, rng):
    """Each row's new tokens: uniform in [q_min, q_max], with the same total for every seed."""
    lo, hi = c["q_min"], c["q_max"]
    qs = [rng.randint(lo, hi) for _ in range(c["rows"])]
    left = c["rows"] * (lo + hi) // 2 - sum(qs)
    while left:
        i = rng.randrange(len(qs))
        q = min(hi, max(lo, qs[i] + left))
        left -= q - qs[i]
        qs[i] = q
    return qs


def _lengths(c, rng):
    ks, qs = [], _new_tokens(c, rng)
    for q in qs:
        if c["spread"] == "lognormal":
            k = round(math.exp(rng.gauss(math.log(max(1.0, min(512.0, c["k_max"] / 8))), 0.83)))
        else:
            k = rng.randint(c["k_min"], c["k_max"])
        ks.append(min(c["k_max"], max(c["k_min"], k, q)))
    return ks + [0] * c["pad_rows"], qs + [1] * c["pad_rows"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    return {"attention": _prepare_attention, "append": _prepare_append, "tables": _prepare_tables}[case["op"]](case, g, rng)


def _prepare_attention(c, g, rng):
    ks, qs = _lengths(c, rng)
    lay = _layout(c["d"], "cuda")
    need = [-(-k // BLOCK) for k in ks]
    width, blocks = max(need), sum(need) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    n = torch.tensor(need, device="cuda")
    col = torch.arange(width, device="cuda")
    table = torch.where(col < n[:, None], order[((n.cumsum(0) - n)[:, None] + col).clamp(max=blocks - 1)], 0)
    i32 = dict(dtype=torch.int32, device="cuda")
    q_lens, k_lens = torch.tensor(qs, **i32), torch.tensor(ks, **i32)
    metadata = {"q_lens": q_lens, "k_lens": k_lens, "q_starts": (q_lens.cumsum(0) - q_lens).to(torch.int32),
                "q_pos_offsets": k_lens - q_lens, "block_table": table, "block_table_row_stride": width,
                "total_query": sum(qs)}
    k_cache, v_cache = _pool(blocks, c, lay, g)
    q = torch.randn(sum(qs), c["hq"], c["d"], generator=g, device="cuda").to(DTYPES[c["dtype"]])
    return {"case": c, "layout": lay, "q": q, "k_cache": k_cache, "v_cache": v_cache, "metadata": metadata,
            "scale": c["d"] ** -0.5, "q_max": max(qs)}


def _prepare_append(c, g, rng):
    n, hq, hkv, d, dtype = c["tokens"], c["hq"], c["hkv"], c["d"], DTYPES[c["dtype"]]
    blocks = n // BLOCK + 40
    # requests' new tokens are runs of neighbouring slots in blocks taken from anywhere in the pool
    order = torch.randperm(blocks, generator=g, device="cuda")
    run = torch.arange(n, device="cuda") + rng.randint(0, 15)
    slots = order[run // BLOCK] * BLOCK + run % BLOCK
    if n <= 256:  # a decode step: one token of each request, all over the pool
        slots = torch.randperm(blocks * BLOCK, generator=g, device="cuda")[:n]
    pos = torch.randint(0, 8192, (n,), generator=g, device="cuda")
    angle = pos.float()[:, None] / 10000.0 ** (torch.arange(0, d, 2, device="cuda").float() / d)
    angle = torch.cat((angle, angle), -1)
    weight = lambda: (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype) if c["norm"] else None  # noqa: E731
    s = {"case": c, "layout": _layout(d, "cuda"), "slots": slots, "eps": 1e-6,
         "qkv": _normal((n, hq + 2 * hkv, d), g, dtype).flatten(1), "cos": angle.cos().to(dtype), "sin": angle.sin().to(dtype),
         "q_weight": weight(), "k_weight": weight()}
    if c["pool"] == "16bit":
        s["k_cache"] = torch.randn(blocks, BLOCK, hkv, d, generator=g, device="cuda").to(dtype)
        s["v_cache"] = torch.randn(blocks, BLOCK, hkv, d, generator=g, device="cuda").to(dtype)
    else:
        s["k_cache"], s["v_cache"] = _pool(blocks, c, s["layout"], g)
    return s


def _prepare_tables(c, g, rng):
    qs = _new_tokens(c, rng)
    ctx = [rng.randint(0, c["ctx_max"]) for _ in range(c["rows"])]
    ctx = [min(x, c["width"] * BLOCK - q) for x, q in zip(ctx, qs)]
    held = sum(-(-x // BLOCK) for x in ctx)
    taken = sum(-(-(x + q) // BLOCK) for x, q in zip(ctx, qs)) - held
    blocks = held + taken + 64
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    n = torch.tensor([-(-x // BLOCK) for x in ctx], device="cuda")
    col = torch.arange(c["width"], device="cuda")
    table = torch.where(col < n[:, None], order[((n.cumsum(0) - n)[:, None] + col).clamp(max=blocks - 1)], 0)
    # the free list is a ring, of which a part is free: its head is anywhere
    ring, head = torch.zeros(blocks, dtype=torch.int32, device="cuda"), rng.randrange(blocks)
    free = order[held:]
    ring[(head + torch.arange(free.shape[0], device="cuda")) % blocks] = free
    i32 = dict(dtype=torch.int32, device="cuda")
    # a fixed-shape batch: its token count is rounded up, and the last places may hold none
    total = sum(qs) + -sum(qs) % 8
    s = {"case": c, "q_lens": torch.tensor(qs, **i32), "context_lens": torch.tensor(ctx, **i32), "block_table": table,
         "free_ids": ring, "free_state": torch.tensor([head, free.shape[0]], **i32), "total_query": total}
    if own:  # the step's output buffers, at fixed addresses, that a serving loop keeps
        import serving_engine_b200 as b200

        s["tables"] = b200.StepTables(c["rows"], total, "cuda")
    return s


# ------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "tables": _plain_tables}[op](state)
    import serving_engine_b200 as b200

    c = state["case"]
    if op == "attention":
        o, lse = b200.paged_flash_attention(state["q"], state["k_cache"], state["v_cache"], state["metadata"], c["hq"],
                                            c["hkv"], state["scale"])
        return [o, lse]
    if op == "append":
        q = b200.qk_norm_rope_append(state["qkv"], state["cos"], state["sin"], state["slots"], state["k_cache"],
                                     state["v_cache"], c["hq"], c["hkv"], state["q_weight"], state["k_weight"],
                                     state["eps"])
        if c["pool"] == "16bit":
            return [q, state["k_cache"], state["v_cache"]]
        k, v = b200.kv_gather_q4(state["k_cache"], state["v_cache"], state["slots"], c["d"], q.dtype)
        return [q, k, v]
    t = state["tables"]
    t.build(state["q_lens"], state["context_lens"], state["block_table"], state["free_ids"], state["free_state"])
    return [t.q_starts, t.k_lens, t.q_pos_offsets, t.item_row, t.positions, t.slot_mapping, state["block_table"],
            t.free_state]


def work(case):
    c = case
    if c["op"] == "attention":
        rng = random.Random(0)  # the mean over the seeds' lengths, by one draw of many rows
        ks, qs = _lengths(dict(c, rows=max(c["rows"], 2000), pad_rows=0), rng)
        scale = c["rows"] / len(ks)
        keys, new = sum(ks) * scale, sum(qs) * scale
        pairs = sum(q * (k - (q - 1) / 2) for k, q in zip(ks, qs)) * scale
        return {"bytes": keys * c["hkv"] * c["d"] * 2 * 9 / 16 + new * c["hq"] * (4 * c["d"] + 4),
                "flops": 4 * pairs * c["hq"] * c["d"]}
    if c["op"] == "append":
        n, hq, hkv, d = c["tokens"], c["hq"], c["hkv"], c["d"]
        # the new tokens' K and V in the pool, and the values of a 4-bit pool that are read back
        kept = 2 * hkv * d * (9 / 16 + 2 if c["pool"] == "4bit" else 2)
        # qkv, cos and sin and the slots in, q out
        return {"bytes": n * ((hq + 2 * hkv) * d * 2 + 4 * d + 8 + hq * d * 2 + kept),
                "flops": n * (hq + 2 * hkv) * d * 12}
    tokens = c["rows"] * (c["q_min"] + c["q_max"]) / 2
    fresh = tokens / BLOCK
    return {"bytes": c["rows"] * 20 + tokens * 20 + fresh * 8 + 16, "flops": c["rows"] * 8 + tokens * 6}


# --------------------------------------------------------------- the same in 64 bits
def _values64(rows, plane, d):
    """One row's blocks [n, heads, 9 * d] as float64 [n * 16, heads, d], read field by field."""
    width = min(d, 128)
    gp, out = width // GROUP, []
    for p in range(d // width):
        codes = rows[..., p * 8 * width:(p + 1) * 8 * width].long()
        pairs = rows[..., 8 * d + p * 64 * gp:8 * d + (p + 1) * 64 * gp].contiguous().view(torch.float16).double()
        lead = codes.shape[:2]
        if plane == "k":  # token, chunk of 16 dims, group, word of 8, odd or even dim, byte
            n = torch.stack((codes % 16, codes // 16), -1).view(*lead, 16, 4, gp, 2, 2, 2, 2)
            n = n.permute(0, 1, 2, 4, 3, 5, 7, 8, 6)  # token, group, chunk, word, byte, nibble, odd
        else:  # pair, chunk of 8 dims (turned by the pair), group, word of 4, token of the pair, byte
            n = torch.stack((codes % 16, codes // 16), -1).view(*lead, 8, 8, gp, 2, 2, 2, 2)
            turned = [[g ^ (2 * (pr % 4) if gp == 2 else 4 * (pr // 2 % 2)) for g in range(8)] for pr in range(8)]
            n = torch.stack([n[:, :, pr][:, :, turned[pr]] for pr in range(8)], 2)
            n = n.permute(0, 1, 2, 6, 4, 3, 5, 7, 8)  # pair, token, group, chunk, word, byte, nibble
        n = n.reshape(*lead, 16, gp, GROUP).double()
        pairs = pairs.view(*lead, 16, gp, 2)
        out.append((n * pairs[..., 0:1] + pairs[..., 1:2]).reshape(*lead, 16, width))
    return torch.cat(out, -1).transpose(1, 2).reshape(-1, rows.shape[1], d)


def _quantised64(x):
    """x [tokens, heads, d] float64 through the 4-bit format and back."""
    x = x.reshape(*x.shape[:-1], -1, GROUP)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale = ((high - low) / 15).half().double()
    low = low.half().double()
    n = torch.nan_to_num((x - low) / scale, nan=0.0, posinf=0.0, neginf=0.0).round().clamp(0, 15)
    return (n * scale + low).flatten(-2)


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    c, d = s["case"], s["case"]["d"]
    if case["op"] == "append":
        n, hq, hkv, half = c["tokens"], c["hq"], c["hkv"], d // 2
        x = s["qkv"].double().view(n, -1, d)
        turn = torch.complex(s["cos"].double()[:, None, :half], s["sin"].double()[:, None, :half])

        def turned(y, w):
            if w is not None:
                y = y / (y.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * w.double()
            z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        q, k, v = turned(x[:, :hq], s["q_weight"]), turned(x[:, hq:hq + hkv], s["k_weight"]), x[:, hq + hkv:]
        if c["pool"] == "4bit":  # the pool takes keys of the element type
            return [q, _quantised64(k.to(s["qkv"].dtype).double()), _quantised64(v)]
        pools = [s["k_cache"].double(), s["v_cache"].double()]
        for pool, new in zip(pools, (k, v)):
            pool.view(-1, *new.shape[1:])[s["slots"]] = new
        return [q, *pools]
    total, hq, group = s["q"].shape[0], c["hq"], c["hq"] // c["hkv"]
    o = torch.zeros(total, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64, device="cuda")
    md = {k: v.tolist() for k, v in s["metadata"].items() if k in ("q_lens", "k_lens", "q_starts", "q_pos_offsets")}
    for r, (nq, nk, start, pos) in enumerate(zip(md["q_lens"], md["k_lens"], md["q_starts"], md["q_pos_offsets"])):
        if nk == 0 or nq == 0:
            continue
        ids = s["metadata"]["block_table"][r, :-(-nk // BLOCK)].long()
        k = _values64(s["k_cache"][ids], "k", d)[:nk]
        v = _values64(s["v_cache"][ids], "v", d)[:nk]
        hidden = torch.arange(nk, device="cuda")[None] > pos + torch.arange(nq, device="cuda")[:, None]
        for h in range(hq):
            x = (s["q"][start:start + nq, h].double() @ k[:, h // group].T) * s["scale"]
            x = x.masked_fill(hidden, -math.inf)
            lse[start:start + nq, h] = x.logsumexp(-1)
            o[start:start + nq, h] = x.softmax(-1) @ v[:, h // group]
    return [o, lse]
