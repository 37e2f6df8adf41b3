"""The 4-bit KV pool on the GPU against the oracle (oracle/q4.py).

What the kernels store is compared byte for byte: quantisation is defined operation by
operation in fp32. Attention is compared with float64. Its bound, with u = 2^-11 the
rounding of fp16 and V the largest |v| a query sees: a probability may be held in fp16
(it weighs a code and its group's offset, each at most 2 V: u * 2 V), scores and sums in
fp32 (2^-13 V for the sizes here), and the result is rounded once to its type (half an
ulp, tests/tolerance.py). LSE is fp32: 1e-4, and 1e-5 of its size.
"""
import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from oracle import q4 as oracle
from tests.tolerance import dtype_key, half_ulp

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rope_tables(n, d, dtype, g):
    pos = torch.randint(0, 5000, (n,), generator=g, device=DEV)
    ang = pos.float()[:, None] / 10000.0 ** (torch.arange(0, d, 2, device=DEV).float() / d)
    ang = torch.cat((ang, ang), -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def junk_pool(nb, h, d, seed):
    """Planes full of random bytes, with NaN pairs among them: what no token wrote must not matter."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, 256, (2, nb, h, 9 * d), generator=g, device=DEV, dtype=torch.uint8)


# ------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 37])
@pytest.mark.parametrize("offset", [0, 1])  # 1: rows that are not 16-byte aligned
def test_kv_append_bytes(dtype, d, n, offset):
    g = torch.Generator(device=DEV).manual_seed(d + n)
    h, nb = 3, 9
    wide = torch.randn(n, 2 * h * d + 3, generator=g, device=DEV).to(dtype) * 3
    k = wide[:, offset:offset + h * d].view(n, h, d)
    v = wide[:, offset + h * d:offset + 2 * h * d].view(n, h, d)
    slots = torch.randperm(nb * 16, generator=g, device=DEV)[:n]
    pool = junk_pool(nb, h, d, 5)
    want = pool.cpu().numpy()
    b200.kv_append_q4(k, v, pool[0], pool[1], slots)
    b200.check_device_errors()
    oracle.write_kv(want[0], want[1], k.float().cpu().numpy(), v.float().cpu().numpy(), slots.tolist())
    assert np.array_equal(pool.cpu().numpy(), want)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        rk, rv = b200.kv_gather_q4(pool[0], pool[1], slots, d, out)
        for got, plane, kind in ((rk, want[0], "k"), (rv, want[1], "v")):
            val = oracle.read(plane, kind, d).reshape(-1, h, d)[slots.tolist()]
            ref = torch.from_numpy(val.astype(np.float32)).to(out)
            # fp32 rounds the product and the sum (2^-23 of each), then the type
            tol = 2.0 ** -22 * np.abs(val).max() + {4: 0, 2: np.abs(val) * (2.0 ** -8 if out is torch.bfloat16 else 2.0 ** -11)}[ref.element_size()]
            assert (np.abs(got.double().cpu().numpy() - val) <= tol).all()


def test_kv_append_error_of_a_value():
    """A value is off by at most half a step, and its group's ends by the rounding of the two parameters."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(64, 2, 128, generator=g, device=DEV).half()
    pool = b200.new_q4_pool(1, 4, 2, 128)[0]
    slots = torch.arange(64, device=DEV)
    b200.kv_append_q4(x, x, pool[0], pool[1], slots)
    k, v = b200.kv_gather_q4(pool[0], pool[1], slots, 128, torch.float32)
    assert torch.equal(k, v)
    grp = x.float().view(64, 2, 2, 64)
    step = (grp.amax(-1) - grp.amin(-1)) / 15
    # codes are taken against the rounded parameters: half a step, and where the rounded range
    # ends inside the group's, what the clamp cuts off: 15 steps * 2^-11 and 2^-11 of the low end
    bound = step * (0.5 + 15 * 2.0 ** -11) + grp.amin(-1).abs() * 2.0 ** -11 + 1e-6
    assert ((k.view_as(grp) - grp).abs() <= bound[..., None]).all()


@pytest.mark.parametrize("kind", ["equal", "tiny", "huge", "inf", "nan", "zero"])
def test_kv_append_special_values(kind):
    d, dtype = 128, torch.bfloat16
    x = torch.randn(4, 1, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    if kind == "equal":
        x[1] = 2.5
    elif kind == "tiny":
        x[1] *= 1e-9
    elif kind == "huge":
        x[1] *= 1e37
    elif kind == "inf":
        x[1, 0, 70] = float("inf")
    elif kind == "nan":
        x[1, 0, 3] = float("nan")
    else:
        x[1] = 0
    pool = junk_pool(1, 1, d, 2)
    want = pool.cpu().numpy()
    slots = torch.tensor([3, 4, 9, 0], device=DEV)
    b200.kv_append_q4(x, x, pool[0], pool[1], slots)
    oracle.write_kv(want[0], want[1], x.float().cpu().numpy(), x.float().cpu().numpy(), slots.tolist())
    assert np.array_equal(pool.cpu().numpy(), want)
    k, _ = b200.kv_gather_q4(pool[0], pool[1], slots, d, torch.float32)
    if kind in ("inf", "nan"):
        nan = torch.isnan(k[1, 0]).view(2, 64)
        assert nan[1 if kind == "inf" else 0].all() and not nan[0 if kind == "inf" else 1].any()
    else:
        assert torch.isfinite(k).all()
    if kind in ("equal", "zero"):
        assert torch.equal(k[1, 0], x[1, 0].float())


def test_slots_out_of_range():
    d, h = 64, 2
    x = torch.randn(4, h, d, device=DEV).bfloat16()
    pool = junk_pool(2, h, d, 9)
    before = pool.clone()
    slots = torch.tensor([-1, 32, 2 ** 40, 5], device=DEV)
    b200.kv_append_q4(x, x, pool[0], pool[1], slots)
    with pytest.raises(RuntimeError, match="slot out of range"):
        b200.check_device_errors()
    assert torch.equal(pool[:, 1], before[:, 1]) and not torch.equal(pool[:, 0], before[:, 0])
    k, v = b200.kv_gather_q4(pool[0], pool[1], slots, d)
    with pytest.raises(RuntimeError, match="slot out of range"):
        b200.check_device_errors()
    assert (k[:3] == 0).all() and (v[:3] == 0).all() and (k[3] != 0).any()
    qkv = torch.randn(4, 4 * h * d // 2 * 2, device=DEV).bfloat16()[:, :3 * h * d]
    cos, sin = rope_tables(4, d, torch.bfloat16, torch.Generator(device=DEV).manual_seed(0))
    before = pool.clone()
    b200.qk_norm_rope_append(qkv, cos, sin, slots, pool[0], pool[1], h, h)
    with pytest.raises(RuntimeError, match="slot out of range"):
        b200.check_device_errors()
    assert torch.equal(pool[:, 1], before[:, 1])


# -------------------------------------------------- norms, rotation and the append
def norm_rope32(x, w, eps, cos, sin):
    """The definition in fp32 on the CPU, operation by operation."""
    half = x.shape[-1] // 2
    x = x.float()
    if w is not None:
        sq = x * x
        sq = sq[..., :half] + sq[..., half:]
        while sq.shape[-1] > 1:
            sq = sq[..., 0::2] + sq[..., 1::2]
        root = (sq * (1.0 / x.shape[-1]) + eps).double().sqrt().float()  # correctly rounded; fp32 sqrt on the CPU is not
        x = x * (torch.ones(()) / root) * w.float()
    a, b = x[..., :half], x[..., half:]
    cos, sin = cos.float()[:, None], sin.float()[:, None]
    return torch.cat((a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]), -1)


def norm_rope64(x, w, eps, cos, sin):
    x = x.double()
    if w is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    half = x.shape[-1] // 2
    rot = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos.double()[:, None] + rot * sin.double()[:, None]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (8, 2, 128), (7, 1, 128), (3, 3, 256)])
@pytest.mark.parametrize("norms", ["both", "none", "q"])
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("offset", [0, 1])
def test_qk_norm_rope_append(dtype, hq, hkv, d, norms, bits, offset):
    g = torch.Generator(device=DEV).manual_seed(hq * d + bits)
    n, nb = 19, 5
    w = (hq + 2 * hkv) * d
    qkv = (torch.randn(n, w + 5, generator=g, device=DEV) * 2 + 0.3).to(dtype)[:, offset:offset + w]
    if offset == 0:
        qkv = qkv.contiguous()
    cos, sin = rope_tables(n, d, dtype, g)
    weight = lambda: (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype)  # noqa: E731
    qw = weight() if norms in ("both", "q") else None
    kw = weight() if norms == "both" else None
    slots = torch.randperm(nb * 16, generator=g, device=DEV)[:n]
    if bits == 4:
        pool = junk_pool(nb, hkv, d, 7)
    else:
        pool = torch.randn(2, nb, 16, hkv, d, generator=g, device=DEV).to(dtype)
    want = pool.cpu().clone()
    q = b200.qk_norm_rope_append(qkv, cos, sin, slots, pool[0], pool[1], hq, hkv, qw, kw, 1e-6)
    b200.check_device_errors()
    c = lambda t: None if t is None else t.cpu()  # noqa: E731
    x = qkv.cpu().reshape(n, hq + 2 * hkv, d)
    args = (1e-6, cos.cpu(), sin.cpu())
    q_ref, k_ref = norm_rope32(x[:, :hq], c(qw), *args).to(dtype), norm_rope32(x[:, hq:hq + hkv], c(kw), *args).to(dtype)
    assert torch.equal(q.cpu(), q_ref)
    if bits == 4:
        oracle.write_kv(want[0].numpy(), want[1].numpy(), k_ref.float().numpy(), x[:, hq + hkv:].float().numpy(),
                        slots.tolist())
    else:
        want[0].view(-1, hkv, d)[slots.cpu()] = k_ref
        want[1].view(-1, hkv, d)[slots.cpu()] = x[:, hq + hkv:]
    assert torch.equal(pool.cpu(), want)
    # and against 64 bits: fp32 arithmetic (under 2^-20 of the largest value of a head), one rounding to the type
    q64 = norm_rope64(x[:, :hq], c(qw), *args)
    tol = torch.from_numpy(half_ulp(q64.numpy(), dtype_key(dtype))) + q64.abs().amax(-1, keepdim=True) * 2.0 ** -20 + 1e-7
    assert ((q.double().cpu() - q64).abs() <= tol).all()


def test_qk_norm_rope_append_without_tokens():
    pool = b200.new_q4_pool(1, 1, 1, 64)[0]
    e = torch.empty(0, 64 * 3, device=DEV, dtype=torch.float16)
    cs = torch.empty(0, 64, device=DEV, dtype=torch.float16)
    q = b200.qk_norm_rope_append(e, cs, cs, torch.empty(0, dtype=torch.int64, device=DEV), pool[0], pool[1], 1, 1)
    assert q.shape == (0, 1, 64)


# ---------------------------------------------------------------------- attention
def make_batch(k_lens, q_lens, hq, hkv, d, dtype, seed=0, gain=1.0, spare=2):
    """Rows over a shuffled pool whose unreached slots are junk, NaN pairs among it."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-k // 16) for k in k_lens]
    nb, width = sum(need) + spare, max(max(need), 1)
    perm = torch.randperm(nb, generator=g, device=DEV).tolist()
    table, slots, at = np.zeros((len(k_lens), width), np.int32), [], 0
    for r, k in enumerate(k_lens):
        ids = perm[at:at + need[r]]
        at += need[r]
        table[r, :need[r]] = ids
        slots += [ids[j // 16] * 16 + j % 16 for j in range(k)]
    pool = junk_pool(nb, hkv, d, seed + 1)
    pool[..., 8 * d:] = 0xFF  # every pair a NaN until a token writes it
    n = len(slots)
    k = torch.randn(n, hkv, d, generator=g, device=DEV) * gain
    k[..., 5::29] += 2.0
    v = torch.randn(n, hkv, d, generator=g, device=DEV)
    if n:
        b200.kv_append_q4(k.to(dtype), v.to(dtype), pool[0], pool[1], torch.tensor(slots, device=DEV))
    q = torch.randn(sum(q_lens), hq, d, generator=g, device=DEV).to(dtype)
    starts = np.concatenate(([0], np.cumsum(q_lens)[:-1]))
    return dict(q=q, pool=pool, table=table, q_lens=list(q_lens), k_lens=list(k_lens), starts=starts.tolist(),
                pos=[k - n for k, n in zip(k_lens, q_lens)], hq=hq, hkv=hkv, scale=d ** -0.5)


def metadata(b):
    i32 = dict(dtype=torch.int32, device=DEV)
    return {"q_lens": torch.tensor(b["q_lens"], **i32), "k_lens": torch.tensor(b["k_lens"], **i32),
            "q_starts": torch.tensor(b["starts"], **i32), "q_pos_offsets": torch.tensor(b["pos"], **i32),
            "block_table": torch.tensor(b["table"], **i32), "block_table_row_stride": b["table"].shape[1],
            "total_query": b["q"].shape[0]}


def check(b, o, lse, causal=True, tokens=None):
    p = b["pool"].cpu().numpy()
    ro, rl, top = oracle.attention(b["q"].double().cpu().numpy(), p[0], p[1], b["table"], b["starts"], b["q_lens"],
                                   b["k_lens"], b["pos"], b["scale"], causal)
    tokens = slice(None) if tokens is None else tokens
    o, lse, ro, rl, top = (x[tokens] for x in (o.double().cpu().numpy(), lse.double().cpu().numpy(), ro, rl, top))
    tol = (2 * 2.0 ** -11 + 2.0 ** -13) * top[..., None] + half_ulp(ro, dtype_key(b["q"].dtype)) + 1e-6
    assert np.isfinite(o).all()
    assert (np.abs(o - ro) <= tol).all(), float((np.abs(o - ro) - tol).max())
    dead = np.isinf(rl)
    assert np.array_equal(np.isneginf(lse), dead)
    assert (np.abs(lse[~dead] - rl[~dead]) <= 1e-4 + 1e-5 * np.abs(rl[~dead])).all()
    assert (o[dead] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (3, 1), (28, 4), (8, 1), (12, 1), (16, 1)])
def test_decode_rows(dtype, d, hq, hkv):
    b = make_batch([1, 16, 17, 130, 0, 700], [1] * 6, hq, hkv, d, dtype, seed=d + hq)
    b["pos"][4] = -1
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), hq, hkv, b["scale"])
    b200.check_device_errors()
    check(b, o, lse)


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 6, 6), (128, 7, 1), (256, 4, 1), (64, 16, 1)])
@pytest.mark.parametrize("q_lens,k_lens", [
    ([3, 1, 8, 5], [40, 1, 8, 333]),          # drafted tokens; a row that is all new
    ([0, 2, 0, 1, 0], [50, 17, 0, 9, 16]),    # rows without tokens
    ([70, 1, 33], [70, 400, 200]),            # chunks next to a decode row
])
def test_rows_of_several_tokens(d, hq, hkv, q_lens, k_lens):
    b = make_batch(k_lens, q_lens, hq, hkv, d, torch.bfloat16, seed=d)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), hq, hkv, b["scale"])
    b200.check_device_errors()
    check(b, o, lse)


@pytest.mark.parametrize("q_lens,k_lens", [([1, 1], [30, 2]), ([9, 40], [25, 40])])
def test_not_causal(q_lens, k_lens):
    b = make_batch(k_lens, q_lens, 4, 2, 128, torch.float16, seed=2)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 4, 2, b["scale"], is_causal=False)
    check(b, o, lse, causal=False)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,k_len", [(1, 9000), (3, 4099)])
def test_long_context(d, rows, k_len):
    """Few rows, a long axis: the keys are split over the GPU and joined."""
    b = make_batch([k_len - 7 * i for i in range(rows)], [1] * rows, 8, 2, d, torch.bfloat16, seed=1)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 8, 2, b["scale"])
    check(b, o, lse)
    again = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 8, 2, b["scale"])
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])  # joined in a fixed order


def test_many_short_rows():
    rng = np.random.default_rng(0)
    ks = rng.integers(1, 90, 700).tolist()
    b = make_batch(ks, [1] * 700, 4, 1, 64, torch.float16, seed=4)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 4, 1, b["scale"])
    check(b, o, lse)


@pytest.mark.parametrize("gain", [30.0, 1e-3])
def test_peaked_and_flat_scores(gain):
    """Scores of hundreds (one key takes all) and of nearly nothing; V of very different sizes in a row."""
    b = make_batch([500, 61, 1000], [1, 4, 1], 4, 1, 128, torch.float16, seed=3, gain=gain)
    k, v = (x for x in b200.kv_gather_q4(b["pool"][0], b["pool"][1], torch.arange(b["pool"].shape[1] * 16, device=DEV), 128, torch.float32))
    size = torch.logspace(-4, 3, v.shape[0], device=DEV)[torch.randperm(v.shape[0], device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))]
    held = torch.isfinite(v).all(-1).all(-1)
    slots = torch.nonzero(held)[:, 0]
    b200.kv_append_q4(k[held].half(), (v * size[:, None, None])[held].half(), b["pool"][0], b["pool"][1], slots)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 4, 1, b["scale"])
    check(b, o, lse)


@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_queries_beyond_fp16(size):
    """bf16 queries that fp16 cannot hold: the largest key takes all, or all keys weigh the same."""
    b = make_batch([77], [2], 2, 1, 64, torch.bfloat16, seed=6)
    b["q"] = (b["q"].float() * size).bfloat16()
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 2, 1, b["scale"])
    p = b["pool"].cpu().numpy()
    ro, rl, top = oracle.attention(b["q"].double().cpu().numpy(), p[0], p[1], b["table"], b["starts"], b["q_lens"],
                                   b["k_lens"], b["pos"], b["scale"])
    tol = (2 * 2.0 ** -11 + 2.0 ** -13) * top[..., None] + half_ulp(ro, "bf16")
    assert (np.abs(o.double().cpu().numpy() - ro) <= tol).all()
    assert (np.abs(lse.double().cpu().numpy() - rl) <= 1e-4 + 1e-5 * np.abs(rl)).all()


def test_strided_inputs_and_given_outputs():
    b = make_batch([40, 90], [1, 3], 4, 2, 128, torch.bfloat16, seed=8)
    wide = torch.randn(4, 4 * 2, 130, device=DEV).bfloat16()
    wide[:, ::2, :128] = b["q"]
    q = wide[:, ::2, :128]
    out = torch.full((6, 4, 200), 7.0, device=DEV, dtype=torch.bfloat16)
    lse = torch.full((6, 9), 7.0, device=DEV)
    md = metadata(b)
    table = torch.zeros(2, 40, dtype=torch.int32, device=DEV)
    table[:, 3:3 + b["table"].shape[1]] = md["block_table"]
    ops_args = (b["pool"][0], b["pool"][1], table[:, 3:3 + b["table"].shape[1]], md["q_starts"], md["q_lens"],
                md["k_lens"], md["q_pos_offsets"], 4, 2, b["scale"])
    o, l = b200.paged_attention_q4(q, *ops_args, out=out[1:5, :, 8:136], lse=lse[1:5, 2:6])
    check(b, o, l)
    assert (out[0] == 7).all() and (out[5] == 7).all() and (out[:, :, :8] == 7).all() and (out[:, :, 136:] == 7).all()
    assert (lse[0] == 7).all() and (lse[:, :2] == 7).all() and (lse[:, 6:] == 7).all()


def test_rows_in_any_order_and_tokens_of_no_row():
    """Row token ranges out of order, with a gap that no row covers."""
    b = make_batch([40, 90, 33], [2, 3, 1], 4, 2, 64, torch.float16, seed=9)
    b["q"] = torch.randn(9, 4, 64, device=DEV).half()
    b["starts"] = [6, 0, 4]
    out = torch.full((9, 4, 64), 5.0, device=DEV, dtype=torch.float16)
    md = metadata(b)
    o, lse = b200.paged_attention_q4(b["q"], b["pool"][0], b["pool"][1], md["block_table"], md["q_starts"], md["q_lens"],
                                     md["k_lens"], md["q_pos_offsets"], 4, 2, b["scale"], out=out)
    b200.check_device_errors()
    check(b, o, lse, tokens=[0, 1, 2, 4, 6, 7])
    assert (out[[3, 5, 8]] == 5).all()


def test_bad_indices_are_reported_and_masked():
    b = make_batch([64, 40], [1, 1], 2, 1, 64, torch.float16, seed=10)
    b["table"][0, 1], b["table"][0, 3] = -3, 10 ** 6
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 2, 1, b["scale"])
    with pytest.raises(RuntimeError, match="block id out of range"):
        b200.check_device_errors()
    check(b, o, lse)
    b = make_batch([64, 40], [1, 1], 2, 1, 64, torch.float16, seed=10)
    md = metadata(b)
    md["k_lens"][1] = 1000  # beyond the table: ends there
    md["q_pos_offsets"][1] = 999
    b["k_lens"][1], b["pos"][1] = 64, 63
    b["table"][1, 3] = 0
    b["pool"][..., 8 * 64:] = torch.where(b["pool"][..., 8 * 64:] == 0xFF, 0, b["pool"][..., 8 * 64:])
    md["block_table"] = torch.tensor(b["table"], device=DEV)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], md, 2, 1, b["scale"])
    with pytest.raises(RuntimeError, match="k_len exceeds"):
        b200.check_device_errors()
    check(b, o, lse)
    md = metadata(b)
    md["q_starts"][0] = 5  # outside q: skipped, the other row unharmed
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], md, 2, 1, b["scale"])
    with pytest.raises(RuntimeError, match="index out of range"):
        b200.check_device_errors()
    check(b, o, lse, tokens=[1])


def test_nan_of_one_row_stays_in_it():
    b = make_batch([64, 40], [1, 1], 2, 1, 128, torch.bfloat16, seed=11)
    slot = int(b["table"][0, 1]) * 16 + 3
    x = torch.full((1, 1, 128), float("nan"), device=DEV).bfloat16()
    b200.kv_append_q4(x, x, b["pool"][0], b["pool"][1], torch.tensor([slot], device=DEV))
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 2, 1, b["scale"])
    assert torch.isnan(o[0]).all()
    check(b, o, lse, tokens=[1])


def test_another_stream_and_a_graph():
    b = make_batch([300, 40, 2000], [1, 2, 1], 8, 2, 128, torch.bfloat16, seed=12)
    md = metadata(b)
    args = (b["q"], b["pool"][0], b["pool"][1], md, 8, 2, b["scale"])
    ref = b200.paged_flash_attention(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = b200.paged_flash_attention(*args)
    s.synchronize()
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = b200.paged_flash_attention(*args)
    for _ in range(3):
        held[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ref[0], held[0]) and torch.equal(ref[1], held[1])


def test_pool_beyond_2_gib():
    """Block ids whose byte offsets pass 2^31 and 2^32 in a plane."""
    h, d = 8, 128
    nb = (1 << 32) // (h * 9 * d) + 64
    pool = torch.empty(2, nb, h, 9 * d, dtype=torch.uint8, device=DEV)
    ids = [nb - 1, 3, (1 << 31) // (h * 9 * d) + 1, nb - 9]
    k_len = 60
    slots = torch.tensor([ids[j // 16] * 16 + j % 16 for j in range(k_len)], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(k_len, h, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    b200.kv_append_q4(k, v, pool[0], pool[1], slots)
    small = torch.zeros(2, 4, h, 9 * d, dtype=torch.uint8, device=DEV)
    b200.kv_append_q4(k, v, small[0], small[1], torch.arange(k_len, device=DEV))
    assert torch.equal(pool[:, ids[:3]], small[:, :3])
    q = torch.randn(1, 32, d, generator=g, device=DEV).bfloat16()
    i32 = dict(dtype=torch.int32, device=DEV)
    rest = (torch.tensor([0], **i32), torch.tensor([1], **i32), torch.tensor([k_len], **i32), torch.tensor([k_len - 1], **i32),
            32, 8, d ** -0.5)
    o, lse = b200.paged_attention_q4(q, pool[0], pool[1], torch.tensor([ids], **i32), *rest)
    o2, lse2 = b200.paged_attention_q4(q, small[0], small[1], torch.tensor([[0, 1, 2, 3]], **i32), *rest)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    b200.check_device_errors()


# ----------------------------------------------------------------------- refusals
def test_refusals():
    pool = b200.new_q4_pool(1, 2, 2, 64)[0]
    x = torch.randn(3, 2, 64, device=DEV).half()
    s = torch.arange(3, device=DEV)
    for args, match in (
            ((x.float(), x.float(), pool[0], pool[1], s), "bf16 or fp16"),
            ((x, x[:2], pool[0], pool[1], s), "must both be"),
            ((x, x, pool[0].int(), pool[1], s), "uint8"),
            ((x, x, pool[0, :, :1], pool[1, :, :1], s), "k_cache must be"),
            ((x[..., ::2].contiguous(), x[..., ::2].contiguous(), pool[0], pool[1], s), "head_dim 32 not supported"),
            ((x, x, pool[0], pool[1], s.int()), "int64"),
            ((x, x, pool[0].cpu(), pool[1], s), "must be on"),
            ((x.transpose(1, 2).contiguous().transpose(1, 2), x, pool[0], pool[1], s), "unit stride")):
        with pytest.raises(ValueError, match=match):
            b200.kv_append_q4(*args)
    with pytest.raises(ValueError, match="unsupported dtype"):
        b200.kv_gather_q4(pool[0], pool[1], s, 64, torch.float64)
    with pytest.raises(ValueError, match="not supported"):
        b200.new_q4_pool(1, 1, 1, 96)
    cos = torch.randn(3, 64, device=DEV).half()
    qkv = torch.randn(3, 64 * 6, device=DEV).half()
    good = dict(qkv=qkv, cos=cos, sin=cos, slot_mapping=s, k_cache=pool[0], v_cache=pool[1], num_q_heads=2, num_kv_heads=2)
    b200.qk_norm_rope_append(**good)
    for change, match in (
            (dict(qkv=qkv[:, :320]), "width"), (dict(cos=cos[:2]), "cos and sin"), (dict(sin=cos.float()), "one dtype"),
            (dict(k_cache=pool[0].half()), "k_cache must be"), (dict(q_weight=cos), "q_weight"),
            (dict(k_weight=torch.ones(32, device=DEV).half()), "k_weight"), (dict(slot_mapping=s[:2]), "slot_mapping"),
            (dict(out=torch.empty(3, 2, 64, device=DEV)), "out must be"), (dict(num_q_heads=3), "width")):
        with pytest.raises(ValueError, match=match):
            b200.qk_norm_rope_append(**{**good, **change})
    b = make_batch([20], [1], 4, 2, 64, torch.half)
    md = metadata(b)
    good = dict(q=b["q"], k_cache=b["pool"][0], v_cache=b["pool"][1], block_table=md["block_table"],
                q_starts=md["q_starts"], q_lens=md["q_lens"], k_lens=md["k_lens"], q_pos_offsets=md["q_pos_offsets"],
                num_q_heads=4, num_kv_heads=2, scale=0.1)
    b200.paged_attention_q4(**good)
    for change, match in (
            (dict(q=b["q"].float()), "bf16 or fp16"), (dict(num_q_heads=5), "q must be"), (dict(num_kv_heads=3), "multiple"),
            (dict(k_lens=md["k_lens"].long()), "int32"), (dict(block_table=md["block_table"][:0]), "block_table"),
            (dict(q_lens=torch.cat([md["q_lens"]] * 2)), "q_lens"), (dict(out=b["q"][:0]), "out must"),
            (dict(lse=torch.empty(1, 4, device=DEV).half()), "lse must"), (dict(k_cache=b["pool"][0].half()), "uint8")):
        with pytest.raises(ValueError, match=match):
            b200.paged_attention_q4(**{**good, **change})
    big = make_batch([20], [1], 17, 1, 64, torch.half)
    with pytest.raises(ValueError, match="group 17"):
        b200.paged_flash_attention(big["q"], big["pool"][0], big["pool"][1], metadata(big), 17, 1, 1.0)


def test_empty_batches():
    pool = b200.new_q4_pool(1, 2, 1, 64)[0]
    i32 = dict(dtype=torch.int32, device=DEV)
    none = torch.empty(0, **i32)
    q = torch.empty(0, 2, 64, device=DEV).half()
    o, lse = b200.paged_attention_q4(q, pool[0], pool[1], torch.empty(0, 4, **i32), none, none, none, none, 2, 1, 1.0)
    assert o.shape == (0, 2, 64) and lse.shape == (0, 2)
    q = torch.randn(1, 2, 64, device=DEV).half()
    z = torch.zeros(1, **i32)
    o, lse = b200.paged_attention_q4(q, pool[0], pool[1], torch.empty(1, 0, **i32), z, z + 1, z, z - 1, 2, 1, 1.0)
    assert (o == 0).all() and torch.isneginf(lse).all()


# ------------------------------------------------------------------- prompt chunks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 8, 2), (128, 7, 1), (64, 3, 3), (128, 16, 1)])
@pytest.mark.parametrize("q_lens,k_lens", [
    ([128], [128]), ([129, 200], [129, 1000]), ([65, 1, 0, 300, 4], [65, 700, 0, 317, 90]), ([257], [600])])
def test_chunks(dtype, d, hq, hkv, q_lens, k_lens):
    """Rows long enough for the tcgen05 kernel, beside rows that are not; tiles that end inside a block."""
    b = make_batch(k_lens, q_lens, hq, hkv, d, dtype, seed=d + hq)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), hq, hkv, b["scale"])
    b200.check_device_errors()
    check(b, o, lse)


@pytest.mark.parametrize("causal", [True, False])
def test_chunks_with_odd_positions(causal):
    """A chunk whose position is not k_len - q_len: tokens that see nothing, and tokens that see all keys."""
    b = make_batch([150, 40], [140, 60], 4, 2, 128, torch.float16, seed=21)
    b["pos"] = [-30, 20]
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 4, 2, b["scale"], is_causal=causal)
    b200.check_device_errors()
    check(b, o, lse, causal=causal)


def test_chunks_negative_scale_and_bad_blocks():
    b = make_batch([400, 300], [100, 90], 4, 1, 64, torch.bfloat16, seed=22)
    b["scale"] = -0.2
    b["table"][0, 3], b["table"][1, 9] = -1, 10 ** 6
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 4, 1, b["scale"])
    with pytest.raises(RuntimeError, match="block id out of range"):
        b200.check_device_errors()
    check(b, o, lse)


def test_chunk_nan_token_is_not_seen_before_it():
    """A token whose K and V are NaN: the chunk's earlier tokens do not see it, its later ones do."""
    b = make_batch([200], [150], 4, 2, 128, torch.bfloat16, seed=23)
    at = 120  # key of the chunk's token 70
    slot = int(b["table"][0, at // 16]) * 16 + at % 16
    x = torch.full((1, 2, 128), float("nan"), device=DEV).bfloat16()
    b200.kv_append_q4(x, x, b["pool"][0], b["pool"][1], torch.tensor([slot], device=DEV))
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 4, 2, b["scale"])
    assert torch.isnan(o[70:]).all()
    check(b, o, lse, tokens=list(range(70)))


@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_chunk_queries_beyond_fp16(size):
    b = make_batch([150], [100], 2, 1, 64, torch.bfloat16, seed=24)
    b["q"] = (b["q"].float() * size).bfloat16()
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 2, 1, b["scale"])
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    if size < 1:  # all scores are next to nothing: the mean of the values seen
        check(b, o, lse)


def test_chunk_values_beyond_fp16():
    """Values between 65504 and what a group's codes can reach are clamped to 65504 for a chunk."""
    n, d = 160, 128
    b = make_batch([n], [n], 1, 1, d, torch.bfloat16, seed=25)
    g = torch.Generator(device=DEV).manual_seed(1)
    v = torch.randn(n, 1, d, generator=g, device=DEV)
    v[:, 0, 3] = 90000.0
    v[:, 0, 70] = -60000.0
    slots = torch.tensor([int(b["table"][0, j // 16]) * 16 + j % 16 for j in range(n)], device=DEV)
    k, _ = b200.kv_gather_q4(b["pool"][0], b["pool"][1], slots, d, torch.float32)
    b200.kv_append_q4(k.bfloat16(), v.bfloat16(), b["pool"][0], b["pool"][1], slots)
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 1, 1, b["scale"])
    assert torch.isfinite(o).all()
    assert ((o[:, 0, 3].float() - 65504).abs() <= 65504 * 2.0 ** -8).all()
    assert ((o[:, 0, 70].float() + 60000).abs() <= 60000 * 2.0 ** -7).all()
