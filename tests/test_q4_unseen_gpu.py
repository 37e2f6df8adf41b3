"""Attention over a 4-bit pool: keys that a query does not see, or that weigh nothing, count for nothing."""
import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from oracle import q4 as oracle
from tests.test_q4_gpu import DEV, make_batch, metadata
from tests.tolerance import dtype_key, half_ulp

pytestmark = pytest.mark.gpu


def run(b, causal=True):
    return b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), b["hq"], b["hkv"], b["scale"],
                                      is_causal=causal)


def slots_of(b, r):
    return [int(b["table"][r, j // 16]) * 16 + j % 16 for j in range(b["k_lens"][r])]


def rewrite_v(b, size):
    """V of normal values, of the given size for each key of each row."""
    g = torch.Generator(device=DEV).manual_seed(5)
    d = b["q"].shape[-1]
    for r in range(len(b["k_lens"])):
        if not b["k_lens"][r]:
            continue
        slots = torch.tensor(slots_of(b, r), device=DEV)
        k, _ = b200.kv_gather_q4(b["pool"][0], b["pool"][1], slots, d, torch.float32)
        v = torch.randn(k.shape, generator=g, device=DEV) * torch.as_tensor(size(r), device=DEV)[:, None, None].float()
        b200.kv_append_q4(k.half(), v.half(), b["pool"][0], b["pool"][1], slots)


def weighted_bound(b, ro, causal=True):
    """What roundings may cost O: p * scale (or p) to 2^-11 of itself, weighing a code (up to 15 scale) and its
    group's offset, so 2 * 2^-11 of the sum of p |v|, |v| the largest of a key's group; 2^-13 of it for scores
    and sums in fp32; what p * scale loses to fp16's subnormals, 2^-20 of the largest p |v| (of any group) for
    each key; half an ulp."""
    p = b["pool"].cpu().numpy()
    d = b["q"].shape[-1]
    q = b["q"].double().cpu().numpy()
    hkv, hq = b["hkv"], b["hq"]
    bound = np.zeros(ro.shape)
    for r in range(len(b["q_lens"])):
        n = b["k_lens"][r]
        if n == 0:
            continue
        ids = b["table"][r][:-(-n // 16)]
        ok = np.repeat((ids >= 0) & (ids < p.shape[1]), 16)[:n]
        safe = np.where((ids >= 0) & (ids < p.shape[1]), ids, 0)
        k = oracle.read(p[0][safe], "k", d).reshape(-1, hkv, d)[:n]
        v = oracle.read(p[1][safe], "v", d).reshape(-1, hkv, d)[:n]
        for i in range(b["q_lens"][r]):
            seen = ok & (np.arange(n) <= b["pos"][r] + i if causal else True)
            if not seen.any():
                continue
            for h in range(hq):
                s = k[seen, h // (hq // hkv)] @ q[b["starts"][r] + i, h] * b["scale"]
                w = np.exp(s - s.max())
                a = np.abs(v[seen, h // (hq // hkv)]).reshape(-1, d // 64, 64).max(-1)  # [keys, groups]
                wa = w[:, None] * a
                of_groups = (2 * 2.0 ** -11 + 2.0 ** -13) * wa.sum(0) + 2.0 ** -20 * wa.max() * len(wa)
                bound[b["starts"][r] + i, h] = np.repeat(of_groups, 64) / w.sum()
    return bound + half_ulp(ro, dtype_key(b["q"].dtype)) + 1e-12


def check(b, o, causal=True, tokens=slice(None)):
    p = b["pool"].cpu().numpy()
    ro, rl, _ = oracle.attention(b["q"].double().cpu().numpy(), p[0], p[1], b["table"], b["starts"], b["q_lens"],
                                 b["k_lens"], b["pos"], b["scale"], causal)
    tol = weighted_bound(b, ro, causal)
    err = np.abs(o.double().cpu().numpy() - ro)
    assert (err <= tol)[tokens].all(), float((err / tol)[tokens].max())


def unseen_pairs(b):
    """[blocks, 16] of the slots that no row holds."""
    mask = torch.ones(b["pool"].shape[1] * 16, dtype=torch.bool, device=DEV)
    for r in range(len(b["k_lens"])):
        if b["k_lens"][r]:
            mask[torch.tensor(slots_of(b, r), device=DEV)] = False
    return mask.view(-1, 16)


def fill_unseen(b, bits):
    """Every (scale, low) pair of slots that no row holds becomes these 16-bit patterns; None: random ones."""
    d = b["q"].shape[-1]
    mask = unseen_pairs(b).cpu()
    pool = b["pool"].clone()
    pairs = pool[..., 8 * d:].contiguous().cpu().view(torch.int16)  # [2, blocks, h, d / 2]
    at = np.array([[oracle.pair_byte(d, r, g) - 8 * d for g in range(d // 64)] for r in range(16)]) // 2
    g = torch.Generator().manual_seed(7)
    for r in range(16):
        for where in (at[r], at[r] + 1):
            new = (torch.randint(-32768, 32768, pairs[..., where].shape, generator=g) if bits is None else
                   torch.full(pairs[..., where].shape, bits[where is not at[r]])).to(torch.int16)
            pairs[..., where] = torch.where(mask[None, :, r, None, None], new, pairs[..., where])
    pool[..., 8 * d:] = pairs.view(torch.uint8).to(DEV)
    return {**b, "pool": pool}


def fp16(x):
    return int(np.float16(x).view(np.int16))


STALE = {"8736": (fp16(8736), fp16(-65504)), "60000": (fp16(60000), fp16(1)), "infinity": (fp16(np.inf), fp16(0)),
         "nan": (-1, -1), "random": None}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 8, 2), (128, 16, 1), (256, 4, 1)])
@pytest.mark.parametrize("q_lens,k_lens", [([1, 1, 1], [10, 130, 700]),          # decode rows
                                           ([3, 1, 5], [43, 17, 333]),           # drafts
                                           ([70, 2, 130], [75, 45, 401])])       # chunks
def test_stale_slots_do_not_matter(dtype, d, hq, hkv, q_lens, k_lens):
    """Whatever the slots past a row's keys hold, the results are the same bits."""
    b = make_batch(k_lens, q_lens, hq, hkv, d, dtype, seed=d)
    rewrite_v(b, lambda r: torch.full((k_lens[r],), 0.02))
    zero = fill_unseen(b, (0, 0))
    o, lse = run(zero)
    check(zero, o)
    for name, bits in STALE.items():
        got = run(fill_unseen(b, bits))
        assert torch.equal(got[0], o) and torch.equal(got[1], lse), name
    b200.check_device_errors()


@pytest.mark.parametrize("d", [64, 128])
def test_blocks_without_data_do_not_matter(d):
    """Bad block ids in mid-row leave what memory held in their place: as if the keys were masked."""
    b = make_batch([400, 90], [1, 3], 4, 2, d, torch.float16, seed=d + 1)
    rewrite_v(b, lambda r: torch.full((b["k_lens"][r],), 0.02))
    b["table"][0, 3], b["table"][0, 24], b["table"][1, 0] = -1, 10 ** 6, -7
    o, lse = run(b)
    big = make_batch([4000] * 8, [1] * 8, 4, 2, d, torch.float16, seed=3)  # leaves large scales behind
    rewrite_v(big, lambda r: torch.full((4000,), 20000.0))
    with pytest.raises(RuntimeError, match="block id out of range"):
        b200.check_device_errors()
    for _ in range(3):
        run(big)
        again = run(b)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    with pytest.raises(RuntimeError, match="block id out of range"):
        b200.check_device_errors()
    check(b, o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,hkv,n", [(64, 4, 1, 8), (128, 8, 2, 6), (128, 8, 1, 2), (128, 4, 1, 90), (256, 4, 4, 3)])
def test_later_tokens_do_not_matter(dtype, d, hq, hkv, n):
    """Of a row's new tokens the last has a V and a K of any size: the tokens before it give the same bits."""
    b = make_batch([77 + n], [n], hq, hkv, d, dtype, seed=d + n)
    rewrite_v(b, lambda r: torch.full((77 + n,), 0.02))
    o, lse = run(b)
    last = torch.tensor(slots_of(b, 0)[-1:], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for k_size, v_size in ((1.0, 60000.0), (100.0, 0.02), (100.0, 60000.0), (1e4, 1.0)):
        k = (torch.randn(1, hkv, d, generator=g, device=DEV) * k_size).clamp(-65504, 65504).half()
        v = (torch.randn(1, hkv, d, generator=g, device=DEV) * v_size).clamp(-65504, 65504).half()
        b200.kv_append_q4(k, v, b["pool"][0], b["pool"][1], last)
        got = run(b)
        assert torch.equal(got[0][:n - 1], o[:n - 1]) and torch.equal(got[1][:n - 1], lse[:n - 1]), (k_size, v_size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,q_len", [(64, 1), (128, 1), (128, 3), (256, 1)])
@pytest.mark.parametrize("order", ["first", "last", "middle"])
@pytest.mark.parametrize("gap", [40.0, 12.0])
def test_keys_of_no_weight_do_not_matter(dtype, d, q_len, order, gap):
    """Keys whose score is `gap` below the others' have a V ten million times theirs: O is still right to
    the rounding of what each key gives it."""
    n = 200
    b = make_batch([n], [q_len], 2, 1, d, dtype, seed=d)
    heavy = torch.zeros(n, dtype=torch.bool)
    heavy[{"first": slice(0, 40), "last": slice(n - 45, n - 5), "middle": slice(60, 100)}[order]] = True
    slots = torch.tensor(slots_of(b, 0), device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    b["q"] = torch.ones(q_len, 2, d, device=DEV, dtype=dtype)
    b["scale"] = 1.0 / d
    k = torch.randn(n, 1, d, generator=g, device=DEV) * 0.1
    k[heavy] -= gap
    v = torch.randn(n, 1, d, generator=g, device=DEV) * torch.where(heavy, 1e4, 1e-3).to(DEV)[:, None, None]
    b200.kv_append_q4(k.half(), v.half(), b["pool"][0], b["pool"][1], slots)
    o, _ = run(b)
    b200.check_device_errors()
    check(b, o)


@pytest.mark.parametrize("d", [128, 256])
def test_groups_of_different_size(d):
    """One group of a head holds values of 10^4, the others of 10^-1: each is right to its own size."""
    n = 300
    b = make_batch([n, 40], [1, 2], 4, 2, d, torch.float16, seed=d)
    slots = torch.tensor(slots_of(b, 0) + slots_of(b, 1), device=DEV)
    k, _ = b200.kv_gather_q4(b["pool"][0], b["pool"][1], slots, d, torch.float32)
    v = torch.randn(k.shape, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    v[..., :64] *= 1e4
    v[..., 64:] *= 0.1
    b200.kv_append_q4(k.half(), v.half(), b["pool"][0], b["pool"][1], slots)
    o, _ = run(b)
    check(b, o)
