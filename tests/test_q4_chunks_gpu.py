"""Prompt chunks over a 4-bit pool (the tcgen05 kernel)."""
import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from oracle import q4 as oracle
from tests.test_q4_gpu import DEV, check, make_batch, metadata
from tests.tolerance import dtype_key, half_ulp

pytestmark = pytest.mark.gpu


def run(b, causal=True):
    return b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), b["hq"], b["hkv"], b["scale"],
                                      is_causal=causal)


def check_with_nan(b, o, lse):
    """NaN where the definition has it and nowhere else; the bound of tests/test_q4_gpu.py, V's largest
    value (below 6 here) in place of the largest that a query sees, for the rest."""
    p = b["pool"].cpu().numpy()
    ro, rl, _ = oracle.attention(b["q"].double().cpu().numpy(), p[0], p[1], b["table"], b["starts"], b["q_lens"],
                                 b["k_lens"], b["pos"], b["scale"])
    o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
    nan = np.isnan(ro)
    assert np.array_equal(np.isnan(o), nan)
    ro, o = np.nan_to_num(ro), np.nan_to_num(o)
    assert (np.abs(o - ro) <= (2 * 2.0 ** -11 + 2.0 ** -13) * 6 + half_ulp(ro, dtype_key(b["q"].dtype)) + 1e-6).all()
    assert (np.abs(lse - rl) <= 1e-4 + 1e-5 * np.abs(rl)).all()
    return nan


def nan_in_v(b, keys):
    """A NaN in one group of one head's V, of each of these keys of row 0."""
    d = b["q"].shape[-1]
    slots = torch.tensor([int(b["table"][0, j // 16]) * 16 + j % 16 for j in keys], device=DEV)
    k, v = b200.kv_gather_q4(b["pool"][0], b["pool"][1], slots, d, torch.float32)
    for i in range(len(keys)):
        v[i, i % 2, d - 1 if i % 2 else 5] = float("nan")  # head 0's first group, head 1's last
    b200.kv_append_q4(k.half(), v.half(), b["pool"][0], b["pool"][1], slots)


@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (128, 8)])
@pytest.mark.parametrize("q_len,k_len,keys", [
    (70, 75, [40]), (300, 300, [130, 290]), (150, 700, [3]), (150, 700, [560, 699]),
    (12, 4000, [3995]), (12, 4000, [1, 3990]),  # one tile of queries, its keys taken in turn
    (40, 6000, [5970]), (40, 6000, [2000])])    # cut by keys
def test_nan_of_a_v_group(d, group, q_len, k_len, keys):
    """A group of V that holds a NaN gives NaN in its own 64 dims, to the queries that see the key, and
    leaves LSE and the other dims alone."""
    b = make_batch([k_len], [q_len], 2 * group, 2, d, torch.bfloat16, seed=d + q_len)
    nan_in_v(b, keys)
    o, lse = run(b)
    nan = check_with_nan(b, o, lse)
    assert nan.any() and not nan.all()
    b200.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (128, 16), (256, 4)])
@pytest.mark.parametrize("q_len,k_len,keys", [(1, 75, [0]), (1, 75, [40, 74]), (3, 3000, [1500, 2998]), (5, 90, [88, 89])])
def test_nan_of_a_v_group_in_rows_of_few_tokens(dtype, d, group, q_len, k_len, keys):
    """As above, and the same of a token whether its row is a chunk or not."""
    b = make_batch([k_len], [q_len], 2 * group, 2, d, dtype, seed=d + q_len)
    nan_in_v(b, keys)
    o, lse = run(b)
    nan = check_with_nan(b, o, lse)
    assert nan.any() and (d == 64 or not nan.all())  # with one group to a head it may be all
    chunk = {**b, "q": b["q"][-1:].repeat(70, 1, 1), "q_lens": [70], "pos": [k_len - 70]}
    many, many_lse = run(chunk)
    assert torch.equal(torch.isnan(many[-1]), torch.isnan(o[-1])) and torch.isfinite(many_lse).all()
    b200.check_device_errors()


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 4), (128, 16, 4)])
def test_the_same_bits_every_time(d, hq, hkv):
    """Copies, decoding and products go on at the same time in warps of their own: what they hand on does
    not depend on which is faster, beside other work or alone."""
    b = make_batch([2500, 700, 1300, 90, 3000], [300, 64, 129, 90, 200], hq, hkv, d, torch.bfloat16, seed=1)
    o, lse = run(b)
    check(b, o, lse)
    side = torch.cuda.Stream()
    busy = torch.randn(1 << 24, device=DEV)
    for i in range(60):
        if i % 2:
            with torch.cuda.stream(side):
                busy.mul_(1.0001)
        again = run(b)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    b200.check_device_errors()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", [(64, 200), (12, 400)])      # two tiles of queries; one, its keys taken in turn
@pytest.mark.parametrize("idle", [(12, 40), (64, 0), (20, 0)])  # a tile for one warpgroup; queries that see no key
def test_units_without_work_for_a_warpgroup(d, first, idle):
    """Many units in a row that one warpgroup of a CTA, or both, have nothing to do for, between units that they
    share: more than there are places to describe units ahead."""
    hkv, group = 4, 4
    rows = [first] * 80 + [idle] * 330 + [first] * 45 + [idle] * 200
    q_lens, k_lens = [q for q, _ in rows], [k for _, k in rows]
    b = make_batch(k_lens, q_lens, hkv * group, hkv, d, torch.float16, seed=d)
    b["pos"] = [k - q if k else 0 for q, k in rows]
    out, lse = run(b)
    b200.check_device_errors()
    slots = (torch.tensor(b["table"], device=DEV).long()[:, :, None] * 16 + torch.arange(16, device=DEV)).view(len(rows), -1)
    for shape in {first, idle}:
        which = [r for r, x in enumerate(rows) if x == shape]
        nq, nk = shape
        tokens = (torch.tensor([b["starts"][r] for r in which], device=DEV)[:, None] + torch.arange(nq, device=DEV)).view(-1)
        o, l = out[tokens].view(len(which), nq, -1, d), lse[tokens].view(len(which), nq, -1)
        if nk == 0:
            assert (o == 0).all() and torch.isneginf(l).all()
            continue
        k, v = b200.kv_gather_q4(b["pool"][0], b["pool"][1], slots[which, :nk].reshape(-1), d, torch.float32)
        k, v = (x.view(len(which), nk, hkv, d).double().repeat_interleave(group, 2) for x in (k, v))
        s = torch.einsum("rqhd,rkhd->rhqk", b["q"][tokens].view(len(which), nq, -1, d).double(), k) * b["scale"]
        s = s.masked_fill(torch.ones(nq, nk, dtype=torch.bool, device=DEV).triu(nk - nq + 1), -torch.inf)
        ref = torch.einsum("rhqk,rkhd->rqhd", s.softmax(-1), v)
        # the bound of tests/test_q4_gpu.py, V below 6
        assert ((o.double() - ref).abs() <= (2 * 2.0 ** -11 + 2.0 ** -13) * 6 + 2.0 ** -11 * ref.abs() + 1e-6).all()
        assert ((l.double() - s.logsumexp(-1).transpose(1, 2)).abs() <= 1e-4).all()
