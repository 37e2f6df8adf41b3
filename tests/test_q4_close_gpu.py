"""Attention over a 4-bit pool against float64 with bounds that follow the roundings closely: what a sum over
many keys, a cut between CTAs or a join may lose shows here."""
import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from oracle import q4 as oracle
from serving_engine_b200.paged_attention import metadata_from_lists
from tests.test_q4_gpu import DEV, make_batch, metadata
from tests.tolerance import dtype_key, half_ulp

pytestmark = pytest.mark.gpu


def filled_pool(blocks, hkv, d, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pool = b200.new_q4_pool(1, blocks, hkv, d)[0]
    for start in range(0, blocks * 16, 16384):
        m = min(16384, blocks * 16 - start)
        k, v = (torch.randn(m, hkv, d, generator=g, device=DEV).half() for _ in range(2))
        b200.kv_append_q4(k, v, pool[0], pool[1], torch.arange(start, start + m, device=DEV))
    return pool, g


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,rows", [(65536, 6), (60001, 2)])
def test_the_mean_of_many_values(d, n, rows):
    """Queries of zero weigh all keys alike. A run adds sums of codes (below 16 for each key) in fp32, in two
    products of 16 keys each, every one off by at most 2^-22 of the sum so far, and takes 8 for each key
    off after 64 keys: 2 * (15 + 8) * 2^-22 * (16 + 32 + 48 + 64) = 1.8e-3 of a scale in 64 keys, 2.8e-5 of a
    scale for each; then fp16's half ulp and the fp32 sums of lows, 2^-18 of V's size."""
    hkv, group = 8, 4
    blocks = -(-n // 16)
    pool, _ = filled_pool(blocks, hkv, d, d + 1)
    _, v = b200.kv_gather_q4(pool[0], pool[1], torch.arange(n, device=DEV), d, torch.float32)
    mean = v.double().mean(0)
    groups = v.view(n, hkv, d // 64, 64)
    scale = ((groups.amax(-1) - groups.amin(-1)) / 15).amax().item()
    md = metadata_from_lists([1] * rows, [n] * rows, list(range(rows)), [n - 1] * rows, [list(range(blocks))] * rows, DEV)
    q = torch.zeros(rows, hkv * group, d, device=DEV).half()
    o, lse = b200.paged_flash_attention(q, pool[0], pool[1], md, hkv * group, hkv, d ** -0.5)
    b200.check_device_errors()
    ref = mean.repeat_interleave(group, 0)[None].expand(rows, -1, -1)
    bound = 2.8e-5 * scale + 2.0 ** -18 * v.abs().amax().item() + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    assert ((o.double() - ref).abs() <= bound).all(), float(((o.double() - ref).abs() / bound).max())
    assert (lse.double() - float(np.log(n))).abs().amax() <= 2e-6 * 12


def reference(q, kk, vv, scale, po, causal):
    """O, LSE, sum p |v|, and the root of sum (p v)^2, which independent errors of each key's term follow."""
    s = torch.einsum("qhd,khd->hqk", q.double(), kk) * scale
    if causal:
        nq, nk = q.shape[0], kk.shape[0]
        s = s.masked_fill(torch.arange(nk, device=DEV)[None] > po + torch.arange(nq, device=DEV)[:, None], -torch.inf)
    p = s.softmax(-1)
    return (torch.einsum("hqk,khd->qhd", p, vv), s.logsumexp(-1).T, torch.einsum("hqk,khd->qhd", p, vv.abs()),
            torch.einsum("hqk,khd->qhd", p.square(), vv.square()).sqrt())


@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (128, 8), (128, 16), (64, 7)])
@pytest.mark.parametrize("q_lens,k_lens", [([40], [9000]), ([100, 13, 7], [5000, 4097, 130]),
                                           ([65, 64, 12], [2049, 64, 7000]), ([3, 1], [6000, 9000])])
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows_of_many_keys(d, group, q_lens, k_lens, causal):
    """Chunks that are cut by keys, and rows of few tokens that are joined. Of each key's term p, V and, through
    its score (off by some 2e-4 where K is rounded once), p again are off by a rounding to 11 bits, 1.2e-4 of it
    in the mean, each on its own: 2.6e-4 of the root of sum (p v)^2 in all, and never 8 times that; then fp16's
    half ulp of O and the fp32 sums."""
    hkv = 2
    hq = hkv * group
    need = [-(-k // 16) for k in k_lens]
    pool, g = filled_pool(sum(need) + 3, hkv, d, d + group)
    ids = torch.randperm(sum(need) + 3, generator=g, device=DEV)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n].tolist())
        at += n
    q = torch.randn(sum(q_lens), hq, d, generator=g, device=DEV).half()
    starts = [sum(q_lens[:i]) for i in range(len(q_lens))]
    pos = [max(k_ - q_, 0) for q_, k_ in zip(q_lens, k_lens)]
    md = metadata_from_lists(q_lens, k_lens, starts, pos, table, DEV)
    scale = d ** -0.5
    o, lse = b200.paged_flash_attention(q, pool[0], pool[1], md, hq, hkv, scale, is_causal=causal)
    b200.check_device_errors()
    for nq, nk, st, po, tb in zip(q_lens, k_lens, starts, pos, table):
        slots = (torch.tensor(tb, device=DEV)[:, None] * 16 + torch.arange(16, device=DEV)).view(-1)[:nk]
        kk, vv = (x.double().repeat_interleave(group, 1)
                  for x in b200.kv_gather_q4(pool[0], pool[1], slots, d, torch.float32))
        ref, ref_lse, size, root = reference(q[st:st + nq], kk, vv, scale, po, causal)
        bound = 2.0 ** -11 * ref.abs() + 8 * 2.6e-4 * root + 2.0 ** -18 * size + 2.0 ** -25
        err = (o[st:st + nq].double() - ref).abs()
        assert (err <= bound).all(), float((err / bound).max())
        assert ((lse[st:st + nq].double() - ref_lse).abs() <= 1e-4).all()


@pytest.mark.parametrize("q_len", [1, 2, 100])
@pytest.mark.parametrize("size", [1e30, 3e4, 1e-30])
def test_queries_of_any_size(q_len, size):
    """bf16 queries that fp16 cannot hold, in rows of few tokens and in chunks: the largest key takes all, or
    all weigh the same."""
    b = make_batch([150], [q_len], 2, 1, 64, torch.bfloat16, seed=24)
    b["q"] = (b["q"].float() * size).bfloat16()
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), 2, 1, b["scale"])
    p = b["pool"].cpu().numpy()
    ro, rl, top = oracle.attention(b["q"].double().cpu().numpy(), p[0], p[1], b["table"], b["starts"], b["q_lens"],
                                   b["k_lens"], b["pos"], b["scale"])
    tol = (2 * 2.0 ** -11 + 2.0 ** -13) * top[..., None] + half_ulp(ro, "bf16") + 1e-6
    assert (np.abs(o.double().cpu().numpy() - ro) <= tol).all()
    assert (np.abs(lse.double().cpu().numpy() - rl) <= 1e-4 + 1e-5 * np.abs(rl)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 2, 70])
@pytest.mark.parametrize("gap", [10.0, 13.3, 14.7])
def test_a_first_key_that_takes_most(dtype, d, q_len, gap):
    """A first key with a score `gap` above all others and a V of next to nothing, as models learn it: O is what
    the others give, and right to its own size though each of them weighs 10^-6 of the first."""
    n, group = 20000, 4
    blocks = -(-n // 16)
    g = torch.Generator(device=DEV).manual_seed(d)
    pool = b200.new_q4_pool(1, blocks, 1, d)[0]
    k = torch.randn(n, 1, d, generator=g, device=DEV) * 0.1
    k[0] = gap
    v = 1 + 0.5 * torch.randn(n, 1, d, generator=g, device=DEV)
    v[0] *= 1e-3
    for start in range(0, n, 8192):
        part = slice(start, min(start + 8192, n))
        b200.kv_append_q4(k[part].to(dtype), v[part].to(dtype), pool[0], pool[1],
                          torch.arange(part.start, part.stop, device=DEV))
    q = (1 + 0.01 * torch.randn(q_len, group, d, generator=g, device=DEV)).to(dtype)
    md = metadata_from_lists([q_len], [n], [0], [n - q_len], [list(range(blocks))], DEV)
    o, lse = b200.paged_flash_attention(q, pool[0], pool[1], md, group, 1, 1.0 / d)
    b200.check_device_errors()
    kk, vv = (x.double().repeat_interleave(group, 1)
              for x in b200.kv_gather_q4(pool[0], pool[1], torch.arange(n, device=DEV), d, torch.float32))
    ref, ref_lse, size, root = reference(q, kk, vv, 1.0 / d, n - q_len, True)
    half = torch.from_numpy(half_ulp(ref.cpu().numpy(), dtype_key(dtype))).to(DEV)
    # roundings of each key's term on its own, as above; of sums, 2^-23 of them for each 16 keys, always down
    bound = half + 8 * 2.6e-4 * root + n / 16 * 2.0 ** -24 * size + 2.0 ** -25
    err = (o.double() - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert ((lse.double() - ref_lse).abs() <= 1e-4 + 1e-5 * ref_lse.abs()).all()
