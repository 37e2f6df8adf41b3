"""Decoding over long rows of a 4-bit pool: what sums of many keys lose."""
import pytest
import torch

import serving_engine_b200 as b200
from serving_engine_b200.paged_attention import metadata_from_lists

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [65536, 65519])
def test_the_mean_of_many_values(d, n):
    """Queries of zero weigh all keys alike, so O is V's mean, some hundredths of V's size, and the
    weights round to nothing: what differs is how the sums are held. Many rows over the same
    blocks make each warp's run long. A run adds sums of codes (below 16 for each key) in fp32,
    each step of 16 keys off by at most 2^-22 of the sum so far, and takes 8 for each key off
    after at most 256 keys: (15 + 8) * 2^-22 * (16 + 32 + ... + 256) = 0.012 of a scale in 256 keys,
    4.7e-5 of a scale for each; then fp16's half ulp and the fp32 sums of lows, 2^-18 of V's size."""
    rows, hkv, group = 6, 8, 4
    blocks = -(-n // 16)
    g = torch.Generator(device=DEV).manual_seed(d)
    pool = b200.new_q4_pool(1, blocks, hkv, d)[0]
    for start in range(0, blocks * 16, 16384):
        m = min(16384, blocks * 16 - start)
        k, v = (torch.randn(m, hkv, d, generator=g, device=DEV).half() for _ in range(2))
        b200.kv_append_q4(k, v, pool[0], pool[1], torch.arange(start, start + m, device=DEV))
    _, v = b200.kv_gather_q4(pool[0], pool[1], torch.arange(n, device=DEV), d, torch.float32)
    mean = v.double().mean(0)
    scale = ((v.view(n, hkv, d // 64, 64).amax(-1) - v.view(n, hkv, d // 64, 64).amin(-1)) / 15).amax().item()
    md = metadata_from_lists([1] * rows, [n] * rows, list(range(rows)), [n - 1] * rows, [list(range(blocks))] * rows, DEV)
    q = torch.zeros(rows, hkv * group, d, device=DEV).half()
    o, lse = b200.paged_flash_attention(q, pool[0], pool[1], md, hkv * group, hkv, d ** -0.5)
    b200.check_device_errors()
    ref = mean.repeat_interleave(group, 0)[None].expand(rows, -1, -1)
    bound = 4.7e-5 * scale + 2.0 ** -18 * v.abs().amax().item() + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    assert ((o.double() - ref).abs() <= bound).all()
    assert (lse.double() - torch.tensor(n, dtype=torch.float64).log().item()).abs().amax() <= 2e-6 * 12


@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (128, 8), (128, 16), (64, 7)])
@pytest.mark.parametrize("q_lens,k_lens", [([40], [9000]), ([100, 13, 7], [5000, 4097, 130]),
                                           ([65, 64, 12], [2049, 64, 7000])])
@pytest.mark.parametrize("causal", [True, False])
def test_few_chunks_of_long_rows(d, group, q_lens, k_lens, causal):
    """Chunks with fewer units than the GPU has CTAs are cut by keys and joined: against float64 over
    what the pool stands for, and twice the same bits."""
    hkv = 2
    hq = hkv * group
    g = torch.Generator(device=DEV).manual_seed(d + group)
    need = [-(-k // 16) for k in k_lens]
    pool = b200.new_q4_pool(1, sum(need) + 3, hkv, d)[0]
    ids = torch.randperm(sum(need) + 3, generator=g, device=DEV)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n].tolist())
        at += n
    k, v = (torch.randn((sum(need) + 3) * 16, hkv, d, generator=g, device=DEV).half() for _ in range(2))
    b200.kv_append_q4(k, v, pool[0], pool[1], torch.arange((sum(need) + 3) * 16, device=DEV))
    total = sum(q_lens)
    q = torch.randn(total, hq, d, generator=g, device=DEV).half()
    starts = [sum(q_lens[:i]) for i in range(len(q_lens))]
    pos = [max(k_ - q_, 0) for q_, k_ in zip(q_lens, k_lens)]
    md = metadata_from_lists(q_lens, k_lens, starts, pos, table, DEV)
    scale = d ** -0.5
    o, lse = b200.paged_flash_attention(q, pool[0], pool[1], md, hq, hkv, scale, is_causal=causal)
    again = b200.paged_flash_attention(q, pool[0], pool[1], md, hq, hkv, scale, is_causal=causal)
    b200.check_device_errors()
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    for r, (nq, nk, st, po, tb) in enumerate(zip(q_lens, k_lens, starts, pos, table)):
        slots = (torch.tensor(tb, device=DEV)[:, None] * 16 + torch.arange(16, device=DEV)).view(-1)[:nk]
        kk, vv = (x.double().repeat_interleave(group, 1) for x in b200.kv_gather_q4(pool[0], pool[1], slots, d, torch.float32))
        s = torch.einsum("qhd,khd->hqk", q[st:st + nq].double(), kk) * scale
        if causal:
            s = s.masked_fill(torch.arange(nk, device=DEV)[None] > po + torch.arange(nq, device=DEV)[:, None], -torch.inf)
        ref = torch.einsum("hqk,khd->qhd", s.softmax(-1), vv)
        # Half an ulp of fp16 for O; K, V and p rounded to fp16 move an output that is a mean of many values by
        # some 2^-11 of V's size (below 5) over the root of the keys that count, and one of few keys by 2^-11 of it.
        bound = 2.0 ** -11 * ref.abs() + 2 * 2.0 ** -11 * 5 + 2.0 ** -24
        assert ((o[st:st + nq].double() - ref).abs() <= bound).all()
        # A score of size sqrt(d) * scale = 1 is off by some 2e-4 where K is rounded once; a row of few keys has it in two parts.
        assert ((lse[st:st + nq].double() - s.logsumexp(-1).T).abs() <= 1e-4).all()
