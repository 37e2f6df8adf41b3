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
