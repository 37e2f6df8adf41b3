"""Sizes that the counts of work have to hold."""
import pytest
import torch

import serving_engine_b200 as b200
from tests.test_q4_gpu import DEV, make_batch, metadata

pytestmark = pytest.mark.gpu


def test_long_chunks_with_a_wide_table():
    """Rows of thousands of tokens whose tables could hold millions of keys: the kernel for rows of few
    tokens, which counts what the tables allow, has none of these."""
    hq = 64
    b = make_batch([4200, 4150], [4200, 4096], hq, hq, 64, torch.bfloat16, seed=1)
    md = metadata(b)
    width = (1 << 18) + 500
    wide = torch.zeros(2, width, dtype=torch.int32, device=DEV)
    wide[:, :b["table"].shape[1]] = md["block_table"]
    md["block_table"], md["block_table_row_stride"] = wide, width
    o, lse = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], md, hq, hq, b["scale"])
    md["block_table"], md["block_table_row_stride"] = metadata(b)["block_table"], b["table"].shape[1]
    want = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], md, hq, hq, b["scale"])
    b200.check_device_errors()
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_overlapping_rows_beyond_32_bits():
    """Rows that all claim all tokens (never valid) come to more work than is counted: an error, no work
    done, and the next call on the stream is right."""
    n, hq, d = 4096, 8, 64
    b = make_batch([8320, 300], [1, 1], hq, hq, d, torch.float16, seed=2)
    want = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), hq, hq, b["scale"])
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.tensor(b["table"][:1], **i32).repeat(n, 1)
    q = torch.zeros(n, hq, d, device=DEV, dtype=torch.float16)
    out = torch.full_like(q, 3.0)
    b200.paged_attention_q4(q, b["pool"][0], b["pool"][1], table, torch.zeros(n, **i32), torch.full((n,), n, **i32),
                            torch.full((n,), 8320, **i32), torch.full((n,), 8320, **i32), hq, hq, b["scale"], out=out)
    with pytest.raises(RuntimeError, match="index out of range"):
        b200.check_device_errors()
    assert (out == 3).all()
    for _ in range(2):
        again = b200.paged_flash_attention(b["q"], b["pool"][0], b["pool"][1], metadata(b), hq, hq, b["scale"])
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    b200.check_device_errors()
