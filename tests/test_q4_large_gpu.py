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
