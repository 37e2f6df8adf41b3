"""The 4-bit pool in the framework's own paths: PagedKVCache, block copies, the registered
attention function's pool, the fused model step, and generation with GPU-built tables."""

import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from serving_engine_b200 import ops
from serving_engine_b200.e2e import random_llama
from serving_engine_b200.llama_step import FusedLlamaStep
from serving_engine_b200.paged_attention import metadata_from_lists
from serving_engine_b200.q4_serve import Q4Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_cache_write_update_and_copy_blocks():
    h, d, layers, nb = 2, 64, 3, 6
    pool = b200.new_q4_pool(layers, nb, h, d)
    cache = b200.PagedKVCache(pool)
    assert cache.is_q4 and cache.num_kv_heads == h and cache.head_dim == d
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(1, h, 20, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    slots = torch.randperm(nb * 16, generator=g, device=DEV)[:20]
    rk, rv = cache.update(k, v, 1, slots, slots)
    want = b200.new_q4_pool(1, nb, h, d)[0]
    b200.kv_append_q4(k[0].transpose(0, 1), v[0].transpose(0, 1), want[0], want[1], slots)
    assert torch.equal(pool[1], want) and (pool[0] == 0).all() and (pool[2] == 0).all()
    ek, ev = b200.kv_gather_q4(want[0], want[1], slots, d, torch.bfloat16)
    assert torch.equal(rk, ek) and torch.equal(rv, ev)
    pool.random_(0, 256)
    ref = pool.clone()
    ref[:, :, [0, 5]] = ref[:, :, [3, 1]]
    cache.copy_blocks([3, 1], [0, 5])
    b200.check_device_errors()
    assert torch.equal(pool, ref)
    with pytest.raises(ValueError, match="pool must be"):
        ops.copy_blocks(pool[0], [1], [2])


def test_slot_minus_one_is_no_token():
    """Tokens of no row (StepTables' padding) are skipped without an error."""
    pool = b200.new_q4_pool(1, 2, 1, 64)[0]
    x = torch.randn(3, 1, 64, device=DEV).half()
    slots = torch.tensor([-1, 7, -1], device=DEV)
    b200.kv_append_q4(x, x, pool[0], pool[1], slots)
    qkv, cs = torch.randn(3, 64 * 4, device=DEV).half(), torch.ones(3, 64, device=DEV).half()
    q = b200.qk_norm_rope_append(qkv, cs, cs * 0, slots, pool[0], pool[1], 2, 1)
    k, _ = b200.kv_gather_q4(pool[0], pool[1], slots, 64)
    b200.check_device_errors()
    assert torch.equal(q, qkv[:, :128].view(3, 2, 64)) and (k[[0, 2]] == 0).all() and (k[1] != 0).any()
    other = pool.clone()
    other[..., :] = 0
    b200.kv_append_q4(qkv[1:2, 128:192].view(1, 1, 64), qkv[1:2, 192:].view(1, 1, 64), other[0], other[1], slots[1:2])
    assert torch.equal(pool, other)


def test_registered_forward_takes_a_q4_pool():
    h, d, n = 2, 128, 40
    cache = b200.PagedKVCache(b200.new_q4_pool(1, 4, h, d))
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(1, 4, n, d, generator=g, device=DEV).bfloat16()
    k, v = (torch.randn(1, h, n, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    table = [2, 0, 3]
    slots = torch.tensor([table[i // 16] * 16 + i % 16 for i in range(n)], device=DEV)
    md = metadata_from_lists([n], [n], [0], [0], [table], DEV)
    module = type("M", (), {"layer_idx": 0})()
    o, _ = b200.b200_paged_attention_forward(module, q, k, v, None, d ** -0.5, cache=cache, write_index=slots, paged_metadata=md)
    kq, vq = b200.kv_gather_q4(*cache.blocks(0), slots, d, torch.float32)
    s = torch.einsum("qhd,khd->hqk", q[0].transpose(0, 1).double(), kq.double().repeat_interleave(2, 1)) * d ** -0.5
    s = s.masked_fill(torch.ones(n, n, device=DEV).triu(1).bool(), -torch.inf)
    ref = torch.einsum("hqk,khd->qhd", s.softmax(-1), vq.double().repeat_interleave(2, 1))
    assert o.shape == (1, n, 4, d)
    # half an ulp of bf16 and fp16 roundings of values up to 4: 2^-8 |O| + 2 * 2^-11 * 4 + 2^-13 * 4
    assert ((o[0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -8 + 2.0 ** -11).all()


def host_step(step, pool, table, ctx, chunks):
    """The same step with tables made on the host."""
    rows = len(chunks)
    lens = [len(c) for c in chunks]
    starts = np.concatenate(([0], np.cumsum(lens)[:-1])).tolist()
    pos = [p for r in range(rows) for p in range(ctx[r], ctx[r] + lens[r])]
    slots = [int(table[r][p // 16]) * 16 + p % 16 for r in range(rows) for p in range(ctx[r], ctx[r] + lens[r])]
    md = metadata_from_lists(lens, [c + n for c, n in zip(ctx, lens)], starts, ctx, [list(t) for t in table], DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int64, device=DEV)  # noqa: E731
    last = t([s + n - 1 for s, n in zip(starts, lens)])
    return step.logits(t([x for c in chunks for x in c]), t(pos), t(slots), pool, md, last)


@pytest.mark.parametrize("norms", [False, True])
def test_generation_with_gpu_tables_equals_host_tables(norms):
    """Prompts in two chunks, then greedy decoding by graph replays: logits and tokens equal those
    of steps whose tables the host makes (attention of the same rows in the same order)."""
    model = random_llama("tiny", 0, torch.bfloat16, DEV)
    if norms:
        g = torch.Generator(device=DEV).manual_seed(3)
        for layer in model.model.layers:
            for name in ("q_norm", "k_norm"):
                w = (1 + 0.2 * torch.randn(64, generator=g, device=DEV)).bfloat16()
                setattr(layer.self_attn, name, type("N", (), {"weight": w})())
    rows, new = 3, 12
    batch = Q4Batch(model, rows, 160, num_blocks=40)
    rng = np.random.default_rng(0)
    first = [rng.integers(0, 1000, n).tolist() for n in (70, 1, 33)]
    second = [rng.integers(0, 1000, n).tolist() for n in (5, 50, 16)]
    # the blocks that StepTables takes: in row order from the head of the free list
    step, pool = FusedLlamaStep(model), torch.zeros_like(batch.pool)
    table, free, ctx = [[] for _ in range(rows)], iter(range(40)), [0] * rows

    def grow(chunks):
        for r, c in enumerate(chunks):
            while len(table[r]) * 16 < ctx[r] + len(c):
                table[r].append(next(free))

    for chunks in (first, second):
        grow(chunks)
        want = host_step(step, pool, table, ctx, chunks)
        ctx = [c + len(x) for c, x in zip(ctx, chunks)]
        got = batch.prefill(chunks)
        assert torch.equal(got, want)
    assert torch.equal(batch.pool, pool)
    tokens = []
    nxt = want.argmax(-1)
    for _ in range(new):
        tokens.append(nxt.tolist())
        chunks = [[t] for t in nxt.tolist()]
        grow(chunks)
        nxt = host_step(step, pool, table, ctx, chunks).argmax(-1)
        ctx = [c + 1 for c in ctx]
    assert batch.decode(new).tolist() == tokens
    b200.check_device_errors()
    assert batch.lens.tolist() == ctx
    assert torch.equal(batch.pool, pool)
    # without a graph the same tokens follow
    again = Q4Batch(model, rows, 160, num_blocks=40)
    again.prefill(first)
    again.prefill(second)
    assert again.decode(new, use_graph=False).tolist() == tokens


def test_q4_pool_is_near_the_16_bit_pool():
    """Logits of a prompt over a 4-bit pool against the same step over a 16-bit pool: within the
    noise of 4 bits (a value is off by up to 1/30 of its group's range, about 0.13 of a standard
    deviation; logits, sums of many, by well under a tenth of their spread)."""
    model = random_llama("tiny", 1, torch.bfloat16, DEV)
    step = FusedLlamaStep(model)
    tokens = [np.random.default_rng(1).integers(0, 1000, 90).tolist()]
    table = [list(range(6))]
    q4 = host_step(step, b200.new_q4_pool(2, 6, 2, 64), table, [0], tokens)
    full = host_step(step, torch.zeros(2, 2, 6, 16, 2, 64, device=DEV, dtype=torch.bfloat16), table, [0], tokens)
    assert (q4 - full).float().norm() <= 0.1 * full.float().norm()


def test_chunk_sizes_are_checked():
    batch = Q4Batch(random_llama("tiny", 0, torch.bfloat16, DEV), 2, 64)
    with pytest.raises(ValueError, match="2 chunks"):
        batch.prefill([[1]])
    with pytest.raises(ValueError, match="at least one token"):
        batch.prefill([[1], []])
