"""Greedy generation for a batch of requests over a KV pool held in 4 bits, with the
step's tables built on the GPU.

``Q4Batch`` holds what a serving loop keeps: the pool, the rows' block tables, lengths
and free blocks (all on the GPU), and a model's fused layers (``FusedLlamaStep``). A
step is: tables from the lengths (``StepTables``), then for each layer the norms and
rotation of queries and keys with the write into the pool (``qk_norm_rope_append``) and
the attention over it (``paged_flash_attention``). Decode steps are one CUDA graph, and
its replays need nothing from the host: tokens, positions, slots, block tables and
lengths follow from the step before on the GPU.

    python -m serving_engine_b200.q4_serve [--rows 64] [--prompt 1024] [--new 128]

runs random prompts through a random-init Llama of the end-to-end configuration's shape
and prints prefill and decode tokens/s beside the pool's size and what a 16-bit one takes.
"""
from __future__ import annotations

import argparse
import time

import torch

from . import ops
from .llama_step import FusedLlamaStep
from .q4 import Workspace, new_q4_pool
from .step_tables import StepTables

BLOCK_SIZE = ops.BLOCK_SIZE


class Q4Batch:
    """``rows`` requests of up to ``max_len`` tokens each over a pool of ``num_blocks``
    blocks (default: enough for all). ``model``: as FusedLlamaStep takes it, on a GPU.
    Batches may run at the same time, each on a stream of its own."""

    def __init__(self, model, rows: int, max_len: int, num_blocks: int | None = None):
        cfg, device = model.config, next(model.parameters()).device
        self.step = FusedLlamaStep(model)
        self.rows, self.device = rows, device
        width = -(-max_len // BLOCK_SIZE)
        num_blocks = rows * width if num_blocks is None else num_blocks
        self.pool = new_q4_pool(cfg.num_hidden_layers, num_blocks, self.step.hkv, self.step.head_dim, device)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.zeros(rows, width, **i32)
        self.lens = torch.zeros(rows, **i32)            # tokens that each row has in the pool
        self.free_ids = torch.arange(num_blocks, **i32)
        self.free_state = torch.tensor([0, num_blocks], **i32)
        self.tokens = torch.zeros(rows, dtype=torch.int64, device=device)  # each row's newest token
        self._ones = torch.ones(rows, **i32)
        self._decode_tables = StepTables(rows, rows, device)
        self._graph = None
        self._workspace = Workspace()  # the graph's: batches on different streams may decode at the same time

    def _advance(self, tables: StepTables) -> None:
        self.lens.copy_(tables.k_lens)
        self.free_state.copy_(tables.free_state)

    def prefill(self, chunks: list[list[int]]) -> torch.Tensor:
        """One step over new tokens of each row (a whole prompt or the next chunk of it, at
        least one token); returns the logits [rows, vocab] after each row's last token."""
        lens = [len(c) for c in chunks]
        if len(chunks) != self.rows or min(lens) < 1:
            raise ValueError(f"Q4Batch.prefill: {self.rows} chunks of at least one token are required")
        host = torch.tensor(lens + [t for c in chunks for t in c], dtype=torch.int64).pin_memory()
        dev = host.to(self.device, non_blocking=True)
        q_lens = dev[:self.rows].to(torch.int32)
        tables = StepTables(self.rows, sum(lens), self.device)
        md = tables.build(q_lens, self.lens, self.block_table, self.free_ids, self.free_state)
        last = (tables.q_starts + q_lens - 1).to(torch.int64)
        logits = self.step.logits(dev[self.rows:], tables.positions, tables.slot_mapping, self.pool, md, last)
        self._advance(tables)
        torch.argmax(logits, dim=-1, out=self.tokens)
        return logits

    def _decode_step(self) -> torch.Tensor:
        t = self._decode_tables
        md = t.build(self._ones, self.lens, self.block_table, self.free_ids, self.free_state)
        logits = self.step.logits(self.tokens, t.positions, t.slot_mapping, self.pool, md)
        self._advance(t)
        torch.argmax(logits, dim=-1, out=self.tokens)
        return logits

    def decode(self, steps: int, use_graph: bool = True) -> torch.Tensor:
        """``steps`` greedy tokens for every row, [steps, rows]. The first call with
        use_graph captures the step (its warm-up advances nothing that it does not put back)."""
        if use_graph and self._graph is None:
            state = (self.lens, self.free_state, self.tokens, self.block_table)
            kept = [t.clone() for t in state]
            side = torch.cuda.Stream(self.device)
            side.wait_stream(torch.cuda.current_stream(self.device))
            with torch.cuda.stream(side), self._workspace:
                self._decode_step()
            torch.cuda.current_stream(self.device).wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side), self._workspace:
                self._decode_step()
            self._graph = graph
            for t, k in zip(state, kept):
                t.copy_(k)
        out = torch.empty(steps, self.rows, dtype=torch.int64, device=self.device)
        for i in range(steps):
            out[i] = self.tokens
            if use_graph:
                self._graph.replay()
            else:
                self._decode_step()
        return out


def main() -> None:
    from .e2e import random_llama

    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=1024)
    ap.add_argument("--new", type=int, default=128)
    a = ap.parse_args()
    model = random_llama("config4", 0, torch.bfloat16, "cuda", init_on_device=True)
    batch = Q4Batch(model, a.rows, a.prompt + a.new + 1)
    gen = torch.Generator().manual_seed(0)
    prompts = torch.randint(0, model.config.vocab_size, (a.rows, a.prompt), generator=gen).tolist()
    batch.prefill([p[:1] for p in prompts])  # warm-up; the prompts' other tokens are timed
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    batch.prefill([p[1:] for p in prompts])
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    batch.decode(1)
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    batch.decode(a.new - 1)
    torch.cuda.synchronize()
    t3 = time.perf_counter()
    ops.check_device_errors(batch.device)
    pool = batch.pool.numel()
    print(f"prefill {a.rows * (a.prompt - 1) / (t1 - t0):,.0f} tokens/s, decode {a.rows * (a.new - 1) / (t3 - t2):,.0f} "
          f"tokens/s; pool {pool / 1e9:.2f} GB, {pool * 32 / 9 / 1e9:.2f} GB in 16 bits")


if __name__ == "__main__":
    main()
