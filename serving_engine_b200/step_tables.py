"""A step's block tables, slots and metadata, built on the GPU from request lengths.

The engine's host code walks every request of a step to extend its block table, place
its tokens and pack the metadata (serving_engine/block_manager.py:87-111,
serving_engine/model_runner.py:127-170, serving_engine/paged_attention_kernel.py:163-200),
then copies the result over. ``StepTables.build`` does the same in one launch from
lengths, tables and a free list that stay on the GPU, so a step can follow another
without the host knowing what was allocated. Its buffers keep their addresses, so a
CUDA graph can hold the call.
"""
from __future__ import annotations

import torch

from . import ops
from ._lib import check, lib

MAX_ROWS = 16384


class StepTables:
    """Output buffers for steps of up to ``rows`` rows (a batch of fixed shape; rows that
    hold no request have q_len 0) and ``tokens`` tokens, and the call that fills them.

    q_starts, k_lens, q_pos_offsets: int32 [rows]; item_row: int32 [tokens] (-1 past the
    rows' tokens); positions, slot_mapping: int64 [tokens] (0 and -1 past them);
    free_state: int32 [2], the free list's head and count after the step.
    """

    def __init__(self, rows: int, tokens: int, device="cuda"):
        if not 0 < rows <= MAX_ROWS or tokens <= 0:
            raise ValueError(f"StepTables: rows must be in [1, {MAX_ROWS}] and tokens positive, got {rows} and {tokens}")
        self.rows, self.tokens = rows, tokens
        wide = torch.zeros(2, tokens, dtype=torch.int64, device=device)
        narrow = torch.zeros(3 * rows + tokens + 2, dtype=torch.int32, device=device)
        self.positions, self.slot_mapping = wide[0], wide[1]
        self.q_starts, self.k_lens, self.q_pos_offsets = narrow[:3 * rows].view(3, rows)
        self.item_row = narrow[3 * rows:3 * rows + tokens]
        self.free_state = narrow[3 * rows + tokens:]
        self.device = wide.device
        self._out = tuple(t.data_ptr() for t in (self.q_starts, self.k_lens, self.q_pos_offsets, self.item_row,
                                                 self.positions, self.slot_mapping, self.free_state))

    def build(self, q_lens: torch.Tensor, context_lens: torch.Tensor, block_table: torch.Tensor,
              free_ids: torch.Tensor, free_state: torch.Tensor) -> dict:
        """Fill the buffers for rows that hold context_lens tokens and add q_lens (int32
        [rows]); new blocks come from the ring free_ids (int32), of which free_state
        (int32 [2]: head, count) are free, and are written into block_table (int32 [rows,
        max_blocks], unit column stride). ``self.free_state`` is the state after the step:
        copy it over free_state, or pass it to another StepTables' next build. Returns the
        metadata dict of build_paged_batch_metadata. One launch.

        The host can follow without reading back: rows take ceil(k_len / 16) -
        ceil(context / 16) blocks each, in row order from the head of the ring.
        """
        dev = self.device
        for name, t, shape in (("q_lens", q_lens, (self.rows,)), ("context_lens", context_lens, (self.rows,)),
                               ("free_state", free_state, (2,))):
            if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"StepTables.build: {name} must be int32 {list(shape)}, contiguous and on {dev}")
        if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != self.rows
                or block_table.shape[1] == 0 or block_table.stride(1) != 1 or block_table.device != dev
                or block_table.stride(0) < block_table.shape[1]):
            raise ValueError(f"StepTables.build: block_table must be int32 [{self.rows}, max_blocks >= 1] on {dev} "
                             "with unit column stride and rows that do not overlap")
        if (free_ids.dtype != torch.int32 or free_ids.dim() != 1 or free_ids.numel() == 0
                or not free_ids.is_contiguous() or free_ids.device != dev):
            raise ValueError(f"StepTables.build: free_ids must be a non-empty int32 vector, contiguous and on {dev}")
        if free_state.data_ptr() == self._out[-1]:
            raise ValueError("StepTables.build: free_state must not be this object's own free_state")
        width = block_table.shape[1]
        st = lib().seb_step_tables(q_lens.data_ptr(), context_lens.data_ptr(), self.rows, self.tokens,
                                   block_table.data_ptr(), block_table.stride(0), width, free_ids.data_ptr(),
                                   free_ids.numel(), free_state.data_ptr(), *self._out,
                                   ops.err_word(dev).data_ptr(), ops._stream(dev))
        check("seb_step_tables", st)
        ops.LAUNCHES[0] += 1
        ops._after(dev)
        return {"q_lens": q_lens, "k_lens": self.k_lens, "q_starts": self.q_starts,
                "q_pos_offsets": self.q_pos_offsets, "block_table": block_table, "block_table_row_stride": width,
                "total_query": self.tokens}
