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

from . import q4
from ._lib import lib

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
        if wide.get_device() < 0:
            raise ValueError(f"StepTables: a CUDA device is required, got {wide.device}")
        self._device = wide.get_device()
        self._out = tuple(t.data_ptr() for t in (self.q_starts, self.k_lens, self.q_pos_offsets, self.item_row,
                                                 self.positions, self.slot_mapping, self.free_state))

    def build(self, q_lens: torch.Tensor, context_lens: torch.Tensor, block_table: torch.Tensor,
              free_ids: torch.Tensor, free_state: torch.Tensor) -> dict:
        """Fill the buffers for rows that hold context_lens tokens and add q_lens (int32
        [rows]); new blocks come from the ring free_ids (int32), of which free_state
        (int32 [2]: head, count) are free, and are written into block_table (int32 [rows,
        max_blocks], unit column stride). ``self.free_state`` is the state after the step:
        copy it over free_state, or pass it to another StepTables' next build. The same goes
        for context_lens and k_lens: this object's own buffers are no input of its build.
        Returns the metadata dict of build_paged_batch_metadata. One launch.

        The host can follow without reading back: rows take ceil(k_len / 16) -
        ceil(context / 16) blocks each, in row order from the head of the ring.
        """
        dev = self._device
        rows = self.rows
        shape, strides = block_table.shape, block_table.stride()
        if not (q_lens.dtype == context_lens.dtype == block_table.dtype == free_ids.dtype == free_state.dtype == torch.int32
                and q_lens.shape == context_lens.shape == (rows,) and free_state.shape == (2,) and free_ids.dim() == 1
                and free_ids.numel() and q_lens.is_contiguous() and context_lens.is_contiguous()
                and free_ids.is_contiguous() and free_state.is_contiguous() and len(shape) == 2 and shape[0] == rows
                and shape[1] and strides[1] == 1 and (rows == 1 or strides[0] >= shape[1])
                and q_lens.get_device() == context_lens.get_device() == block_table.get_device()
                == free_ids.get_device() == free_state.get_device() == dev):
            self._refuse(q_lens, context_lens, block_table, free_ids, free_state)
        if free_state.data_ptr() == self._out[-1]:
            raise ValueError("StepTables.build: free_state must not be this object's own free_state")
        width = shape[1]
        st = lib().seb_step_tables(q_lens.data_ptr(), context_lens.data_ptr(), rows, self.tokens,
                                   block_table.data_ptr(), max(strides[0], width), width, free_ids.data_ptr(),
                                   free_ids.numel(), free_state.data_ptr(), *self._out, q4._err_ptr(dev),
                                   q4._raw_stream(dev))
        q4._done("seb_step_tables", st, dev)
        return {"q_lens": q_lens, "k_lens": self.k_lens, "q_starts": self.q_starts,
                "q_pos_offsets": self.q_pos_offsets, "block_table": block_table, "block_table_row_stride": width,
                "total_query": self.tokens}

    def _refuse(self, q_lens, context_lens, block_table, free_ids, free_state):
        """Says what is wrong with build's arguments."""
        dev, rows = self.device, self.rows
        for name, t, shape in (("q_lens", q_lens, (rows,)), ("context_lens", context_lens, (rows,)),
                               ("free_state", free_state, (2,))):
            if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"StepTables.build: {name} must be int32 {list(shape)}, contiguous and on {dev}")
        if (free_ids.dtype != torch.int32 or free_ids.dim() != 1 or free_ids.numel() == 0
                or not free_ids.is_contiguous() or free_ids.device != dev):
            raise ValueError(f"StepTables.build: free_ids must be a non-empty int32 vector, contiguous and on {dev}")
        raise ValueError(f"StepTables.build: block_table must be int32 [{rows}, max_blocks >= 1] on {dev} with unit "
                         "column stride and rows that do not overlap")
