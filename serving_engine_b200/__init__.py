"""B200 (sm_100a) paged-KV attention backend for the serving engine.

Public API mirrors the reference's hot-path modules:

* ``paged_flash_attention`` / ``build_paged_batch_metadata``
  (serving_engine/paged_attention_kernel.py)
* ``PagedKVCache`` (serving_engine/model_runner.py:_PagedKVCache) and the
  attention function registered as ``"paged|b200"``
* tensor ops ``kv_append``, ``copy_blocks``, ``paged_decode``, ``paged_prefill``
  over the C ABI in include/serving_engine_b200.h, and the decode-layer fusions
  ``rope_kv_append``, ``add_rmsnorm``, ``swiglu`` used by the tensor-parallel
  decoder;
* a KV pool held in 4 bits: ``new_q4_pool``, ``kv_append_q4``, ``kv_gather_q4``,
  ``qk_norm_rope_append`` (head norms, rotary embedding and the write to a 4-bit or
  16-bit pool), ``paged_attention_q4`` (``paged_flash_attention``, ``PagedKVCache`` and
  the registered attention function take such a pool as well), and ``StepTables``, a
  step's tables built on the GPU; ``q4_serve.Q4Batch`` runs a model with all of them.

Importing the package does not load the CUDA library; the first op does, and
raises if it has not been built (``python -m serving_engine_b200.build``).
"""
from .kv_cache import PAGED_B200_ATTN_IMPL, PagedKVCache, b200_paged_attention_forward, register
from .ops import (add_rmsnorm, check_device_errors, copy_blocks, kv_append, paged_decode, paged_prefill,
                  rope_kv_append, swiglu)
from .paged_attention import (PAGED_K_TILE_SIZE, PAGED_Q_TILE_SIZE, build_paged_batch_metadata,
                              metadata_from_lists, paged_flash_attention)
from .q4 import kv_append_q4, kv_gather_q4, new_q4_pool, paged_attention_q4, qk_norm_rope_append
from .step_tables import StepTables

__all__ = [
    "PAGED_B200_ATTN_IMPL",
    "PAGED_K_TILE_SIZE",
    "PAGED_Q_TILE_SIZE",
    "PagedKVCache",
    "StepTables",
    "add_rmsnorm",
    "b200_paged_attention_forward",
    "build_paged_batch_metadata",
    "check_device_errors",
    "copy_blocks",
    "kv_append",
    "kv_append_q4",
    "kv_gather_q4",
    "metadata_from_lists",
    "new_q4_pool",
    "paged_attention_q4",
    "paged_decode",
    "paged_flash_attention",
    "paged_prefill",
    "qk_norm_rope_append",
    "register",
    "rope_kv_append",
    "swiglu",
]
