"""The 4-bit KV pool: its tensors, and the ops that write it, read it and attend over it.

One layer of the pool is two uint8 planes (K and V) of shape [num_blocks, kv heads,
9 * head_dim]; ``new_q4_pool`` makes the pool of a model, [layers, 2, num_blocks, kv
heads, 9 * head_dim]. Every 64 values of a token's head share a scale and a lowest
value in fp16 and take 4 bits each, 4.5 bits in all: 3.6 times the tokens of a 16-bit
pool, and as much less to read in a decode step. include/serving_engine_b200.h states
what each call computes and csrc/q4_format.cuh the order of the bytes.

The ops follow ``ops``: shapes, dtypes and devices are checked on the host without a
sync, work goes to the current stream, out-of-range indices met at run time are
reported by ``check_device_errors``. bf16 and fp16, head_dim 64, 128 and 256.
"""
from __future__ import annotations

import functools
import itertools
import threading
import weakref

import torch

from . import ops
from ._lib import Q4_COUNTER_SLOTS, SEB_BF16, SEB_F16, check, lib
from .ops import BLOCK_SIZE, LAUNCHES, _nvtx, dtype_code, err_word

HEAD_DIMS = (64, 128, 256)
_HALF = {torch.bfloat16: SEB_BF16, torch.float16: SEB_F16}


def row_bytes(head_dim: int) -> int:
    """Bytes of one kv head of one block in one plane: 8 * head_dim of codes, head_dim of (scale, low) pairs."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"4-bit KV pool: head_dim {head_dim} not supported {HEAD_DIMS}")
    return 9 * head_dim


def new_q4_pool(num_layers: int, num_blocks: int, num_kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A zeroed 4-bit pool for a model: uint8 [layers, 2, num_blocks, kv heads, 9 * head_dim]."""
    return torch.zeros(num_layers, 2, num_blocks, num_kv_heads, row_bytes(head_dim), dtype=torch.uint8, device=device)


# A stream's workspace and counter slot on a device (or a Workspace's, under a negative number). Slots are handed out under the lock, and one at a
# time: two calls that overlap on the GPU with one slot would join sums that are not complete. A workspace
# that a larger call outgrew stays allocated: a captured CUDA graph may hold its address.
_lock = threading.Lock()
_slots: dict[tuple[int, int], int] = {}
_workspaces: dict[tuple[int, int], tuple[torch.Tensor, int]] = {}
_retired: list[torch.Tensor] = []
_own = threading.local()  # .key: the Workspace that this thread's calls use
_own_keys = itertools.count(1)
_gone: list[int] = []  # Workspaces that are no more
_idle: dict[int, list[int]] = {}  # by device: slots that they left


class Workspace:
    """A workspace and counters of its own: calls that a thread issues ``with`` it use these and not their
    stream's. For a CUDA graph, which holds those of its capture and may be replayed beside other calls and
    other graphs of the same capture stream. Keep it as long as the graph."""

    def __init__(self):
        self._key = -next(_own_keys)
        weakref.finalize(self, _gone.append, self._key)

    def __enter__(self):
        _own.outer = (getattr(_own, "key", None), getattr(_own, "outer", None))
        _own.key = self._key
        return self

    def __exit__(self, *exc):
        _own.key, _own.outer = _own.outer


def _slot(device: int, stream: int) -> int:
    with _lock:
        while _gone:
            key = _gone.pop()
            for at in [at for at in _slots if at[1] == key]:
                _idle.setdefault(at[0], []).append(_slots.pop(at))
                _workspaces.pop(at, None)
        slot = _slots.get((device, stream))
        if slot is None:
            idle = _idle.get(device, [])
            taken = {s for (d, _), s in _slots.items() if d == device}.union(idle)
            slot = next((s for s in range(Q4_COUNTER_SLOTS) if s not in taken), None)
            if slot is None and idle:
                torch.cuda.synchronize(device)  # the last calls of the one that left it may still run
                slot = idle.pop()
            if slot is None:
                raise RuntimeError(f"paged_attention_q4: all {Q4_COUNTER_SLOTS} counter slots of device {device} belong to "
                                   "streams and Workspaces; issue the calls on fewer streams")
            _slots[device, stream] = slot
    return slot


def _workspace(device: int, stream: int, nbytes: int) -> tuple[torch.Tensor, int]:
    """The stream's own workspace and counters, so calls on different streams may overlap."""
    held = _workspaces.get((device, stream))
    if held is None or held[0].numel() < nbytes:
        slot = _slot(device, stream)
        with torch.inference_mode(False):
            ws = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device))
        with _lock:
            held = _workspaces.get((device, stream))
            if held is None or held[0].numel() < nbytes:
                if held is not None:
                    _retired.append(held[0])
                held = _workspaces[device, stream] = (ws, slot)
    return held


@functools.lru_cache(maxsize=4096)
def _attention_workspace_bytes(device: int, rows: int, total_query: int, num_q_heads: int, num_kv_heads: int,
                               head_dim: int) -> int:
    """By device: the library's answer depends on the device's SMs."""
    return int(lib().seb_paged_attention_q4_workspace_size(rows, total_query, num_q_heads, num_kv_heads, head_dim))


# The host's part of a call is what a small call costs, so the checks below read each
# attribute once and only work out a message when something is wrong.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _device(name: str, *tensors: torch.Tensor) -> int:
    """The index of the CUDA device that all the tensors are on."""
    device = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != device or device < 0:
            ops._require_cuda(name, *tensors)
    return device


def _half(name: str, *tensors: torch.Tensor) -> int:
    """The code of the 16-bit dtype that all the tensors have."""
    dtype = tensors[0].dtype
    for t in tensors:
        if t.dtype != dtype or dtype not in _HALF:
            ops._half_dtype(name, *tensors)
    return _HALF[dtype]


def _err_ptr(device: int) -> int:
    word = ops._err_words.get(device)
    return (err_word(torch.device("cuda", device)) if word is None else word).data_ptr()


def _done(name: str, status: int, device: int, launches: int = 1) -> None:
    if status:
        check(name, status)
    LAUNCHES[0] += launches
    if ops.DEBUG:
        ops._after(torch.device("cuda", device))


def _check_planes(name: str, k_cache: torch.Tensor, v_cache: torch.Tensor, num_kv_heads: int, head_dim: int) -> None:
    shape = k_cache.shape
    if (head_dim in HEAD_DIMS and len(shape) == 3 and shape[1] == num_kv_heads and shape[2] == 9 * head_dim
            and k_cache.dtype == v_cache.dtype == torch.uint8 and v_cache.shape == shape and k_cache.is_contiguous()
            and v_cache.is_contiguous()):
        return
    want = row_bytes(head_dim)
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise ValueError(f"{name}: a 4-bit pool is uint8, got {k_cache.dtype} and {v_cache.dtype}")
    if len(shape) != 3 or shape[1] != num_kv_heads or shape[2] != want:
        raise ValueError(f"{name}: k_cache must be [num_blocks, {num_kv_heads}, {want}], got {tuple(shape)}")
    raise ValueError(f"{name}: k_cache and v_cache must be contiguous and of equal shape")


def _aligned(t: torch.Tensor) -> bool:
    """Whether a [tokens, heads, head_dim] tensor's rows are 16-byte aligned."""
    token, head, _ = t.stride()
    return t.data_ptr() % 16 == 0 and token % 8 == 0 and head % 8 == 0


def _check_slots(name: str, slots: torch.Tensor, n: int) -> torch.Tensor:
    if slots.dtype != torch.int64 or slots.shape != (n,):
        raise ValueError(f"{name}: slot_mapping must be int64 [{n}]")
    return slots if slots.is_contiguous() else slots.contiguous()


@_nvtx
def kv_append_q4(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slot_mapping: torch.Tensor) -> None:
    """``kv_append`` into a 4-bit pool: quantises k_new, v_new [n_tokens, H, D] (unit
    stride on D, any token and head strides) into the slots slot_mapping, int64
    [n_tokens], of the planes k_cache, v_cache [num_blocks, H, 9 * D]. One launch."""
    device = _device("kv_append_q4", k_new, v_new, k_cache, v_cache, slot_mapping)
    dt = _half("kv_append_q4", k_new, v_new)
    if k_new.dim() != 3 or v_new.shape != k_new.shape:
        raise ValueError(f"kv_append_q4: k_new/v_new must both be [n_tokens, H, D], got {tuple(k_new.shape)} "
                         f"and {tuple(v_new.shape)}")
    n, h, d = k_new.shape
    _check_planes("kv_append_q4", k_cache, v_cache, h, d)
    ks, vs = k_new.stride(), v_new.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("kv_append_q4: new K/V must have unit stride on head_dim")
    slot_mapping = _check_slots("kv_append_q4", slot_mapping, n)
    if n == 0:
        return
    st = lib().seb_kv_append_q4(
        k_new.data_ptr(), ks[0], ks[1], v_new.data_ptr(), vs[0], vs[1], n, slot_mapping.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), k_cache.shape[0], h, d, dt, _err_ptr(device), _raw_stream(device))
    _done("seb_kv_append_q4", st, device)


@_nvtx
def kv_gather_q4(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V values that the pool's slots (int64 [n]) stand for, each [n, kv heads,
    head_dim] of ``dtype`` (fp32, fp16 or bf16; computed in fp32, rounded once). One launch."""
    device = _device("kv_gather_q4", k_cache, v_cache, slots)
    if k_cache.dim() != 3:
        raise ValueError(f"kv_gather_q4: k_cache must be [num_blocks, kv heads, 9 * head_dim], got {tuple(k_cache.shape)}")
    blocks, h, _ = k_cache.shape
    n = slots.numel()
    _check_planes("kv_gather_q4", k_cache, v_cache, h, head_dim)
    slots = _check_slots("kv_gather_q4", slots, n)
    kv = k_cache.new_empty((2, n, h, head_dim), dtype=dtype)
    dt = dtype_code(kv)
    k, v = kv.unbind(0)
    if n == 0:
        return k, v
    st = lib().seb_kv_gather_q4(k_cache.data_ptr(), v_cache.data_ptr(), blocks, h, head_dim, slots.data_ptr(), n,
                                k.data_ptr(), v.data_ptr(), dt, _err_ptr(device), _raw_stream(device))
    _done("seb_kv_gather_q4", st, device)
    return k, v


@_nvtx
def qk_norm_rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, slot_mapping: torch.Tensor,
                        k_cache: torch.Tensor, v_cache: torch.Tensor, num_q_heads: int, num_kv_heads: int,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm of every query and key head, the rotary embedding and the KV write in one
    launch: returns q [n_tokens, num_q_heads, head_dim] and writes K and V of token t to
    slot slot_mapping[t] of a 16-bit pool ([num_blocks, 16, kv heads, head_dim] of qkv's
    dtype) or of a 4-bit one (uint8 [num_blocks, kv heads, 9 * head_dim]).

    qkv: [n_tokens, (num_q_heads + 2 * num_kv_heads) * head_dim], q heads, then k, then v;
    cos/sin: [n_tokens, head_dim] (any leading views that flatten to that); q_weight,
    k_weight: [head_dim] norm weights, None where the model has no such norm. Computed in
    fp32 and rounded once (rope_kv_append rounds every product as the eager ops do).
    """
    name = "qk_norm_rope_append"
    weights = [w for w in (q_weight, k_weight) if w is not None]
    device = _device(name, qkv, cos, sin, slot_mapping, k_cache, v_cache, *weights)
    q4_pool = k_cache.dtype == torch.uint8
    if v_cache.dtype != k_cache.dtype:
        raise ValueError(f"{name}: k_cache must be of v_cache's dtype, got {k_cache.dtype} and {v_cache.dtype}")
    dt = _half(name, qkv, cos, sin, *weights) if q4_pool else _half(name, qkv, cos, sin, k_cache, *weights)
    if qkv.dim() != 2 or qkv.stride(1) != 1:
        raise ValueError(f"{name}: qkv must be [n_tokens, width] with unit column stride")
    (n, width), d = qkv.shape, cos.shape[-1]
    if d not in HEAD_DIMS:
        raise ValueError(f"{name}: head_dim {d} not supported {HEAD_DIMS}")
    if num_q_heads <= 0 or num_kv_heads <= 0 or width != (num_q_heads + 2 * num_kv_heads) * d:
        raise ValueError(f"{name}: qkv width {width} != ({num_q_heads} + 2 x {num_kv_heads}) x {d}")
    if q4_pool:
        _check_planes(name, k_cache, v_cache, num_kv_heads, d)
    else:
        if k_cache.dim() != 4 or tuple(k_cache.shape[1:]) != (BLOCK_SIZE, num_kv_heads, d):
            raise ValueError(f"{name}: k_cache must be [num_blocks, {BLOCK_SIZE}, {num_kv_heads}, {d}], "
                             f"got {tuple(k_cache.shape)}")
        if v_cache.shape != k_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
            raise ValueError(f"{name}: k_cache and v_cache must be contiguous and of equal shape")
    if cos.dim() != 2:
        cos = cos.reshape(-1, d)
    if sin.dim() != 2:
        sin = sin.reshape(-1, sin.shape[-1])
    cs = cos.stride()
    if cos.shape != (n, d) or sin.shape != (n, d) or sin.stride() != cs or cs[1] != 1:
        raise ValueError(f"{name}: cos and sin must be [n_tokens={n}, head_dim={d}] with equal strides")
    for what, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or not w.is_contiguous()):
            raise ValueError(f"{name}: {what} must be [{d}] and contiguous")
    slot_mapping = _check_slots(name, slot_mapping, n)
    if out is None:
        out = qkv.new_empty((n, num_q_heads, d))
    elif (out.shape != (n, num_q_heads, d) or out.stride(2) != 1 or out.stride(1) != d or out.dtype != qkv.dtype
          or out.get_device() != device):
        raise ValueError(f"{name}: out must be [n_tokens, num_q_heads, head_dim] of qkv's dtype and device "
                         "with contiguous heads")
    if n == 0:
        return out
    st = lib().seb_qk_norm_rope_append(
        qkv.data_ptr(), qkv.stride(0), n, num_q_heads, num_kv_heads, d, cos.data_ptr(), sin.data_ptr(), cs[0],
        None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
        slot_mapping.data_ptr(), out.data_ptr(), out.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
        k_cache.shape[0], 4 if q4_pool else 16, dt, _err_ptr(device), _raw_stream(device))
    _done("seb_qk_norm_rope_append", st, device)
    return out


def _refuse_attention(q, block_table, arrays, rows, num_q_heads, num_kv_heads, out, lse):
    """Says what is wrong with paged_attention_q4's arguments; returns if nothing is."""
    name = "paged_attention_q4"
    if q.dim() != 3 or q.stride(2) != 1 or q.shape[1] != num_q_heads:
        raise ValueError(f"{name}: q must be [total_query, {num_q_heads}, head_dim] with unit inner stride, "
                         f"got {tuple(q.shape)}")
    if num_kv_heads <= 0 or num_q_heads % num_kv_heads:
        raise ValueError(f"{name}: num_q_heads {num_q_heads} not a multiple of num_kv_heads {num_kv_heads}")
    for what, t in zip(("q_starts", "q_lens", "k_lens", "q_pos_offsets"), arrays):
        if t.dtype != torch.int32 or t.shape != (rows,) or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be int32 [{rows}] and contiguous")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != rows:
        raise ValueError(f"{name}: block_table must be int32 [{rows}, max_blocks], got {tuple(block_table.shape)}")
    device = q.get_device()
    if out is not None and (out.shape != q.shape or out.stride(2) != 1 or out.dtype != q.dtype or out.get_device() != device):
        raise ValueError(f"{name}: out must match q, with unit stride on head_dim")
    if lse is not None and (lse.shape != (q.shape[0], num_q_heads) or lse.dtype != torch.float32 or lse.stride(1) != 1
                            or lse.get_device() != device):
        raise ValueError(f"{name}: lse must be fp32 [{q.shape[0]}, {num_q_heads}] with unit column stride")


@_nvtx
def paged_attention_q4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                       q_starts: torch.Tensor, q_lens: torch.Tensor, k_lens: torch.Tensor,
                       q_pos_offsets: torch.Tensor, num_q_heads: int, num_kv_heads: int, scale: float,
                       is_causal: bool = True, out: torch.Tensor | None = None,
                       lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Paged attention over a 4-bit pool for rows of any length (decode rows, drafted
    tokens, prefill chunks, mixed): (out like q, lse fp32 [total_query, num_q_heads]).

    q: [total_query, num_q_heads, D] with unit stride on D; the planes as in
    ``kv_append_q4``; block_table int32 [rows, max_blocks]; the other arrays int32 [rows].
    A query that sees no key gets 0 and -inf; tokens of no row keep what out held.

    Every stream has its own workspace and counters: calls on different streams may overlap
    (on 128 streams of a device; a call on one more raises RuntimeError). A CUDA
    graph holds the workspace of the stream it was captured on; graphs captured on one
    stream must not be replayed at the same time, nor beside calls on that stream, unless
    each is captured ``with`` a ``q4.Workspace`` of its own.
    """
    arrays = (q_starts, q_lens, k_lens, q_pos_offsets)
    device = _device("paged_attention_q4", q, k_cache, v_cache, block_table, *arrays)
    dt = _half("paged_attention_q4", q)
    rows = q_starts.numel()
    _refuse_attention(q, block_table, arrays, rows, num_q_heads, num_kv_heads, out, lse)
    total_q, _, d = q.shape
    _check_planes("paged_attention_q4", k_cache, v_cache, num_kv_heads, d)
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    if not _aligned(q):
        q = q.contiguous()
        if not _aligned(q):
            q = q.clone()
    if out is None:
        out = q.new_empty((total_q, num_q_heads, d))
    if lse is None:
        lse = q.new_empty((total_q, num_q_heads), dtype=torch.float32)
    max_blocks = block_table.shape[1]
    if rows == 0 or total_q == 0:
        return out, lse
    if max_blocks == 0:  # no row has a key
        out.zero_()
        lse.fill_(float("-inf"))
        return out, lse
    result = out
    if not _aligned(out):
        out = result.clone(memory_format=torch.contiguous_format)
    stream = _raw_stream(device)
    ws, slot = _workspace(device, getattr(_own, "key", None) or stream,
                          _attention_workspace_bytes(device, rows, total_q, num_q_heads, num_kv_heads, d))
    qs, os = q.stride(), out.stride()
    st = lib().seb_paged_attention_q4(
        q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0],
        block_table.data_ptr(), block_table.stride(0), max_blocks, q_starts.data_ptr(), q_lens.data_ptr(),
        k_lens.data_ptr(), q_pos_offsets.data_ptr(), rows, total_q, num_q_heads, num_kv_heads, d, dt, scale,
        1 if is_causal else 0, out.data_ptr(), os[0], os[1], lse.data_ptr(), lse.stride(0), ws.data_ptr(), ws.numel(),
        slot, _err_ptr(device), stream)
    # rows of many tokens have their own kernel
    _done("seb_paged_attention_q4", st, device, 2 if total_q > rows and d <= 128 else 1)
    if result is not out:
        result.copy_(out)
    return result, lse
