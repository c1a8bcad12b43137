"""The 4-bit paged K/V cache: block plan, rows in and out, attention.

A pool is a uint8 tensor [blocks, kv_heads, 36 * head_dim] (:func:`kv4_pool`):
32-token blocks at 4.5 bits an element, against 16 in the FP16 pool of
:class:`DecodeContext`. A serving step with it:

    slots, positions, cu = plan_blocks(add, seq_lens, block_table, free_list, free_top, tokens)
    for each layer:                                  # one pool a layer, one plan for all
        pack_kv4(pool, key, value, slots)            # the step's rows
        out = attention_kv4(query, pool, block_table, seq_lens)

:func:`unpack_kv4` reads rows back (a cached prefix for the next chunk of its
prompt). All calls are asynchronous on the current stream of the tensors'
device, never synchronise or copy to the host, and can be captured in a CUDA
graph. A ``status`` word (int32 [1], optional) collects the SA_DEV_* bits that
the kernels raise; the formats and rules stand in include/sa_b200.h.
"""
from __future__ import annotations

import functools
import math

import torch

from ._lib import SA_TYPE_BF16, SA_TYPE_F16, SA_TYPE_F32, check, load

_TYPES = {torch.float32: SA_TYPE_F32, torch.float16: SA_TYPE_F16, torch.bfloat16: SA_TYPE_BF16}


def _tensor(t, dtype, dim, name, index=None) -> int:
    """The address of a contiguous CUDA tensor of the given type and rank (on
    device `index`)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with {dim} dimension(s)")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    return t.data_ptr()


def _rows(t, dim, name, index) -> int:
    """The address of a CUDA tensor whose last axis is contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.dim() != dim or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} must have {dim} dimensions, the last one contiguous")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    return t.data_ptr()


def _status(status, index):
    return None if status is None else _tensor(status, torch.int32, 1, "status", index)


def _public_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The current stream's handle without a Stream object around it (0.1 us, not 2.2).
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _call(index, what, fn, *args) -> None:
    """fn(*args, stream) with the current stream of device `index`, made current for the call."""
    if index == torch.cuda.current_device():
        status = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _stream_of(index))
    if status:
        check(status, what)


def _pool_dims(pool) -> tuple[int, int, int, int]:
    """(address, blocks, KV heads, head_dim) of a pool tensor."""
    ptr = _tensor(pool, torch.uint8, 3, "pool")
    blocks, heads, nbytes = pool.shape
    if nbytes % 36:
        raise ValueError("pool must be [blocks, kv_heads, 36 * head_dim]")
    return ptr, blocks, heads, nbytes // 36


def kv4_pool(blocks: int, kv_heads: int, head_dim: int = 128, device=None) -> torch.Tensor:
    """A zeroed pool of `blocks` 32-token blocks (every slot holds zero rows)."""
    nbytes = load().sa_kv4_entry_bytes(head_dim)
    if nbytes == 0:
        raise ValueError("head_dim must be 64, 128 or 256")
    return torch.zeros(blocks, kv_heads, nbytes, dtype=torch.uint8,
                       device="cuda" if device is None else device)


def plan_blocks(add: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
                free_list: torch.Tensor, free_top: torch.Tensor, max_tokens: int,
                status: torch.Tensor | None = None
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Grow and shrink a batch's requests by ``add`` tokens each (int32 [requests]).

    ``seq_lens`` [requests], ``block_table`` [requests, blocks], ``free_list``
    [pool blocks] and ``free_top`` [1] (int32) are the state, changed in place.
    Returns (slots [max_tokens], positions [max_tokens], cu_tokens [requests +
    1]): the slots and positions of the new tokens request by request, -1 and 0
    behind the last, and each request's first row. A request whose growth does
    not fit is left as it was, its slots are -1 and a status bit is set; those
    that shrink or end always do (sa_plan_blocks). A batch without requests is
    an empty plan.
    """
    ptr = _tensor(add, torch.int32, 1, "add")
    dev = add.get_device()
    n = add.shape[0]
    lens = _tensor(seq_lens, torch.int32, 1, "seq_lens", dev)
    table = _tensor(block_table, torch.int32, 2, "block_table", dev)
    free = _tensor(free_list, torch.int32, 1, "free_list", dev)
    top = _tensor(free_top, torch.int32, 1, "free_top", dev)
    if seq_lens.shape[0] != n or block_table.shape[0] != n or free_top.shape[0] != 1:
        raise ValueError("add, seq_lens and block_table must have a row a request, free_top one element")
    if max_tokens < 0:
        raise ValueError("max_tokens must not be negative")
    if n == 0:  # an idle batch
        _status(status, dev)
        return add.new_full((max_tokens,), -1), add.new_zeros(max_tokens), add.new_zeros(1)
    slots, positions, cu = add.new_empty(max_tokens), add.new_empty(max_tokens), add.new_empty(n + 1)
    _call(dev, "plan_blocks", load().sa_plan_blocks, ptr, n, lens, table, block_table.shape[1], free,
          free_list.shape[0], top, max_tokens, slots.data_ptr(), positions.data_ptr(), cu.data_ptr(),
          _status(status, dev))
    return slots, positions, cu


def pack_kv4(pool: torch.Tensor, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor,
             status: torch.Tensor | None = None) -> None:
    """Quantise rows ``key`` and ``value`` [tokens, kv_heads, head_dim] (one type
    of float32, float16, bfloat16; any strides along tokens and heads) into
    ``slots`` [tokens] int32 of ``pool``; rows with a negative slot are skipped
    (sa_pack_kv4)."""
    ptr, blocks, heads, d = _pool_dims(pool)
    dev = pool.get_device()
    k, v = _rows(key, 3, "key", dev), _rows(value, 3, "value", dev)
    at = _tensor(slots, torch.int32, 1, "slots", dev)
    tokens = slots.shape[0]
    if key.shape != (tokens, heads, d) or value.shape != key.shape or key.dtype != value.dtype:
        raise ValueError(f"key and value must be [{tokens}, {heads}, {d}] of one type")
    _call(dev, "pack_kv4", load().sa_pack_kv4, ptr, blocks, k, v, _TYPES[key.dtype], key.stride(0),
          key.stride(1), value.stride(0), value.stride(1), at, tokens, heads, d,
          _status(status, dev))


def unpack_kv4(pool: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
               status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows held in ``slots`` [tokens] int32: (key, value) [tokens, kv_heads,
    head_dim] of ``dtype``, zeros where the slot is negative (sa_unpack_kv4)."""
    ptr, blocks, heads, d = _pool_dims(pool)
    dev = pool.get_device()
    at = _tensor(slots, torch.int32, 1, "slots", dev)
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    tokens = slots.shape[0]
    key = pool.new_empty((tokens, heads, d), dtype=dtype)
    value = key.new_empty((tokens, heads, d))
    _call(dev, "unpack_kv4", load().sa_unpack_kv4, ptr, blocks, at, tokens, heads, d, key.data_ptr(),
          value.data_ptr(), _TYPES[dtype], _status(status, dev))
    return key, value


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n, new, qh, heads, d, index) -> int:
    with torch.cuda.device(index):
        return load().sa_attention_kv4_workspace_size(n, new, qh, heads, d)


def attention_kv4(query: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, scale: float | None = None,
                  selected: torch.Tensor | None = None,
                  selected_count: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None, return_lse: bool = False,
                  status: torch.Tensor | None = None):
    """Attention of the newest tokens over a 4-bit pool.

    ``query`` [requests, query_heads, head_dim] (one new token each) or
    [requests, new_tokens, query_heads, head_dim]: float32, float16 or bfloat16,
    any strides but along head_dim. ``seq_lens`` [requests] count the new tokens;
    new token i of a request stands at ``seq_lens - new_tokens + i`` and sees
    what is not behind it. ``selected`` [requests, groups, budget] int32 with
    ``selected_count`` [requests, groups] restricts the attention to those
    logical blocks (ascending; as from select_shared_blocks) and the block of
    the newest token. Returns the output in the query's shape and type
    (``out_dtype`` for a float32 query), and with ``return_lse`` also the
    log-sum-exp of the logits, FP32, without head_dim (sa_attention_kv4). There
    is no backward pass: a query that requires grad is refused in grad mode.
    """
    ptr, blocks, heads, d = _pool_dims(pool)
    dev = pool.get_device()
    lead = 4 if isinstance(query, torch.Tensor) and query.dim() == 4 else 3
    q = _rows(query, lead, "query", dev)
    if query.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("attention_kv4 has no backward pass: call it under torch.no_grad() or detach the query")
    n, qh = query.shape[0], query.shape[-2]
    new = query.shape[1] if lead == 4 else 1
    table = _tensor(block_table, torch.int32, 2, "block_table", dev)
    lens = _tensor(seq_lens, torch.int32, 1, "seq_lens", dev)
    if query.shape[-1] != d or block_table.shape[0] != n or seq_lens.shape[0] != n:
        raise ValueError("query, block_table and seq_lens must have a row a request, and query the "
                         "pool's head_dim")
    ids = counts = None
    groups = budget = 0
    if selected is not None:
        ids = _tensor(selected, torch.int32, 3, "selected", dev)
        counts = _tensor(selected_count, torch.int32, 2, "selected_count", dev)
        _, groups, budget = selected.shape
        if selected.shape[0] != n or selected_count.shape != (n, groups):
            raise ValueError("selected must be [requests, groups, budget], selected_count [requests, groups]")
    elif selected_count is not None:
        raise ValueError("selected_count without selected")
    lib = load()
    out_dtype = query.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    shape = query.shape
    out = query.new_empty(shape, dtype=out_dtype)
    lse = query.new_empty(shape[:-1], dtype=torch.float32) if return_lse else None
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if n == 0:  # an idle batch
        _status(status, dev)
        return (out, lse) if return_lse else out
    if block_table.shape[1] == 0:  # no request holds a block: a column without one stands for it
        block_table = block_table.new_full((n, 1), -1)
        table = block_table.data_ptr()
    if selected is not None and budget == 0:  # lists without room: the block of the newest token alone
        selected, selected_count = seq_lens.new_zeros(n, groups, 1), seq_lens.new_zeros(n, groups)
        ids, counts, budget = selected.data_ptr(), selected_count.data_ptr(), 1
    ws_bytes = _workspace_bytes(n, new, qh, heads, d, dev)
    ws = pool.new_empty(ws_bytes or 16)
    _call(dev, "attention_kv4", lib.sa_attention_kv4, q, _TYPES[query.dtype], query.stride(0),
          query.stride(1) if lead == 4 else 0, query.stride(-2), ptr, blocks, table,
          block_table.shape[1], lens, ids, counts, groups, budget, n, new, qh, heads, d, scale,
          out.data_ptr(), _TYPES[out_dtype], None if lse is None else lse.data_ptr(), ws.data_ptr(),
          ws_bytes, _status(status, dev))
    return (out, lse) if return_lse else out
