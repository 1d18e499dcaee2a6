"""Serving attention: a paged K/V cache (block tables and slots, writes, attention
of new tokens over it) and attention to an encoder's states of another length.

No counterpart in the reference. As in the package: launch_* binds one C entry
point, takes tensors or device pointers and launches on `stream` (None: the
current one); the functions without launch_ take torch tensors, check them and
run on the current stream of the tensors' device. Forward only.

    cache = paged_cache(k_cache, v_cache)
    step = paged_slots(cached, new, block_table, free_blocks, block_size, max_tokens)
    paged_append(k, v, step.slot_map, cache)
    o = attention_paged(q, cache, block_table, step.query_starts, step.kv_lens, max_query_len)
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple, Optional

import cuda_fused_attention_amd as _fa

DTYPE_BF16 = 0
DTYPE_FP16 = 1


def _strides(value):
    """A (batch, head, row) tuple in elements as the struct; None: contiguous."""
    return None if value is None else ctypes.byref(_fa.Strides(*value))


class PagedCache:
    """The two tensors of a paged cache and the description of them that the C
    entry points take. Build it with paged_cache and keep it."""

    __slots__ = ("k", "v", "info", "ref", "dtype", "device", "num_blocks", "heads_kv", "block_size", "head_dim")

    def __init__(self, k, v, info):
        self.k, self.v, self.info, self.ref = k, v, info, ctypes.byref(info)
        self.dtype, self.device = k.dtype, k.device
        self.num_blocks, self.heads_kv, self.block_size, self.head_dim = k.shape


class PagedSlots(NamedTuple):
    """What paged_slots writes beside the block table."""

    query_starts: object  # int32 [num_seqs + 1]
    kv_lens: object       # int32 [num_seqs]
    slot_map: object      # int64 [max_tokens]
    blocks_taken: object  # int32 [1]


# ---------------------------------------------------------------- C entry points
def launch_paged_slots(cached_lens, new_lens, block_table, free_blocks, query_starts, kv_lens, slot_map, blocks_taken,
                       num_seqs: int, table_width: int, table_stride: int, num_free: int, block_size: int,
                       max_tokens: int, stream=None) -> bool:
    p = _fa._ptr
    st = _fa.lib().fa_launch_paged_slots(p(cached_lens), p(new_lens), p(block_table), p(free_blocks), p(query_starts),
                                         p(kv_lens), p(slot_map), p(blocks_taken), num_seqs, table_width, table_stride,
                                         num_free, block_size, max_tokens, _fa._stream(stream))
    return _fa._check(st, "fa_launch_paged_slots")


def launch_paged_append(k, v, slot_map, cache: PagedCache, tokens: int, k_strides=None, v_strides=None,
                        stream=None) -> bool:
    p = _fa._ptr
    st = _fa.lib().fa_launch_paged_append(p(k), p(v), p(slot_map), cache.ref, tokens, _strides(k_strides),
                                          _strides(v_strides), _fa._stream(stream))
    return _fa._check(st, "fa_launch_paged_append")


def attention_paged_workspace_bytes(tokens: int, num_seqs: int, heads: int, heads_kv: int, head_dim: int,
                                    max_query_len: int, max_kv_len: int) -> int:
    return int(_fa.lib().fa_attention_paged_workspace_bytes(tokens, num_seqs, heads, heads_kv, head_dim, max_query_len,
                                                            max_kv_len))


def _config(call, *sizes):
    rows, splits = ctypes.c_int(), ctypes.c_int()
    if not _fa._check(getattr(_fa.lib(), call)(*sizes, ctypes.byref(rows), ctypes.byref(splits)), call):
        return None
    return rows.value, splits.value


def attention_paged_config(tokens: int, num_seqs: int, heads: int, heads_kv: int, head_dim: int, max_query_len: int,
                           max_kv_len: int):
    """(rows per workgroup, most chunks of a sequence's keys), or None for an
    unsupported head_dim."""
    return _config("fa_attention_paged_config", tokens, num_seqs, heads, heads_kv, head_dim, max_query_len, max_kv_len)


def launch_attention_paged(q, cache: PagedCache, o, workspace, workspace_bytes: int, block_table, query_starts, kv_lens,
                           num_seqs: int, tokens: int, heads: int, table_width: int, table_stride: int,
                           max_query_len: int, max_kv_len: int, causal: bool, q_strides=None, o_strides=None,
                           stream=None) -> bool:
    p = _fa._ptr
    st = _fa.lib().fa_launch_attention_paged(p(q), cache.ref, p(o), p(workspace), workspace_bytes, p(block_table),
                                             p(query_starts), p(kv_lens), num_seqs, tokens, heads, table_width,
                                             table_stride, max_query_len, max_kv_len, int(causal), _strides(q_strides),
                                             _strides(o_strides), _fa._stream(stream))
    return _fa._check(st, "fa_launch_attention_paged")


def attention_cross_workspace_bytes(batch: int, heads: int, heads_kv: int, q_len: int, kv_len: int, head_dim: int) -> int:
    return int(_fa.lib().fa_attention_cross_workspace_bytes(batch, heads, heads_kv, q_len, kv_len, head_dim))


def attention_cross_config(batch: int, heads: int, heads_kv: int, q_len: int, kv_len: int, head_dim: int):
    """As attention_paged_config."""
    return _config("fa_attention_cross_config", batch, heads, heads_kv, q_len, kv_len, head_dim)


def launch_attention_cross(q, k, v, o, workspace, workspace_bytes: int, kv_lens, batch: int, heads: int, heads_kv: int,
                           q_len: int, kv_len: int, head_dim: int, dtype: int, q_strides=None, k_strides=None,
                           v_strides=None, o_strides=None, stream=None) -> bool:
    p = _fa._ptr
    st = _fa.lib().fa_launch_attention_cross(p(q), p(k), p(v), p(o), p(workspace), workspace_bytes, p(kv_lens), batch,
                                             heads, heads_kv, q_len, kv_len, head_dim, dtype, _strides(q_strides),
                                             _strides(k_strides), _strides(v_strides), _strides(o_strides),
                                             _fa._stream(stream))
    return _fa._check(st, "fa_launch_attention_cross")


# ---------------------------------------------------------------- torch convenience
def _dtype_id(dtype) -> int:
    import torch

    if dtype == torch.bfloat16:
        return DTYPE_BF16
    if dtype == torch.float16:
        return DTYPE_FP16
    raise ValueError(f"bf16 or fp16 tensors are needed, not {dtype}")


def _on(device):
    """The context in which `device` is the current one."""
    import torch

    if device.type != "cuda":
        raise ValueError("CUDA tensors are needed")
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _int32(x, name: str, shape, device):
    """`x` is a contiguous int32 tensor of this shape on this device."""
    import torch

    _need(x.dtype == torch.int32 and x.device == device and tuple(x.shape) == shape and x.is_contiguous(),
          f"{name} must be a contiguous int32 tensor {list(shape)} on {device}")


def _table(block_table, num_seqs, device):
    """(width, row stride) of a block table."""
    import torch

    _need(block_table.dtype == torch.int32 and block_table.device == device and block_table.dim() == 2
          and block_table.shape[0] == num_seqs, f"block_table must be an int32 tensor [{num_seqs}, width] on {device}")
    width = block_table.shape[1]
    stride = block_table.stride(0) if num_seqs > 1 else max(width, 1)
    _need(width <= 1 or block_table.stride(1) == 1, "block_table rows must be contiguous")
    _need(stride >= width, "block_table rows must not overlap")
    return width, stride


def _stride(x, dim: int) -> int:
    """The distance along `dim`; where it has one entry, whose stride means nothing,
    one row."""
    return x.stride(dim) if x.shape[dim] > 1 else x.shape[-1]


def _row_strides(x, name: str):
    """Strides (0, head, row) of a [rows, heads, dim] tensor."""
    _need(x.stride(2) == 1, f"{name}: head_dim must be contiguous")
    return 0, _stride(x, 1), _stride(x, 0)


def _head_strides(x, name: str):
    """Strides (batch, head, row) of a [batch, heads, rows, dim] tensor."""
    _need(x.stride(3) == 1, f"{name}: head_dim must be contiguous")
    return _stride(x, 0), _stride(x, 1), _stride(x, 2)


def paged_cache(k_cache, v_cache) -> PagedCache:
    """A cache of two tensors [num_blocks, heads_kv, block_size, head_dim] (bf16 or
    fp16, equal strides, head_dim contiguous). Pages that hold their tokens' heads
    side by side, [num_blocks, block_size, heads_kv, head_dim], come as
    .transpose(1, 2)."""
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "k_cache, v_cache: [num_blocks, heads_kv, block_size, head_dim]")
    _need(k_cache.dtype == v_cache.dtype and k_cache.device == v_cache.device, "k_cache and v_cache differ in type or device")
    _need(k_cache.is_cuda, "CUDA tensors are needed")
    _need(k_cache.stride(3) == 1 and v_cache.stride(3) == 1
          and all(_stride(k_cache, d) == _stride(v_cache, d) for d in range(3)),
          "k_cache and v_cache must have equal strides, head_dim contiguous")
    num_blocks, heads_kv, block_size, head_dim = k_cache.shape
    block, head, token = (_stride(k_cache, d) for d in range(3))
    info = _fa.PagedCacheInfo(k_cache.data_ptr(), v_cache.data_ptr(), block, head, token, num_blocks, heads_kv, block_size,
                              head_dim, _dtype_id(k_cache.dtype))
    return PagedCache(k_cache, v_cache, info)


def paged_slots_buffers(num_seqs: int, max_tokens: int, device="cuda") -> PagedSlots:
    """Buffers that paged_slots can write again and again (`out`)."""
    import torch

    def ints(n, dtype=torch.int32):
        return torch.empty(n, dtype=dtype, device=device)

    return PagedSlots(ints(num_seqs + 1), ints(num_seqs), ints(max_tokens, torch.int64), ints(1))


def paged_slots(cached_lens, new_lens, block_table, free_blocks, block_size: int, max_tokens: int,
                out: Optional[PagedSlots] = None) -> PagedSlots:
    """Block tables and slot maps from request lengths: sequence s holds
    cached_lens[s] tokens and gets new_lens[s] more. Entries of block_table
    [num_seqs, width] for the blocks that the new tokens open are taken from
    free_blocks, in order; every new token gets its slot in slot_map (-1: none).
    All int32; what happens at the ends is written at fa_launch_paged_slots."""
    import torch

    device = cached_lens.device
    _need(cached_lens.dim() == 1 and free_blocks.dim() == 1, "cached_lens and free_blocks must be vectors")
    num_seqs = cached_lens.shape[0]
    _int32(cached_lens, "cached_lens", (num_seqs,), device)
    _int32(new_lens, "new_lens", (num_seqs,), device)
    _int32(free_blocks, "free_blocks", (free_blocks.shape[0],), device)
    width, stride = _table(block_table, num_seqs, device)
    with _on(device):
        if out is None:
            out = paged_slots_buffers(num_seqs, max_tokens, device)
        _int32(out.query_starts, "query_starts", (num_seqs + 1,), device)
        _int32(out.kv_lens, "kv_lens", (num_seqs,), device)
        _int32(out.blocks_taken, "blocks_taken", (1,), device)
        slots = out.slot_map
        _need(slots.dtype == torch.int64 and slots.device == device and tuple(slots.shape) == (max_tokens,)
              and slots.is_contiguous(), f"slot_map must be a contiguous int64 tensor [{max_tokens}] on {device}")
        launch_paged_slots(cached_lens, new_lens, block_table, free_blocks, out.query_starts, out.kv_lens, slots,
                           out.blocks_taken, num_seqs, width, stride, free_blocks.shape[0], block_size, max_tokens)
    return out


def paged_append(k, v, slot_map, cache: PagedCache) -> None:
    """New rows k, v [tokens, heads_kv, head_dim] into the cache's slots slot_map
    (int64 [tokens]; negative or past the cache: skipped)."""
    import torch

    shape = (slot_map.shape[0], cache.heads_kv, cache.head_dim)
    for x, name in ((k, "k"), (v, "v")):
        _need(tuple(x.shape) == shape and x.dtype == cache.dtype and x.device == cache.device,
              f"{name} must be a {cache.dtype} tensor {list(shape)} on {cache.device}")
    _need(slot_map.dtype == torch.int64 and slot_map.device == cache.device and slot_map.dim() == 1
          and slot_map.is_contiguous(), f"slot_map must be a contiguous int64 vector on {cache.device}")
    with _on(cache.device):
        launch_paged_append(k, v, slot_map, cache, shape[0], _row_strides(k, "k"), _row_strides(v, "v"))


def _workspace(workspace, nbytes: int, device):
    """(workspace, its bytes): the caller's, or a new one."""
    import torch

    if workspace is None:
        if nbytes == 0:
            return None, 0
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _need(workspace.device == device and workspace.is_contiguous(), f"workspace must be a contiguous tensor on {device}")
    have = workspace.numel() * workspace.element_size()
    _need(have >= nbytes, f"workspace holds {have} bytes, {nbytes} are needed")
    return workspace, have


def attention_paged_workspace(q, cache: PagedCache, num_seqs: int, max_query_len: int, max_kv_len: int):
    """A workspace for attention_paged calls of these sizes (None: they need none)."""
    import torch

    with _on(q.device):
        n = attention_paged_workspace_bytes(q.shape[0], num_seqs, q.shape[1], cache.heads_kv, cache.head_dim, max_query_len,
                                            max_kv_len)
        return torch.empty(n, dtype=torch.uint8, device=q.device) if n else None


def attention_paged(q, cache: PagedCache, block_table, query_starts, kv_lens, max_query_len: int,
                    max_kv_len: Optional[int] = None, causal: bool = True, out=None, workspace=None):
    """softmax(q K^T / sqrt(head_dim)) V of new tokens q [tokens, heads, head_dim] over
    the cache. Sequence s has the rows query_starts[s] .. query_starts[s+1] - 1, the
    last of its kv_lens[s] tokens; their keys are in the cache already (paged_append),
    in the pages block_table[s] names. causal: each sees the tokens up to itself;
    else all kv_lens[s]. A row that sees nothing is 0; rows of no sequence, and past
    max_query_len of one, stay as they were in `out`. max_kv_len (default: the
    table's width) only decides how the work is split. `workspace`: from
    attention_paged_workspace, one per call that may run at the same time; a new one
    if not given. Returns O, like q."""
    import torch

    device = cache.device
    _need(q.dim() == 3 and q.shape[2] == cache.head_dim and q.dtype == cache.dtype and q.device == device,
          f"q must be a {cache.dtype} tensor [tokens, heads, {cache.head_dim}] on {device}")
    tokens, heads, head_dim = q.shape
    _need(kv_lens.dim() == 1, "kv_lens must be a vector")
    num_seqs = kv_lens.shape[0]
    _int32(kv_lens, "kv_lens", (num_seqs,), device)
    _int32(query_starts, "query_starts", (num_seqs + 1,), device)
    width, stride = _table(block_table, num_seqs, device)
    if max_kv_len is None:
        max_kv_len = width * cache.block_size
    with _on(device):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device, "out must be like q")
        nbytes = attention_paged_workspace_bytes(tokens, num_seqs, heads, cache.heads_kv, head_dim, max_query_len, max_kv_len)
        workspace, have = _workspace(workspace, nbytes, device)
        if not launch_attention_paged(q, cache, out, workspace, have, block_table, query_starts, kv_lens, num_seqs, tokens,
                                      heads, width, stride, max_query_len, max_kv_len, causal, _row_strides(q, "q"),
                                      _row_strides(out, "out")):
            raise ValueError(f"head_dim {head_dim} is not supported")
    return out


def attention_cross_workspace(q, k):
    """A workspace for attention_cross calls of these shapes (None: they need none)."""
    import torch

    with _on(q.device):
        n = attention_cross_workspace_bytes(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3])
        return torch.empty(n, dtype=torch.uint8, device=q.device) if n else None


def attention_cross(q, k, v, kv_lens=None, out=None, workspace=None):
    """softmax(q k^T / sqrt(head_dim)) v of queries q [batch, heads, q_len, head_dim] to
    an encoder's states k, v [batch, heads_kv, kv_len, head_dim] (bf16 or fp16, any
    strides with head_dim contiguous). kv_lens (int32 [batch]): the states of each
    entry; what lies behind them is padding. A row without states is 0. `workspace`:
    from attention_cross_workspace, one per call that may run at the same time; a new
    one if not given. Returns O, like q."""
    import torch

    device = q.device
    dtype = _dtype_id(q.dtype)
    _need(q.dim() == 4 and k.dim() == 4 and k.shape == v.shape, "q, k, v: [batch, heads, length, head_dim]")
    batch, heads, q_len, head_dim = q.shape
    heads_kv, kv_len = k.shape[1], k.shape[2]
    _need(k.shape[0] == batch and k.shape[3] == head_dim, "q, k and v differ in batch or head_dim")
    for x, name in ((k, "k"), (v, "v")):
        _need(x.dtype == q.dtype and x.device == device, f"{name} must be a {q.dtype} tensor on {device}")
    if kv_lens is not None:
        _int32(kv_lens, "kv_lens", (batch,), device)
    with _on(device):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == device, "out must be like q")
        nbytes = attention_cross_workspace_bytes(batch, heads, heads_kv, q_len, kv_len, head_dim)
        workspace, have = _workspace(workspace, nbytes, device)
        if not launch_attention_cross(q, k, v, out, workspace, have, kv_lens, batch, heads, heads_kv, q_len, kv_len, head_dim,
                                      dtype, _head_strides(q, "q"), _head_strides(k, "k"), _head_strides(v, "v"),
                                      _head_strides(out, "out")):
            raise ValueError(f"head_dim {head_dim} is not supported")
    return out
