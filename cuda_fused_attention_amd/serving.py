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

import ctypes
from typing import Optional

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


class PagedSlots:
    """What paged_slots writes beside the block table: query_starts int32
    [num_seqs + 1], kv_lens int32 [num_seqs], slot_map int64 [max_tokens] and
    blocks_taken int32 [1], contiguous on one device. Checked when it is made."""

    __slots__ = ("query_starts", "kv_lens", "slot_map", "blocks_taken", "num_seqs", "max_tokens", "device")

    def __init__(self, query_starts, kv_lens, slot_map, blocks_taken):
        torch = _torch or _bind()
        device, num_seqs, max_tokens = kv_lens.device, kv_lens.numel(), slot_map.numel()
        for x, n, dtype, name in ((query_starts, num_seqs + 1, torch.int32, "query_starts"),
                                  (kv_lens, num_seqs, torch.int32, "kv_lens"),
                                  (slot_map, max_tokens, torch.int64, "slot_map"),
                                  (blocks_taken, 1, torch.int32, "blocks_taken")):
            _vector(x, n, device, dtype, name)
        for name, value in (("query_starts", query_starts), ("kv_lens", kv_lens), ("slot_map", slot_map),
                            ("blocks_taken", blocks_taken), ("num_seqs", num_seqs), ("max_tokens", max_tokens),
                            ("device", device)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError("PagedSlots cannot be changed")


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
    out = [ctypes.c_int() for _ in range(3)]
    if not _fa._check(getattr(_fa.lib(), call)(*sizes, *map(ctypes.byref, out)), call):
        return None
    return tuple(x.value for x in out)


def attention_paged_config(tokens: int, num_seqs: int, heads: int, heads_kv: int, head_dim: int, max_query_len: int,
                           max_kv_len: int):
    """(rows per workgroup, wave groups that share its keys, most chunks of a
    sequence's keys), or None for an unsupported head_dim."""
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
# torch, the element types, the current device and its current stream as raw values,
# and the library, bound on first use (torch is imported only for torch callers).
# These functions are on the path of every decoding step: they call the C entry
# points without the wrappers above, and a check costs its comparisons and builds no
# message (7.8 -> 6 us for paged_slots, of which its kernel's launch is 3.5).
_torch = None
_dtype_ids = {}
_device_index = None
_raw_stream = None
_lib = None


def _bind():
    global _torch, _dtype_ids, _device_index, _raw_stream, _lib
    import torch

    _dtype_ids = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_FP16}
    _device_index = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if _raw_stream is None:
        _raw_stream = lambda index: int(torch.cuda.current_stream(index).cuda_stream)  # noqa: E731
    _lib = _fa.lib()
    _torch = torch
    return torch


def _dtype_id(dtype) -> int:
    if dtype not in _dtype_ids:
        raise ValueError(f"bf16 or fp16 tensors are needed, not {dtype}")
    return _dtype_ids[dtype]


def _other_device(device):
    """A context in which `device`, another GPU than the current one, is current."""
    if device.type != "cuda":
        raise ValueError("CUDA tensors are needed")
    return _torch.cuda.device(device)


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _vector(x, n: int, device, dtype, name: str):
    """`x` is a contiguous vector of n integers on this device."""
    if x.dtype is not dtype or x.dim() != 1 or x.numel() != n or not x.is_contiguous() or x.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor [{n}] on {device}")


def _table(table, num_seqs: int, device):
    """(width, row stride) of a block table."""
    if table.dtype is not _torch.int32 or table.dim() != 2 or table.device != device:
        raise ValueError(f"block_table must be an int32 tensor [{num_seqs}, width] on {device}")
    rows, width = table.shape
    if rows != num_seqs:
        raise ValueError(f"block_table has {rows} rows for {num_seqs} sequences")
    stride, column = table.stride()
    if num_seqs < 2:
        stride = max(width, 1)
    if (width > 1 and column != 1) or stride < width:
        raise ValueError("block_table: entries of a row must be contiguous, rows must not overlap")
    return width, stride


def _strides_of(x, name: str):
    """Strides (batch, head, row) of a [batch, heads, rows, dim] tensor, (0, head, row)
    of a [rows, heads, dim] one. Along an axis of one entry, whose stride means
    nothing, one row."""
    shape, stride = x.shape, x.stride()
    dim = shape[-1]
    if stride[-1] != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    if len(shape) == 3:
        return 0, stride[1] if shape[1] > 1 else dim, stride[0] if shape[0] > 1 else dim
    return (stride[0] if shape[0] > 1 else dim, stride[1] if shape[1] > 1 else dim, stride[2] if shape[2] > 1 else dim)


def _strides_arg(x, name: str):
    """The strides as a C entry point takes them: none for a contiguous tensor."""
    return None if x.is_contiguous() else ctypes.byref(_fa.Strides(*_strides_of(x, name)))


def _like_q(out, q):
    if out.dtype is not q.dtype or out.shape != q.shape or out.device != q.device:
        raise ValueError("out must have q's shape, type and device")


def _workspace_room(workspace, device) -> int:
    if workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on {device}")
    return workspace.nbytes


def _refused(status: int, what: str, head_dim: int, workspace, have: int, need: int):
    if status == _fa.FA_ERROR_UNSUPPORTED:
        raise ValueError(f"head_dim {head_dim} is not supported")
    if workspace is not None and have < need:
        raise ValueError(f"workspace holds {have} bytes, {need} are needed")
    raise _fa.FaError(status, what)


def paged_cache(k_cache, v_cache) -> PagedCache:
    """A cache of two tensors [num_blocks, heads_kv, block_size, head_dim] (bf16 or
    fp16, equal strides, head_dim contiguous). Pages that hold their tokens' heads
    side by side, [num_blocks, block_size, heads_kv, head_dim], come as
    .transpose(1, 2)."""
    if _torch is None:
        _bind()
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "k_cache, v_cache: [num_blocks, heads_kv, block_size, head_dim]")
    _need(k_cache.dtype == v_cache.dtype and k_cache.device == v_cache.device, "k_cache and v_cache differ in type or device")
    _need(k_cache.is_cuda, "CUDA tensors are needed")
    block, head, token = _strides_of(k_cache, "k_cache")
    _need((block, head, token) == _strides_of(v_cache, "v_cache"), "k_cache and v_cache must have equal strides")
    num_blocks, heads_kv, block_size, head_dim = k_cache.shape
    info = _fa.PagedCacheInfo(k_cache.data_ptr(), v_cache.data_ptr(), block, head, token, num_blocks, heads_kv, block_size,
                              head_dim, _dtype_id(k_cache.dtype))
    return PagedCache(k_cache, v_cache, info)


def paged_slots_buffers(num_seqs: int, max_tokens: int, device="cuda") -> PagedSlots:
    """Buffers that paged_slots can write again and again (`out`)."""
    torch = _torch or _bind()

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
    torch = _torch or _bind()
    device = cached_lens.device
    index = device.index
    if index is None or index != _device_index():
        with _other_device(device):
            return paged_slots(cached_lens, new_lens, block_table, free_blocks, block_size, max_tokens, out)
    num_seqs, num_free = cached_lens.numel(), free_blocks.numel()
    if out is None:
        out = paged_slots_buffers(num_seqs, max_tokens, device)
    elif out.num_seqs != num_seqs or out.max_tokens != max_tokens or out.device != device:
        raise ValueError(f"out is for {out.num_seqs} sequences and {out.max_tokens} tokens on {out.device}")
    int32 = torch.int32
    _vector(cached_lens, num_seqs, device, int32, "cached_lens")
    _vector(new_lens, num_seqs, device, int32, "new_lens")
    _vector(free_blocks, num_free, device, int32, "free_blocks")
    width, stride = _table(block_table, num_seqs, device)
    status = _lib.fa_launch_paged_slots(
        cached_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), free_blocks.data_ptr(),
        out.query_starts.data_ptr(), out.kv_lens.data_ptr(), out.slot_map.data_ptr(), out.blocks_taken.data_ptr(), num_seqs,
        width, stride, num_free, block_size, max_tokens, _raw_stream(index))
    if status:
        raise _fa.FaError(status, "fa_launch_paged_slots")
    return out


def paged_append(k, v, slot_map, cache: PagedCache) -> None:
    """New rows k, v [tokens, heads_kv, head_dim] into the cache's slots slot_map
    (int64 [tokens]; negative or past the cache: skipped)."""
    device = cache.device
    index = device.index
    if index is None or index != _device_index():
        with _other_device(device):
            return paged_append(k, v, slot_map, cache)
    tokens = slot_map.numel()
    _vector(slot_map, tokens, device, _torch.int64, "slot_map")
    shape = (tokens, cache.heads_kv, cache.head_dim)
    dtype = cache.dtype
    if (k.dtype is not dtype or v.dtype is not dtype or k.shape != shape or v.shape != shape or k.device != device
            or v.device != device):
        raise ValueError(f"k and v must be {dtype} tensors {list(shape)} on {device}")
    status = _lib.fa_launch_paged_append(k.data_ptr(), v.data_ptr(), slot_map.data_ptr(), cache.ref, tokens,
                                         _strides_arg(k, "k"), _strides_arg(v, "v"), _raw_stream(index))
    if status:
        raise _fa.FaError(status, "fa_launch_paged_append")


def attention_paged_workspace(q, cache: PagedCache, num_seqs: int, max_query_len: int, max_kv_len: int):
    """A workspace for attention_paged calls of these sizes (None: they need none)."""
    with _torch.cuda.device(q.device):
        n = attention_paged_workspace_bytes(q.shape[0], num_seqs, q.shape[1], cache.heads_kv, cache.head_dim, max_query_len,
                                            max_kv_len)
        return _torch.empty(n, dtype=_torch.uint8, device=q.device) if n else None


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
    device = cache.device
    index = device.index
    if index is None or index != _device_index():
        with _other_device(device):
            return attention_paged(q, cache, block_table, query_starts, kv_lens, max_query_len, max_kv_len, causal, out,
                                   workspace)
    if q.dim() != 3 or q.dtype is not cache.dtype or q.device != device:
        raise ValueError(f"q must be a {cache.dtype} tensor [tokens, heads, {cache.head_dim}] on {device}")
    tokens, heads, head_dim = q.shape
    if head_dim != cache.head_dim:
        raise ValueError(f"q has head_dim {head_dim}, the cache {cache.head_dim}")
    num_seqs = kv_lens.numel()
    _vector(kv_lens, num_seqs, device, _torch.int32, "kv_lens")
    _vector(query_starts, num_seqs + 1, device, _torch.int32, "query_starts")
    width, stride = _table(block_table, num_seqs, device)
    if max_kv_len is None:
        max_kv_len = width * cache.block_size
    if out is None:
        out = _torch.empty_like(q, memory_format=_torch.contiguous_format)
    else:
        _like_q(out, q)

    room, have = workspace, 0
    if workspace is not None:
        have = _workspace_room(workspace, device)
    else:
        have = attention_paged_workspace_bytes(tokens, num_seqs, heads, cache.heads_kv, head_dim, max_query_len, max_kv_len)
        if have:
            room = _torch.empty(have, dtype=_torch.uint8, device=device)
    status = _lib.fa_launch_attention_paged(
        q.data_ptr(), cache.ref, out.data_ptr(), None if room is None else room.data_ptr(), have, block_table.data_ptr(),
        query_starts.data_ptr(), kv_lens.data_ptr(), num_seqs, tokens, heads, width, stride, max_query_len, max_kv_len,
        1 if causal else 0, _strides_arg(q, "q"), _strides_arg(out, "out"), _raw_stream(index))
    if status:
        need = attention_paged_workspace_bytes(tokens, num_seqs, heads, cache.heads_kv, head_dim, max_query_len, max_kv_len)
        _refused(status, "fa_launch_attention_paged", head_dim, workspace, have, need)
    return out


def attention_cross_workspace(q, k):
    """A workspace for attention_cross calls of these shapes (None: they need none)."""
    torch = _torch or _bind()
    with torch.cuda.device(q.device):
        n = attention_cross_workspace_bytes(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3])
        return torch.empty(n, dtype=torch.uint8, device=q.device) if n else None


def attention_cross(q, k, v, kv_lens=None, out=None, workspace=None):
    """softmax(q k^T / sqrt(head_dim)) v of queries q [batch, heads, q_len, head_dim] to
    an encoder's states k, v [batch, heads_kv, kv_len, head_dim] (bf16 or fp16, any
    strides with head_dim contiguous). kv_lens (int32 [batch]): the states of each
    entry; what lies behind them is padding. A row without states is 0. `workspace`:
    from attention_cross_workspace, one per call that may run at the same time; a new
    one if not given. Returns O, like q."""
    torch = _torch or _bind()
    device = q.device
    index = device.index
    if index is None or index != _device_index():
        with _other_device(device):
            return attention_cross(q, k, v, kv_lens, out, workspace)
    dtype = q.dtype
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q, k, v: [batch, heads, length, head_dim], k and v alike")
    batch, heads, q_len, head_dim = q.shape
    k_batch, heads_kv, kv_len, k_dim = k.shape
    if k_batch != batch or k_dim != head_dim:
        raise ValueError("q, k and v differ in batch or head_dim")
    if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device:
        raise ValueError("q, k and v differ in type or device")
    if kv_lens is not None:
        _vector(kv_lens, batch, device, torch.int32, "kv_lens")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _like_q(out, q)

    room, have = workspace, 0
    if workspace is not None:
        have = _workspace_room(workspace, device)
    else:
        have = attention_cross_workspace_bytes(batch, heads, heads_kv, q_len, kv_len, head_dim)
        if have:
            room = torch.empty(have, dtype=torch.uint8, device=device)
    status = _lib.fa_launch_attention_cross(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None if room is None else room.data_ptr(), have,
        None if kv_lens is None else kv_lens.data_ptr(), batch, heads, heads_kv, q_len, kv_len, head_dim, _dtype_id(dtype),
        _strides_arg(q, "q"), _strides_arg(k, "k"), _strides_arg(v, "v"),
        _strides_arg(out, "out"), _raw_stream(index))
    if status:
        need = attention_cross_workspace_bytes(batch, heads, heads_kv, q_len, kv_len, head_dim)
        _refused(status, "fa_launch_attention_cross", head_dim, workspace, have, need)
    return out
