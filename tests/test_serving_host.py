"""CPU tests of the serving operators' host side: what is refused before any
launch, the workspace and configuration queries, and the plain forms that the GPU
tests compare with. Pointers are made up; nothing is launched."""
import ctypes
import re

import pytest
import torch

import serving_ref as ref

INVALID = 1  # hipErrorInvalidValue
CONFIGS = {64: {(64, 1), (128, 1), (64, 2)}, 128: {(64, 1), (128, 1), (64, 2), (256, 1)}}  # (rows, wave groups)
P = 1 << 20  # a device pointer that nobody follows: every call below is refused


@pytest.fixture(scope="module")
def fa(fa_lib):
    fa_lib.get_last_error()
    return fa_lib


def cache_info(fa, **more):
    values = dict(k=P, v=P, block_stride=4 * 16 * 64, head_stride=16 * 64, token_stride=64, num_blocks=10, heads_kv=4,
                  block_size=16, head_dim=64, dtype=fa.DTYPE_BF16)
    values.update(more)
    return fa.PagedCacheInfo(**values)


def refused(fa, status):
    """The call was refused, and the calling thread's error says so."""
    assert status == INVALID
    assert fa.get_last_error() == INVALID
    return True


def paged_status(fa, cache=None, **more):
    a = dict(q=P, o=P, workspace=None, workspace_bytes=0, table=P, starts=P, lens=P, seqs=2, tokens=5, heads=8, width=3,
             stride=3, max_q=3, max_kv=48, causal=1, q_strides=None, o_strides=None)
    a.update(more)
    info = cache_info(fa) if cache is None else cache

    def s(x):
        return None if x is None else ctypes.byref(fa.Strides(*x))

    return fa.lib().fa_launch_attention_paged(
        a["q"], ctypes.byref(info), a["o"], a["workspace"], a["workspace_bytes"], a["table"], a["starts"], a["lens"],
        a["seqs"], a["tokens"], a["heads"], a["width"], a["stride"], a["max_q"], a["max_kv"], a["causal"],
        s(a["q_strides"]), s(a["o_strides"]), None)


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(dtype=-1), dict(block_size=8), dict(block_size=24), dict(block_size=0), dict(block_size=-16),
    dict(block_size=1 << 21), dict(num_blocks=-1), dict(heads_kv=-1), dict(heads_kv=0), dict(heads_kv=3), dict(k=None),
    dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(token_stride=56), dict(token_stride=68), dict(token_stride=0),
    dict(token_stride=1 << 26), dict(block_stride=4), dict(block_stride=-64), dict(block_stride=(1 << 34) + 8),
    dict(head_stride=12), dict(head_stride=-8), dict(block_size=1 << 20, token_stride=2048),
])
def test_paged_refuses_a_bad_cache(fa, bad):
    assert refused(fa, paged_status(fa, cache_info(fa, **bad)))
    if bad not in (dict(heads_kv=0), dict(heads_kv=3)):  # an append has no query heads
        info = cache_info(fa, **bad)
        assert refused(fa, fa.lib().fa_launch_paged_append(P, P, P, ctypes.byref(info), 3, None, None, None))


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(o=None), dict(starts=None), dict(lens=None), dict(table=None), dict(q=P + 2), dict(o=P + 8),
    dict(seqs=-1), dict(tokens=-1), dict(heads=-1), dict(max_q=-1), dict(max_kv=-1), dict(width=-1), dict(stride=-3),
    dict(heads=6), dict(heads=65540), dict(q_strides=(0, 64, 4)), dict(q_strides=(0, 60, 512)), dict(o_strides=(0, 64, 514)),
    dict(o_strides=(0, 2, 512)), dict(width=1 << 27, stride=1 << 27), dict(tokens=1 << 30, max_q=1 << 30),
    dict(tokens=1 << 30, seqs=1 << 30, max_q=1),  # more workgroups than a grid holds
])
def test_paged_refuses_bad_arguments(fa, bad):
    assert refused(fa, paged_status(fa, **bad))


def test_paged_workspace_is_checked(fa):
    sizes = dict(tokens=1, seqs=1, max_q=1, max_kv=8192, width=512, stride=512)
    need = fa.attention_paged_workspace_bytes(1, 1, 8, 4, 64, 1, 8192)
    rows, groups, splits = fa.attention_paged_config(1, 1, 8, 4, 64, 1, 8192)
    assert splits > 1 and need == 8 * splits * (64 + 2) * 4
    for ws, size in ((None, 0), (None, need), (P, need - 1), (P + 8, need)):
        assert refused(fa, paged_status(fa, workspace=ws, workspace_bytes=size, **sizes))


def test_calls_without_work_return(fa):
    L = fa.lib()
    assert paged_status(fa, seqs=0) == 0 and paged_status(fa, tokens=0) == 0 and paged_status(fa, heads=0) == 0
    assert paged_status(fa, max_q=0) == 0
    info = cache_info(fa)
    assert L.fa_launch_paged_append(None, None, None, ctypes.byref(info), 0, None, None, None) == 0
    info = cache_info(fa, heads_kv=0, k=None, v=None)
    assert L.fa_launch_paged_append(None, None, None, ctypes.byref(info), 5, None, None, None) == 0
    for batch, heads, q_len in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        assert cross_status(fa, batch=batch, heads=heads, q_len=q_len) == 0
    assert fa.peek_at_last_error() == 0


def test_unsupported_head_dims(fa):
    for d in (8, 32, 96, 192, 256):
        info = cache_info(fa, head_dim=d, token_stride=d, head_stride=16 * d, block_stride=64 * d)
        assert paged_status(fa, info) == fa.FA_ERROR_UNSUPPORTED
        assert cross_status(fa, head_dim=d) == fa.FA_ERROR_UNSUPPORTED
        assert fa.attention_paged_config(1, 1, 8, 4, d, 1, 64) is None
        assert fa.attention_cross_config(1, 8, 4, 1, 64, d) is None
    assert fa.peek_at_last_error() == 0


def cross_status(fa, **more):
    a = dict(q=P, k=P, v=P, o=P, workspace=None, workspace_bytes=0, lens=None, batch=2, heads=8, heads_kv=4, q_len=5,
             kv_len=7, head_dim=64, dtype=0, qs=None, ks=None, vs=None, os=None)
    a.update(more)

    def s(x):
        return None if x is None else ctypes.byref(fa.Strides(*x))

    return fa.lib().fa_launch_attention_cross(
        a["q"], a["k"], a["v"], a["o"], a["workspace"], a["workspace_bytes"], a["lens"], a["batch"], a["heads"],
        a["heads_kv"], a["q_len"], a["kv_len"], a["head_dim"], a["dtype"], s(a["qs"]), s(a["ks"]), s(a["vs"]), s(a["os"]),
        None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(q=P + 8), dict(k=P + 2), dict(v=P + 4), dict(o=P + 1),
    dict(batch=-1), dict(heads=-1), dict(heads_kv=-1), dict(heads_kv=0), dict(heads_kv=3), dict(q_len=-1), dict(kv_len=-1),
    dict(dtype=2), dict(ks=(0, 448, 0)), dict(vs=(0, 448, 32)), dict(ks=(4, 448, 64)), dict(qs=(0, 0, 4)),
    dict(os=(0, 12, 64)), dict(ks=(0, 0, 1 << 26)), dict(heads=65540, heads_kv=4), dict(kv_len=(1 << 30) + 1),
    dict(q_len=1 << 30, heads=8, heads_kv=4), dict(q_len=1 << 29, heads=4, batch=1 << 10),
    dict(q_len=1, kv_len=8192, batch=1), dict(q_len=1, kv_len=8192, batch=1, workspace=P, workspace_bytes=64),
])
def test_cross_refuses_bad_arguments(fa, bad):
    assert refused(fa, cross_status(fa, **bad))


@pytest.mark.parametrize("bad", [
    dict(seqs=-1), dict(width=-1), dict(stride=-1), dict(free=-1), dict(block=15), dict(block=48), dict(block=0),
    dict(tokens=-1), dict(stride=2), dict(cached=None), dict(new=None), dict(table=None), dict(free_p=None),
    dict(starts=None), dict(lens=None), dict(slots=None), dict(taken=None),
])
def test_slots_refuses_bad_arguments(fa, bad):
    a = dict(cached=P, new=P, table=P, free_p=P, starts=P, lens=P, slots=P, taken=P, seqs=2, width=3, stride=3, free=4,
             block=16, tokens=8)
    a.update(bad)
    assert refused(fa, fa.lib().fa_launch_paged_slots(
        a["cached"], a["new"], a["table"], a["free_p"], a["starts"], a["lens"], a["slots"], a["taken"], a["seqs"],
        a["width"], a["stride"], a["free"], a["block"], a["tokens"], None))


def test_append_refuses_bad_arguments(fa):
    L, info = fa.lib(), cache_info(fa)
    ref_ = ctypes.byref(info)

    def strides(*x):
        return ctypes.byref(fa.Strides(*x))

    for args in ((None, P, P, ref_, 3, None, None), (P, None, P, ref_, 3, None, None), (P, P, None, ref_, 3, None, None),
                 (P + 8, P, P, ref_, 3, None, None), (P, P + 2, P, ref_, 3, None, None), (P, P, P, ref_, -1, None, None),
                 (P, P, P, ref_, 3, strides(0, 64, 260), None), (P, P, P, ref_, 3, None, strides(0, 4, 256)),
                 (P, P, P, None, 3, None, None)):
        assert refused(fa, L.fa_launch_paged_append(*args, None))


def test_configurations(fa):
    """Rows and chunks over the range: the rows cover a block, chunks stay within the
    joins' limit, and a launch without chunks needs no workspace."""
    for heads, heads_kv in ((8, 8), (32, 8), (64, 1), (7, 7)):
        for dim in (64, 128):
            for seqs, q in ((1, 1), (1, 7), (3, 40), (64, 1), (300, 2), (1, 2048), (8, 512)):
                for kv in (0, 1, 31, 500, 4096, 70000, 1 << 20, 1 << 30):
                    tokens = seqs * q
                    rows, groups, splits = fa.attention_paged_config(tokens, seqs, heads, heads_kv, dim, q, kv)
                    need = fa.attention_paged_workspace_bytes(tokens, seqs, heads, heads_kv, dim, q, kv)
                    assert (rows, groups) in CONFIGS[dim] and 1 <= splits <= 256
                    assert need == (tokens * heads * splits * (dim + 2) * 4 if splits > 1 else 0)
                    rows, groups, splits = fa.attention_cross_config(seqs, heads, heads_kv, q, kv, dim)
                    need = fa.attention_cross_workspace_bytes(seqs, heads, heads_kv, q, kv, dim)
                    assert (rows, groups) in CONFIGS[dim] and 1 <= splits <= 256
                    assert need == (tokens * heads * splits * (dim + 2) * 4 if splits > 1 else 0)
    for bad in ((0, 1, 8, 8, 64, 1, 10), (1, 0, 8, 8, 64, 1, 10), (1, 1, 8, 3, 64, 1, 10), (1, 1, 8, 0, 64, 1, 10),
                (1, 1, 8, 8, 64, 0, 10), (1, 1, 8, 8, 64, 1, -1)):
        assert fa.attention_paged_workspace_bytes(*bad) == 0
        with pytest.raises(fa.FaError):
            fa.attention_paged_config(*bad)
    fa.get_last_error()


def test_chunks_stay_within_the_grid(fa):
    """Launches so large that chunks would pass the grid's limit take none."""
    for seqs, heads, kv in ((1 << 16, 128, 4096), (1 << 17, 64, 1 << 20), (200000, 32, 70000)):
        rows, groups, splits = fa.attention_paged_config(seqs, seqs, heads, heads, 128, 1, kv)
        assert seqs * heads * splits * rows * 2 * groups <= 2 ** 31 - 1
        assert splits == 1 or seqs * heads * 256 <= 2 ** 31 - 1
        rows, groups, splits = fa.attention_cross_config(seqs, heads, heads, 1, kv, 128)
        assert seqs * heads * splits * rows * 2 * groups <= 2 ** 31 - 1


def test_header_is_plain_c(tmp_path):
    import os
    import subprocess

    src = tmp_path / "caller.c"
    src.write_text('#include "fa_mi355x.h"\n'
                   "int main(void) { fa_paged_cache c = {0}; fa_strides s = {0, 64, 128}; c.dtype = FA_DTYPE_FP16;\n"
                   "  return fa_launch_paged_append(0, 0, 0, &c, 0, &s, &s, 0); }\n")
    include = os.path.join(os.path.dirname(__file__), "..", "include")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", f"-I{include}", str(src)], check=True)


def test_structs_match_the_header(fa):
    """The ctypes mirrors have the header's fields in the header's order."""
    import os

    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "fa_mi355x.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, mirror in (("fa_strides", fa.Strides), ("fa_paged_cache", fa.PagedCacheInfo)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = [(t.strip(), f) for t, f in re.findall(r"((?:long long|void\*|int))\s+(\w+);", body)]
        want = {"long long": ctypes.c_longlong, "void*": ctypes.c_void_p, "int": ctypes.c_int}
        assert [(f, want[t]) for t, f in fields] == list(mirror._fields_)


def test_python_refuses_before_the_library(fa):
    cpu = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fa.paged_cache(cpu, cpu)
    with pytest.raises(ValueError):
        fa.attention_cross(cpu, cpu, cpu)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        fa.paged_slots(one, one, one[None], one, 16, 4)
    out = fa.paged_slots_buffers(3, 8, device="cpu")
    assert (out.num_seqs, out.max_tokens) == (3, 8)
    with pytest.raises(AttributeError):
        out.kv_lens = one
    for i, x in ((0, one), (1, one.long()), (2, torch.zeros(8, dtype=torch.int32)), (3, torch.ones(2, dtype=torch.int32))):
        parts = [out.query_starts, out.kv_lens, out.slot_map, out.blocks_taken]
        parts[i] = x
        with pytest.raises(ValueError):
            fa.PagedSlots(*parts)


# ---------------------------------------------------------------- the plain forms
def test_plain_attention_against_torch():
    """The 64-bit form against torch's own softmax and products, and its zero rows."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((n, 64), generator=g).to(torch.bfloat16) for n in (9, 33, 33))
    limits = torch.tensor([0, 1, 2, 5, 16, 31, 32, 33, 40])
    o, tol = ref.attend(q, k, v, limits)
    assert (o[0] == 0).all() and (tol[0] == 0).all()
    for i in range(1, 9):
        n = min(int(limits[i]), 33)
        w = torch.softmax(q[i].double() @ k[:n].double().T / 8.0, -1)
        assert torch.allclose(o[i], w @ v[:n].double(), rtol=1e-12, atol=1e-12)
    assert (tol[1:] > 0).all() and (tol[1:] < 0.05).all()
    assert torch.allclose(o[1], v[0].double())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mistake", ["key dropped", "key too many", "scale"])
def test_tolerance_sees_mistakes(dtype, mistake):
    """The comparison fails where the oracle's side has one key too few or too many,
    or another scale; and passes for the same rounded the way the kernels round."""
    g = torch.Generator().manual_seed(2)
    t = ref.TYPES[dtype]
    q, k, v = (torch.randn((n, 64), generator=g).to(t) for n in (40, 60, 60))
    limits = torch.arange(10, 50)
    o, tol = ref.attend(q, k, v, limits)
    s = (q.float() @ k.float().T / 8.0).masked_fill(torch.arange(60)[None] >= limits[:, None], -float("inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True)).to(t).float()
    ref.check((p @ v.float() / p.sum(-1, keepdim=True)).to(t), o, tol, "rounded")
    if mistake == "scale":
        bad, _ = ref.attend((q.float() * 1.05).to(t), k, v, limits)
    else:
        bad, _ = ref.attend(q, k, v, limits + (1 if mistake == "key too many" else -1))
    with pytest.raises(AssertionError):
        ref.check(bad.to(t), o, tol, mistake)


def test_plain_slots_by_hand():
    table, starts, kv, slot, taken = ref.slots([3, 16, 0], [2, 1, 0], [[7, -1], [4, -1], [-1, -1]], [9, 8], 16, 5)
    assert table == [[7, -1], [4, 9], [-1, -1]] and starts == [0, 2, 3, 3] and kv == [5, 17, 0]
    assert slot == [7 * 16 + 3, 7 * 16 + 4, 9 * 16, -1, -1] and taken == 1
