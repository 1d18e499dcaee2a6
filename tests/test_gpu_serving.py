"""Serving operators on the GPU against plain forms in 64 bits (serving_ref.py),
at the lengths, masks, layouts and pages where they can go wrong."""
import math

import pytest
import torch

import serving_ref as ref
from gpu_common import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa(fa_lib):
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X")
    return fa_lib


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def heads_view(x, layout):
    return x if layout == "HND" else x.transpose(1, 2).contiguous().transpose(1, 2)


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


class Paged:
    """A batch over a cache whose unused slots hold NaN."""

    def __init__(self, fa, cached, new, heads, heads_kv, dim, block, dtype, layout="HND", seed=1, extra_rows=0,
                 extra_width=0, scale=1.0, fill=float("nan")):
        g = gen(seed)
        self.kv = [c + n for c, n in zip(cached, new)]
        need = [-(-x // block) for x in self.kv]
        blocks = sum(need) + 3
        self.block, self.dtype = block, ref.TYPES[dtype]
        shape = (blocks, heads_kv, block, dim)
        self.k, self.v = (heads_view(torch.full(shape, fill, device="cuda", dtype=self.dtype), layout) for _ in range(2))
        order = torch.randperm(blocks, device="cuda", generator=g).tolist()
        width = max(max(need, default=0), 1) + extra_width
        table = [[-7] * width for _ in need]
        at = 0
        for s, n in enumerate(need):
            for b in range(n):
                table[s][b] = order[at]
                count = min(block, self.kv[s] - b * block)
                self.k[order[at], :, :count] = randn((heads_kv, count, dim), self.dtype, g, scale)
                self.v[order[at], :, :count] = randn((heads_kv, count, dim), self.dtype, g)
                at += 1
        self.table = ints(table).reshape(len(need), width)
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.q = randn((self.starts[-1] + extra_rows, heads, dim), self.dtype, g, scale)
        self.max_new = max(new, default=0)
        self.cache = fa.paged_cache(self.k, self.v)

    def run(self, fa, causal=True, out=None, max_kv_len=None, **more):
        if out is None:
            out = torch.full_like(self.q, float("nan"))
        fa.attention_paged(self.q, self.cache, self.table, ints(self.starts), ints(self.kv), self.max_new, max_kv_len,
                           causal=causal, out=out, **more)
        torch.cuda.synchronize()
        return out

    def check(self, fa, causal=True, what="", **more):
        got = self.run(fa, causal, **more)
        want, tol, inside = ref.paged(self.q, self.k, self.v, self.table, self.starts, self.kv, self.block, causal)
        ref.check(got[inside], want[inside], tol[inside], what)
        assert got[~inside].isnan().all(), "rows of no sequence were written"
        return got


# ---------------------------------------------------------------- block tables and slots
@pytest.mark.parametrize("cached,new,block", [
    ([0], [1], 16), ([15], [1], 16), ([16], [1], 16), ([17], [40], 16), ([0], [0], 16), ([5], [0], 32),
    ([0, 0, 7, 31, 32, 33, 64], [0, 5, 0, 1, 1, 100, 0], 32),
    ([100] * 64, [1] * 64, 128),
])
def test_slots_small(fa, cached, new, block):
    say("slots", cached, new, block)
    _check_slots(fa, cached, new, block)


def _check_slots(fa, cached, new, block, free_cut=0, width_cut=0, pad=5, row_gap=0, out=None, token_cut=0):
    cached_p, new_p = [max(c, 0) for c in cached], [max(n, 0) for n in new]
    have = [-(-c // block) for c in cached_p]
    need = [-(-(c + n) // block) for c, n in zip(cached_p, new_p)]
    width = max(max(need, default=1), 1) - width_cut
    pages = torch.randperm(sum(need) + 9, generator=torch.Generator().manual_seed(3)).tolist()
    table = [[-5] * width for _ in cached]
    at = 0
    for s, n in enumerate(have):
        for b in range(min(n, width)):
            table[s][b] = pages[at]
            at += 1
    free = pages[at:at + max(0, sum(need) - sum(have) - free_cut)]
    tokens = max(0, sum(new_p) + pad - token_cut)
    want = ref.slots(cached, new, table, free, block, tokens)
    wide = torch.full((len(cached), width + row_gap), -9, dtype=torch.int32, device="cuda")
    dev = wide[:, :width]
    if cached:
        dev.copy_(ints(table))
    got = fa.paged_slots(ints(cached), ints(new), dev, ints(free), block, tokens, out=out)
    torch.cuda.synchronize()
    assert dev.tolist() == want[0]
    assert (wide[:, width:] == -9).all()
    assert got.query_starts.tolist() == want[1] and got.kv_lens.tolist() == want[2]
    assert got.slot_map.tolist() == want[3] and got.blocks_taken.tolist() == [want[4]]


@pytest.mark.parametrize("seqs,block,seed", [(1, 16, 1), (63, 16, 2), (64, 32, 3), (65, 16, 4), (255, 16, 5), (256, 64, 6),
                                              (257, 16, 7), (1023, 16, 8), (1025, 32, 9), (2500, 16, 10)])
def test_slots_many(fa, seqs, block, seed):
    import random

    rng = random.Random(seed)
    cached = [rng.choice([0, rng.randint(0, 300)]) for _ in range(seqs)]
    new = [rng.choice([0, 1, 1, 1, rng.randint(0, 90)]) for _ in range(seqs)]
    say("slots", seqs, block, seed)
    _check_slots(fa, cached, new, block)
    _check_slots(fa, cached, new, block, row_gap=3, token_cut=min(40, sum(new)), pad=0)


def test_slots_ends(fa):
    """A short free list, a narrow table, negative lengths, no sequence, one long prompt."""
    cached, new = [3, 40, 0, 16], [20, 33, 64, 1]
    for cut in (1, 3, 100):
        say("slots free cut", cut)
        _check_slots(fa, cached, new, 16, free_cut=cut)
    for cut in (1, 2, 3):
        say("slots width cut", cut)
        _check_slots(fa, cached, new, 16, width_cut=cut)
    _check_slots(fa, [-3, 5, -1], [4, -9, -2], 16)
    _check_slots(fa, [], [], 16)
    _check_slots(fa, [7], [70000], 16)
    _check_slots(fa, [0] * 300, [200] * 300, 64, pad=0)


# ---------------------------------------------------------------- cache writes
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("tokens,heads_kv,dim,block", [(1, 1, 64, 16), (7, 8, 128, 16), (129, 5, 64, 32), (33, 2, 8, 16),
                                                       (1000, 4, 96, 128), (3, 16, 128, 1024)])
def test_append(fa, dtype, layout, tokens, heads_kv, dim, block):
    say("append", dtype, layout, tokens, heads_kv, dim, block)
    g, t = gen(tokens), ref.TYPES[dtype]
    blocks = -(-tokens // block) + 2
    k, v = (heads_view(randn((blocks, heads_kv, block, dim), t, g), layout) for _ in range(2))
    slots = torch.randperm(blocks * block, device="cuda", generator=g)[:tokens].contiguous()
    slots[tokens // 2] = -1
    if tokens > 4:
        slots[0], slots[4] = blocks * block, -(2 ** 62)
        slots[1] = 2 ** 62
    qkv = randn((tokens, heads_kv + 2 * heads_kv, dim), t, g)
    new_k, new_v = qkv[:, heads_kv:2 * heads_kv], qkv[:, 2 * heads_kv:]
    want_k, want_v = k.clone(), v.clone()
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * block:
            want_k[s // block, :, s % block] = new_k[i]
            want_v[s // block, :, s % block] = new_v[i]
    fa.paged_append(new_k, new_v, slots, fa.paged_cache(k, v))
    torch.cuda.synchronize()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    fa.paged_append(new_k[:0], new_v[:0], slots[:0], fa.paged_cache(k, v))
    torch.cuda.synchronize()
    assert torch.equal(k, want_k)


# ---------------------------------------------------------------- attention over the cache
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,heads_kv", [(1, 1), (8, 8), (8, 2), (7, 1), (12, 4)])
def test_paged_decode(fa, dtype, dim, heads, heads_kv):
    cached = [0, 1, 14, 15, 16, 30, 31, 32, 33, 63, 64, 65, 200, 511]
    for layout, block in (("HND", 16), ("NHD", 32), ("HND", 128)):
        say("decode", dtype, dim, heads, heads_kv, layout, block)
        Paged(fa, cached, [1] * len(cached), heads, heads_kv, dim, block, dtype, layout, seed=block).check(fa, what="decode")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_chunks(fa, dtype, dim, causal):
    """Chunks of every size class of the row blocks, beside decoding sequences."""
    for cached, new, heads, heads_kv in (
            ([0, 3, 100], [1, 2, 3], 4, 2), ([70, 0, 33, 5], [33, 64, 1, 9], 1, 1), ([0, 500, 17], [130, 65, 127], 4, 4),
            ([200, 1, 0, 31], [257, 1, 300, 16], 6, 2), ([0], [1100], 2, 1), ([900, 4], [40, 1], 16, 1)):
        for layout, block in (("HND", 16), ("NHD", 64)):
            say("chunks", dtype, dim, causal, cached, new, heads, heads_kv, layout, block)
            Paged(fa, cached, new, heads, heads_kv, dim, block, dtype, layout, seed=len(cached),
                  extra_rows=3).check(fa, causal, "chunks")


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("fp16", 64), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_splits(fa, dtype, dim, causal):
    """Long caches, whose keys are split over workgroups and joined; short ones beside
    them, and a hint that is far off."""
    for cached, new, heads, heads_kv in (([4000], [1], 4, 2), ([3000, 0, 257, 512, 2047], [1, 1, 1, 1, 1], 8, 1),
                                         ([2500, 100], [70, 40], 2, 1), ([5000], [300], 1, 1), ([2222, 0], [9, 9], 4, 1)):
        b = Paged(fa, cached, new, heads, heads_kv, dim, 16, dtype, seed=7, extra_rows=2)
        rows, groups, splits = fa.attention_paged_config(b.q.shape[0], len(new), heads, heads_kv, dim, b.max_new, max(b.kv))
        say("splits", dtype, dim, causal, cached, new, rows, groups, splits)
        assert splits > 1
        b.check(fa, causal, "splits")
        b.check(fa, causal, "splits, long hint", max_kv_len=100000)
        b.check(fa, causal, "splits, short hint", max_kv_len=600)
        b.check(fa, causal, "splits, no hint", max_kv_len=0)


def test_paged_empty_rows(fa):
    """No keys, more new tokens than keys, no new tokens, no sequences."""
    b = Paged(fa, [0, 5, 0, 40], [0, 3, 70, 1], 4, 2, 64, 16, "bf16", extra_rows=4)
    b.kv[1], b.kv[2], b.kv[3] = 0, 50, -3  # lengths below the new tokens': the first rows see nothing
    say("empty rows")
    got = b.check(fa, True, "empty")
    assert (got[:3] == 0).all() and (got[3:23] == 0).all() and (got[73] == 0).all()
    b.check(fa, False, "empty, all keys")
    out = torch.full_like(b.q, 7.0)
    fa.attention_paged(b.q, b.cache, b.table[:0], ints([0]), ints([]), 1, out=out)
    fa.attention_paged(b.q[:0], b.cache, b.table, ints([0] * 5), ints(b.kv), 1, out=out[:0])
    fa.attention_paged(b.q, b.cache, b.table, ints(b.starts), ints(b.kv), 0, out=out)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


def test_paged_pages_outside_the_cache(fa):
    """A page that does not exist holds zeros; keys past the table do not exist."""
    for dim, cached, new in ((64, [40, 700], [1, 3]), (128, [33, 100], [200, 17])):
        b = Paged(fa, cached, new, 4, 2, dim, 16, "bf16", seed=5)
        b.table[0, 1] = -1
        b.table[1, 0] = b.cache.num_blocks
        b.table[1, 3] = 2 ** 31 - 1
        b.table[1, 4] = -2 ** 31
        say("pages", dim)
        b.check(fa, True, "pages")
        b.table = b.table[:, :5]
        b.check(fa, True, "narrow table")
        b.check(fa, False, "narrow table, all keys")
    b.table = b.table[:, :0]
    got = b.run(fa)
    assert (got == 0).all()


def test_paged_rows_past_max_query_len(fa):
    b = Paged(fa, [10, 20], [9, 4], 4, 2, 64, 16, "bf16")
    for limit in (4, 6, 100):
        b.max_new = limit
        say("max_query_len", limit)
        got = b.run(fa)
        want, tol, _ = ref.paged(b.q, b.k, b.v, b.table, b.starts, b.kv, 16, True)
        n = min(limit, 9)
        ref.check(got[:n], want[:n], tol[:n], "first rows")
        ref.check(got[9:], want[9:], tol[9:], "second sequence")
        assert got[n:9].isnan().all()


@pytest.mark.parametrize("causal", [True, False])
def test_paged_many_sequences(fa, causal):
    """Row blocks that are found among many sequences, some of them without new tokens."""
    import random

    rng = random.Random(4)
    for seqs, top in ((70, 150), (300, 90)):
        new = [rng.choice([0, 1, 1, 2, rng.randint(0, 5)]) for _ in range(seqs)]
        for s in rng.sample(range(seqs), 5):
            new[s] = rng.randint(40, top)
        cached = [rng.randint(0, 50) for _ in range(seqs)]
        say("many", seqs, causal)
        Paged(fa, cached, new, 4, 1, 64, 16, "bf16", seed=seqs, extra_rows=7).check(fa, causal, "many sequences")


def test_paged_rows_before_the_first_sequence(fa):
    """Starts that begin past 0: the rows before them belong to no sequence."""
    for new in ([1, 1, 1], [70, 3, 200], [5, 0, 1]):
        b = Paged(fa, [9, 40, 0], new, 4, 2, 64, 16, "bf16", extra_rows=80)
        b.starts = [x + 77 for x in b.starts]
        say("starts past 0", new)
        b.check(fa, True, "starts past 0")


def test_paged_in_place(fa):
    """O over q: a workgroup writes the rows that it alone has read."""
    for cached, new in (([30, 200], [90, 1]), ([3000], [2])):
        b = Paged(fa, cached, new, 4, 2, 64, 16, "bf16")
        q = b.q.clone()
        say("in place", cached, new)
        got = b.run(fa, out=b.q)
        want, tol, _ = ref.paged(q, b.k, b.v, b.table, b.starts, b.kv, 16, True)
        ref.check(got, want, tol, "in place")


def test_paged_views(fa):
    """Strided q and out, a wide table's columns, a cache between other data."""
    b = Paged(fa, [30, 0, 77], [5, 40, 1], 4, 2, 64, 16, "bf16", "NHD", extra_rows=1)
    qkv = torch.zeros((b.q.shape[0], 9, 64), dtype=b.dtype, device="cuda")
    qkv[:, 2:6] = b.q
    b.q = qkv[:, 2:6]
    wide = torch.full((3, b.table.shape[1] + 5), -3, dtype=torch.int32, device="cuda")
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide[:, :b.table.shape[1]]
    both = torch.full((b.k.shape[0], 3, 16, 2, 64), float("nan"), dtype=b.dtype, device="cuda")
    both[:, 0], both[:, 2] = b.k.transpose(1, 2), b.v.transpose(1, 2)
    b.cache = fa.paged_cache(both[:, 0].transpose(1, 2), both[:, 2].transpose(1, 2))
    room = torch.full((b.q.shape[0], 6, 64), float("nan"), dtype=b.dtype, device="cuda")
    say("views")
    b.check(fa, True, "views", out=room[:, 1:5])
    assert room[:, 0].isnan().all() and room[:, 5].isnan().all()


def test_paged_past_32_bits(fa):
    """Pages whose bytes lie past 2^32, and a page and a head stride that span it."""
    dim, block, heads_kv = 128, 16, 2
    room = torch.zeros(3 * 2 ** 30, dtype=torch.bfloat16, device="cuda")  # 6 GiB
    g = gen(2)
    page = 1 << 28  # elements from page to page
    shape, strides = (10, heads_kv, block, dim), (page, 1 << 27, dim, 1)
    k = room.as_strided(shape, strides)
    v = room[1 << 20:].as_strided(shape, strides)
    for c in (k, v):
        c.copy_(randn(shape, torch.bfloat16, g))
    table = ints([[9, 0, 8, 3, 7], [1, 9, 2, 8, 5]])
    starts, kv = [0, 1, 40], [70, 79]
    q = randn((40, 4, dim), torch.bfloat16, g)
    say("past 32 bits")
    got = fa.attention_paged(q, fa.paged_cache(k, v), table, ints(starts), ints(kv), 39)
    torch.cuda.synchronize()
    want, tol, _ = ref.paged(q, k, v, table, starts, kv, block, True)
    ref.check(got, want, tol, "past 32 bits")
    slots = ints([9 * 16 + 3, 8 * 16 + 15], torch.int64)
    rows = randn((2, heads_kv, dim), torch.bfloat16, g)
    fa.paged_append(rows, rows, slots, fa.paged_cache(k, v))
    torch.cuda.synchronize()
    assert torch.equal(k[9, :, 3], rows[0]) and torch.equal(v[8, :, 15], rows[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_paged_large_scores(fa, dtype):
    """Scores whose maximum keeps growing along a row, and far apart."""
    b = Paged(fa, [1500, 60], [3, 50], 4, 2, 64, 16, dtype, seed=11, scale=4.0)
    say("large scores", dtype)
    b.check(fa, True, "large scores")


# (batch, heads, key heads, new tokens, keys) that take each of the workgroups (rows,
# wave groups), with and without chunks
SHAPES = {
    64: [(200, 4, 4, 1, 33), (4, 16, 16, 1, 1500), (1, 1, 1, 1, 260), (64, 4, 2, 1, 1500), (1, 2, 2, 1000, 90),
         (1, 1, 1, 1, 33), (1, 1, 1, 1, 700), (3, 10, 5, 301, 533)],
    128: [(1, 1, 1, 1, 33), (1, 1, 1, 1, 260), (64, 8, 8, 1, 33), (16, 4, 4, 1, 700), (1, 8, 8, 1, 3000), (4, 4, 4, 1, 1500),
          (1, 1, 1, 17, 90), (200, 2, 2, 1, 33), (64, 4, 4, 130, 260), (2, 32, 16, 1000, 33), (4, 4, 2, 1000, 3000),
          (1, 4, 2, 400, 700), (8, 4, 4, 400, 6000)],
}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["paged", "cross"])
def test_every_configuration(fa, dtype, dim, kind):
    seen = set()
    for batch, heads, heads_kv, n, kv in SHAPES[dim]:
        if kind == "paged":
            if batch * n * heads * kv > 6e7:
                continue
            b = Paged(fa, [kv] * batch, [n] * batch, heads, heads_kv, dim, 16, dtype, seed=n)
            config = fa.attention_paged_config(batch * n, batch, heads, heads_kv, dim, n, kv + n)
            say("configuration", kind, dtype, dim, batch, heads, heads_kv, n, kv, config)
            b.check(fa, True, f"{config}", max_kv_len=kv + n)
        else:
            g, t = gen(n), ref.TYPES[dtype]
            q, k, v = (randn((batch, h, m, dim), t, g) for h, m in ((heads, n), (heads_kv, kv), (heads_kv, kv)))
            config = fa.attention_cross_config(batch, heads, heads_kv, n, kv, dim)
            say("configuration", kind, dtype, dim, batch, heads, heads_kv, n, kv, config)
            out = torch.full_like(q, float("nan"))
            fa.attention_cross(q, k, v, out=out)
            torch.cuda.synchronize()
            want, tol = ref.cross(q, k, v, [kv] * batch)
            ref.check(out, want, tol, f"cross {config}")
        seen.add((config[0], config[1], config[2] > 1))
    say("seen", kind, dim, sorted(seen))
    rows = {64: [(64, 1), (128, 1), (64, 2)], 128: [(64, 1), (128, 1), (64, 2), (256, 1)]}[dim]
    assert seen == {(*r, chunks) for r in rows for chunks in (False, True)}


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("top", [10, 24, 34])
def test_paged_one_key_takes_all(fa, dtype, dim, top):
    """Scores j * 2^top / sqrt(dim) for key j: every row's result is the value of the
    last key that it sees, exactly, though the base moves at every tile and (from 2^28
    on) is coarser than the distance of two scores is to a weight."""
    if dtype == "fp16" and top > 24:
        top = 24  # j 2^a and 2^b in fp16
    for new in (1, 70, 200):
        b = Paged(fa, [240 - new], [new], 2, 1, dim, 16, dtype, seed=new)
        low = min(top // 2, 6 if dtype == "fp16" else top)
        b.q[:], b.k[:] = 0, 0
        b.q[..., 0] = 2.0 ** (top - low) if dtype == "bf16" else 2.0 ** min(top - low, 15)
        for j in range(240):
            b.k[b.table[0, j // 16], :, j % 16, 0] = j * 2.0 ** low
        say("one key", dtype, dim, top, new)
        for hint in (None, 5000):
            got = b.run(fa, max_kv_len=hint)
            last = torch.arange(240 - new, 240, device="cuda")
            want = b.v[b.table[0].long()[last // 16], 0, last % 16]
            assert torch.equal(got[:, 0], want) and torch.equal(got[:, 1], want)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_not_finite_queries(fa, value):
    """A query row that is not finite makes its own row NaN, and no other."""
    b = Paged(fa, [40, 1500], [50, 3], 4, 2, 64, 16, "bf16", seed=2)
    want, tol, _ = ref.paged(b.q, b.k, b.v, b.table, b.starts, b.kv, 16, True)
    for row, h in ((7, 1), (33, 3), (51, 0)):
        b.q[row, h, 9] = value
    say("not finite q", value)
    for hint in (None, 200):
        got = b.run(fa, max_kv_len=hint)
        bad = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
        for row, h in ((7, 1), (33, 3), (51, 0)):
            bad[row, h] = True
        assert got[bad].isnan().all()
        ref.check(got[~bad], want[~bad], tol[~bad], "other rows")


def _check_not_finite(b, got, causal):
    """Rows against sums over the keys that each sees: infinities and NaN where one of
    those holds them, the usual tolerance elsewhere. fp16 weights are multiples of 2^-24
    where the row's largest is 2^8 or more, so a key of less than 2^-33 of the largest
    weighs 0, and 0 times an infinity is NaN: below 2^-32 either is right."""
    heads, group = b.q.shape[1], b.q.shape[1] // b.k.shape[1]
    clean_v = torch.where(b.v.isfinite(), b.v, 0)
    clean_k = torch.where(b.k.isfinite(), b.k, 0)
    want, tol, _ = ref.paged(b.q, clean_k, clean_v, b.table, b.starts, b.kv, b.block, causal)
    for s, kv in enumerate(b.kv):
        a, n = b.starts[s], b.starts[s + 1] - b.starts[s]
        pos = torch.arange(kv, device="cuda")
        page = b.table[s].long()[pos // b.block]
        first = kv - n + 1 if causal else kv
        for h in range(heads):
            v = b.v[page, h // group, pos % b.block].double()
            bad_k = ~b.k[page, h // group, pos % b.block].isfinite().all(-1)
            for i in range(n):
                seen = slice(0, first + (i if causal else 0))
                extra = torch.where(v[seen].isfinite(), 0.0, v[seen]).sum(0)
                if bad_k[seen].any():
                    extra = torch.full_like(extra, float("nan"))
                got_row, want_row, t = got[a + i, h].double(), want[a + i, h], tol[a + i, h]
                fine = extra == 0
                inf = extra.isinf()
                if b.dtype == torch.float16 and inf.any():
                    k = clean_k[page, h // group, pos % b.block].double()[seen]
                    score = torch.mv(k, b.q[a + i, h].double()) / math.sqrt(k.shape[1])
                    lost = score - score.amax() < -32 * math.log(2)
                    vanished = (v[seen].isinf() & lost[:, None]).any(0)
                    assert (got_row[inf & vanished].isinf() | got_row[inf & vanished].isnan()).all(), (s, i, h)
                    got_row = torch.where(vanished, extra, got_row)
                assert (got_row.isnan() == extra.isnan()).all(), (s, i, h)
                assert (got_row[inf] == extra[inf]).all(), (s, i, h)
                ref.check(got_row[fine], want_row[fine], t[fine], f"sequence {s} row {i} head {h}")


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("fp16", 128), ("bf16", 128)])
@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_paged_infinities_and_nan_in_v(fa, dtype, dim, scale):
    """A value that is not finite reaches the rows that see its key, and no other: in
    the tile of the diagonal, beside it, with rising scores, and a page of zeros there."""
    for cached, new, heads, heads_kv in (([0, 13], [40, 33], 2, 1), ([100], [70], 2, 2), ([5, 0], [3, 140], 4, 1)):
        b = Paged(fa, cached, new, heads, heads_kv, dim, 16, dtype, seed=21, scale=scale, extra_rows=1)
        for s, (at, value, d) in enumerate([(-1, math.nan, 3), (-2, math.inf, 7), (-20, -math.inf, 11), (-33, math.inf, 11)]):
            for q in range(len(new)):
                p = b.kv[q] + at
                if p >= 0:
                    b.v[b.table[q, p // 16], :, p % 16, d + 16 * (s % 2)] = value
        say("not finite v", dtype, dim, scale, cached, new)
        _check_not_finite(b, b.run(fa), True)
        _check_not_finite(b, b.run(fa, max_kv_len=4096), True)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_paged_not_finite_keys(fa, value):
    """A key that is not finite makes the rows that see it NaN, and no other."""
    b = Paged(fa, [20, 3], [70, 35], 2, 1, 64, 16, "bf16", seed=5)
    for q, p in ((0, 60), (1, 37)):
        b.k[b.table[q, p // 16], :, p % 16, 5] = math.nan
    b.v[b.table[0, 50 // 16], :, 50 % 16, 9] = value
    say("not finite k", value)
    _check_not_finite(b, b.run(fa), True)


def test_paged_left_out_tile_with_a_missing_page(fa):
    """The tile of the diagonal holds a NaN, and half of it lies in a page of zeros."""
    b = Paged(fa, [0], [64], 2, 1, 64, 16, "bf16", seed=6)
    b.v[b.table[0, 3], :, 15, 4] = math.nan
    b.table[0, 2] = -1
    say("left out, missing page")
    got = b.run(fa)
    v = b.v.clone()
    v[b.table[0, 3], :, 15, 4] = 0
    want, tol, _ = ref.paged(b.q, b.k, v, b.table, b.starts, b.kv, 16, True)
    assert got[63, :, 4].isnan().all()
    ref.check(got[:63], want[:63], tol[:63], "left out")


# ---------------------------------------------------------------- attention to an encoder's states
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,kv_len", [(1, 1), (1, 700), (3, 31), (17, 32), (33, 33), (64, 65), (100, 1), (129, 257),
                                          (300, 95), (1, 3001), (40, 2048)])
def test_cross(fa, dtype, dim, q_len, kv_len):
    for batch, heads, heads_kv, layout, padded in ((1, 1, 1, "HND", False), (3, 6, 2, "NHD", True), (2, 5, 5, "HND", True)):
        say("cross", dtype, dim, q_len, kv_len, batch, heads, heads_kv, layout, padded)
        g, t = gen(q_len * 7 + kv_len), ref.TYPES[dtype]
        q = heads_view(randn((batch, heads, q_len, dim), t, g), layout)
        k, v = (heads_view(randn((batch, heads_kv, kv_len, dim), t, g), layout) for _ in range(2))
        lens = [kv_len] * batch
        if padded:
            lens = [kv_len, max(0, kv_len - 5), 0, 1][:batch]
            for b, m in enumerate(lens):  # the padding is never used
                k[b, :, m:], v[b, :, m:] = float("nan"), float("inf")
        out = torch.full_like(q, float("nan"))
        fa.attention_cross(q, k, v, ints(lens) if padded else None, out=out)
        torch.cuda.synchronize()
        want, tol = ref.cross(q, k, v, lens)
        ref.check(out, want, tol, "cross")


def test_cross_ends(fa):
    """No states, lengths out of range, nothing to do, shared states (stride 0)."""
    g = gen(1)
    q = randn((3, 4, 9, 64), torch.bfloat16, g)
    k, v = (randn((1, 2, 50, 64), torch.bfloat16, g) for _ in range(2))
    ke, ve = k.expand(3, 2, 50, 64), v.expand(3, 2, 50, 64)
    say("cross ends")
    got = fa.attention_cross(q, ke, ve, ints([-4, 50, 1000]))
    torch.cuda.synchronize()
    want, tol = ref.cross(q, ke, ve, [0, 50, 50])
    ref.check(got, want, tol, "lengths")
    none = fa.attention_cross(q, ke[:, :, :0], ve[:, :, :0])
    torch.cuda.synchronize()
    assert (none == 0).all()
    assert fa.attention_cross(q[:0], ke[:0], ve[:0]).shape[0] == 0
    assert fa.attention_cross(q[:, :, :0], ke, ve).shape[2] == 0


def test_cross_is_the_self_attention(fa):
    """With as many keys as queries: the fused forward's result, each within its rounding."""
    g = gen(8)
    q, k, v = (randn((2, 4, 384, 128), torch.bfloat16, g) for _ in range(3))
    say("cross as self")
    got = fa.attention_cross(q, k, v)
    base = fa.attention_forward(q, k, v)
    torch.cuda.synchronize()
    _, tol = ref.cross(q, k, v, [384, 384])
    ref.check(got, base.double(), 2 * tol, "self")


# ---------------------------------------------------------------- how they are called
def _serve(fa, layout, dtype, steps, graph):
    """A prompt in chunks, then decoding, each step: slots, writes, attention."""
    dim, heads, heads_kv, block, seqs, t = 64, 4, 2, 16, 3, ref.TYPES[dtype]
    g = gen(3)
    k, v = (heads_view(torch.full((40, heads_kv, block, dim), float("nan"), device="cuda", dtype=t), layout) for _ in range(2))
    cache = fa.paged_cache(k, v)
    table = torch.full((seqs, 12), -1, dtype=torch.int32, device="cuda")
    pages = torch.randperm(40, device="cuda", generator=g).to(torch.int32)
    cached, new = torch.zeros(seqs, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda")
    free = pages.clone()
    rows = 64
    q, nk, nv = (torch.zeros((rows, n, dim), device="cuda", dtype=t) for n in (heads, heads_kv, heads_kv))
    bufs = fa.paged_slots_buffers(seqs, rows)
    out = torch.empty_like(q)
    ws = fa.attention_paged_workspace(q, cache, seqs, 50, 12 * block)

    def step():
        fa.paged_slots(cached, new, table, free, block, rows, out=bufs)
        fa.paged_append(nk, nv, bufs.slot_map, cache)
        fa.attention_paged(q, cache, table, bufs.query_starts, bufs.kv_lens, 50, out=out, workspace=ws)

    captured = None
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            step()
    results, taken = [], 0
    history = [[torch.zeros((0, heads_kv, dim), dtype=t, device="cuda")] * 2 for _ in range(seqs)]
    lens = [0] * seqs
    for counts in steps:
        cached.copy_(ints(lens))
        new.copy_(ints(counts))
        free.copy_(torch.roll(pages, -taken))
        for x in (q, nk, nv):
            x.copy_(randn(x.shape, t, g))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        captured.replay() if graph else step()
        torch.cuda.synchronize()
        taken += int(bufs.blocks_taken)
        at = 0
        for s, n in enumerate(counts):
            history[s] = [torch.cat([history[s][0], nk[at:at + n]]), torch.cat([history[s][1], nv[at:at + n]])]
            for h in range(heads):
                limits = lens[s] + 1 + torch.arange(n, device="cuda")
                want, tol = ref.attend(q[at:at + n, h], history[s][0][:, h // 2], history[s][1][:, h // 2], limits)
                ref.check(out[at:at + n, h], want, tol, f"step {counts} sequence {s}")
            lens[s] += n
            at += n
        assert out[at:].isnan().all()
        results.append(out.clone())
    return results


STEPS = [[40, 1, 0], [1, 17, 0], [1, 1, 50], [1, 1, 1], [0, 1, 1], [1, 0, 30], [1, 1, 1]]


@pytest.mark.parametrize("layout,dtype", [("HND", "bf16"), ("NHD", "fp16")])
def test_serving_run(fa, layout, dtype):
    say("serving run", layout, dtype)
    eager = _serve(fa, layout, dtype, STEPS, False)
    say("serving run captured", layout, dtype)
    replayed = _serve(fa, layout, dtype, STEPS, True)
    for a, b in zip(eager, replayed):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_streams_and_repeats(fa):
    """On another stream than the current one, and bitwise the same every time, with a
    split launch's workspace full of NaN at the start."""
    b = Paged(fa, [3000, 20], [1, 30], 4, 1, 128, 16, "bf16", seed=9)
    ws = fa.attention_paged_workspace(b.q, b.cache, 2, b.max_new, max(b.kv))
    assert ws is not None
    ws.fill_(255)
    first = b.run(fa, workspace=ws, max_kv_len=max(b.kv))
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = b.run(fa, workspace=ws, max_kv_len=max(b.kv))
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first.view(torch.int16), again.view(torch.int16))
    say("streams")


def test_two_streams_at_once(fa):
    """Calls that overlap, each with a workspace of its own or one that it allocates."""
    batches = [Paged(fa, [2500 + 100 * i, 30], [1, 20 + i], 4, 1, 64, 16, "bf16", seed=i) for i in range(4)]
    alone = [b.run(fa) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    outs = [torch.full_like(b.q, float("nan")) for b in batches]
    args = [(ints(b.starts), ints(b.kv)) for b in batches]
    torch.cuda.synchronize()
    say("two streams")
    for _ in range(5):
        for b, s, o, (starts, kv) in zip(batches, streams, outs, args):
            with torch.cuda.stream(s):
                fa.attention_paged(b.q, b.cache, b.table, starts, kv, b.max_new, out=o)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert torch.equal(a.view(torch.int16), o.view(torch.int16))


def test_cross_in_a_graph(fa):
    """A captured call follows its tensors' values and lengths; two graphs with a
    workspace each."""
    g = gen(4)
    q, k, v = (randn((4, 2, n, 64), torch.bfloat16, g) for n in (1, 2000, 2000))
    lens = ints([2000, 1, 700, 0])
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        out, ws = torch.empty_like(q), fa.attention_cross_workspace(q, k)
        assert ws is not None
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fa.attention_cross(q, k, v, lens, out=out, workspace=ws)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fa.attention_cross(q, k, v, lens, out=out, workspace=ws)
        graphs.append((graph, out, ws))
    for now in ([2000, 1, 700, 0], [5, 2000, 0, 1999], [0, 0, 0, 0], [33, 32, 31, 64]):
        lens.copy_(ints(now))
        q.copy_(randn(q.shape, torch.bfloat16, g))
        eager = fa.attention_cross(q, k, v, lens)
        torch.cuda.synchronize()
        say("cross graph", now)
        for graph, out, ws in graphs:
            out.fill_(float("nan"))
            ws.fill_(255)
            torch.cuda.synchronize()
            graph.replay()
        torch.cuda.synchronize()
        want, tol = ref.cross(q, k, v, now)
        ref.check(eager, want, tol, "eager")
        for _, out, _ in graphs:
            assert torch.equal(out.view(torch.int16), eager.view(torch.int16))


@pytest.mark.parametrize("dim", [64, 128])
def test_paged_joins(fa, dim):
    """Few and many chunks of few and many rows: both ways to join them."""
    for cached, new, heads, heads_kv in (([800], [1], 2, 2), ([6000], [1], 8, 1), ([6000], [9], 4, 1), ([5000], [20], 6, 1),
                                         ([900], [30], 2, 1), ([2000, 5], [14, 1], 4, 1)):
        b = Paged(fa, cached, new, heads, heads_kv, dim, 32, "bf16", seed=len(cached) + new[0])
        config = fa.attention_paged_config(b.q.shape[0], len(new), heads, heads_kv, dim, b.max_new, max(b.kv))
        say("joins", dim, cached, new, heads, heads_kv, config)
        b.check(fa, True, f"joins {config}", max_kv_len=max(b.kv))


@pytest.mark.parametrize("heads,new", [(2, 1), (2, 5), (40, 3)])
def test_paged_long_cache(fa, heads, new):
    """300000 cached tokens, as many chunks as a join takes."""
    b = Paged(fa, [300000], [new], heads, 1, 64, 1024, "bf16", seed=3)
    say("long cache", heads, new, fa.attention_paged_config(new, 1, heads, 1, 64, new, b.kv[0]))
    b.check(fa, True, "long cache")


@pytest.mark.parametrize("dim,heads,heads_kv,block", [(64, 100, 1, 16), (128, 64, 1, 2048), (64, 36, 2, 64)])
def test_paged_wide_groups(fa, dim, heads, heads_kv, block):
    """More query heads on a key head than a wave has rows."""
    for cached, new in (([70, 5], [1, 3]), ([0, 200], [40, 9]), ([1300], [2])):
        say("wide groups", dim, heads, heads_kv, block, cached, new)
        Paged(fa, cached, new, heads, heads_kv, dim, block, "bf16", seed=heads).check(fa, True, "wide groups")


def test_paged_thousands_of_sequences(fa):
    """More sequences than two rounds of the search tell apart."""
    import random

    rng = random.Random(8)
    new = [rng.choice([0, 1, 2, 40]) for _ in range(4300)]
    cached = [rng.choice([0, 3, 20]) for _ in new]
    say("thousands of sequences")
    b = Paged(fa, cached, new, 4, 1, 64, 16, "bf16", seed=8, extra_rows=9)
    b.check(fa, True, "thousands of sequences")


def test_refusals(fa):
    b = Paged(fa, [10], [2], 4, 2, 64, 16, "bf16")
    starts, kv = ints(b.starts), ints(b.kv)

    def call(q=b.q, cache=b.cache, table=b.table, starts=starts, kv=kv, n=2, **more):
        return fa.attention_paged(q, cache, table, starts, kv, n, **more)

    for bad in (dict(q=b.q.half()), dict(q=b.q[:, :, :32]), dict(q=b.q.cpu()), dict(table=b.table.long()),
                dict(starts=starts[:1]), dict(kv=kv.long()), dict(out=b.q.half()), dict(table=b.table[:0]),
                dict(q=b.q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(fa.FaError):
        call(q=randn((2, 3, 64), torch.bfloat16, gen(1)))  # heads no multiple of the key heads
    with pytest.raises(fa.FaError):
        call(n=-1)
    long = Paged(fa, [5000], [1], 4, 2, 64, 16, "bf16")
    with pytest.raises(ValueError):
        fa.attention_paged(long.q, long.cache, long.table, ints(long.starts), ints(long.kv), 1,
                           workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    odd = torch.zeros((4, 2, 16, 96), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        fa.attention_paged(torch.zeros((1, 2, 96), dtype=torch.bfloat16, device="cuda"), fa.paged_cache(odd, odd),
                           ints([[0]]), ints([0, 1]), ints([1]), 1)
    with pytest.raises(ValueError):
        fa.paged_cache(b.k, b.v.transpose(1, 2).contiguous().transpose(1, 2) if b.k.is_contiguous() else b.v.contiguous())
    with pytest.raises(ValueError):
        fa.paged_cache(b.k.float(), b.v.float())
    q, k = torch.zeros((1, 4, 3, 64), device="cuda"), torch.zeros((1, 2, 5, 64), device="cuda")
    with pytest.raises(ValueError):
        fa.attention_cross(q, k, k)
    q, k = q.bfloat16(), k.bfloat16()
    with pytest.raises(ValueError):
        fa.attention_cross(q, k.half(), k.half())
    with pytest.raises(ValueError):
        fa.attention_cross(q, k, k, ints([5, 5]))
    with pytest.raises(fa.FaError):
        fa.attention_cross(q, k[:, :, :1].expand(1, 2, 5, 64), k)  # key rows on top of each other
    with pytest.raises(ValueError):
        fa.paged_slots(ints([1]), ints([1, 2]), ints([[0]]), ints([1]), 16, 4)
    with pytest.raises(fa.FaError):
        fa.paged_slots(ints([1]), ints([1]), ints([[0]]), ints([1]), 24, 4)
    with pytest.raises(ValueError):
        fa.paged_append(q[0], q[0], ints([0, 1, 2, 3]), b.cache)
    torch.cuda.synchronize()
