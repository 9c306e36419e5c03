"""Page cache and rotary positions on the GPU against the plain model of page_model.py: pages and tables exactly, turned
values within the roundings that page_model.tolerance adds up."""
import ctypes as C
import sys

import numpy as np
import pytest

import multimesh_jax_amd as mm
from multimesh_jax_amd import _binding as B

import page_model as pm

pytestmark = pytest.mark.gpu


def say(msg):
    print("[gpu-test] " + msg, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    c = mm.ReshardContext(0)
    yield c
    c.close()


def whole(ctx, values, type="S32"):
    """A store in one buffer that holds `values`."""
    values = np.ascontiguousarray(values)
    shape = mm.sharded_shape(type, [(n, 1, i) for i, n in enumerate(values.shape)], 0, 1)
    s = ctx.CreateStore(shape)
    if values.size:
        ctx.AssembleShards(shape, 0, values.view(np.uint8).reshape(-1), existing_store=s)
    return s


def split(ctx, values, type, cut, n_dev, minor_to_major=None, start=0):
    """A store with dim `cut` of `values` over n_dev devices, padded with 0x5a bytes where the tiles do not divide."""
    dims = [(n, n_dev if i == cut else 1, i) for i, n in enumerate(values.shape)]
    shape = mm.sharded_shape(type, dims, start, n_dev, minor_to_major)
    s = ctx.CreateStore(shape)
    ext = -(-values.shape[cut] // n_dev)
    for k in range(n_dev):
        local = list(values.shape)
        local[cut] = ext
        tile = np.full(int(np.prod(local)) * values.itemsize, 0x5A, np.uint8).view(values.dtype).reshape(local)
        part = values[(slice(None),) * cut + (slice(k * ext, (k + 1) * ext),)]
        tile[(slice(None),) * cut + (slice(0, part.shape[cut]),)] = part
        if minor_to_major is not None:
            tile = tile.transpose(list(minor_to_major)[::-1])
        if tile.size:
            ctx.AssembleShards(shape, start + k, np.ascontiguousarray(tile).view(np.uint8).reshape(-1), existing_store=s)
    return s


def joined(ctx, store, like, cut, n_dev, minor_to_major=None, start=0):
    """(the array of a store made by split, its padding as bytes)"""
    ext = -(-like.shape[cut] // n_dev)
    parts, pad = [], []
    for k in range(n_dev):
        local = list(like.shape)
        local[cut] = ext
        raw = ctx.ReadShard(store, start + k, like.dtype)
        if minor_to_major is not None:
            order = list(minor_to_major)[::-1]
            raw = raw.reshape([local[i] for i in order]).transpose(np.argsort(order))
        raw = raw.reshape(local)
        n = max(0, min(ext, like.shape[cut] - k * ext))
        parts.append(raw[(slice(None),) * cut + (slice(0, n),)])
        pad.append(np.ascontiguousarray(raw[(slice(None),) * cut + (slice(n, None),)]).view(np.uint8).reshape(-1))
    return np.concatenate(parts, cut), np.concatenate(pad)


class Pair:
    """A page cache on the GPU and its model, from the same beginnings."""

    def __init__(self, ctx, S, Bl, P, T, shape, type, n_pools=2, n_dev=1, cut=1, layout=None, seed=0):
        rng = np.random.Generator(np.random.PCG64(seed))
        self.ctx, self.cut, self.n_dev, self.layout = ctx, cut, n_dev, layout
        raw = pm.RAW[type]
        pools = [rng.integers(0, 256, size=int(np.prod((P,) + shape)) * np.dtype(raw).itemsize, dtype=np.uint8).view(raw).reshape((P,) + shape)
                 for _ in range(n_pools)]
        self.pools = [split(ctx, p, type, cut, n_dev, layout) for p in pools]
        self.model = pm.Cache(S, Bl, P, T, pools)
        self.table, self.lengths, self.refs = (whole(ctx, a) for a in (self.model.table, self.model.lengths, self.model.refs))
        self.cache = ctx.CreatePages(self.pools, self.table, self.lengths, self.refs, page_tokens=T)

    def ids(self, values):
        return whole(self.ctx, np.asarray(values, dtype=np.int32))

    def op(self, name, *args):
        getattr(self.cache, name.capitalize())(*[self.ids(a) for a in args])
        getattr(self.model, name)(*args)

    def tables(self):
        n = self.model
        return (self.ctx.ReadShard(self.table, 0, np.int32).reshape(n.S, n.B), self.ctx.ReadShard(self.lengths, 0, np.int32),
                self.ctx.ReadShard(self.refs, 0, np.int32))

    def check(self, pools=True):
        table, lengths, refs = self.tables()
        assert np.array_equal(lengths, self.model.lengths)
        assert np.array_equal(refs, self.model.refs)
        assert np.array_equal(table, self.model.table)
        for s, want in zip(self.pools, self.model.pools) if pools else ():
            got, pad = joined(self.ctx, s, want, self.cut, self.n_dev, self.layout)
            assert np.array_equal(got, want)
        assert self.cache.Status() == ([], int((self.model.refs > 0).sum()))

    def close(self):
        self.cache.Destroy()
        for s in self.pools + [self.table, self.lengths, self.refs]:
            self.ctx.Free(s)


CACHES = {
    # pages, tokens, rest of the page's shape, type, pools, devices, sharded dim
    "bf16 pages of 4 KiB, heads on 2 devices": dict(S=40, Bl=20, P=301, T=16, shape=(16, 4, 64), type="BF16", n_dev=2, cut=2),
    "odd pages of 21 bytes": dict(S=30, Bl=40, P=500, T=3, shape=(3, 7), type="U8", n_pools=3, cut=1),
    "one token and 12 bytes a page, uneven heads": dict(S=25, Bl=60, P=900, T=1, shape=(1, 3, 2), type="F16", n_dev=2, cut=2),
    "pages over a chunk, heads before tokens": dict(S=12, Bl=9, P=70, T=5, shape=(5, 6, 100), type="F32", n_dev=3, cut=2,
                                                    layout=(3, 1, 2, 0)),
    "pages of 9 bytes": dict(S=20, Bl=30, P=400, T=3, shape=(3, 3), type="U8", n_pools=1, cut=1),
    "three segments of pages, 8-byte values": dict(S=300, Bl=50, P=9001, T=2, shape=(2, 1), type="F64", n_pools=1, cut=1),
}


@pytest.mark.parametrize("name", CACHES)
def test_a_run_of_page_operators(ctx, name):
    """Sequences come, grow, fork, end; pages are copied and compacted: after every call the tables, and at the end of
    every round the pages, are those of the model."""
    say("page operators: " + name)
    p = Pair(ctx, **CACHES[name], seed=len(name))
    m, rng = p.model, np.random.Generator(np.random.PCG64(7))
    for round in range(4):
        empty = rng.permutation(np.flatnonzero(m.lengths == 0))
        n = min(len(empty), m.S // 4)
        room = len(m.free_pages()) // max(1, 2 * n) * m.T
        p.op("extend", empty[:n], rng.integers(0, min(m.B * m.T, max(room, 1)) + 1, n))
        p.check(pools=False)
        live = np.flatnonzero(m.lengths > 0)
        # one token each: where the last page is full, a page each
        grow = [s for s in live if m.lengths[s] < m.B * m.T and
                (m.lengths[s] % m.T == 0 or m.refs[m.table[s, m.lengths[s] // m.T]] == 1)][:len(m.free_pages())]
        p.op("extend", grow, np.ones(len(grow), dtype=np.int32))
        p.check(pools=False)
        empty = rng.permutation(np.flatnonzero(m.lengths == 0))[:min(10, len(m.free_pages()))]
        if len(live):
            p.op("fork", rng.choice(live, len(empty)), empty)
        p.check()
        p.op("free", rng.permutation(np.flatnonzero(m.lengths > 0))[::2])
        p.check(pools=False)
        used, free = np.flatnonzero(m.refs > 0), m.free_pages()
        n = min(len(used), len(free), 40)
        if n:
            p.op("copy", np.append(rng.choice(used, n - 1), used[0]), rng.permutation(free)[:n])
        p.check()
        p.op("compact")
        p.check()
        p.op("compact")  # nothing left to move
        p.check()
    p.op("free", np.arange(m.S))
    assert (m.refs == 0).all()
    p.check()
    p.close()


def test_few_and_many_entries(ctx):
    """No entries, one, and more than a workgroup has threads; rows that fill exactly; a pool given out to its last page."""
    p = Pair(ctx, S=3000, Bl=4, P=6000, T=4, shape=(4, 1, 1), type="U8", n_pools=1, seed=3)
    for name, args in (("extend", ([], [])), ("fork", ([], [])), ("free", ([],)), ("copy", ([], []))):
        p.op(name, *args)
    p.check()
    rng = np.random.Generator(np.random.PCG64(3))
    p.op("extend", rng.permutation(2000), np.tile([16, 0, 5, 1, 7], 400))  # up to full rows, 2000 + 1200 + ... pages
    p.check()
    left = len(p.model.free_pages())
    p.op("fork", np.full(left % 900 + 100, 7), 2000 + np.arange(left % 900 + 100))
    p.check()
    p.op("free", rng.permutation(3000))
    p.check()
    p.op("extend", np.arange(1500), np.full(1500, 16))  # every page
    assert not len(p.model.free_pages())
    p.check()
    p.op("compact")
    p.check()
    p.close()


def test_rows_longer_than_a_workgroup(ctx):
    p = Pair(ctx, S=6, Bl=5000, P=9000, T=1, shape=(1, 1), type="U8", n_pools=1, seed=5)
    p.op("extend", [1, 4], [3000, 4321])
    p.op("fork", [4, 1], [0, 2])
    p.op("free", [4])
    p.op("compact")
    p.check()
    p.op("free", [1, 2, 0])
    p.check()
    p.close()


BAD = [
    ("extend", ([0, 99], [1, 1]), {"BAD_SEQUENCE"}),
    ("extend", ([0, -2], [1, 1]), {"BAD_SEQUENCE"}),
    ("extend", ([3, 4, 3], [1, 1, 1]), {"REPEATED"}),
    ("extend", ([3], [-1]), {"TOO_LONG"}),
    ("extend", ([3], [33]), {"TOO_LONG"}),
    ("extend", ([0], [2 ** 31 - 1]), {"TOO_LONG"}),
    ("extend", ([3, 4, 5], [32, 32, 32]), {"OUT_OF_PAGES"}),
    ("fork", ([0, 0], [3, 99]), {"BAD_SEQUENCE"}),
    ("fork", ([-5], [3]), {"BAD_SEQUENCE"}),
    ("fork", ([0, 1], [3, 3]), {"REPEATED"}),
    ("fork", ([0], [1]), {"NOT_EMPTY"}),
    ("fork", ([0], [0]), {"NOT_EMPTY"}),
    ("copy", ([0, 1], [20, 20]), {"REPEATED"}),
    ("copy", ([0, 20], [20, 21]), {"OVERLAP"}),
    ("copy", ([0, 1], [1, 0]), {"OVERLAP"}),
    ("copy", ([0, 24], [20, 21]), {"BAD_PAGE"}),
    ("copy", ([0, 1], [-2, 21]), {"BAD_PAGE"}),
    ("copy", ([0, -1], [22, 21]), {"BAD_PAGE"}),
]


@pytest.mark.parametrize("name,args,flags", BAD, ids=["%s %s" % (n, sorted(f)[0]) + str(i) for i, (n, _, f) in enumerate(BAD)])
def test_a_call_with_a_bad_entry_changes_nothing(ctx, name, args, flags):
    p = Pair(ctx, S=8, Bl=8, P=24, T=4, shape=(4, 2, 8), type="BF16", seed=9)
    p.op("extend", [0, 1], [13, 20])
    say("%s %s" % (name, args))
    getattr(p.cache, name.capitalize())(*[p.ids(a) for a in args])
    got, used = p.cache.Status()
    assert set(got) == flags and used == 9
    p.check()  # the status is cleared, and everything is as it was
    p.op("fork", [0, 1, 0], [2, 3, 4])  # and the marks of the refused call are gone
    p.op("copy", [0], [23])
    p.check()
    p.close()


def test_free_takes_a_sequence_once_and_skips_bad_entries(ctx):
    p = Pair(ctx, S=8, Bl=8, P=24, T=4, shape=(4, 2, 8), type="BF16", seed=9)
    p.op("extend", [0, 1, 2], [13, 20, 4])
    p.cache.Free(p.ids([1, 99, 1, 5, -2, 1]))
    p.model.free([1])
    got, used = p.cache.Status()
    assert got == ["BAD_SEQUENCE"] and used == 5
    p.check()
    p.close()


def test_entries_that_are_none_are_passed_over(ctx):
    """A batch smaller than the arrays: MMR_PAGES_NONE stands where there is no entry, whatever stands beside it."""
    none = B.MMR_PAGES_NONE
    p = Pair(ctx, S=8, Bl=8, P=40, T=4, shape=(4, 2, 8), type="BF16", seed=9)
    p.cache.Extend(p.ids([none, 0, none, 1, 2, none]), p.ids([99999, 13, -7, 20, 4, 1]))
    p.model.extend([0, 1, 2], [13, 20, 4])
    p.check()
    p.cache.Fork(p.ids([99, 0, -4]), p.ids([none, 3, none]))
    p.model.fork([0], [3])
    p.check()
    p.cache.Copy(p.ids([0, 1, -9]), p.ids([30, none, none]))
    p.model.copy([0], [30])
    p.cache.Copy(p.ids([0, -9] * 18 + [2]), p.ids([none, none] * 18 + [31]))
    p.model.copy([2], [31])
    p.cache.Free(p.ids([none, 2, none]))
    p.model.free([2])
    p.check()
    k = values(np.random.Generator(np.random.PCG64(1)), (5, 2, 8), "BF16")
    p.cache.Write(p.ids([none, 1, none]), p.ids([0, 2, 3, 5]), 0, split(ctx, k, "BF16", 1, 1))
    p.model.pools[0][p.model.table[1, 4], 3] = k[2]
    p.check()
    for call in (p.cache.Extend, p.cache.Fork, p.cache.Copy):
        call(p.ids([0, 1]), p.ids([none, none])) if call != p.cache.Extend else call(p.ids([none, none]), p.ids([0, 1]))
    p.check()
    p.close()


def test_calls_from_two_threads(ctx):
    """Two threads on one cache: every call is whole, whichever comes first."""
    import threading
    p = Pair(ctx, S=64, Bl=8, P=400, T=4, shape=(4, 8), type="BF16", n_pools=1, seed=9)
    ids = [[p.ids([s, s + 1]) for s in range(t * 32, t * 32 + 32, 2)] for t in range(2)]
    counts = p.ids([6, 9])

    def work(t):
        for a in ids[t]:
            p.cache.Extend(a, counts)
        for a in ids[t][::2]:
            p.cache.Free(a)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    table, lengths, refs = p.tables()
    want = np.array([0 if s // 2 % 2 == 0 else (6, 9)[s % 2] for s in range(64)])
    assert np.array_equal(lengths, want)
    held = np.concatenate([table[s, :p.model.blocks(n)] for s, n in enumerate(want)])
    assert len(set(held)) == len(held) and refs.sum() == len(held) and (refs[held] == 1).all()
    assert p.cache.Status() == ([], len(held))
    p.close()


def test_a_shared_tail_is_not_extended(ctx):
    p = Pair(ctx, S=4, Bl=8, P=24, T=4, shape=(4, 8), type="BF16", seed=9)
    p.op("extend", [0], [6])
    p.model.refs[1] = 2  # somebody else keeps the partly filled page
    ctx.AssembleShards(p.refs.shape, 0, p.model.refs.view(np.uint8), existing_store=p.refs)
    p.cache.Extend(p.ids([0]), p.ids([1]))
    assert p.cache.Status() == (["SHARED_TAIL"], 2)
    p.op("extend", [0], [0])  # nothing is written
    p.check()
    p.close()


def test_pages_beyond_four_gigabytes(ctx):
    """Offsets of pages past 2^32 bytes."""
    P, page = 70001, 65536
    pool = ctx.CreateStore(mm.sharded_shape("U8", [(P, 1, 0), (16, 1, 1), (4096, 1, 2)], 0, 1))
    tables = [whole(ctx, np.zeros(s, np.int32)) for s in ((4, 4), (4,), (P,))]
    cache = ctx.CreatePages([pool], *tables, page_tokens=16)
    pattern = np.random.Generator(np.random.PCG64(1)).integers(0, 256, page, dtype=np.uint8)
    ctx.AssembleShards(pool.shape, 0, pattern, existing_store=pool)
    say("copy to page %d and back" % (P - 1))
    cache.Copy(whole(ctx, np.array([0], np.int32)), whole(ctx, np.array([P - 1], np.int32)))
    cache.Copy(whole(ctx, np.array([P - 1], np.int32)), whole(ctx, np.array([2], np.int32)))
    out = np.empty(3 * page, np.uint8)
    B.check(B.load().mmr_store_read_shard(ctx._h, pool._h, 0, out.ctypes.data, out.nbytes))
    assert np.array_equal(out, np.concatenate([pattern, np.zeros(page, np.uint8), pattern]))
    assert cache.Status() == ([], 0)
    cache.Destroy()
    for s in [pool] + tables:
        ctx.Free(s)
    ctx.ClearStoreCache()


# ---------------------------------------------------------------- rotary positions

def values(rng, shape, type):
    return pm.to_bits(rng.standard_normal(shape, dtype=np.float32), type)


def compare(got, want, size, type, magnitude=1.0):
    err = np.abs(pm.from_bits(got, type) - want)
    tol = pm.tolerance(want, size, type, magnitude)
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (worst, err[worst], tol[worst])


PARTS = dict(scaling="parts", factor=8.0, original_positions=4096, low_turns=1.0, high_turns=32.0)
ROTARY = [
    # shape, seq dim, sharded dim, devices, layout, rotary dim, interleaved, type, scaling, magnitude, offset
    ((2, 4, 37, 128), 2, 2, 4, None, 128, False, "BF16", {}, 1.0, 0),
    ((2, 37, 5, 128), 1, 1, 3, None, 64, True, "F16", PARTS, 1.2, 0),
    ((3, 5, 64, 84), 2, 1, 2, None, 60, True, "F32", dict(scaling="linear", factor=4.0), 1.0, 1 << 20),
    ((33, 3, 48), 0, 0, 2, None, 16, False, "F32", {}, 0.5, -17),
    ((33, 3, 50), 0, 1, 3, None, 10, False, "BF16", {}, 1.0, 3),
    ((1, 70), 0, 0, 1, None, 70, True, "F16", {}, 1.0, 2 ** 31 - 1),
    ((5, 2, 9, 96), 2, 0, 2, (3, 1, 2, 0), 96, False, "BF16", {}, 1.0, -2 ** 31),
    ((4, 40, 128), 1, 1, 8, None, 128, True, "BF16", PARTS, 1.0, 100000),
    ((2, 19, 40, 24), 1, 2, 2, None, 24, False, "F16", {}, 1.0, 5),
    ((6, 3, 600), 0, 0, 2, None, 600, False, "F32", {}, 1.0, 0),
    ((6, 3, 1100), 0, 0, 1, None, 1100, False, "F32", dict(frequencies=True), 1.0, 9),
    ((7, 2, 2), 0, 0, 1, None, 2, False, "BF16", {}, 1.0, 0),
    # turned parts of 8, 4 and 2 bytes' multiples, rests of many and of few bytes
    ((9, 3, 40), 0, 0, 2, None, 40, False, "BF16", {}, 1.0, 0),
    ((9, 3, 45), 0, 1, 2, None, 12, False, "BF16", {}, 1.0, 100),
    ((9, 3, 21), 0, 0, 1, None, 20, True, "F16", {}, 1.0, 0),
    ((9, 3, 31), 0, 0, 1, None, 6, True, "F32", {}, 1.0, 0),
    ((9, 3, 31), 0, 0, 1, None, 28, False, "F32", {}, 1.0, 0),
    ((9, 3, 16), 0, 0, 1, None, 14, True, "BF16", {}, 1.0, 50),
    ((9, 3, 35), 0, 0, 1, None, 6, False, "F16", {}, 1.0, 50),
    ((40, 3, 16), 0, 0, 20, None, 16, False, "BF16", {}, 1.0, 0),   # 20 buffers: more than one launch takes
    ((1, 1, 8), 0, 0, 1, None, 8, True, "F16", {}, 1.0, 12345),
    ((300, 9, 32, 128), 1, 1, 3, None, 128, False, "BF16", {}, 1.0, 7),  # 22 MB
    ((2, 2100, 33, 128), 1, 2, 1, None, 128, False, "F32", {}, 1.0, 7),  # 71 MB: results past the caches, 33 heads
]


@pytest.mark.parametrize("case", ROTARY, ids=[str(i) for i in range(len(ROTARY))])
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_rotary_positions(ctx, case, backward, in_place):
    shape, seq_dim, cut, n_dev, layout, R, interleaved, type, scaling, magnitude, offset = case
    say("rotary %s backward %s in place %s" % (case, backward, in_place))
    rng = np.random.Generator(np.random.PCG64(abs(hash(str(case))) % 1000))
    x = values(rng, shape, type)
    sx = split(ctx, x, type, cut, n_dev, layout)
    out = sx if in_place else split(ctx, np.zeros_like(x), type, cut, n_dev, layout)
    before = joined(ctx, out, x, cut, n_dev, layout)[1]
    if "frequencies" in scaling:
        f = rng.uniform(-2, 2, R // 2)
        plan = ctx.CreateRotary(R, interleaved=interleaved, magnitude=magnitude, frequencies=f)
        freq = f.astype(np.longdouble)
    else:
        plan = ctx.CreateRotary(R, interleaved=interleaved, magnitude=magnitude, **scaling)
        freq = pm.frequencies(R, **scaling)
    ctx.ApplyRotary(plan, sx, out, seq_dim=seq_dim, offset=offset, backward=backward)
    got, pad = joined(ctx, out, x, cut, n_dev, layout)
    place = [1] * (len(shape) - 1)
    place[seq_dim] = shape[seq_dim]
    positions = (offset + np.arange(shape[seq_dim])).reshape(place)
    want, size = pm.turn(pm.from_bits(x, type), positions, freq, interleaved, magnitude, backward)
    compare(got, want, size, type, magnitude)
    assert np.array_equal(got[..., R:], x[..., R:])  # what is not turned passes bit for bit
    assert np.array_equal(pad, before)               # and padding is left alone
    if not in_place:
        assert np.array_equal(joined(ctx, sx, x, cut, n_dev, layout)[0], x)
        ctx.Free(out)
    ctx.Free(sx)
    plan.Destroy()


@pytest.mark.parametrize("rank,spread", [(1, "alike"), (1, "everywhere"), (2, "alike"), (2, "everywhere")])
@pytest.mark.parametrize("heads_first", [False, True])
def test_rotary_positions_from_a_store(ctx, rank, spread, heads_first):
    rng = np.random.Generator(np.random.PCG64(rank))
    batch, heads, seq, dim, n_dev = 3, 5, 22, 64, 4
    shape = (batch, heads, seq, dim) if heads_first else (batch, seq, heads, dim)
    at = 2 if heads_first else 1
    x = values(rng, shape, "F32")
    pos = rng.integers(-50, 100000, size=(seq,) if rank == 1 else (batch, seq), dtype=np.int32)
    sx, out = (split(ctx, v, "F32", at, n_dev) for v in (x, np.zeros_like(x)))
    if spread == "alike":
        ps = split(ctx, pos, "S32", rank - 1, n_dev)
    else:  # a copy on every device
        dims = [(n, 1, i) for i, n in enumerate(pos.shape)] + [(1, n_dev, rank)]
        d = mm.sharded_shape("S32", dims, 0, n_dev)
        ps = ctx.CreateStore(d)
        for k in range(n_dev):
            ctx.AssembleShards(d, k, pos.view(np.uint8).reshape(-1), existing_store=ps)
    plan = ctx.CreateRotary(dim)
    ctx.ApplyRotary(plan, sx, out, seq_dim=at, positions=ps)
    p = pos.reshape((1, seq) if rank == 1 else (batch, seq))
    p = p[:, None, :] if heads_first else p[:, :, None]
    want, size = pm.turn(pm.from_bits(x, "F32"), np.broadcast_to(p, shape[:-1]), pm.frequencies(dim))
    compare(joined(ctx, out, x, at, n_dev)[0], want, size, "F32")
    plan.Destroy()


def test_the_gradient_is_that_of_differences(ctx):
    """sum(w * rotary(x)) moved along single elements of x: the result is linear in x, so the central difference is exact
    but for rounding: two values of y within 2^-22 of sizes up to 8, divided by the step of 2."""
    rng = np.random.Generator(np.random.PCG64(4))
    shape, R = (9, 2, 40), 24
    x, w = rng.standard_normal(shape, dtype=np.float32), rng.standard_normal(shape, dtype=np.float32)
    plan = ctx.CreateRotary(R, interleaved=True, magnitude=1.5, **PARTS)

    def apply(v, backward=False):
        s, o = split(ctx, v.view(np.uint32), "F32", 0, 2), split(ctx, np.zeros(shape, np.uint32), "F32", 0, 2)
        ctx.ApplyRotary(plan, s, o, seq_dim=0, offset=777, backward=backward)
        y = joined(ctx, o, v.view(np.uint32), 0, 2)[0].view(np.float32).astype(np.float64)
        ctx.Free(s)
        ctx.Free(o)
        return y

    dx = apply(w, backward=True)
    for _ in range(25):
        at = tuple(rng.integers(0, n) for n in shape)
        up, down = x.copy(), x.copy()
        up[at] += 1
        down[at] -= 1
        step = float(up[at]) - float(down[at])
        diff = ((apply(up) - apply(down)) * w).sum() / step
        assert abs(diff - dx[at]) <= 2 * np.abs(w).max() * 2 * 8 * 2.0 ** -22, (at, diff, dx[at])
    # and the adjoint: <w, y(x)> = <dx, x>
    lhs, rhs = (apply(x) * w).sum(), (dx * x).sum()
    assert abs(lhs - rhs) <= x.size * 1.5 * 2.0 ** -22 * np.abs(x).max() * np.abs(w).max()


# ---------------------------------------------------------------- new tokens into pages

WRITE = [
    # heads, query heads, dim, rotary dim, interleaved, type, devices, layout, T, counts
    (8, 32, 128, 128, False, "BF16", 1, None, 16, [1] * 20),
    (4, 8, 64, 32, True, "F16", 2, None, 8, [17, 0, 1, 40]),
    (3, 6, 20, 20, False, "F32", 1, None, 5, [9, 1]),
    (2, 2, 96, 96, True, "BF16", 2, (3, 1, 2, 0), 4, [1, 1, 3]),
    (5, 5, 22, 6, True, "BF16", 3, None, 1, [3, 2]),
    (2, 4, 128, None, False, "BF16", 2, None, 16, [33, 1]),
    (3, 3, 7, None, False, "F8E4M3FN", 1, None, 3, [4, 5, 0]),
    (1, 16, 128, 128, False, "F16", 1, None, 64, [700]),
    (16, 24, 64, 64, False, "BF16", 8, None, 16, [1, 1, 1, 1, 1]),  # 24 buffers: more than one launch takes
    (2, 2, 32, 32, False, "F32", 1, None, 2, [1] * 130),            # more sequences than a wave has lanes
    (3, 3, 32, 16, True, "F32", 1, None, 2, [0, 2] * 70 + [0, 0, 5]),
]


@pytest.mark.parametrize("case", WRITE, ids=[str(i) for i in range(len(WRITE))])
@pytest.mark.parametrize("padding", [0, 3])
def test_new_tokens_are_turned_and_written(ctx, case, padding):
    heads, qheads, dim, R, interleaved, type, n_dev, layout, T, counts = case
    say("write %s padding %d" % (case, padding))
    rng = np.random.Generator(np.random.PCG64(len(counts)))
    n = len(counts)
    S, Bl = n + 2, -(-(max(counts) + 40) // T)
    p = Pair(ctx, S=S, Bl=Bl, P=S * Bl, T=T, shape=(T, heads, dim), type=type, n_pools=3, n_dev=n_dev, cut=2, layout=layout, seed=1)
    seqs = rng.permutation(S)[:n]
    p.op("extend", np.arange(S), rng.integers(0, 40, S))
    p.op("extend", seqs, counts)
    begins = padding + np.concatenate([[0], np.cumsum(counts)])
    tokens = int(begins[-1]) + padding
    raw = pm.RAW[type]
    some = lambda h: (rng.integers(0, 256, (tokens, h, dim), dtype=np.uint8) if raw == np.uint8 else values(rng, (tokens, h, dim), type))  # noqa: E731
    k, v, q = some(heads), some(heads), some(qheads)
    sk, sv = split(ctx, k, type, 1, n_dev), split(ctx, v, type, 1, n_dev)
    plan = ctx.CreateRotary(R, interleaved=interleaved, magnitude=1.25) if R else None
    if plan:
        sq, so = split(ctx, q, type, 1, n_dev), split(ctx, np.zeros_like(q), type, 1, n_dev)
        p.cache.Write(p.ids(seqs), p.ids(begins), 2, sk, 0, sv, rotary=plan, q=sq, q_out=so)
    else:
        p.cache.Write(p.ids(seqs), p.ids(begins), 2, sk, 0, sv)
    places = p.model.places(seqs, begins)
    positions = np.zeros(tokens, np.int64)
    for t, (pos, page, row) in places.items():
        positions[t] = pos
        p.model.pools[0][page, row] = v[t]
        p.model.pools[2][page, row] = k[t]
    if plan:
        freq = pm.frequencies(R)
        got = joined(ctx, p.pools[2], p.model.pools[2], 2, n_dev, layout)[0]
        want, size = pm.turn(pm.from_bits(k, type), positions[:, None], freq, interleaved, 1.25)
        for t, (pos, page, row) in places.items():
            compare(got[page, row], want[t], size[t], type, 1.25)
            assert np.array_equal(got[page, row][:, R:], k[t][:, R:])
            p.model.pools[2][page, row] = got[page, row]
        got = joined(ctx, so, q, 1, n_dev)[0]
        want, size = pm.turn(pm.from_bits(q, type), positions[:, None], freq, interleaved, 1.25)
        inside = sorted(places)
        compare(got[inside], want[inside], size[inside], type, 1.25)
        outside = [t for t in range(tokens) if t not in places]
        assert not got[outside].any()  # rows of padding are left as they were
        p.cache.Write(p.ids(seqs), p.ids(begins), 2, sk, rotary=plan, q=sq, q_out=sq)  # in place, and without values
        again = joined(ctx, sq, q, 1, n_dev)[0]
        assert np.array_equal(again[inside], got[inside]) and np.array_equal(again[outside], q[outside])
    p.check()  # every other row of every page is as it was
    p.close()


def test_bad_entries_of_a_write_are_skipped(ctx):
    p = Pair(ctx, S=6, Bl=4, P=12, T=4, shape=(4, 2, 16), type="BF16", seed=2)
    p.op("extend", [0, 1, 2], [5, 6, 3])
    p.model.table[1, 1] = 12  # outside the pool
    ctx.AssembleShards(p.table.shape, 0, p.model.table.view(np.uint8).reshape(-1), existing_store=p.table)
    rng = np.random.Generator(np.random.PCG64(2))
    k = values(rng, (12, 2, 16), "BF16")
    sk = split(ctx, k, "BF16", 1, 1)
    # sequence 0: its 2 last; an id outside; sequence 1: 3 of which 2 stand in the bad page; sequence 2: more than it holds
    p.cache.Write(p.ids([0, 6, 1, 2]), p.ids([0, 2, 4, 7, 12]), 1, sk)
    m = p.model
    m.pools[1][m.table[0, 0], 3], m.pools[1][m.table[0, 1], 0] = k[0], k[1]
    m.pools[1][m.table[1, 0], 3] = k[4]
    for i, t in enumerate((9, 10, 11)):
        m.pools[1][m.table[2, 0], i] = k[t]
    got, used = p.cache.Status()
    assert set(got) == {"BAD_SEQUENCE", "BAD_PAGE", "TOO_LONG"}
    p.check()
    p.close()


# ---------------------------------------------------------------- together

def test_a_prefill_mesh_hands_over_to_a_decode_mesh(ctx):
    """As they would be used: keys, values and queries of two prompts come from a mesh that shards the sequence, by a
    reshard, to one that shards the heads; they are turned, written, forked into beams, decoded on for some steps, beams
    end, the cache is compacted, and what every sequence then holds in its pages is what a contiguous cache would hold."""
    rng = np.random.Generator(np.random.PCG64(11))
    heads, qheads, dim, T, n_dev, layers = 4, 8, 64, 8, 2, 2
    S, Bl, P = 8, 12, 64
    type = "BF16"
    p = Pair(ctx, S=S, Bl=Bl, P=P, T=T, shape=(T, heads, dim), type=type, n_pools=2 * layers, n_dev=n_dev, cut=2, seed=4)
    plan = ctx.CreateRotary(dim)
    freq = pm.frequencies(dim)
    held = {s: [[] for _ in range(2 * layers)] for s in range(S)}  # what a contiguous cache holds: (values, sizes or None)

    def step(seqs, counts):
        p.op("extend", seqs, counts)
        begins = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        tokens = int(begins[-1])
        places = p.model.places(seqs, begins)
        position = np.array([places[t][0] for t in range(tokens)])
        for layer in range(layers):
            stores = []
            for h in (qheads, heads, heads):
                whole_ = values(rng, (tokens, h, dim), type)
                src = split(ctx, whole_, type, 0, 2, start=8)           # tokens over the prefill mesh, devices 8 and 9
                dst = split(ctx, np.zeros_like(whole_), type, 1, n_dev)  # heads over the decode mesh
                ctx.Reshard(src, dst)
                stores.append((whole_, dst))
            (q, sq), (k, sk), (v, sv) = stores
            p.cache.Write(p.ids(seqs), p.ids(begins), 2 * layer, sk, 2 * layer + 1, sv, rotary=plan, q=sq, q_out=sq)
            want, size = pm.turn(pm.from_bits(q, type), position[:, None], freq)
            compare(joined(ctx, sq, q, 1, n_dev)[0], want, size, type)
            want, size = pm.turn(pm.from_bits(k, type), position[:, None], freq)
            for j, s in enumerate(seqs):
                for t in range(begins[j], begins[j + 1]):
                    held[s][2 * layer].append((want[t], size[t]))
                    held[s][2 * layer + 1].append((pm.from_bits(v[t], type), None))
        # the model does not turn: it takes the pages as they are now, which are compared row by row at the end
        for i, s in enumerate(p.pools):
            p.model.pools[i][:] = joined(ctx, s, p.model.pools[i], 2, n_dev)[0]

    def fork(parents, children):
        p.op("fork", parents, children)
        for a, b in zip(parents, children):
            held[b] = [list(rows) for rows in held[a]]

    def free(seqs):
        p.op("free", seqs)
        for s in seqs:
            held[s] = [[] for _ in range(2 * layers)]

    step([0, 3], [21, 16])
    fork([0, 0, 3], [1, 2, 5])
    for _ in range(5):
        step([5, 0, 1, 2, 3], [1, 1, 1, 1, 1])
    free([0, 3])
    fork([2], [0])
    step([0, 2], [4, 1])
    free([1])
    p.op("compact")
    step([7], [9])
    p.check()
    pools = [joined(ctx, s, w, 2, n_dev)[0] for s, w in zip(p.pools, p.model.pools)]
    for s in range(S):
        assert p.model.lengths[s] == len(held[s][0])
        for i in range(2 * layers):
            for t, (want, size) in enumerate(held[s][i]):
                row = pools[i][p.model.table[s, t // T], t % T]
                if size is None:
                    assert np.array_equal(pm.from_bits(row, type), want)
                else:
                    compare(row, want, size, type)
    assert p.model.lengths.sum() > 0
    p.close()


def hip_graph_functions():
    hip = C.CDLL("libamdhip64.so.7")  # the runtime the library already loaded
    for name, args in (("hipStreamBeginCapture", [C.c_void_p, C.c_int]), ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]),
                       ("hipGraphInstantiate", [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]),
                       ("hipGraphLaunch", [C.c_void_p, C.c_void_p]), ("hipGraphExecDestroy", [C.c_void_p]),
                       ("hipGraphDestroy", [C.c_void_p])):
        getattr(hip, name).restype, getattr(hip, name).argtypes = C.c_int, args
    return hip


def test_a_scheduler_step_replays_from_a_hip_graph():
    """extend, write, fork, free, copy, compact and a rotation captured once, replayed with other arguments in the same
    arrays and eager calls in between; every replay gives what the model gives."""
    hip = hip_graph_functions()
    with mm.ReshardContext(0) as ctx:
        p = Pair(ctx, S=16, Bl=8, P=96, T=4, shape=(4, 2, 16), type="BF16", n_dev=2, cut=2, seed=6)
        rng = np.random.Generator(np.random.PCG64(6))
        names = ("seqs", "counts", "begins", "parents", "children", "ends", "src", "dst")
        n = dict(seqs=3, counts=3, begins=4, parents=2, children=2, ends=2, src=1, dst=1)
        arrays = {k: p.ids(np.zeros(n[k])) for k in names}
        tokens = 12
        k = values(rng, (tokens, 2, 16), "BF16")
        sk = split(ctx, k, "BF16", 1, 2)
        x = values(rng, (tokens, 2, 16), "F32")
        sx, so = split(ctx, x, "F32", 0, 2), split(ctx, np.zeros_like(x), "F32", 0, 2)
        plan = ctx.CreateRotary(16)
        stream = ctx.stream

        def issue():
            p.cache.Extend(arrays["seqs"], arrays["counts"])
            p.cache.Write(arrays["seqs"], arrays["begins"], 0, sk)
            p.cache.Fork(arrays["parents"], arrays["children"])
            p.cache.Free(arrays["ends"])
            p.cache.Copy(arrays["src"], arrays["dst"])
            p.cache.Compact()
            ctx.ApplyRotary(plan, sx, so, seq_dim=0, offset=3)

        ctx.Sync()
        allocations = ctx.stats["device_allocations"]
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        issue()
        with pytest.raises(mm.MmrError, match="capturing"):
            p.cache.Status()
        with pytest.raises(mm.MmrError, match="capturing"):
            ctx.CreateRotary(8)
        with pytest.raises(mm.MmrError, match="capturing"):
            ctx.CreatePages(p.pools, p.table, p.lengths, p.refs, page_tokens=4)
        graph, exe = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0 and graph.value
        assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        assert ctx.stats["device_allocations"] == allocations
        p.check()  # nothing has run
        m = p.model
        for replay in range(4):
            seqs = rng.permutation([s for s in range(16) if m.lengths[s] < 12])[:3]
            counts = rng.multinomial(10, [0.3, 0.3, 0.4])
            begins = 1 + np.concatenate([[0], np.cumsum(counts)])
            for name, v in (("seqs", seqs), ("counts", counts), ("begins", begins)):
                ctx.AssembleShards(arrays[name].shape, 0, np.asarray(v, np.int32).view(np.uint8), existing_store=arrays[name])
            m.extend(seqs, counts)
            for t, (pos, page, row) in m.places(seqs, begins).items():
                m.pools[0][page, row] = k[t]
            empty = rng.permutation(np.flatnonzero(m.lengths == 0))[:2]
            live = np.flatnonzero(m.lengths > 0)
            parents = rng.choice(live, 2)
            ends = rng.choice(live, 2, replace=False)
            for name, v in (("parents", parents), ("children", empty), ("ends", ends)):
                ctx.AssembleShards(arrays[name].shape, 0, np.asarray(v, np.int32).view(np.uint8), existing_store=arrays[name])
            m.fork(parents, empty)
            m.free(ends)
            src, dst = np.flatnonzero(m.refs > 0)[:1], m.free_pages()[-1:]
            for name, v in (("src", src), ("dst", dst)):
                ctx.AssembleShards(arrays[name].shape, 0, np.asarray(v, np.int32).view(np.uint8), existing_store=arrays[name])
            m.copy(src, dst)
            m.compact()
            x = values(rng, x.shape, "F32")
            for d in range(2):
                ctx.AssembleShards(sx.shape, d, np.ascontiguousarray(x[6 * d:6 * d + 6]).view(np.uint8).reshape(-1), existing_store=sx)
            say("graph replay %d" % replay)
            assert hip.hipGraphLaunch(exe, stream) == 0
            p.check()
            want, size = pm.turn(pm.from_bits(x, "F32"), 3 + np.arange(tokens)[:, None], pm.frequencies(16))
            compare(joined(ctx, so, x, 0, 2)[0], want, size, "F32")
            p.op("free", rng.permutation(np.flatnonzero(m.lengths > 0))[:1])  # eager, between the replays
            p.check()
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0


def test_stores_that_move_or_go(ctx):
    """A pool that was offloaded comes back elsewhere and the cache follows; while it is away, and once a store of the
    cache is freed, calls are refused."""
    p = Pair(ctx, S=4, Bl=4, P=16, T=4, shape=(4, 8, 16), type="BF16", n_dev=2, cut=2, seed=8)
    p.op("extend", [0], [6])
    ctx.OffloadDtoH([p.pools[1]])
    with pytest.raises(mm.MmrError, match="offloaded"):
        p.cache.Fork(p.ids([0]), p.ids([1]))
    taken = ctx.CreateStore(p.pools[1].shape, allocate_from_cache=True)  # takes the device buffer the offload gave up
    ctx.OffloadHtoD([p.pools[1]])
    p.op("fork", [0], [1])
    p.check()
    ctx.Free(taken)
    ctx.Free(p.lengths)
    with pytest.raises(mm.MmrError, match="lengths store .* was freed") as e:
        p.cache.Compact()
    assert e.value.status_name == "NOT_FOUND"


def test_two_contexts_at_once():
    """Caches of two contexts, calls in turn without waiting: neither disturbs the other."""
    with mm.ReshardContext(0) as a, mm.ReshardContext(0) as b:
        pairs = [Pair(c, S=32, Bl=10, P=250, T=4, shape=(4, 4, 64), type="BF16", seed=i) for i, c in enumerate((a, b))]
        for i in range(6):
            for p in pairs:
                empty = np.flatnonzero(p.model.lengths == 0)
                p.op("extend", empty[:3], [5 + i, 11, 1])
                p.op("fork", empty[:2], empty[3:5])
                p.op("free", [empty[0]])
                p.op("compact")
        for p in pairs:
            p.check()


REFUSALS = [
    ("pages of 0 tokens", lambda c, s: c.CreatePages([s["pool"]], s["table"], s["lengths"], s["refs"], page_tokens=0)),
    ("0 pools", lambda c, s: c.CreatePages([], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("same store", lambda c, s: c.CreatePages([s["pool"], s["pool"]], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("one of the tables", lambda c, s: c.CreatePages([s["refs"]], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("stores of their own", lambda c, s: c.CreatePages([s["pool"]], s["table"], s["refs"], s["refs"], page_tokens=4)),
    ("not S32", lambda c, s: c.CreatePages([s["pool"]], s["table"], s["lengths"], s["f32"], page_tokens=4)),
    ("rank 1, not 2", lambda c, s: c.CreatePages([s["pool"]], s["lengths"], s["lengths"], s["refs"], page_tokens=4)),
    ("lengths of 16", lambda c, s: c.CreatePages([s["pool"]], s["table"], s["refs"], s["lengths"], page_tokens=4)),
    ("not the 16 pages", lambda c, s: c.CreatePages([s["x"]], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("not the slowest", lambda c, s: c.CreatePages([s["inner"]], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("unsharded", lambda c, s: c.CreatePages([s["cutpages"]], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("spread over 2 devices", lambda c, s: c.CreatePages([s["pool"]], s["cuttable"], s["lengths"], s["refs"], page_tokens=4)),
    ("another context", lambda c, s: c.CreatePages([s["foreign"]], s["table"], s["lengths"], s["refs"], page_tokens=4)),
    ("entries, at most 4", lambda c, s: s["cache"].Free(s["many"])),
    ("entries, at most 16", lambda c, s: s["cache"].Copy(s["many"], s["many"])),
    ("sequences is null", lambda c, s: s["cache"].Free((0, 1))),
    ("4-byte aligned", lambda c, s: s["cache"].Free((1234561, 1))),
    ("pool 3 of 1", lambda c, s: s["cache"].Write(s["one"], s["two"], 3, s["k"])),
    ("not .pages", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["x3"])),
    ("type of the k store", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["kf32"])),
    ("rank 4, not", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["x"])),
    ("come together", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["k"], q=s["k"], rotary=s["plan"])),
    ("without a rotary plan", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["k"], q=s["k"], q_out=s["k"])),
    ("same pool", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["k"], 0, s["k"])),
    ("different devices|sharded differently", lambda c, s: s["cache"].Write(s["one"], s["two"], 0, s["k2"])),
    ("not even", lambda c, s: c.CreateRotary(7)),
    ("not even", lambda c, s: c.CreateRotary(0)),
    ("base", lambda c, s: c.CreateRotary(8, base=0.0)),
    ("base", lambda c, s: c.CreateRotary(8, base=float("nan"))),
    ("magnitude", lambda c, s: c.CreateRotary(8, magnitude=float("inf"))),
    ("factor", lambda c, s: c.CreateRotary(8, scaling="linear", factor=0.0)),
    ("parts from", lambda c, s: c.CreateRotary(8, scaling="parts", factor=2.0, original_positions=0, low_turns=1, high_turns=2)),
    ("parts from", lambda c, s: c.CreateRotary(8, scaling="parts", factor=2.0, original_positions=9, low_turns=2, high_turns=2)),
    ("not finite", lambda c, s: c.CreateRotary(2, frequencies=[float("inf")])),
    ("rows of 16", lambda c, s: c.ApplyRotary(s["wide"], s["x"], seq_dim=1)),
    ("turn F32", lambda c, s: c.ApplyRotary(s["plan"], s["table"], seq_dim=0)),
    ("rank 1, not", lambda c, s: c.ApplyRotary(s["plan"], s["refs"], seq_dim=0)),
    ("seq_dim 3", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=3)),
    ("seq_dim -1", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=-1)),
    ("different descriptors", lambda c, s: c.ApplyRotary(s["plan"], s["x"], s["x3"], seq_dim=1)),
    ("minor-most", lambda c, s: c.ApplyRotary(s["plan"], s["inner"], seq_dim=1)),
    ("last dim .* sharded", lambda c, s: c.ApplyRotary(s["plan"], s["cutrow"], seq_dim=0)),
    ("offset", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=1, offset=1 << 31)),
    ("and an offset", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=1, offset=1, positions=s["lengths"])),
    ("positions of 16, sequence of 5", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=1, positions=s["refs"])),
    ("not S32", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=1, positions=s["f32"])),
    ("take dim 0", lambda c, s: c.ApplyRotary(s["plan"], s["x"], seq_dim=0, positions=s["table"])),
    ("another part of the sequence|on 1 devices", lambda c, s: c.ApplyRotary(s["plan"], s["xcut"], seq_dim=1, positions=s["five"])),
    ("another part of the sequence", lambda c, s: c.ApplyRotary(s["plan"], s["quad"], seq_dim=1, positions=s["crossed"])),
    ("another context", lambda c, s: c.ApplyRotary(s["plan"], s["foreign"], seq_dim=0)),
]


def test_calls_that_the_host_refuses():
    """Every refusal by its message; none of them launches anything."""
    with mm.ReshardContext(0) as c, mm.ReshardContext(0) as other:
        z = lambda *s: np.zeros(s, np.int32)  # noqa: E731
        h = lambda *s: np.zeros(s, np.uint16)  # noqa: E731
        s = dict(table=whole(c, z(4, 5)), lengths=whole(c, z(4)), refs=whole(c, z(16)), f32=whole(c, z(16), "F32"),
                 many=whole(c, z(17)), one=whole(c, z(1)), two=whole(c, z(2)), five=whole(c, z(5)),
                 pool=whole(c, h(16, 4, 2, 16), "BF16"), x=whole(c, h(3, 5, 2, 16), "BF16"), x3=whole(c, h(3, 5, 16), "BF16"),
                 k=whole(c, h(9, 2, 16), "BF16"), kf32=whole(c, np.zeros((9, 2, 16), np.uint32), "F32"),
                 k2=split(c, h(9, 2, 16), "BF16", 1, 2), inner=split(c, h(16, 4, 2), "BF16", 1, 1, (0, 1, 2)),
                 cutpages=split(c, h(16, 4, 2), "BF16", 0, 2), cuttable=split(c, z(4, 5), "S32", 0, 2),
                 cutrow=split(c, h(16, 4, 16), "BF16", 2, 2), xcut=split(c, h(3, 5, 2, 16), "BF16", 1, 2),
                 foreign=whole(other, h(16, 4, 2, 16), "BF16"), plan=c.CreateRotary(16), wide=c.CreateRotary(18))
        # the two tiles of the sequence in the other order: 2 x 2 devices, the sequence the major digit here, the minor one there
        s["quad"] = c.CreateStore(mm.sharded_shape("BF16", [(3, 1, 0), (6, 2, 1), (2, 2, 2), (16, 1, 3)], 0, 4))
        s["crossed"] = c.CreateStore(mm.sharded_shape("S32", [(6, 2, 1), (1, 2, 0)], 0, 4))
        s["cache"] = c.CreatePages([s["pool"]], s["table"], s["lengths"], s["refs"], page_tokens=4)
        c.Sync()
        launches = c.stats["kernel_launches"]
        for match, call in REFUSALS:
            with pytest.raises(mm.MmrError, match=match) as e:
                call(c, s)
            assert e.value.status_name in ("INVALID_ARGUMENT", "UNSUPPORTED")
        assert c.stats["kernel_launches"] == launches
        for call, error in ((lambda: s["cache"].Free([0]), TypeError), (lambda: s["cache"].Free(np.zeros(1, np.int32)), TypeError),
                            (lambda: s["cache"].Free(s["table"]), ValueError), (lambda: s["cache"].Free(s["f32"]), ValueError),
                            (lambda: s["cache"].Free(whole(other, z(1))), ValueError),
                            (lambda: s["cache"].Extend(s["one"], s["two"]), ValueError),
                            (lambda: s["cache"].Write(s["one"], s["one"], 0, s["k"]), ValueError),
                            (lambda: c.CreateRotary(8, frequencies=[1.0]), ValueError)):
            with pytest.raises(error):
                call()
        assert s["cache"].Status() == ([], 0)


def test_layout_and_stream_of_the_caller(ctx):
    """A context on a caller's stream, ids as (address, entries)."""
    hip = C.CDLL("libamdhip64.so.7")
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    with mm.ReshardContext(0, hip_stream=stream.value) as c:
        p = Pair(c, S=6, Bl=6, P=30, T=4, shape=(4, 2, 8), type="F32", seed=1)
        seqs, counts = p.ids([2, 4, 0, 5]), p.ids([7, 3, 8, 1])
        at = c.SliceLocalShard(0, seqs), c.SliceLocalShard(0, counts)
        p.cache.Extend((at[0], 3), (at[1], 3))  # the first three
        p.model.extend([2, 4, 0], [7, 3, 8])
        p.cache.Free((at[0] + 4, 1))
        p.model.free([4])
        p.check()
    assert hip.hipStreamDestroy(stream) == 0
