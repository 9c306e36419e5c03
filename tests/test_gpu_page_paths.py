"""Page operators on the GPU where a call takes another form than small ones do (more launches, more segments of pages, more
chunks), on both sides of each limit, and on tables that are out of step with themselves."""
import ctypes as C

import numpy as np
import pytest

import multimesh_jax_amd as mm

import page_model as pm
import test_gpu_pages as base
from test_gpu_pages import Pair, compare, ctx, say, split, values, whole  # noqa: F401  (ctx is the fixture)

pytestmark = pytest.mark.gpu


def put(p, name):
    """The model's table, lengths or refs, into the store."""
    p.ctx.AssembleShards(getattr(p, name).shape, 0, np.ascontiguousarray(getattr(p.model, name)).view(np.uint8).reshape(-1),
                         existing_store=getattr(p, name))


# the plan of a fork checks up to 4,096 places of the parents' rows itself and scans up to two segments of 4,096 pages
FORKS = {"the plan checks": dict(Bl=8, P=24), "a launch checks": dict(Bl=1500, P=24), "a launch checks and scans": dict(Bl=8, P=9001)}


@pytest.mark.parametrize("form", FORKS)
@pytest.mark.parametrize("page,id,users,flag", [(0, -1, 1, "BAD_PAGE"), (2, "P", 1, "BAD_PAGE"), (1, None, 0, "BAD_COUNT"),
                                                (3, None, 0, "BAD_COUNT"), (3, -9, 1, "BAD_PAGE")])
def test_a_fork_of_a_bad_row_changes_nothing(ctx, form, page, id, users, flag):  # noqa: F811
    """Sequence 1 holds three full pages and a partly filled one; one of them is not there, or has no user."""
    say("fork of a bad row, %s: page %d" % (form, page))
    p = Pair(ctx, S=8, T=4, shape=(4, 2, 8), type="BF16", seed=9, **FORKS[form])
    p.op("extend", [1, 0], [14, 9])
    row, refs = p.model.table.copy(), p.model.refs.copy()
    held = row[1, page]
    if id is not None:
        p.model.table[1, page] = p.model.P if id == "P" else id
    p.model.refs[held] = users
    put(p, "table")
    put(p, "refs")
    p.cache.Fork(p.ids([0, 1, 0]), p.ids([3, 4, 5]))
    assert p.cache.Status() == ([flag], int((p.model.refs > 0).sum()))
    p.check()
    p.model.table[:], p.model.refs[:] = row, refs
    put(p, "table")
    put(p, "refs")
    p.op("fork", [0, 1, 0], [3, 4, 5])  # and nothing of the refusal is left
    p.check()
    p.close()


# a compact of more than 16,384 pages lists its moves in a launch of its own, one of more than 8,192 scans in one
@pytest.mark.parametrize("P", [24, 9001, 20001])
@pytest.mark.parametrize("id,flag", [(0, "BAD_COUNT"), (5, "BAD_COUNT"), (7, "BAD_COUNT"), ("last", "BAD_COUNT"), ("P", "BAD_PAGE"), (-1, "BAD_PAGE")])
def test_a_compact_keeps_a_bad_id_and_tells(ctx, P, id, flag):  # noqa: F811
    """A row names a page that is not there, or that nobody uses, before and behind the pages in use."""
    say("compact of a bad row, %d pages: %s" % (P, id))
    p = Pair(ctx, S=8, Bl=6, P=P, T=4, shape=(4, 2, 8), type="BF16", seed=9)
    m = p.model
    for s, n, row in ((0, 14, [1, P - 2, 8, 3]), (3, 9, [P - 3, 6, P - 5]), (5, 4, [2])):
        m.lengths[s], m.table[s, :len(row)] = n, row
        m.refs[row] += 1
    for name in ("table", "lengths", "refs"):
        put(p, name)
    p.op("compact")
    p.check()
    m.refs[m.table[5, 0]] = 0  # sequence 5 names what is no longer its own
    for s, n, row in ((0, 14, [1, P - 2, 8, 3]), (3, 9, [P - 3, 6, P - 5])):
        m.table[s, :len(row)] = row
    m.refs[:] = 0
    m.refs[m.table[0, :4]] += 1
    m.refs[m.table[3, :3]] += 1  # 7 pages in use
    bad = {"P": P, "last": P - 1}.get(id, id)
    m.table[5, 0] = bad
    for name in ("table", "refs"):
        put(p, name)
    m.table[5, 0] = 0
    p.op("compact")
    m.table[5, 0] = bad
    assert p.cache.Status() == ([flag], 7)
    p.check()
    p.close()


def test_a_free_of_rows_out_of_step(ctx):  # noqa: F811
    """An id outside, a page that nobody uses, a page that more rows name than use it: told, and no count below zero."""
    p = Pair(ctx, S=8, Bl=6, P=24, T=4, shape=(4, 2, 8), type="BF16", seed=9)
    m = p.model
    p.op("extend", [0, 1, 2, 3], [8, 9, 12, 5])
    row = m.table.copy()
    m.table[0, 1] = 24
    m.refs[row[1, 0]] = 0
    m.table[2, 2] = m.table[3, 0]
    for name in ("table", "refs"):
        put(p, name)
    for seqs, flag in (([0], "BAD_PAGE"), ([1], "BAD_COUNT"), ([2, 3], "BAD_COUNT")):
        p.cache.Free(p.ids(seqs))
        for s in seqs:
            for page in m.table[s, :m.blocks(m.lengths[s])]:
                if page < 24 and m.refs[page] > 0:
                    m.refs[page] -= 1
            m.lengths[s] = 0
        assert p.cache.Status() == ([flag], int((m.refs > 0).sum()))
        p.check()
    p.close()


def adopted(c, type, shape, values, devices):
    """A store of `shape` whose devices[i] is the row of `values` that device i holds, every row in one buffer however many
    devices share it -> (the store, the store that owns the buffers)."""
    raw = np.ascontiguousarray(values)
    own = whole(c, raw.view(np.uint8).reshape(len(raw), -1), "U8")
    at, size = c.SliceLocalShard(0, own), raw[0].nbytes
    assert size % 16 == 0
    return c.AdoptShards(shape, [at + size * d for d in devices]), own


@pytest.mark.parametrize("replicas_major", [False, True])
@pytest.mark.parametrize("R,interleaved", [(16, False), (10, True)])
def test_replicas_in_one_buffer_are_turned_once(ctx, replicas_major, R, interleaved):  # noqa: F811
    """Two halves of a sequence on two devices each, both in the buffer of the half; in place, and into such a store."""
    rng = np.random.Generator(np.random.PCG64(5))
    digits = [(3, 1, 0), (14, 2, 1), (16, 1, 2), (1, 2, 3)] if not replicas_major else [(3, 1, 1), (14, 2, 2), (16, 1, 3), (1, 2, 0)]
    shape = mm.sharded_shape("BF16", digits, 0, 4)
    half_of = [0, 0, 1, 1] if not replicas_major else [0, 1, 0, 1]
    x = values(rng, (3, 14, 16), "BF16")
    halves = np.stack([x[:, :7], x[:, 7:]])
    sx, own = adopted(ctx, "BF16", shape, halves, half_of)
    so, own2 = adopted(ctx, "BF16", shape, np.zeros_like(halves), half_of)
    plan = ctx.CreateRotary(R, interleaved=interleaved, magnitude=1.5)
    ctx.ApplyRotary(plan, sx, so, seq_dim=1, offset=9)
    ctx.ApplyRotary(plan, sx, seq_dim=1, offset=9)
    want, size = pm.turn(pm.from_bits(x, "BF16"), 9 + np.arange(14)[None, :], pm.frequencies(R), interleaved, 1.5)
    for o in (own2, own):
        got = ctx.ReadShard(o, 0, np.uint16).reshape(halves.shape)
        got = np.concatenate([got[0], got[1]], 1)
        compare(got, want, size, "BF16", 1.5)
        assert np.array_equal(got[..., R:], x[..., R:])
    plan.Destroy()
    for s in (sx, so, own, own2):
        ctx.Free(s)


def test_queries_of_replicas_in_one_buffer_are_turned_once(ctx):  # noqa: F811
    p = Pair(ctx, S=4, Bl=4, P=16, T=4, shape=(4, 2, 16), type="BF16", n_pools=1, n_dev=2, cut=2, seed=3)
    p.op("extend", [2, 0], [5, 3])
    rng = np.random.Generator(np.random.PCG64(3))
    k, q = values(rng, (8, 2, 16), "BF16"), values(rng, (1, 8, 3, 16), "BF16")
    sq, own = adopted(ctx, "BF16", mm.sharded_shape("BF16", [(8, 1, 0), (3, 1, 1), (16, 1, 2), (1, 3, 3)], 0, 3), q, [0, 0, 0])
    plan = ctx.CreateRotary(16)
    p.cache.Write(p.ids([2, 0]), p.ids([0, 5, 8]), 0, split(ctx, k, "BF16", 1, 2), rotary=plan, q=sq, q_out=sq)
    position = np.append(np.arange(5), np.arange(3))
    want, size = pm.turn(pm.from_bits(q[0], "BF16"), position[:, None], pm.frequencies(16))
    compare(ctx.ReadShard(own, 0, np.uint16).reshape(8, 3, 16), want, size, "BF16")
    assert p.cache.Status() == ([], 3)
    p.close()


def test_tiles_that_lie_over_one_another_are_refused(ctx):  # noqa: F811
    """Two parts of an array in one buffer, or replicas that do not begin together, as a result or in place."""
    own = whole(ctx, np.zeros(4096, np.uint8), "U8")
    at = ctx.SliceLocalShard(0, own)
    parts = mm.sharded_shape("BF16", [(6, 2, 0), (2, 1, 1), (16, 1, 2)], 0, 2)     # 192 bytes each
    copies = mm.sharded_shape("BF16", [(3, 1, 0), (2, 1, 1), (16, 1, 2), (1, 2, 3)], 0, 2)
    plan = ctx.CreateRotary(16)
    ctx.Sync()
    launches = ctx.stats["kernel_launches"]
    for shape, ptrs in ((parts, [at, at]), (parts, [at, at + 176]), (copies, [at, at + 16]), (copies, [at + 176, at])):
        s = ctx.AdoptShards(shape, ptrs)
        apart = ctx.AdoptShards(shape, [at + 1024, at + 1024 + 192])
        for x in (s, apart):
            with pytest.raises(mm.MmrError, match="overlap") as e:
                ctx.ApplyRotary(plan, x, s, seq_dim=0)
            assert e.value.status_name == "INVALID_ARGUMENT"
        assert ctx.stats["kernel_launches"] == launches
        ctx.ApplyRotary(plan, s, apart, seq_dim=0)  # only read
        launches = ctx.stats["kernel_launches"]
        ctx.Free(s)
        ctx.Free(apart)
    plan.Destroy()


def test_queries_are_not_turned_into_the_keys_or_values(ctx):  # noqa: F811
    """They are read while the queries are written."""
    p = Pair(ctx, S=4, Bl=4, P=16, T=4, shape=(4, 2, 16), type="BF16", seed=3)
    p.op("extend", [2], [5])
    k, v = (split(ctx, values(np.random.Generator(np.random.PCG64(s)), (5, 2, 16), "BF16"), "BF16", 1, 1) for s in range(2))
    plan = ctx.CreateRotary(16)
    ctx.Sync()
    launches = ctx.stats["kernel_launches"]
    for q, q_out, what in ((k, k, "k"), (v, k, "k"), (v, v, "v"), (k, v, "v")):
        ids = p.ids([2]), p.ids([0, 5])
        with pytest.raises(mm.MmrError, match="q_out is also the %s store" % what) as e:
            p.cache.Write(*ids, 0, k, 1, v, rotary=plan, q=q, q_out=q_out)
        assert e.value.status_name == "INVALID_ARGUMENT"
    assert ctx.stats["kernel_launches"] == launches
    p.check()
    plan.Destroy()
    p.close()


@pytest.mark.parametrize("magnitude", [3.5e38, 1e300, -1.0, float("nan")])
def test_magnitudes_that_32_bits_do_not_hold_are_refused(ctx, magnitude):  # noqa: F811
    with pytest.raises(mm.MmrError, match="magnitude") as e:
        ctx.CreateRotary(8, magnitude=magnitude)
    assert e.value.status_name == "INVALID_ARGUMENT"
    ctx.CreateRotary(8, magnitude=3.4e38).Destroy()
    ctx.CreateRotary(8, magnitude=0.0).Destroy()


# ---------------------------------------------------------------- forms of the launches

def test_extend_in_two_launches(ctx):  # noqa: F811
    """More than 16,384 pages may be given out, so the tables are written by a launch of their own where it is more than
    4,096 pages, by the plan where it is not; too few pages for all, and a bad entry, change nothing."""
    p = Pair(ctx, S=6000, Bl=8, P=40000, T=4, shape=(4, 1, 4), type="U8", n_pools=1, seed=3)
    m, rng = p.model, np.random.Generator(np.random.PCG64(3))
    some = rng.permutation(6000)
    p.op("extend", some[:2500], rng.integers(0, 16, 2500))       # about 5,000 pages, in five segments and more
    p.check()
    p.op("free", some[:2500:3])
    p.op("extend", some[:5000], rng.integers(0, 16, 5000))       # more sequences than the launch has workgroups
    assert (m.refs > 0).sum() > 12000
    p.check()
    p.op("extend", rng.permutation(6000), np.ones(6000, int))    # a step of decoding: under 4,096 fresh pages
    p.check()
    for seqs, counts, flag in ((np.arange(6000), np.full(6000, 32) - m.lengths, "OUT_OF_PAGES"),
                               (np.append(np.arange(4000), 7), np.full(4001, 1), "REPEATED")):
        p.cache.Extend(p.ids(seqs), p.ids(counts))
        assert p.cache.Status() == ([flag], int((m.refs > 0).sum()))
        p.check()
    p.op("extend", [int(np.argmin(m.lengths))], [5])
    p.check()
    p.close()


def test_fork_and_compact_of_more_sequences_than_workgroups(ctx):  # noqa: F811
    p = Pair(ctx, S=11000, Bl=6, P=30000, T=4, shape=(4, 1, 5), type="U8", n_pools=2, seed=4)
    m, rng = p.model, np.random.Generator(np.random.PCG64(4))
    p.op("extend", np.arange(5000), rng.integers(0, 21, 5000))
    p.op("fork", rng.integers(0, 5000, 5500), 5000 + rng.permutation(6000)[:5500])
    p.check()
    p.op("free", rng.permutation(11000)[:6000])
    p.op("compact")  # lists its moves in a launch of its own
    p.check()
    p.close()


# page, as (tokens, rest): one of 14 pieces in a pool's buffer is more than 64 pairs may check in one launch
COPIES = {"few pairs of long pages": (140, (4, 7000, 2), 64), "by destination": (600, (4, 3), 100), "in the given order": (3000, (4, 3), 100),
          "by destination, more than one round": (9000, (4, 8), 3000), "in the given order, more than one round": (20000, (4, 8), 2000)}


@pytest.mark.parametrize("name", COPIES)
def test_copies_that_are_planned(ctx, name):  # noqa: F811
    """Copies that one launch does not check: results, entries that are none or copy a page onto itself, refusals."""
    P, shape, n = COPIES[name]
    p = Pair(ctx, S=4, Bl=4, P=P, T=4, shape=shape, type="U8", n_pools=2, seed=5)
    rng = np.random.Generator(np.random.PCG64(5))
    say("planned copy, " + name)
    ids = rng.permutation(P)
    dst, src = ids[:n], rng.choice(ids[n:], n)
    a, b = p.ids(src), p.ids(dst)
    before = ctx.stats["kernel_launches"]
    p.cache.Copy(a, b)
    p.model.copy(src, dst)
    assert ctx.stats["kernel_launches"] == before + 2  # the plan and the move
    p.check()
    src[3], dst[5], src[5] = dst[3], -1, P + 7  # onto itself; no entry
    p.cache.Copy(p.ids(src), p.ids(dst))
    on = dst >= 0
    p.model.copy(src[on], dst[on])
    p.check()
    for at, (s, d), flag in ((9, (src[9], dst[10]), "REPEATED"), (9, (dst[20], dst[9]), "OVERLAP"), (n - 1, (src[0], P), "BAD_PAGE"),
                             (0, (-1, dst[0]), "BAD_PAGE"), (n // 2, (P, dst[n // 2]), "BAD_PAGE")):
        a, b = src.copy(), dst.copy()
        a[at], b[at] = s, d
        p.cache.Copy(p.ids(a), p.ids(b))
        assert p.cache.Status() == ([flag], 0)
        p.check()
    p.op("copy", src[on][::-1].copy(), dst[on][::-1].copy())  # and no mark is left
    p.check()
    p.close()


@pytest.mark.parametrize("bytes", [20000, 20007, 8192, 8200])
def test_pages_of_several_pieces_beside_small_ones(ctx, bytes):  # noqa: F811
    """Fork, copy (in one launch and planned) and compact of pools whose pages are more than one 8-KiB piece, with a pool of
    small pages in the same cache."""
    P, T = 90, 1
    p = Pair(ctx, S=20, Bl=8, P=P, T=T, shape=(T, bytes), type="U8", n_pools=2, seed=6)
    rng = np.random.Generator(np.random.PCG64(6))
    p.cache.Destroy()
    for size in (48, 7):
        small = rng.integers(0, 256, (P, T, size), dtype=np.uint8)
        p.model.pools.append(small)
        p.pools.append(split(ctx, small.copy(), "U8", 1, 1))
    p.cache = ctx.CreatePages(p.pools, p.table, p.lengths, p.refs, page_tokens=T)
    m = p.model
    p.op("extend", [0, 1, 2], [8, 5, 7])
    p.op("copy", [0, 9, 12], [60, 70, 89])
    p.check()
    p.op("copy", np.arange(20).repeat(4)[:70], 20 + np.arange(70))
    p.check()
    p.op("fork", [1, 1, 0], [4, 5, 6])
    p.op("free", [0, 1])
    p.op("compact")
    p.check()
    p.close()
    # partly filled pages: a fork copies one a child
    p = Pair(ctx, S=9, Bl=4, P=30, T=3, shape=(3, bytes), type="U8", n_pools=1, seed=7)
    p.op("extend", [0, 1], [8, 4])
    p.op("fork", [0, 1, 1], [4, 5, 6])
    p.check()
    p.close()


def test_more_pieces_than_workgroups(ctx):  # noqa: F811
    """264,000 pieces; a launch has 262,144 workgroups, which then loop."""
    P, n, words = 66000, 33000, 129 * 4
    page = lambda i: (np.arange(P * words, dtype=np.uint32) * np.uint32(2654435761) + np.uint32(i * 977)).reshape(P, 1, words)  # noqa: E731
    pools = []
    for i in range(8):
        pools.append(split(ctx, page(i), "U32", 1, 1))
    tables = [whole(ctx, np.zeros(s, np.int32)) for s in ((4, 4), (4,), (P,))]
    cache = ctx.CreatePages(pools, *tables, page_tokens=1)
    rng = np.random.Generator(np.random.PCG64(8))
    ids = rng.permutation(P).astype(np.int32)
    say("a copy of 264,000 pieces")
    cache.Copy(whole(ctx, ids[:n]), whole(ctx, ids[n:]))
    assert cache.Status() == ([], 0)
    for i, s in enumerate(pools):
        want = page(i)
        want[ids[n:]] = want[ids[:n]]
        assert np.array_equal(ctx.ReadShard(s, 0, np.uint32).reshape(want.shape), want)
    cache.Destroy()
    for s in pools + tables:
        ctx.Free(s)
    ctx.ClearStoreCache()


def turned(ctx, case, backward, seed, launches=None):  # noqa: F811
    shape, seq_dim, cut, n_dev, layout, R, interleaved, type, scaling, magnitude, offset = case
    rng = np.random.Generator(np.random.PCG64(seed))
    x = values(rng, shape, type)
    sx, out = split(ctx, x, type, cut, n_dev, layout), split(ctx, np.zeros_like(x), type, cut, n_dev, layout)
    more, freq = dict(scaling), None
    if more.pop("frequencies", False):
        more["frequencies"] = rng.uniform(-2, 2, R // 2)
        freq = more["frequencies"].astype(np.longdouble)
    plan = ctx.CreateRotary(R, interleaved=interleaved, magnitude=magnitude, **more)
    before = ctx.stats["kernel_launches"]
    ctx.ApplyRotary(plan, sx, out, seq_dim=seq_dim, offset=offset, backward=backward)
    assert launches is None or ctx.stats["kernel_launches"] == before + launches
    place = [1] * (len(shape) - 1)
    place[seq_dim] = shape[seq_dim]
    got = base.joined(ctx, out, x, cut, n_dev, layout)[0]
    want, size = pm.turn(pm.from_bits(x, type), (offset + np.arange(shape[seq_dim])).reshape(place),
                         pm.frequencies(R, **scaling) if freq is None else freq, interleaved, magnitude, backward)
    compare(got, want, size, type, magnitude)
    assert np.array_equal(got[..., R:], x[..., R:])
    plan.Destroy()
    for s in (sx, out):
        ctx.Free(s)


@pytest.mark.parametrize("i", range(len(base.ROTARY)))
def test_rotary_positions_of_fixed_values(ctx, i):  # noqa: F811
    turned(ctx, base.ROTARY[i], i % 2 == 1, 100 + i)


@pytest.mark.parametrize("n_dev,launches", [(8, 1), (9, 1), (24, 1), (25, 2), (60, 3)])
@pytest.mark.parametrize("type,R", [("BF16", 16), ("F32", 6)])
def test_rotary_positions_on_many_devices(ctx, n_dev, launches, type, R):  # noqa: F811
    """A launch takes 24 buffers."""
    turned(ctx, ((n_dev * 3 - 2, 3, 16), 0, 0, n_dev, None, R, False, type, {}, 1.0, 5), False, n_dev, launches)


MIXED = [
    (2, 4, 32, 32, False, "BF16", 1, None, 16, [512] + [1] * 300),              # a prompt beside a step of decoding
    (2, 4, 32, 16, True, "F16", 2, None, 8, [1] * 90 + [70, 1, 1, 0, 33] + [1] * 90),
    (9, 9, 16, 16, False, "F32", 9, None, 4, [5, 1, 1]),                        # 27 buffers: two launches
    (30, 60, 8, 8, True, "BF16", 30, None, 4, [2, 1, 9]),
]


@pytest.mark.parametrize("i", range(len(MIXED)))
@pytest.mark.parametrize("padding", [0, 3])
def test_prompts_and_single_tokens_in_one_write(ctx, i, padding):  # noqa: F811
    base.test_new_tokens_are_turned_and_written(ctx, MIXED[i], padding)


@pytest.mark.parametrize("form", ["a launch checks", "a launch checks and scans"])
def test_the_longer_forms_replay_from_a_hip_graph(form):
    """fork with its check in a launch of its own, a planned copy and a compact, captured once: replays that are carried out
    and one whose fork is refused for a bad row, with eager calls in between."""
    hip = base.hip_graph_functions()
    with mm.ReshardContext(0) as c:
        size = dict(FORKS[form])
        size["P"] = max(size["P"], 400)
        p = Pair(c, S=24, T=4, shape=(4, 2, 8), type="BF16", seed=9, **size)
        m, rng = p.model, np.random.Generator(np.random.PCG64(9))
        p.op("extend", np.arange(6), [14, 9, 20, 1, 16, 7])
        arrays = {k: p.ids(np.zeros(n)) for k, n in dict(parents=3, children=3, src=70, dst=70).items()}
        c.Sync()
        graph, exe = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(c.stream, 0) == 0
        p.cache.Fork(arrays["parents"], arrays["children"])
        p.cache.Copy(arrays["src"], arrays["dst"])
        p.cache.Compact()
        assert hip.hipStreamEndCapture(c.stream, C.byref(graph)) == 0 and graph.value
        assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        for replay in range(4):
            parents, children = rng.choice(np.flatnonzero(m.lengths > 0), 3), np.flatnonzero(m.lengths == 0)[:3]
            if replay == 2:
                parents[1] = 0
            ids = rng.permutation(np.arange(100, 400))
            for name, v in (("parents", parents), ("children", children), ("src", ids[70:140]), ("dst", ids[:70])):
                c.AssembleShards(arrays[name].shape, 0, np.asarray(v, np.int32).view(np.uint8), existing_store=arrays[name])
            say("graph of the longer forms, %s, replay %d" % (form, replay))
            if replay == 2:  # the first, full page of one parent is not there
                held = m.table[0, 0]
                m.table[0, 0] = m.P
                put(p, "table")
            assert hip.hipGraphLaunch(exe, c.stream) == 0
            if replay == 2:
                m.table[0, 0] = held
                m.copy(ids[70:140], ids[:70])
                m.compact()
                assert p.cache.Status()[0] == ["BAD_PAGE"]
                assert p.tables()[0][0, 0] == m.P  # compact leaves it too; the page itself is where the model has it
                put(p, "table")
            else:
                m.fork(parents, children)
                m.copy(ids[70:140], ids[:70])
                m.compact()
            p.check()
            p.op("free", [int(np.flatnonzero(m.lengths > 0)[-1])])  # eager, between the replays
            p.check()
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0
