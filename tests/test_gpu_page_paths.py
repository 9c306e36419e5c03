"""Page operators on the GPU where a call takes another form than small ones do (more launches, more segments of pages, more
chunks), on both sides of each limit, and on tables that are out of step with themselves."""
import numpy as np
import pytest

from test_gpu_pages import Pair, ctx, say  # noqa: F401  (ctx is the fixture)

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
