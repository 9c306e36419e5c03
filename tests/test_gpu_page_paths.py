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
