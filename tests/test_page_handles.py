"""Handles that are gone, in arguments that may be left out: refused, not taken for left out (no GPU: the C entry points are
replaced by ones that note what they are given)."""
import ctypes as C
import weakref

import pytest

import multimesh_jax_amd as mm
from multimesh_jax_amd import api


class Noted:
    """Stands for the library: every entry point takes anything, notes it and reports success."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0
        return entry


def null(a):
    return a is None or (isinstance(a, C.c_void_p) and not a.value)


def context(monkeypatch):
    ctx = mm.ReshardContext.__new__(mm.ReshardContext)
    ctx._lib, ctx._h, ctx._handles, ctx.hip_device = Noted(), C.c_void_p(8), weakref.WeakSet(), 0
    monkeypatch.setattr(api.B, "load", lambda: ctx._lib)
    return ctx


def store(ctx, address):
    return api.StoreHandle(ctx, C.c_void_p(address), None, "s")


@pytest.fixture
def world(monkeypatch):
    ctx = context(monkeypatch)
    w = dict(ctx=ctx, cache=api.PageCache(ctx, C.c_void_p(16)), plan=api.RotaryPlan(ctx, C.c_void_p(24)),
             **{name: store(ctx, 32 + 8 * i) for i, name in enumerate(("k", "v", "q", "q_out", "x", "out", "positions"))})
    ctx._lib.calls.clear()
    yield w
    ctx._h = None


def write(w, **without):
    args = dict(v_pool=1, v=w["v"], rotary=w["plan"], q=w["q"], q_out=w["q_out"])
    args.update(without)
    w["cache"].Write((64, 1), (72, 2), 0, w["k"], **args)


def rotate(w, **more):
    args = dict(out=w["out"], seq_dim=1, positions=w["positions"])
    args.update(more)
    w["ctx"].ApplyRotary(w["plan"], w["x"], **args)


def test_what_is_given_arrives(world):
    write(world)
    rotate(world)
    (name, a), (name2, b) = world["ctx"]._lib.calls
    assert name == "mmr_pages_write" and [x.value for x in (a[0], a[5], a[7], a[8], a[9], a[10])] == [16, 32, 40, 24, 48, 56]
    assert name2 == "mmr_rotary_apply" and [x.value for x in (b[0], b[1], b[2], b[4])] == [24, 64, 72, 80]
    write(world, v=None, rotary=None, q=None, q_out=None)
    rotate(world, out=None, positions=None)
    a, b = (args for _, args in world["ctx"]._lib.calls[2:])
    assert all(null(a[i]) for i in (7, 8, 9, 10)) and b[2].value == b[1].value and null(b[4])


@pytest.mark.parametrize("call,gone", [(write, ["v"]), (write, ["plan"]), (write, ["q"]), (write, ["q_out"]), (write, ["q", "q_out"]),
                                       (write, ["k"]), (write, ["cache"]), (rotate, ["positions"]), (rotate, ["out"]), (rotate, ["x"]),
                                       (rotate, ["plan"])])
@pytest.mark.parametrize("how", ["freed", "closed"])
def test_what_is_gone_is_never_taken_for_left_out(world, monkeypatch, call, gone, how):
    """Freed or destroyed, or of another context that was closed: an error here, or null where the C entry point takes no null."""
    lib = world["ctx"]._lib
    if how == "closed":
        other = context(monkeypatch)
        for name in gone:
            world[name] = (api.RotaryPlan(other, C.c_void_p(80)) if name == "plan" else api.PageCache(other, C.c_void_p(80)) if name == "cache"
                           else store(other, 80))
            if name == "cache":
                world[name]._lib = lib
        other.close()
    else:
        for name in gone:
            if name in ("plan", "cache"):
                world[name].Destroy()
            else:
                world["ctx"].Free(world[name])
    lib.calls.clear()
    needed = {write: {"cache": 0, "k": 5}, rotate: {"plan": 0, "x": 1, "out": 2}}[call]
    if set(gone) <= set(needed):
        call(world)
        (_, args), = lib.calls
        assert all(null(args[needed[name]]) for name in gone)
    else:
        with pytest.raises(ValueError, match="freed|destroyed"):
            call(world)
        assert not lib.calls


def test_calls_after_the_context_is_closed(world):
    """Nothing that the context made reaches a C entry point."""
    ctx, cache, plan = world["ctx"], world["cache"], world["plan"]
    lib = ctx._lib
    ctx.close()
    ctx.close()
    assert [name for name, _ in lib.calls] == ["mmr_context_destroy"]
    lib.calls.clear()
    for call in (lambda: cache.Compact(), lambda: cache.Free((64, 1)), lambda: cache.Extend((64, 1), (72, 1)),
                 lambda: cache.Status(), lambda: cache.Destroy(), lambda: plan.Destroy(), lambda: ctx.Reshard(world["k"], world["v"])):
        call()
    assert len(lib.calls) == 7 and all(null(args[0]) for _, args in lib.calls)
    assert all(null(a) for a in lib.calls[-1][1])
