"""How products of 8-bit rows would run (tcx_hip_linear8_plan): the tile, the split of the
sums, the launches and the workspace. No kernel runs here."""

from __future__ import annotations

import ctypes

import pytest

import block8_ways as ways
import tensorcx_hip_capi as capi


def plan(rows, outputs, features, gated=False, **more):
    return capi.linear8_plan(capi.linear8_desc(rows, features, outputs), gated, **more)


def way(p):
    return p.tile_rows, p.tile_outputs, p.sets, p.units, p.splits > 1


def test_plan_refuses():
    desc, out = capi.linear8_desc(2, 300, 5), capi.Linear8Plan()
    raw = capi.lib().tcx_hip_linear8_plan
    assert raw(None, 0, 0, ctypes.byref(out)) == raw(ctypes.byref(desc), 0, 0, None) == capi.TCX_INVALID_ARGUMENT
    for sizes in ((0, 5, 300), (2, 0, 300), (2, 5, 0), (-1, 5, 300), (2, 5, 1 << 22), (1 << 30, 5, 300)):
        for gated in (False, True):
            with pytest.raises(capi.HipError) as error:
                plan(*sizes, gated)
            assert error.value.code == capi.TCX_INVALID_ARGUMENT


@pytest.mark.parametrize("gated,taken,shape", [(False, *x) for x in ways.flat(ways.LINEAR)] +
                         [(True, *x) for x in ways.flat(ways.GATED) + ways.flat(ways.GATED_ONE_LAUNCH)], ids=str)
def test_sizes_take_their_ways(gated, taken, shape):
    """The sizes that the GPU tests run are on the ways that they are there for."""
    p = plan(*shape, gated)
    assert way(p) == taken
    one_launch = (taken in ways.GATED_ONE_LAUNCH and shape in ways.GATED_ONE_LAUNCH[taken]) if gated else p.splits == 1
    assert p.launches == (1 if one_launch else 2)
    assert p.workspace_bytes == (0 if one_launch else p.splits * shape[0] * shape[1] * (2 if gated else 1) * 4)
    assert p.workspace_bytes == capi.linear8_workspace_bytes(capi.linear8_desc(shape[0], shape[2], shape[1]), gated)


def test_split_as_far_as_the_workspace_goes():
    for shape in ((100, 300, 8192), (64, 4096, 11264), (614, 1878, 7432), (5972, 674, 6026), (35, 16925, 2764)):
        full = plan(*shape)
        assert full.splits > 1
        for share in (2, 3, 10):
            part = plan(*shape, workspace_bytes=full.workspace_bytes // share)
            assert part.workspace_bytes <= full.workspace_bytes // share
        none = plan(*shape, workspace_bytes=0)
        assert (none.splits, none.launches, none.workspace_bytes) == (1, 1, 0)


def test_gated_plans_need_their_workspace():
    """A gated product runs one way: the workspace at hand does not change it."""
    for shape in ((16, 4500, 4000), (972, 2055, 6498), (100, 3000, 1000)):
        full, none = plan(*shape, True), plan(*shape, True, workspace_bytes=0)
        assert (way(full), full.splits, full.workspace_bytes) == (way(none), none.splits, none.workspace_bytes)
