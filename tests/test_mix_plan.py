"""CPU: how the bf16 channel-mixing kernels divide their products, and that the GPU tests reach every way of doing it."""
import ctypes

import pytest

import mix_strict as M
from mappedconvolutions_b200 import _lib


def chosen(case):
    act = case[7] is not None or case[4]
    names = [p for p in M.PRODUCTS if (act or p != "act") and (case[4] or p not in ("gate", "weight_out"))]
    return {p: M.plan(_lib.lib(), M.path_desc(case), p, 148) for p in names}


@pytest.mark.parametrize("i", range(len(M.PATHS)))
def test_plans_of_the_tested_shapes(i):
    case, want = M.PATHS[i]
    got = chosen(case)
    assert {k: got[k][0] for k in want} == want


def test_every_way_is_reached():
    seen = {k: set() for k in ("layer", "gate", "act", "gate_bwd", "outer")}
    for case, _ in M.PATHS:
        for p, (way, work) in chosen(case).items():
            if p.startswith("weight"):
                seen["outer"].add((way, work > 12))  # more blocks of pixels than any ring of stages holds
                continue
            bn, tiles, group = way
            kind = "gate" if p == "gate" else "layer" if p != "act" else "gate_bwd" if case[4] else "act"
            stays = "travel" if group == 0 else "one" if tiles == 1 else "several tiles" if group > 1 else "several groups"
            seen[kind].add((bn, stays, work > 1))
    assert {(bn, "one", True) for bn in (64, 128, 256)} <= seen["layer"]
    assert {(bn, "one", True) for bn in (64, 256)} <= seen["act"]
    for kind in ("layer", "act"):
        assert {(256, "several tiles", True), (128, "several tiles", True), (256, "several groups", True),
                (256, "travel", True)} <= seen[kind]
    assert {(64, "one", True), (128, "several groups", True), (128, "travel", True)} <= seen["gate"]
    assert (64, "travel", True) in seen["gate_bwd"]
    assert {((r, c), True) for r in (256, 512) for c in (128, 256)} <= seen["outer"]


def test_more_channel_tiles_than_pairs_of_blocks():
    case = next(c for c, _ in M.PATHS if c[5] == 9700)
    (bn, tiles, group), work = chosen(case)["output"]
    assert tiles > 74 and group == 0 and work > 1


def test_refusals():
    L, v = _lib.lib(), (ctypes.c_int32 * 6)()
    d = lambda **k: _lib.McMixDesc(**{**dict(B=1, S=1000, C_in=8, C_out=8, hidden=0, act=1, dtype=_lib.MC_BF16, layout=0), **k})
    assert L.mc_mix_plan(d(), 0, 148, v) == 0
    for bad in (dict(B=0), dict(C_in=0), dict(hidden=-1), dict(act=9)):
        assert L.mc_mix_plan(d(**bad), 0, 148, v) == -1
    assert L.mc_mix_plan(d(dtype=_lib.MC_F32), 0, 148, v) == -2 and L.mc_mix_plan(d(S=1 << 31), 0, 148, v) == -6
    for product in (-1, 1, 5, 6):  # (a pointwise layer has no gate and no second weight)
        assert L.mc_mix_plan(d(), product, 148, v) == -1
    assert L.mc_mix_plan(d(act=0), 2, 148, v) == -1 and L.mc_mix_plan(d(act=0, hidden=8), 2, 148, v) == 0  # nor, without one, an activation's gradient
    assert L.mc_mix_plan(d(), 0, -1, v) == -1 and L.mc_mix_plan(d(), 0, 1, v) == -1 and L.mc_mix_plan(d(), 0, 148, None) == -1
