"""Work-item tables of the score-rule attention, on the CPU: every visible (query, key) pair is covered by exactly one work
item, no item leaves its segment, forward and backward forms, whole and cut sweeps; refusals of the builders."""
import ctypes as C

import numpy as np
import pytest

from long_vita_amd import _lib

I32P = C.POINTER(C.c_int32)


def table(cu, causal, band, prefix, backward, piece):
    cu = np.asarray(cu, np.int32)
    pre = None if prefix is None else np.asarray(prefix, np.int32)
    pp = None if pre is None else pre.ctypes.data_as(I32P)
    nc, ws = C.c_int(0), C.c_int(0)
    fn = _lib.lib().lv_build_score_blocks

    def call(d, nd, c, ncb):
        return _lib.check(fn(cu.ctypes.data_as(I32P), len(cu) - 1, int(causal), band, pp, int(backward), piece, d, nd, c, ncb, C.byref(nc), C.byref(ws)), "t")
    n = call(None, 0, None, 0)
    desc, comb = np.zeros((max(n, 1), 8), np.int32), np.zeros((max(nc.value, 1), 4), np.int32)
    assert call(desc.ctypes.data_as(I32P), desc.shape[0], comb.ctypes.data_as(I32P), comb.shape[0]) == n
    return desc[:n], comb[:nc.value], ws.value


def mask(cu, causal, band, prefix):
    T = cu[-1]
    m = np.zeros((T, T), bool)
    for s, (a, z) in enumerate(zip(cu[:-1], cu[1:])):
        i, j = np.arange(z - a)[:, None], np.arange(z - a)[None, :]
        see = np.ones((z - a, z - a), bool)
        if causal:
            see = (j <= i) | (j < (prefix[s] if prefix is not None else 0))
        if band >= 0:
            see = see & (j >= i - band)
        m[a:z, a:z] = see
    return m


RULES = [
    ([0, 1], True, -1, None), ([0, 700], True, -1, None), ([3, 3, 260, 517, 1300], True, -1, None), ([0, 300, 777], False, -1, None),
    ([0, 600, 1111], True, -1, [256, 1000]), ([0, 513], True, -1, [1]), ([0, 513, 514], True, -1, [0, 0]), ([0, 900], True, -1, [899]),
    ([0, 900], True, 0, None), ([0, 900], True, 63, None), ([0, 300, 1000], True, 400, None), ([0], True, -1, None),
]


@pytest.mark.parametrize("piece", [0, 1, 3, 1 << 22], ids=["whole", "shortest", "middling", "one_piece"])
@pytest.mark.parametrize("backward", [False, True], ids=["fwd", "bwd"])
@pytest.mark.parametrize("cu,causal,band,prefix", RULES)
def test_every_visible_pair_once(cu, causal, band, prefix, backward, piece):
    piece *= 32 if backward else 64
    desc, comb, ws_rows = table(cu, causal, band, prefix, backward, piece)
    own = 128 if backward else 256
    want = mask(cu, causal, band, prefix)
    seen = np.zeros(want.shape, np.int32)
    spots = set()
    for a0, an, b0, bn, shift, delta, band_p1, pre in desc:
        seg = [s for s in range(len(cu) - 1) if cu[s] <= a0 < cu[s + 1]]
        assert len(seg) == 1 and 1 <= an <= own and a0 + an <= cu[seg[0] + 1]
        assert bn >= 0 and b0 >= cu[seg[0]] and b0 + bn <= cu[seg[0] + 1]
        i, j = (np.arange(bn)[:, None], np.arange(an)[None, :]) if backward else (np.arange(an)[:, None], np.arange(bn)[None, :])
        vis = (j <= i + shift) | (j < pre)
        if band_p1:
            vis &= j >= i + shift - (band_p1 - 1)
        q0, k0 = (b0, a0) if backward else (a0, b0)
        seen[q0:q0 + i.shape[0], k0:k0 + j.shape[1]] += vis
        assert band_p1 == (band + 1 if band >= 0 else 0)
        spots.add(a0 + delta)
        if piece == 0:
            assert delta == 0
    assert np.array_equal(seen, want.astype(np.int32))
    if piece:     # every item has workspace rows of its own, and the combine table points at all of them
        assert len(spots) == len(desc) and all(0 <= s and s + own <= ws_rows for s in spots)
        rows = {ws0 + p * own for _, _, ws0, n in comb for p in range(n)}
        assert rows == spots
        assert sorted((a, n) for a, n, _, _ in comb.tolist()) == sorted({(a, n) for a, n in desc[:, :2].tolist()})


def test_heaviest_first_and_room():
    desc, _, _ = table([0, 5000], True, -1, [800], False, 0)
    work = desc[:, 1].astype(np.int64) * desc[:, 3]
    assert (np.diff(work) <= 0).all()
    cu = np.asarray([0, 5000], np.int32)
    out = np.zeros((2, 8), np.int32)
    rc = _lib.lib().lv_build_score_blocks(cu.ctypes.data_as(I32P), 1, 1, -1, None, 0, 0, out.ctypes.data_as(I32P), 2, None, 0, None, None)
    assert rc == -3 and b"room for 2" in _lib.lib().lvattn_last_error()


@pytest.mark.parametrize("cu,causal,band,prefix,backward,piece", [
    ([0, 5, 4], 1, -1, None, 0, 0), ([-1, 5], 1, -1, None, 0, 0), ([0, 5], 0, 3, None, 0, 0), ([0, 5], 1, 3, [1], 0, 0),
    ([0, 5], 0, -1, [1], 0, 0), ([0, 5], 1, -1, [-1], 0, 0), ([0, 5], 1, -1, None, 0, 32), ([0, 5], 1, -1, None, 1, 48), ([0, 5], 1, -1, None, 0, -64)])
def test_builder_refusals(cu, causal, band, prefix, backward, piece):
    cu = np.asarray(cu, np.int32)
    pre = None if prefix is None else np.asarray(prefix, np.int32)
    rc = _lib.lib().lv_build_score_blocks(cu.ctypes.data_as(I32P), len(cu) - 1, causal, band, None if pre is None else pre.ctypes.data_as(I32P), backward,
                                          piece, None, 0, None, 0, None, None)
    assert rc == -1 and _lib.lib().lvattn_last_error()


def test_plan_cuts_few_long_sweeps_only():
    cu = np.asarray([0, 8192], np.int32)
    fn = _lib.lib().lv_plan_score_split
    assert fn(cu.ctypes.data_as(I32P), 1, 1, -1, None, 0, 5, 1, 256) > 0
    assert fn(cu.ctypes.data_as(I32P), 1, 1, -1, None, 0, 40, 8, 256) == 0
    assert fn(cu.ctypes.data_as(I32P), 1, 1, -1, None, 0, 5, 2, 256) == -1


def test_entry_points_refuse_bad_rules():
    L = _lib.lib()
    ones = [16] * 3
    common = [16, None, 0, 16, 16, 1, 8, 8, 4, 2, 64] + [256, 64] * 4 + [8]
    assert L.lvattn_fwd_score(*ones, *common, 1.0, -1.0, None, None) == -1 and b"softcap" in L.lvattn_last_error()
    assert L.lvattn_fwd_score(*ones, *common, 1.0, float("nan"), None, None) == -1
    assert L.lvattn_fwd_score(*ones, *common, float("inf"), 0.0, None, None) == -1 and b"softmax_scale" in L.lvattn_last_error()
    assert L.lvattn_fwd_score(None, 16, 16, *common, 1.0, 0.0, None, None) == -1
