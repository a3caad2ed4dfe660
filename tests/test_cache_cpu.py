"""What the C entry points of the operators on ragged KV caches refuse before anything is launched, and the workspace sizes
they ask for (no GPU: nothing that is refused reaches a kernel)."""
import pytest

from long_vita_amd import _lib

EINVAL, ESIZE = -1, -3
P = 1 << 12        # a well-aligned address that is never read


def tree(**kw):
    a = dict(q=P, k=P, v=P, out=P, lse=None, lens=P, parents=None, pbs=0, ws=P, wsb=1 << 40, batch=2, n=3, rows=20, hq=4, hkv=2, d=64, q_bs=768, q_ns=256, q_hs=64,
             k_bs=2560, k_rs=128, k_hs=64, v_bs=2560, v_rs=128, v_hs=64, o_bs=768, o_ns=256, o_hs=64, scale=0.1, cap=0.0, slopes=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().lvattn_tree(*a.values())


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lens=None), dict(ws=None), dict(ws=P + 8), dict(q=P + 2), dict(k=P + 8),
                                 dict(batch=0), dict(batch=513), dict(n=0), dict(n=257, rows=300), dict(rows=2), dict(hq=5), dict(hkv=0), dict(d=96), dict(q_ns=257),
                                 dict(q_bs=-8), dict(k_bs=-8), dict(k_rs=132), dict(v_hs=65), dict(pbs=-1), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("nan"))])
def test_tree_refuses(bad):
    assert tree(**bad) == EINVAL and _lib.lib().lvattn_last_error()


def test_tree_workspace():
    L = _lib.lib()
    need = L.lvattn_tree_workspace_bytes(2, 3, 20, 4, 2, 64)
    assert need > 0 and tree(wsb=need - 1) == ESIZE and str(need).encode() in L.lvattn_last_error()
    for bad in ((0, 3, 20, 4, 2, 64), (2, 0, 20, 4, 2, 64), (2, 3, 2, 4, 2, 64), (2, 3, 20, 5, 2, 64), (2, 3, 20, 4, 2, 80)):
        assert L.lvattn_tree_workspace_bytes(*bad) == 0
    # bounded by the chip, not by the cache: a million keys need no more than a hundred thousand
    assert L.lvattn_tree_workspace_bytes(1, 8, 1 << 20, 40, 8, 128) == L.lvattn_tree_workspace_bytes(1, 8, 100000, 40, 8, 128)


def accept(**kw):
    a = dict(k=P, v=P, w=None, lens=P, path=P, cnt=P, batch=2, n=5, rows=20, hkv=2, d=64, k_bs=2560, k_rs=128, k_hs=64, v_bs=2560, v_rs=128, v_hs=64, w_bs=40, w_hs=20,
             stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().lv_tree_accept(*a.values())


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(lens=None), dict(path=None), dict(cnt=None), dict(k=P + 8), dict(v_rs=129), dict(d=80), dict(batch=0),
                                 dict(hkv=0), dict(n=0), dict(n=21)])
def test_accept_refuses(bad):
    assert accept(**bad) == EINVAL and _lib.lib().lvattn_last_error()


def weights(**kw):
    a = dict(q=P, k=P, lse=P, rho=None, w_in=P, w_out=P, lens=P, parents=None, pbs=0, ws=P, wsb=1 << 40, batch=2, n=3, rows=20, hq=4, hkv=2, d=64, q_bs=768, q_ns=256,
             q_hs=64, k_bs=2560, k_rs=128, k_hs=64, wi_bs=40, wi_hs=20, wo_bs=40, wo_hs=20, scale=0.1, cap=0.0, slopes=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().lv_key_weights(*a.values())


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(lse=None), dict(w_in=None), dict(w_out=None), dict(lens=None), dict(k=P + 8), dict(q_bs=-8), dict(q_ns=3),
                                 dict(k_bs=4), dict(k_rs=130), dict(batch=0), dict(n=0), dict(rows=2), dict(hq=3), dict(d=32), dict(pbs=-1), dict(q_ns=1 << 30),
                                 dict(parents=P, n=257, rows=400), dict(scale=float("nan")), dict(cap=float("inf")), dict(batch=40000, hkv=2)])
def test_weights_refuse(bad):
    assert weights(**bad) == EINVAL and _lib.lib().lvattn_last_error()


def test_weights_workspace():
    L = _lib.lib()
    assert L.lv_key_weights_workspace_bytes(4, 1, 70000, 40, 8) == 0 == L.lv_key_weights_workspace_bytes(4, 25, 70000, 40, 8)
    need = L.lv_key_weights_workspace_bytes(1, 900, 900, 40, 8)
    assert need > 0
    big = dict(batch=1, n=900, rows=900, hq=40, hkv=8, d=128, q_ns=5120, q_hs=128, k_rs=1024, k_hs=128)
    assert weights(**big, wsb=need - 1) == ESIZE and weights(**big, ws=None) == EINVAL and weights(**big, ws=P + 4) == EINVAL


def index(**kw):
    a = dict(w=P, lens=P, index=P, new_lens=None, ws=P, wsb=1 << 40, batch=2, rows=100, hkv=2, keep=30, sink=4, recent=8, w_bs=200, w_hs=100, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().lv_evict_index(*a.values())


@pytest.mark.parametrize("bad", [dict(w=None), dict(lens=None), dict(index=None), dict(batch=0), dict(rows=0), dict(hkv=0), dict(batch=40000), dict(keep=0), dict(keep=101),
                                 dict(sink=-1), dict(recent=-1), dict(sink=20, recent=11), dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)])
def test_evict_index_refuses(bad):
    assert index(**bad) == EINVAL and _lib.lib().lvattn_last_error()


def test_evict_workspace():
    L = _lib.lib()
    assert L.lv_evict_workspace_bytes(8, 4096, 8) == 0
    need = L.lv_evict_workspace_bytes(2, 50000, 2)
    assert need > 0 and index(rows=50000, wsb=need - 1) == ESIZE and index(rows=50000, ws=None) == ESIZE


def take(**kw):
    a = dict(k=P, v=P, w=P, index=P, ko=P, vo=P, wo=P, batch=2, hkv=2, d=64, keep=30, zero=1, k_bs=2560, k_rs=128, k_hs=64, v_bs=2560, v_rs=128, v_hs=64, w_bs=200,
             w_hs=100, ko_bs=2560, ko_rs=128, ko_hs=64, vo_bs=2560, vo_rs=128, vo_hs=64, wo_bs=60, wo_hs=30, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().lv_evict_take(*a.values())


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(w=None), dict(index=None), dict(ko=None), dict(vo=None), dict(wo=None), dict(d=256), dict(batch=0),
                                 dict(batch=70000), dict(hkv=0), dict(keep=0), dict(k=P + 2), dict(vo=P + 8), dict(k_rs=127), dict(ko_hs=63), dict(v_bs=4)])
def test_evict_take_refuses(bad):
    assert take(**bad) == EINVAL and _lib.lib().lvattn_last_error()
