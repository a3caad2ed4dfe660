"""The work-item tables that captured calls of score_attention keep (no GPU: captures and their ends are played by the test)."""
import gc
import weakref

import pytest
import torch

from long_vita_amd import ops


@pytest.fixture
def played(monkeypatch):
    """Tables on the CPU; ``state`` says whether and in which capture the stream is."""
    state = {"capture": 0, "ended": [], "watched": []}
    real = ops._lib.lib()

    class Lib:
        def __getattr__(self, name):
            return getattr(real, name)

        @staticmethod
        def lv_capture_ended(ids, room):
            n = min(room, len(state["ended"]))
            for i in range(n):
                ids[i] = state["ended"].pop(0)
            return n

        @staticmethod
        def lv_capture_watch(stream):
            state["watched"].append(state["capture"])
            return 0
    lib = Lib()
    monkeypatch.setattr(ops._lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_to_device", lambda host, device: torch.from_numpy(host.copy()))
    monkeypatch.setattr(ops, "_capture_number", lambda: state["capture"], raising=False)
    monkeypatch.setattr(ops, "_captured_tables", {})
    monkeypatch.setattr(ops, "_watched_captures", set(), raising=False)
    monkeypatch.setattr(ops, "_blocks", ops._BlockCache(4))
    monkeypatch.setattr(ops, "_ended_tables", {}, raising=False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: state.__setitem__("waits", state.get("waits", 0) + (state["capture"] == 0)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capture"] != 0)
    return state


def table(cu, backward=False):
    return ops._ScoreRule(cu, True, None, None, 30.0).tables(backward, 0, "cuda:0")


def test_second_graph_of_a_packing_leaves_the_first_its_table(played):
    first = weakref.ref(table((0, 100)))
    played["capture"] = 1
    assert table((0, 100)) is first()
    played["capture"] = 0
    for n in range(5):                       # the table's turn in the cache is over
        table((0, 200 + n))
    again = table((0, 100))
    assert again is not first()
    played["capture"] = 2
    assert table((0, 100)) is again
    gc.collect()
    assert first() is not None               # graph 1 still reads it


def test_tables_go_with_their_graph(played):
    kept = []
    for graph in (1, 2, 3):
        played["capture"] = 0
        for backward in (False, True):
            table((0, 100 * graph), backward)
        played["capture"] = graph
        for _layer in range(3):
            for backward in (False, True):
                kept.append(weakref.ref(table((0, 100 * graph), backward)))
    assert played["watched"] == [1, 2, 3]    # one object per graph, however many calls it captured
    played["capture"] = 0
    for n in range(5):
        table((0, 900 + n))
    gc.collect()
    assert all(t() is not None for t in kept) and len(ops._captured_tables) == 6
    played["ended"] += [1, 3]
    table((0, 999))                          # the next table that is built lets go
    gc.collect()
    assert [t() is not None for t in kept] == [False] * 6 + [True] * 6 + [False] * 6 and played["waits"] == 1
    played["ended"].append(2)
    played["capture"] = 4
    table((0, 999))                          # inside a capture there is no waiting for a last replay: the tables stay
    gc.collect()
    assert all(t() for t in kept[6:12]) and [k[0] for k in ops._captured_tables] == [4]
    played["capture"] = 0
    table((0, 998))
    gc.collect()
    assert not any(t() for t in kept) and played["waits"] == 2


def test_many_graphs_end_at_once(played):
    table((0, 64))
    for graph in range(1, 151):
        played["capture"] = graph
        table((0, 64))
    assert len(ops._captured_tables) == 150
    played["ended"] += list(range(1, 150))
    played["capture"] = 0
    table((0, 65))
    assert [k[0] for k in ops._captured_tables] == [150]
