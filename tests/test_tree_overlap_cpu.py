"""tree_attention's refusal of buffers that meet (no GPU: what is not refused reaches a library that launches nothing)."""
import pytest
import torch

from long_vita_amd import _lib, ops


@pytest.fixture
def launches(monkeypatch):
    """Calls that would have been launched; the sizes asked of the library are real."""
    real, calls = _lib.lib(), []

    class Lib:
        def __getattr__(self, name):
            return getattr(real, name)

        def lvattn_tree(self, *args):
            calls.append(args)
            return 0
    lib = Lib()
    monkeypatch.setattr(ops._lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    return calls


B, N, ROWS, HQ, HKV, D = 2, 3, 20, 4, 2, 64
NEED = 1 << 20


def setup():
    kv = torch.zeros(B, ROWS, 2, HKV, D, dtype=torch.bfloat16)
    qo = torch.zeros(B, N, 2 * HQ, D, dtype=torch.bfloat16)
    return kv, qo, torch.tensor([5, 9], dtype=torch.int32)


def test_interleaved_buffers_are_taken(launches):
    kv, qo, lens = setup()
    assert ops.tree_workspace_bytes(B, N, ROWS, HQ, HKV, D) <= NEED
    out = qo[:, :, HQ:]
    res, lse = ops.tree_attention(qo[:, :, :HQ], kv[:, :, 0], kv[:, :, 1], lens, out=out, lse=torch.zeros(B, N, HQ), return_lse=True,
                                  workspace=torch.zeros(NEED, dtype=torch.uint8))
    assert res is out and len(launches) == 1


big = torch.zeros(4 << 20, dtype=torch.uint8)


@pytest.mark.parametrize("name,kw", [
    ("out_one_head_into_q", lambda kv, qo: dict(out=qo[:, :, 1:HQ + 1])),
    ("out_last_head_of_q", lambda kv, qo: dict(out=qo[:, :, HQ - 1:2 * HQ - 1])),
    ("out_one_row_into_k", lambda kv, qo: dict(out=kv.view(B, ROWS, 2 * HKV, D)[:, 1:1 + N])),
    ("out_in_v", lambda kv, qo: dict(out=kv.view(-1)[HKV * D:][:B * N * HQ * D].view(B, N, HQ, D))),
    ("out_behind_q_of_other_strides", lambda kv, qo: dict(out=qo.view(-1)[8:8 + B * N * HQ * D].view(B, N, HQ, D))),
    ("lse_in_q", lambda kv, qo: dict(lse=qo.view(torch.float32).view(-1)[4:4 + B * N * HQ].view(B, N, HQ))),
    ("lse_in_out", lambda kv, qo: dict(out=qo[:, :, HQ:], lse=qo.view(torch.float32).view(-1)[HQ * D // 2:][:B * N * HQ].view(B, N, HQ))),
    ("workspace_holds_out", lambda kv, qo: dict(workspace=big, out=big.view(torch.bfloat16)[4096:4096 + B * N * HQ * D].view(B, N, HQ, D))),
    ("workspace_holds_lse", lambda kv, qo: dict(workspace=big, lse=big.view(torch.float32)[4096:4096 + B * N * HQ].view(B, N, HQ)))])
def test_buffers_that_meet(launches, name, kw):
    kv, qo, lens = setup()
    with pytest.raises(_lib.LvAttnError, match="overlap"):
        ops.tree_attention(qo[:, :, :HQ], kv[:, :, 0], kv[:, :, 1], lens, return_lse=True, **kw(kv, qo))
    assert not launches


@pytest.mark.parametrize("which", ["q", "lens", "parents", "slopes"])
def test_workspace_that_holds_inputs(launches, which):
    kv, qo, lens = setup()
    args = dict(q=qo[:, :, :HQ], k=kv[:, :, 0], v=kv[:, :, 1], cache_lens=lens, parents=torch.tensor([-1, 0, 1], dtype=torch.int32), alibi_slopes=torch.zeros(HQ))
    inside = {"q": lambda: big.view(torch.bfloat16)[:B * N * HQ * D].view(B, N, HQ, D), "lens": lambda: big.view(torch.int32)[8:10],
              "parents": lambda: big.view(torch.int32)[:N], "slopes": lambda: big.view(torch.float32)[64:64 + HQ]}[which]()
    args[{"lens": "cache_lens", "slopes": "alibi_slopes"}.get(which, which)] = inside
    with pytest.raises(_lib.LvAttnError, match="overlap"):
        ops.tree_attention(**args, workspace=big)
    assert not launches
