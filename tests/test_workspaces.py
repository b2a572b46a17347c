"""What calls on a (device, stream) share: the header with the error word, and
the layer's scratch. The bookkeeping is host code, checked here without a GPU;
tests/test_gpu_error_word.py has the rest."""
import gc
import struct
import weakref

import pytest
import torch

from trials_b200 import _lib, moe

P = 256
CPU = torch.device("cpu")


@pytest.fixture
def spaces(monkeypatch):
    state = {"stream": 1, "capturing": False}
    monkeypatch.setattr(moe, "_stream", lambda device: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    return moe._Workspaces(), state


def test_scratch_grows_and_is_let_go(spaces):
    ws, _ = spaces
    first = ws.get(CPU, 1000)
    assert ws.get(CPU, 500) is first
    gone = weakref.ref(first)
    del first
    assert ws.get(CPU, 2000).numel() == 2000
    gc.collect()
    assert gone() is None


def test_scratch_of_a_captured_call_is_kept(spaces):
    ws, state = spaces
    ws.get(CPU, 1000)                  # made by an eager call
    state["capturing"] = True
    held = weakref.ref(ws.get(CPU, 800))
    state["capturing"] = False
    ws.get(CPU, 2000)
    gc.collect()
    assert held() is not None and held().numel() == 1000
    second = weakref.ref(ws.get(CPU, 100))  # no graph has seen this one
    ws.get(CPU, 3000)
    gc.collect()
    assert second() is None and held() is not None


def test_streams_have_scratch_of_their_own(spaces):
    ws, state = spaces
    one = ws.get(CPU, 100)
    state["stream"] = 2
    assert ws.get(CPU, 100) is not one


def test_header_is_made_once(monkeypatch):
    made = []

    class Lib:
        @staticmethod
        def b200moe_header_create(ref):
            made.append(ref)
            ref._obj.value = 4096 * len(made)
            return _lib.OK

    class Guard:
        def __init__(self, index):
            pass

        __enter__ = __exit__ = lambda *a: None

    monkeypatch.setattr(_lib, "lib", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    ws = moe._Workspaces()
    assert [ws.header_ptr(0, 7), ws.header_ptr(0, 7), ws.header_ptr(1, 7), ws.header_ptr(0, 7)] == [4096, 4096, 8192, 4096]
    assert len(made) == 2


def layer_call(hidden=P, hidden_q=0, hidden_scale=0, M=4, H=256, I=128, E=8, k=2, logits=0, groups=0, topk_groups=0,
               scoring=1, w=P, ids=P, header=P, work=P, nwork=1 << 30):
    return _lib.lib().b200moe_layer_call(struct.pack(
        "15qd13q", hidden, hidden_q, hidden_scale, M, H, I, E, k, logits, 0, groups, topk_groups, scoring, 0, 1, 1.0,
        w, P, P, P, P, ids, 0, E, P, header, work, nwork, 0))


@pytest.mark.parametrize("kw", [
    dict(hidden=0), dict(hidden_q=P, hidden_scale=P), dict(hidden=0, hidden_q=P), dict(header=0), dict(header=P + 4),
    dict(w=0), dict(ids=0), dict(M=-1), dict(E=0), dict(k=0), dict(work=0), dict(work=P + 8),
    dict(logits=P, scoring=2), dict(logits=P, groups=3, topk_groups=1), dict(logits=P, groups=-1, topk_groups=1),
    dict(logits=P, groups=4, topk_groups=5)])
def test_layer_call_invalid_arguments(kw):
    assert layer_call(**kw) == _lib.ERR_INVALID_ARG


def test_layer_call_sizes():
    assert layer_call(H=200) == _lib.ERR_UNSUPPORTED
    assert layer_call(E=4096) == _lib.ERR_UNSUPPORTED
    assert layer_call(logits=P, E=2048) == _lib.ERR_UNSUPPORTED
    assert layer_call(nwork=1000) == _lib.ERR_WORKSPACE
    assert layer_call(M=0, hidden=0, header=0) == _lib.OK
    assert _lib.lib().b200moe_layer_call(None) == _lib.ERR_INVALID_ARG
    assert _lib.lib().b200moe_header_create(None) == _lib.ERR_INVALID_ARG


def test_groups_must_be_positive():
    with pytest.raises(ValueError):
        moe._check_groups(0, 0)
