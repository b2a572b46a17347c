"""Refusals of group-limited routing, checked on the host (no GPU needed)."""
import struct

import pytest
import torch

from trials_b200 import _lib, moe, stages

P = 256


def call(M=4, E=64, G=8, T=3, k=6, scoring=1, bias=P, logits=P, w=P, ids=P):
    args = (logits, 0, M, E, G, T, k, scoring, bias, 1, 1.0, w, ids, None)
    return _lib.lib().b200moe_router_topk_grouped(struct.pack("10qd3q", *(0 if a is None else a for a in args)))


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(E=0), dict(k=0), dict(k=65), dict(scoring=2), dict(scoring=0), dict(logits=None), dict(w=None),
    dict(ids=None), dict(E=-(1 << 32)), dict(T=(1 << 32) + 3), dict(G=0), dict(G=7), dict(G=-8), dict(T=0), dict(T=9), dict(T=1, k=9)])
def test_invalid_arguments(kw):
    assert call(**kw) == _lib.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(E=2048), dict(E=(1 << 32) + 64, k=1), dict(k=17, T=8), dict(G=64, T=64)])
def test_unsupported_sizes(kw):
    assert call(**kw) == _lib.ERR_UNSUPPORTED


def test_fused_entries_check_the_groups_too():
    L = _lib.lib()
    assert L.b200moe_route_logits_grouped(P, 0, 4, 64, 7, 3, 6, 1, P, 1, 1.0, P, P, None, 64, 32, P, 1 << 20, P, P, P,
                                          1 << 20, P, P, P, P, P, 1 << 20, P, None) == _lib.ERR_INVALID_ARG
    assert L.b200moe_layer_logits_grouped(P, 4, 256, 128, 64, 6, P, 0, 8, 9, 1, P, 1, 1.0, P, P, P, P, None, 64, P, P,
                                          P, P, 1 << 30, None) == _lib.ERR_INVALID_ARG


def test_empty_batch_launches_nothing():
    assert call(M=0, logits=None, w=None, ids=None) == _lib.OK
    assert _lib.lib().b200moe_router_topk_grouped(None) == _lib.ERR_INVALID_ARG


def test_python_arguments():
    assert moe._check_groups(None, None) is False and moe._check_groups(8, 4) is True
    for pair in ((8, None), (None, 4)):
        with pytest.raises(ValueError):
            moe._check_groups(*pair)
    with pytest.raises(ValueError, match="CUDA"):
        moe.select_experts(torch.zeros(2, 8), 2, num_expert_group=2, topk_group=1)


def test_router_bias_covers_the_experts():
    """A bias may be longer than the experts (padded); the kernels read the first ones."""
    long = torch.arange(96, dtype=torch.float32)
    got = moe._router_bias(long, torch.device("cpu"), long.get_device(), 64)
    assert torch.equal(got[:64], long[:64])
    odd = torch.arange(192, dtype=torch.bfloat16)[::2]
    got = moe._router_bias(odd, torch.device("cpu"), None, 64)
    assert got.dtype == torch.float32 and got.is_contiguous() and torch.equal(got[:64], odd[:64].float())
    assert moe._router_bias(None, torch.device("cpu"), None, 64) is None
    with pytest.raises(ValueError, match="64"):
        moe._router_bias(long[:63], torch.device("cpu"), None, 64)


@pytest.mark.parametrize("kw", [dict(logits=P + 2), dict(logits=P + 1), dict(bias=P + 2), dict(w=P + 1), dict(ids=P + 2)])
def test_pointers_must_be_aligned(kw):
    assert call(**kw) == _lib.ERR_UNSUPPORTED


class Entered(Exception):
    pass


class OnDevice1:
    """Stands for a tensor on a device that is not the current one."""
    device = torch.device("cuda", 1)
    dtype = torch.float32
    shape = (4, 64)

    def get_device(self):
        return 1


@pytest.mark.parametrize("groups", [{}, dict(num_expert_group=8, topk_group=4)])
def test_calls_go_to_the_device_of_their_tensors(monkeypatch, groups):
    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            raise Entered(self.device)

        def __exit__(self, *a):
            pass

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for module in (moe, stages):
        monkeypatch.setattr(module, "_require_cuda", lambda *t: torch.device("cuda", 1))
    x = OnDevice1()
    for call in (lambda: moe.select_experts(x, 6, "sigmoid", **groups),
                 lambda: moe.moe_layer_from_logits(x, x, x, x, x, x, 6, **groups),
                 lambda: stages.route_logits(x, 6, 32, **groups),
                 lambda: moe.moe_decode_megakernel_full(x, x, x, x, x, x, x)):
        with pytest.raises(Entered) as e:
            call()
        assert getattr(e.value.args[0], "index", e.value.args[0]) == 1
