"""Refusals of group-limited routing, checked on the host (no GPU needed)."""
import struct

import pytest
import torch

from trials_b200 import _lib, moe

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
