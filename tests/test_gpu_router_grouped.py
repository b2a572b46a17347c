"""Group-limited routing against its definition in 64 bits: the selection has
to be the exact one, near ties included.

Weights: an expf (2 ulp) or a sigmoid (expf, sum, division), a sum of at most 16
of them, a division and the scaling: below 16 roundings of 2^-24 each, so within
2^-20 of the value."""
import contextlib

import numpy as np
import pytest
import torch

from trials_b200 import _lib, fp8_mlp, layer_error_word, moe, read_device_error, stages, synth

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]


def exact(logits, groups, topk_group, k, scoring, bias, renorm, scale):
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    M, E = x.shape
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            s = 1 / (1 + np.exp(-x))
        else:
            top = x.max(1, keepdims=True)
            e = np.where(x == -np.inf, 0.0, np.where(x == top, 1.0, np.exp(x - top)))
            s = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
        if bias is not None:
            c = s + bias.double().cpu().numpy()
            c = np.where(np.isnan(c), -np.inf, c)
            g = -np.sort(-c.reshape(M, groups, -1), axis=2)
            score = g[..., 0] + g[..., 1] if E // groups > 1 else g[..., 0]
            score = np.where(np.isnan(score), -np.inf, score)
        else:
            c = x
            score = x.reshape(M, groups, -1).max(2)
        taken = np.argsort(-score, axis=1, kind="stable")[:, :topk_group]
        alive = np.zeros((M, groups), bool)
        np.put_along_axis(alive, taken, True, 1)
        alive = alive.repeat(E // groups, 1)
        # closed experts behind open ones of -inf
        order = np.lexsort((np.broadcast_to(np.arange(E), c.shape), -c, ~alive), axis=1)
        ids = order[:, :k]
        w = np.take_along_axis(s, ids, 1)
        if renorm:
            t = w.sum(1, keepdims=True)
            w = np.where(t > 0, w / np.where(t > 0, t, 1), 0.0)
    return ids, w * scale


def check(logits, groups, topk_group, k, scoring, bias=None, renorm=True, scale=1.0):
    w, ids = moe.select_experts(logits, k, scoring, bias, renorm, scale, num_expert_group=groups, topk_group=topk_group)
    eids, ew = exact(logits, groups, topk_group, k, scoring, bias, renorm, scale)
    assert np.array_equal(ids.cpu().numpy(), eids)
    w = w.double().cpu().numpy()
    assert (np.abs(w - ew) <= 2.0 ** -20 * ew + 1e-37).all()


SHAPES = [  # M, E, groups, topk_group, k
    (1, 256, 8, 4, 8), (300, 256, 8, 4, 8), (77, 160, 8, 3, 6), (33, 64, 4, 1, 6), (129, 1024, 32, 5, 16),
    (64, 512, 16, 16, 10), (50, 60, 6, 2, 4), (50, 60, 5, 3, 16), (9, 8, 8, 2, 2), (20, 96, 3, 2, 6), (10, 30, 15, 4, 3),
    (40, 7, 1, 1, 7), (16, 1, 1, 1, 1), (25, 330, 2, 1, 8), (31, 1000, 10, 3, 16), (2000, 128, 4, 2, 5),
    # lanes not all full, lanes across groups
    (60, 250, 5, 2, 9), (55, 312, 4, 1, 16), (80, 336, 16, 9, 7), (30, 992, 31, 4, 8), (40, 1020, 17, 5, 8),
    (21, 900, 12, 4, 8), (64, 40, 8, 2, 2)]


@pytest.mark.parametrize("M,E,G,T,k", SHAPES)
@pytest.mark.parametrize("scoring,bias,dtype,renorm", [
    ("sigmoid", True, torch.float32, True), ("sigmoid", True, torch.bfloat16, False),
    ("sigmoid", False, torch.bfloat16, True), ("softmax", False, torch.float32, False),
    ("softmax", False, torch.bfloat16, True)])
def test_selection_and_weights(cuda_device, M, E, G, T, k, scoring, bias, dtype, renorm):
    g = torch.Generator().manual_seed(M + E + G + T + k)
    x = (torch.randn(M, E, generator=g) * 2).to(dtype).to(cuda_device)
    b = (torch.randn(E, generator=g) * 0.2).to(cuda_device) if bias else None
    check(x, G, T, k, scoring, b, renorm, 2.5)


@pytest.mark.parametrize("M,E,G,T,k", SHAPES)
def test_near_ties_are_told_apart(cuda_device, M, E, G, T, k):
    """Biases that make every c the same up to their own rounding (3e-8)."""
    g = torch.Generator().manual_seed(E)
    row = torch.randn(E, generator=g)
    b = (0.75 - torch.sigmoid(row.double())).float()
    x = row.repeat(M, 1)
    x += (torch.randn(M, E, generator=g) * 1e-7) * (torch.arange(M) % 2)[:, None]
    check(x.to(cuda_device), G, T, k, "sigmoid", b.to(cuda_device))
    # scores of groups that nearly cancel: large biases of both signs
    b = torch.where(torch.arange(E) % 2 == 0, 1000.0, -1000.0) + torch.rand(E, generator=g)
    check(x.to(cuda_device), G, T, k, "sigmoid", b.to(cuda_device))


@pytest.mark.parametrize("M,E,G,T,k", [(6, 256, 8, 4, 8), (6, 60, 6, 2, 4), (6, 512, 16, 3, 16)])
@pytest.mark.parametrize("scoring,bias", [("sigmoid", True), ("sigmoid", False), ("softmax", False)])
@pytest.mark.parametrize("renorm", [True, False])
def test_equal_masked_and_bad_logits(cuda_device, M, E, G, T, k, scoring, bias, renorm):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(M, E, generator=torch.Generator().manual_seed(3))
    x[0] = 0.5                                    # all equal
    x[1] = -inf                                   # nothing left
    x[2, E // 2:] = -inf                          # half masked
    x[3] = torch.finfo(torch.float32).min         # masked by the lowest value
    x[3, 5] = 1.0
    x[4, ::3] = nan
    x[5, 1:: E // 4] = inf
    b = None
    if bias:
        b = torch.zeros(E)
        b[7] = -inf
    check(x.to(cuda_device), G, T, k, scoring, None if b is None else b.to(cuda_device), renorm)
    signed = torch.zeros(2, E)
    signed[:, ::2] = -0.0
    check(signed.to(cuda_device), G, T, k, scoring, None, renorm)


def test_bad_biases(cuda_device):
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    b = torch.zeros(64)
    b[3], b[17], b[40] = float("inf"), float("nan"), -float("inf")
    check(x, 8, 3, 6, "sigmoid", b.to(cuda_device))


def test_refusals_on_device(cuda_device):
    x = torch.randn(4, 64, device=cuda_device)
    for kw in (dict(num_expert_group=8), dict(num_expert_group=7, topk_group=2), dict(num_expert_group=8, topk_group=9)):
        with pytest.raises(ValueError):
            moe.select_experts(x, 4, "sigmoid", **kw)
    with pytest.raises(ValueError):  # a bias that does not cover the experts
        moe.select_experts(x, 4, "sigmoid", torch.zeros(32, device=cuda_device), num_expert_group=8, topk_group=2)
    with pytest.raises(ValueError):
        stages.route_logits(x, 4, 32, correction_bias=torch.zeros(32, device=cuda_device), num_expert_group=8,
                            topk_group=2)
    with pytest.raises(ValueError):
        stages.LayerPipeline(8, 256, 128, 64, 4, device=cuda_device,
                             router={"correction_bias": torch.zeros(32), "num_expert_group": 8, "topk_group": 2})
    with pytest.raises(NotImplementedError):
        moe.select_experts(x.half(), 4, "sigmoid", num_expert_group=8, topk_group=2)


def test_bias_of_another_type_or_layout(cuda_device):
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(8)).to(cuda_device)
    b = torch.randn(128, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)[::2]
    check(x, 8, 3, 6, "sigmoid", b)  # bf16, strided, on the host
    buf = torch.zeros(65, device=cuda_device)
    buf[1:] = b.to(cuda_device)
    check(x, 8, 3, 6, "sigmoid", buf[1:])  # 4-byte aligned
    wide = torch.zeros(50 * 64 + 1, device=cuda_device)[1:].view(50, 64)
    wide.copy_(x)
    check(wide, 8, 3, 6, "sigmoid", buf[1:])


def test_one_group_is_ungrouped_routing(cuda_device):
    x = torch.randn(500, 256, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    w, ids = moe.select_experts(x, 8, "softmax")
    w1, ids1 = moe.select_experts(x, 8, "softmax", num_expert_group=1, topk_group=1)
    assert torch.equal(ids, ids1) and torch.allclose(w, w1, rtol=1e-5, atol=0)


def test_layouts_streams_and_graphs(cuda_device):
    x = torch.randn(64, 256, generator=torch.Generator().manual_seed(4)).to(cuda_device)
    kw = dict(scoring_func="sigmoid", num_expert_group=8, topk_group=4)
    w, ids = moe.select_experts(x, 8, **kw)
    w2, ids2 = moe.select_experts(torch.cat([x, x], 1)[:, :256], 8, **kw)
    assert torch.equal(w, w2) and torch.equal(ids, ids2)
    assert moe.select_experts(x[:0], 8, **kw)[0].shape == (0, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w3, ids3 = moe.select_experts(x, 8, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(w, w3) and torch.equal(ids, ids3)
    buf = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w4, ids4 = moe.select_experts(buf, 8, **kw)
    buf.copy_(x)
    graph.replay()
    assert torch.equal(w, w4) and torch.equal(ids, ids4)


@pytest.mark.parametrize("M,E,G,T,k,scoring,bias,dtype,tile", [
    (1, 256, 8, 4, 8, "sigmoid", True, torch.float32, 32), (64, 256, 8, 4, 8, "sigmoid", True, torch.bfloat16, 32),
    (300, 1024, 16, 3, 16, "softmax", False, torch.float32, 32), (2048, 256, 8, 4, 8, "sigmoid", True, torch.float32, 128),
    (5000, 96, 6, 2, 6, "sigmoid", False, torch.float32, 128), (3000, 512, 8, 2, 6, "softmax", False, torch.float32, 128)])
def test_route_logits_equals_router_then_route(cuda_device, M, E, G, T, k, scoring, bias, dtype, tile):
    g = torch.Generator().manual_seed(M)
    x = (torch.randn(M, E, generator=g) * 2).to(dtype).to(cuda_device)
    b = (torch.randn(E, generator=g) * 0.1).to(cuda_device) if bias else None
    w_ref, ids_ref = moe.select_experts(x, k, scoring, b, True, 2.5, num_expert_group=G, topk_group=T)
    r_ref = stages.route(ids_ref, E, tile)
    for _ in range(2):
        r, w, ids = stages.route_logits(x, k, tile, scoring, b, True, 2.5, num_expert_group=G, topk_group=T)
        assert torch.equal(ids, ids_ref) and torch.equal(w, w_ref)
        assert torch.equal(r.counts, r_ref.counts)
        assert torch.equal(r.sorted_ids, r_ref.sorted_ids) and torch.equal(r.slot_pos, r_ref.slot_pos)
        assert read_device_error(r.err) == 0


@contextlib.contextmanager
def launch_mode(mode):
    prev = _lib.lib().b200moe_set_layer_launch(mode)
    try:
        yield
    finally:
        _lib.lib().b200moe_set_layer_launch(prev)


@pytest.mark.parametrize("M", [1, 24, 300])
def test_block_of_router_experts_and_shared_expert(cuda_device, M):
    """Router with groups, routed experts and the shared expert in one call:
    the same bits as the calls one by one, whichever way the layer launches."""
    H, I, E, k = 512, 256, 32, 4
    L = synth.make_layer(synth.LayerShape(M=M, H=H, I=I, E=E, topk=k), moe.per_block_quant_fp8, seed=M,
                         device=cuda_device)
    w = (L.w13, L.w13_scale, L.w2, L.w2_scale)
    g = torch.Generator(device=cuda_device).manual_seed(M)
    logits = torch.randn(M, E, generator=g, device=cuda_device)
    bias = torch.randn(E, generator=g, device=cuda_device) * 0.1
    groups = dict(num_expert_group=4, topk_group=2)
    s13 = moe.per_block_quant_fp8(torch.randn(2 * 384, H, generator=g, device=cuda_device).to(torch.bfloat16) * 0.05)
    s2 = moe.per_block_quant_fp8(torch.randn(H, 384, generator=g, device=cuda_device).to(torch.bfloat16) * 0.05)
    shared = (*s13, *s2)
    tw, ids = moe.select_experts(logits, k, "sigmoid", bias, True, 2.5, **groups)
    routed = moe.moe_decode_megakernel_full(L.hidden, *w, tw, ids)
    want = fp8_mlp(L.hidden, *shared, residual=routed)
    for mode in (0, 1):
        with launch_mode(mode):
            for extra, ref in (({}, routed), ({"shared_expert": shared}, want)):
                out, tw1, ids1 = moe.moe_layer_from_logits(L.hidden, logits, *w, k, "sigmoid", bias, True, 2.5,
                                                           **groups, **extra)
                assert torch.equal(ids1, ids) and torch.equal(tw1, tw) and torch.equal(out, ref)
    router = dict(scoring_func="sigmoid", correction_bias=bias, routed_scaling_factor=2.5, **groups)
    for mode in (0, 1):
        with launch_mode(mode):
            pipe = stages.LayerPipeline(M, H, I, E, k, cuda_device, router=router)
            assert torch.equal(pipe.run_from_logits(L.hidden, logits, *w), routed)
    # the whole block in a graph
    buf, graph = torch.zeros_like(L.hidden), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _, _ = moe.moe_layer_from_logits(buf, logits, *w, k, "sigmoid", bias, True, 2.5, **groups,
                                              shared_expert=shared)
    buf.copy_(L.hidden)
    graph.replay()
    assert torch.equal(out, want)
    assert read_device_error(layer_error_word(cuda_device)) == 0


def test_expert_map(cuda_device):
    M, E, k = 100, 32, 4
    L = synth.make_layer(synth.LayerShape(M=M, H=512, I=256, E=16, topk=k), moe.per_block_quant_fp8, seed=5,
                         device=cuda_device)
    w = (L.w13, L.w13_scale, L.w2, L.w2_scale)
    logits = torch.randn(M, E, generator=torch.Generator().manual_seed(6)).to(cuda_device)
    emap = torch.full((E,), -1, dtype=torch.int32)
    emap[::2] = torch.arange(16, dtype=torch.int32)
    groups = dict(num_expert_group=4, topk_group=2)
    out, tw, ids = moe.moe_layer_from_logits(L.hidden, logits, *w, k, "sigmoid", expert_map=emap, **groups)
    tw1, ids1 = moe.select_experts(logits, k, "sigmoid", **groups)
    assert torch.equal(ids, ids1) and torch.equal(tw, tw1)
    ref = moe.moe_layer_ep_local(L.hidden, *w, tw, ids, emap.to(cuda_device), E)
    assert torch.equal(out, ref)
