"""A correction bias padded past the experts routes like its first entries, with
groups and without, in every call that takes one."""
import pytest
import torch

from trials_b200 import moe, per_block_quant_fp8, stages, synth

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]


@pytest.mark.parametrize("groups", [{}, dict(num_expert_group=4, topk_group=2)])
def test_padded_bias(cuda_device, groups):
    M, E, k = 24, 32, 4
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.randn(M, E, generator=g, device=cuda_device)
    padded = torch.randn(E + 16, generator=g, device=cuda_device)
    bias = padded[:E].clone()
    w, ids = moe.select_experts(x, k, "sigmoid", bias, **groups)
    got = moe.select_experts(x, k, "sigmoid", padded, **groups)
    assert torch.equal(got[0], w) and torch.equal(got[1], ids)
    _, tw, routed = stages.route_logits(x, k, 32, correction_bias=padded, **groups)
    assert torch.equal(tw, w) and torch.equal(routed, ids)
    L = synth.make_layer(synth.LayerShape(M=M, H=512, I=256, E=E, topk=k), per_block_quant_fp8, seed=2,
                         device=cuda_device)
    ws = (L.w13, L.w13_scale, L.w2, L.w2_scale)
    want = moe.moe_decode_megakernel_full(L.hidden, *ws, w, ids)
    out, tw, routed = moe.moe_layer_from_logits(L.hidden, x, *ws, k, "sigmoid", padded, **groups)
    assert torch.equal(out, want) and torch.equal(tw, w) and torch.equal(routed, ids)
    pipe = stages.LayerPipeline(M, 512, 256, E, k, cuda_device, router=dict(correction_bias=padded, **groups))
    assert torch.equal(pipe.run_from_logits(L.hidden, x, *ws), want)
    with pytest.raises(ValueError):
        moe.select_experts(x, k, "sigmoid", bias[:E - 1], **groups)
