"""Group-limited sigmoid routing of logits far below zero, whose scores fp32 cannot
hold: the renormalised weights are ratios of the scores, so they are those of 64
bits (within 2^-20, as everywhere) as long as 64 bits hold the scores; a row
whose scores are all 0 there has weights 0."""
import numpy as np
import pytest
import torch

from trials_b200 import moe

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]


def exact(x, ids, scale):
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-x.double().cpu().numpy()))
    w = np.take_along_axis(s, ids.cpu().numpy().astype(np.int64), 1)
    t = w.sum(1, keepdims=True)
    return np.where(t > 0, w / np.where(t > 0, t, 1), 0.0) * scale


@pytest.mark.parametrize("E,G,T,k", [(256, 8, 4, 8), (60, 6, 2, 4), (1024, 16, 3, 16)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_below_zero(cuda_device, E, G, T, k, bias, dtype):
    g = torch.Generator().manual_seed(E)
    centre = torch.tensor([-30.0, -60.0, -69.0, -80.0, -88.0, -95.0, -104.0, -200.0, -650.0, -740.0, -5000.0])
    x = centre.repeat_interleave(8)[:, None] + torch.randn(88, E, generator=g) * 4
    x = torch.cat([x, torch.full((1, E), torch.finfo(dtype).min), torch.full((1, E), float("-inf")),
                   torch.full((1, E), -100.0)]).to(dtype)
    x[0, 3], x[40, 7] = float("nan"), float("-inf")
    x = x.to(cuda_device)
    b = (torch.randn(E, generator=g) * 0.1).to(cuda_device) if bias else None
    w, ids = moe.select_experts(x, k, "sigmoid", b, True, 2.5, num_expert_group=G, topk_group=T)
    want = exact(torch.nan_to_num(x.float(), nan=float("-inf"), neginf=float("-inf")), ids, 2.5)
    got = w.double().cpu().numpy()
    # below 1e-30 of the whole, fp32's own range may end
    assert (np.abs(got - want) <= 2.0 ** -20 * want + 1e-30).all()
    assert np.allclose(got[-1], 2.5 / k, rtol=1e-6) and (got[-2] == 0).all() and (got[-3] == 0).all()
