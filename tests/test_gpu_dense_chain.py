"""Products back to back on one stream, each reading what the one before has just
written into buffers that every step uses again: the same bits as with a
synchronisation between the steps."""
import pytest
import torch

from trials_b200 import (fp8_block_linear, fp8_gate_up, fp8_mlp, layer_error_word, per_block_quant_fp8,
                         read_device_error)

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]


def weight(dev, N, K, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return per_block_quant_fp8((torch.randn(N, K, generator=g, device=dev) * K ** -0.5).to(torch.bfloat16))


@pytest.mark.parametrize("M", [1, 12, 64, 200, 2500])
def test_chain(cuda_device, M):
    H, I, steps = 1024, 768, 12
    layers = [(*weight(cuda_device, 2 * I, H, 10 * i), *weight(cuda_device, H, I, 10 * i + 1),
               *weight(cuda_device, H, H, 10 * i + 2)) for i in range(steps)]
    x = torch.randn(M, H, generator=torch.Generator(device=cuda_device).manual_seed(M), device=cuda_device)
    x = x.to(torch.bfloat16)

    def run(sync):
        h, y = x.clone(), torch.empty_like(x)
        seen = []
        for w13, s13, w2, s2, w, s in layers:
            h.copy_(x)  # silu(gate) * up grows like a square: a chain through all steps overflows
            fp8_mlp(h, w13, s13, w2, s2, residual=h, out=h)
            sync()
            fp8_block_linear(h, w, s, residual=h, out=y)
            sync()
            q, qs = fp8_gate_up(y, w13, s13)
            sync()
            fp8_block_linear(q, w2, s2, x_scale=qs, residual=y, out=h)
            sync()
            seen.append((q, qs, h.clone(), y.clone()))
        return seen

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        got = run(lambda: None)
        for a, b in zip(got, want):
            assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))
    assert all(t.float().isfinite().all() for step in want for t in step)
    assert read_device_error(layer_error_word(cuda_device)) == 0
