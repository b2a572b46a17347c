"""A row's product does not depend on the batch it stands in beyond the rounding
of its sums: batches of other sizes take other kernels and add in another order.

Both results lie within (256 + 2 * K/128 + 2) u S of the exact one (u = 2^-24, S
the sum of the magnitudes; the bound of tests/test_gpu_dense.py), so within twice
that of each other."""
import pytest
import torch

from trials_b200 import fp8_block_linear, fp8_gate_up, per_block_quant_fp8, per_token_group_quant_fp8

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
U = 2.0 ** -24
BATCHES = (1, 2, 16, 17, 40, 64, 65, 130, 200, 333, 700, 1300)


def values(q, s, rows):
    r = s.double().repeat_interleave(rows, 0)[:q.shape[0]]
    return q.double() * r.repeat_interleave(128, 1)


@pytest.mark.parametrize("N,K", [(1000, 2048), (4096, 1024), (130, 4096), (2048, 384)])
def test_rows_across_batch_sizes(cuda_device, N, K):
    M = 2500
    g = torch.Generator(device=cuda_device).manual_seed(N + K)
    x = torch.randn(M, K, generator=g, device=cuda_device).to(torch.bfloat16)
    w, ws = per_block_quant_fp8((torch.randn(N, K, generator=g, device=cuda_device) * K ** -0.5).to(torch.bfloat16))
    xq, xs = per_token_group_quant_fp8(x)
    S = values(xq, xs, 1).abs() @ values(w, ws, 128).abs().t()
    bound = 2 * (256 + 2 * (K // 128) + 2) * U * S
    whole = fp8_block_linear(x, w, ws, out_dtype=torch.float32).double()
    for m in BATCHES:
        for first in (0, 777):
            part = fp8_block_linear(x[first:first + m], w, ws, out_dtype=torch.float32).double()
            assert ((part - whole[first:first + m]).abs() <= bound[first:first + m]).all()


@pytest.mark.parametrize("M,N,K", [(300, 12544, 512), (600, 15104, 256), (1100, 32768, 256), (1100, 16381, 384)])
def test_odd_numbers_of_token_tiles(cuda_device, M, N, K):
    """From one round of tiles to many, with half of a pair's last tile empty."""
    g = torch.Generator(device=cuda_device).manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g, device=cuda_device).to(torch.bfloat16)
    w, ws = per_block_quant_fp8((torch.randn(N, K, generator=g, device=cuda_device) * K ** -0.5).to(torch.bfloat16))
    xq, xs = per_token_group_quant_fp8(x)
    a, b = values(xq, xs, 1), values(w, ws, 128)
    bound = (256 + 2 * (K // 128) + 2) * U * (a.abs() @ b.abs().t())
    got = fp8_block_linear(x, w, ws, out_dtype=torch.float32)
    assert ((got.double() - a @ b.t()).abs() <= bound).all()
    res = torch.randn(M, N, generator=g, device=cuda_device).to(torch.bfloat16)
    assert torch.equal(fp8_block_linear(x, w, ws, residual=res), (got + res.float()).to(torch.bfloat16))


def test_gate_up_rows_across_batch_sizes(cuda_device):
    """Scales within the bound of both products' errors (d silu(g) <= 1.1 dg; silu good
    to 2^-20), as in tests/test_gpu_dense.py, on each side."""
    M, H, I = 1600, 1024, 512
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(M, H, generator=g, device=cuda_device).to(torch.bfloat16)
    w, ws = per_block_quant_fp8((torch.randn(2 * I, H, generator=g, device=cuda_device) * H ** -0.5).to(torch.bfloat16))
    xq, xs = per_token_group_quant_fp8(x)
    a, b = values(xq, xs, 1), values(w, ws, 128)
    y, e = a @ b.t(), (256 + 2 * (H // 128) + 2) * U * (a.abs() @ b.abs().t())
    gate, up, eg, eu = y[:, 0::2], y[:, 1::2], e[:, 0::2], e[:, 1::2]
    sg = gate / (1 + torch.exp(-gate))
    ev = 1.1 * eg * up.abs() + sg.abs() * eu + 1.1 * eg * eu + 2.0 ** -20 * (sg * up).abs()
    s64 = ((sg * up).abs().view(M, -1, 128).amax(2) / 448).clamp_min(1e-12)
    bound = 2 * (ev.view(M, -1, 128).amax(2) / 448 + 4 * U * s64)
    _, whole = fp8_gate_up(x, w, ws)
    for m in BATCHES:
        _, part = fp8_gate_up(x[300:300 + m], w, ws)
        assert ((part.double() - whole[300:300 + m].double()).abs() <= bound[300:300 + m]).all()
