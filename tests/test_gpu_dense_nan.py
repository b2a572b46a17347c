"""NaN and infinities through the dense FP8 products: what is broken in a token's
row, or in a weight, shows in the outputs it reaches and nowhere else, as in
  s = max(amax / 448, 1e-12), q = e4m3(clamp(v / s)), y = sum xs ws xq wq."""
import pytest
import torch

from trials_b200 import (fp8_block_linear, fp8_gate_up, fp8_mlp, layer_error_word, per_block_quant_fp8,
                         per_token_group_quant_fp8, read_device_error)

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
FP8 = torch.float8_e4m3fn

# The kernels: rows quantised in the product, split, token-major tiles of 128 and
# 256 columns (gate/up: of 256), pairs.
SIZES = [(5, 512, 256), (12, 1024, 2560), (40, 1024, 512), (300, 1024, 4096), (200, 4096, 2048), (3000, 512, 2048),
         (2500, 640, 640)]


def weight(dev, N, K, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return per_block_quant_fp8((torch.randn(N, K, generator=g, device=dev) * K ** -0.5).to(torch.bfloat16))


def rows(dev, M, K):
    g = torch.Generator(device=dev).manual_seed(M)
    return torch.randn(M, K, generator=g, device=dev).to(torch.bfloat16)


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def nan_rows(t):
    return t.float().isnan()


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(cuda_device, M, N, K, fp8, dtype):
    w, ws = weight(cuda_device, N, K)
    x = rows(cuda_device, M, K)
    bad = x.clone()
    bad[2, 100], bad[3, K - 1] = float("nan"), float("-inf")
    if fp8:
        x, xs = per_token_group_quant_fp8(x)
        bad, bs = x.clone(), xs.clone()
        bad.view(torch.uint8)[2, 100], bs[3, K // 128 - 1] = 0xFF, float("nan")
        xs = dict(x_scale=xs)
        bs = dict(x_scale=bs)
    else:
        xs = bs = {}
    res = torch.ones(M, N, dtype=torch.bfloat16, device=cuda_device)
    want = fp8_block_linear(x, w, ws, residual=res, out_dtype=dtype, **xs)
    got = fp8_block_linear(bad, w, ws, residual=res, out_dtype=dtype, **bs)
    keep = [r for r in range(M) if r not in (2, 3)]
    assert want.isfinite().all() and same(got[keep], want[keep])
    assert got[2:4].isnan().all()


@pytest.mark.parametrize("M,I,H", [(m, n // 2, k) for m, n, k in SIZES])
@pytest.mark.parametrize("fp8", [False, True])
def test_gate_up_and_mlp_rows(cuda_device, M, I, H, fp8):
    I = max(I // 128, 1) * 128
    w13, s13 = weight(cuda_device, 2 * I, H)
    w2, s2 = weight(cuda_device, H, I, 1)
    x = rows(cuda_device, M, H)
    bad = x.clone()
    bad[2, 100], bad[3, H - 1] = float("nan"), float("inf")
    if fp8:
        x, xs = per_token_group_quant_fp8(x)
        bad, bs = x.clone(), xs.clone()
        bad.view(torch.uint8)[2, 100], bs[3, 0] = 0x7F, float("inf")
        xs, bs = dict(x_scale=xs), dict(x_scale=bs)
    else:
        xs = bs = {}
    q, s = fp8_gate_up(x, w13, s13, **xs)
    qb, sb = fp8_gate_up(bad, w13, s13, **bs)
    keep = [r for r in range(M) if r not in (2, 3)]
    assert same(qb[keep], q[keep]) and same(sb[keep], s[keep]) and s.isfinite().all()
    assert sb[2].isnan().all() and nan_rows(qb[2]).all()
    assert not sb[3].isfinite().any()
    res = torch.ones(M, H, dtype=torch.bfloat16, device=cuda_device)
    y = fp8_mlp(x, w13, s13, w2, s2, residual=res, **xs)
    yb = fp8_mlp(bad, w13, s13, w2, s2, residual=res, **bs)
    assert same(yb[keep], y[keep]) and yb[2].isnan().all() and not yb[3].isfinite().any()
    assert read_device_error(layer_error_word(cuda_device)) == 0


@pytest.mark.parametrize("M,I,H", [(5, 384, 512), (40, 384, 1024), (200, 2048, 1152), (3000, 2048, 512)])
@pytest.mark.parametrize("row", [10, 11])  # a gate row and an up row
def test_nan_in_one_column_reaches_its_group(cuda_device, M, I, H, row):
    w13, s13 = weight(cuda_device, 2 * I, H)
    x = rows(cuda_device, M, H)
    q, s = fp8_gate_up(x, w13, s13)
    w13.view(torch.uint8)[256 + row, 7] = 0x7F  # column 128 + row / 2: the second group
    qb, sb = fp8_gate_up(x, w13, s13)
    assert sb[:, 1].isnan().all() and nan_rows(qb[:, 128:256]).all()
    keep = [g for g in range(I // 128) if g != 1]
    assert same(sb[:, keep], s[:, keep])
    assert same(qb[:, :128].contiguous(), q[:, :128].contiguous())
    assert same(qb[:, 256:].contiguous(), q[:, 256:].contiguous())


@pytest.mark.parametrize("M,I,H", [(5, 128, 256), (40, 128, 256), (300, 2048, 512), (3000, 2048, 512)])
def test_overflow_of_the_product(cuda_device, M, I, H):
    """Gates of +inf: values of +-inf, an infinite scale, zeros beside NaN. Gates
    of -inf: silu is -0, and -0 times an infinite up is NaN."""
    x = torch.zeros(M, H, dtype=torch.bfloat16, device=cuda_device)
    x[:, 0] = 1.0
    w = torch.zeros(2 * I, H, device=cuda_device)
    w[0::2, 0], w[1::2, 0] = 1.0, 0.5
    w13, s13 = per_block_quant_fp8(w.to(torch.bfloat16))
    s13 = s13.clone()
    q, s = fp8_gate_up(x, w13, s13)
    assert s.isfinite().all() and (s[0] == s).all()
    x[1, 0] = 3e38
    s13 *= 4
    q, s = fp8_gate_up(x, w13, s13)  # row 1: gate 1.2e39
    assert s[1].isinf().all() and nan_rows(q[1]).all()
    assert s[2:].isfinite().all() and s[0].isfinite().all() and not nan_rows(q[2:]).any()
    x[1, 0] = -3e38
    q, s = fp8_gate_up(x, w13, s13)
    assert s[2:].isfinite().all() and not nan_rows(q[2:]).any()
    # gate -inf, up -6e38 = -inf: -0 * -inf
    assert s[1].isnan().all() and nan_rows(q[1]).all()


def test_the_row_quantiser_itself_is_as_before(cuda_device):
    """per_token_group_quant_fp8 and the routed layer keep their rule: the largest
    number counts and NaN becomes -448."""
    x = rows(cuda_device, 8, 256)
    x[2, 5] = 0.0
    want, ws = per_token_group_quant_fp8(x)
    x[2, 5] = float("nan")
    q, s = per_token_group_quant_fp8(x)
    assert q[2, 5].float() == -448 and same(s, ws)
    q[2, 5] = want[2, 5]
    assert same(q, want)
