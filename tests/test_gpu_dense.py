"""Dense FP8 products against their definition in 64 bits.

Bounds. u = 2^-24. An e4m3 product is exact in fp32; a K block's partial takes
128 additions, each off by at most 2u of the sum of magnitudes S (the tensor
core may truncate), and its promotion a rounding of the scales' product and of
the fma, so |y - exact| <= (256 + 2 * K/128 + 2) u S in fp32; the residual adds
one rounding, a bf16 result one of 2^-8 of its value."""
import pytest
import torch

from oracle import moe_oracle as orc
from trials_b200 import (_lib, fp8_block_linear, fp8_gate_up, fp8_mlp, layer_error_word, moe,
                         per_block_quant_fp8, per_token_group_quant_fp8, read_device_error)

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
FP8 = torch.float8_e4m3fn
U = 2.0 ** -24


def make(dev, M, N, K, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(M, K, generator=g, device=dev) * torch.exp(torch.randn(M, 1, generator=g, device=dev)))
    w = torch.randn(N, K, generator=g, device=dev) * K ** -0.5
    w *= 1 + (torch.arange(N, device=dev)[:, None] // 128) % 3  # blocks of different size
    wq, ws = per_block_quant_fp8(w.to(torch.bfloat16))
    return x.to(torch.bfloat16), wq, ws


def values(q, s, rows):
    N, K = q.shape
    r = s.double().repeat_interleave(rows, 0)[:N] if rows > 1 else s.double()
    return q.double() * r.repeat_interleave(128, 1)


def exact(xq, xs, wq, ws):
    """(y, bound of the fp32 result) in 64 bits."""
    a, b = values(xq, xs, 1), values(wq, ws, 128)
    K = xq.shape[1]
    return a @ b.t(), (256 + 2 * (K // 128) + 2) * U * (a.abs() @ b.abs().t())


def check(out, y, bound):
    assert out.shape == y.shape
    if out.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (y.abs() + bound)
    off = (out.double() - y).abs()
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), float((off / bound).max())


SHAPES = [(1, 128, 128), (1, 4096, 1024), (2, 6144, 2048), (3, 256, 6144), (11, 4096, 512), (2, 1, 128), (7, 300, 256), (16, 256, 6144), (17, 129, 384), (33, 576, 896),
          (64, 2048, 2048), (65, 257, 512), (100, 8, 1152), (127, 1000, 256), (128, 512, 640), (129, 383, 2048),
          (255, 64, 128), (300, 1280, 768), (512, 640, 1024), (1000, 384, 512), (2100, 520, 384), (5000, 130, 256),
          # 128-column tiles: split, one each over two rounds, and pairs past that
          (300, 1000, 1152), (777, 77, 768), (20000, 24, 256), (40000, 128, 128),
          # rows quantised in the product, as many as there may be
          (4, 4096, 6144), (12, 5000, 1024),
          # pairs: whole and partial boxes of the output
          (5000, 328, 256), (4100, 776, 512), (9000, 256, 1024)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(cuda_device, M, N, K):
    x, wq, ws = make(cuda_device, M, N, K, M + N + K)
    xq, xs = per_token_group_quant_fp8(x)
    y, bound = exact(xq, xs, wq, ws)
    f32 = fp8_block_linear(xq, wq, ws, x_scale=xs, out_dtype=torch.float32)
    check(f32, y, bound)
    # bf16 rows are quantised the same way; the same product rounded once
    assert torch.equal(fp8_block_linear(x, wq, ws, out_dtype=torch.float32), f32)
    assert torch.equal(fp8_block_linear(x, wq, ws), f32.to(torch.bfloat16))
    res = torch.randn(M, N, device=cuda_device).to(torch.bfloat16)
    with_res = fp8_block_linear(xq, wq, ws, x_scale=xs, residual=res)
    assert torch.equal(with_res, (f32 + res.float()).to(torch.bfloat16))
    with_res32 = fp8_block_linear(xq, wq, ws, x_scale=xs, residual=res, out_dtype=torch.float32)
    assert torch.equal(with_res32, f32 + res.float())
    into = res.clone()
    assert fp8_block_linear(x, wq, ws, residual=into, out=into) is into
    assert torch.equal(into, with_res)
    assert read_device_error(layer_error_word(cuda_device)) == 0


@pytest.mark.parametrize("M,H,I", [(1, 256, 128), (1, 6144, 512), (2, 6144, 2048), (5, 4096, 512), (3, 640, 256), (16, 1024, 384), (63, 256, 1280), (64, 2048, 256),
                                   (65, 384, 128), (128, 512, 512), (200, 1152, 640), (513, 256, 384),
                                   (1500, 384, 256)])
def test_gate_up(cuda_device, M, H, I):
    """s and q against silu(gate) * up in 64 bits. d silu(g) <= 1.1 dg, silu
    itself is good to 2^-20 of its value, so v = silu(g) u is off by at most
    e = 1.1 eg |u| + |silu(g)| eu + 1.1 eg eu + 2^-20 |v|; s by the largest e of
    its group over 448 and two roundings; q stands for v / s within half a step
    of e4m3 (2^-4 of the value, 2^-10 below its normal range)."""
    x, wq, ws = make(cuda_device, M, 2 * I, H, M + H + I)
    xq, xs = per_token_group_quant_fp8(x)
    y, b = exact(xq, xs, wq, ws)
    g, u, eg, eu = y[:, 0::2], y[:, 1::2], b[:, 0::2], b[:, 1::2]
    sg = g / (1 + torch.exp(-g))
    v = sg * u
    e = 1.1 * eg * u.abs() + sg.abs() * eu + 1.1 * eg * eu + 2.0 ** -20 * v.abs()
    q, s = fp8_gate_up(xq, wq, ws, x_scale=xs)
    assert q.dtype == FP8 and q.shape == (M, I) and s.shape == (M, I // 128)
    vg, egr = v.view(M, -1, 128), e.view(M, -1, 128)
    s64 = (vg.abs().amax(2) / 448).clamp_min(1e-12)
    assert ((s.double() - s64).abs() <= egr.amax(2) / 448 + 4 * U * s64).all()
    sd = s.double().repeat_interleave(128, 1)
    got = q.double()
    step = torch.maximum(2.0 ** -4 * (v / sd).abs(), torch.full_like(v, 2.0 ** -10))
    off = (got - (v / sd).clamp(-448, 448)).abs()
    assert (off <= step * (1 + 2.0 ** -3) + e / sd * (1 + 2.0 ** -3)).all()
    q2, s2 = fp8_gate_up(x, wq, ws)  # bf16 rows
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


@pytest.mark.parametrize("M,H,I", [(1, 256, 128), (1, 6144, 2048), (5, 512, 384), (64, 1024, 512), (100, 640, 256),
                                   (300, 256, 640), (1200, 512, 256)])
def test_mlp_is_gate_up_then_linear(cuda_device, M, H, I):
    x, w13, s13 = make(cuda_device, M, 2 * I, H, M)
    _, w2, s2 = make(cuda_device, 1, H, I, M + 1)
    res = torch.randn(M, H, device=cuda_device).to(torch.bfloat16)
    q, s = fp8_gate_up(x, w13, s13)
    want = fp8_block_linear(q, w2, s2, x_scale=s, residual=res)
    assert torch.equal(fp8_mlp(x, w13, s13, w2, s2, residual=res), want)
    xq, xs = per_token_group_quant_fp8(x)
    assert torch.equal(fp8_mlp(xq, w13, s13, w2, s2, x_scale=xs, residual=res), want)
    assert torch.equal(fp8_mlp(x, w13, s13, w2, s2), fp8_block_linear(q, w2, s2, x_scale=s))
    y, bound = exact(q, s, w2, s2)
    check(want, y + res.double(), bound + U * (y + res.double()).abs())
    # a row's result does not depend on the batch it is in beyond rounding of the partial sums
    out = res.clone()
    assert fp8_mlp(x, w13, s13, w2, s2, residual=out, out=out) is out
    assert torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 40, 200])
def test_mlp_is_a_one_expert_layer(cuda_device, M):
    """The same expert through the routed layer (one expert, weight 1)."""
    H, I = 512, 256
    x, w13, s13 = make(cuda_device, M, 2 * I, H, M)
    _, w2, s2 = make(cuda_device, 1, H, I, 9)
    ids = torch.zeros(M, 1, dtype=torch.int32, device=cuda_device)
    tw = torch.ones(M, 1, device=cuda_device)
    ref = moe.moe_decode_megakernel_full(x, w13[None], s13[None], w2[None], s2[None], tw, ids)
    assert orc.rel_l2(fp8_mlp(x, w13, s13, w2, s2).float(), ref.float()) < 5e-3


def test_empty_batch(cuda_device):
    x, w13, s13 = make(cuda_device, 1, 256, 256)
    assert fp8_block_linear(x[:0], w13, s13).shape == (0, 256)
    q, s = fp8_gate_up(x[:0], w13, s13)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    _, w2, s2 = make(cuda_device, 1, 256, 128)
    assert fp8_mlp(x[:0], w13, s13, w2, s2).shape == (0, 256)


@pytest.mark.parametrize("M,N", [(3, 200), (130, 200), (130, 264), (70, 512), (5000, 328)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_surroundings(cuda_device, M, N, dtype):
    """Row strides of every operand; nothing outside the result is written."""
    K = 384
    x, wq, ws = make(cuda_device, M, N, K)
    xq, xs = per_token_group_quant_fp8(x)
    want = fp8_block_linear(xq, wq, ws, x_scale=xs, out_dtype=dtype)
    wide = torch.zeros(M, K + 128, dtype=FP8, device=cuda_device)
    wide[:, :K] = xq
    wide_w = torch.zeros(N, K + 64, dtype=FP8, device=cuda_device)
    wide_w[:, :K] = wq
    wide_s = torch.full((M, 7), -1.0, device=cuda_device)
    wide_s[:, 2:5] = xs
    for extra in (5, 8):  # rows of out that start aligned, and that do not
        buf = torch.full((M + 2, N + extra), 7.0, dtype=dtype, device=cuda_device)
        out = buf[1:M + 1, :N]
        assert fp8_block_linear(wide[:, :K], wide_w[:, :K], ws, x_scale=wide_s[:, 2:5], out=out, out_dtype=dtype) is out
        assert torch.equal(out, want)
        rest = buf.clone()
        rest[1:M + 1, :N] = 7.0
        assert (rest == 7.0).all()
    # layouts that have to be copied first
    assert torch.equal(fp8_block_linear(xq.t().contiguous().t(), wq, ws, x_scale=xs.t().contiguous().t(),
                                        out_dtype=dtype), want)
    bx = torch.zeros(M, K + 3, dtype=torch.bfloat16, device=cuda_device)
    bx[:, 3:] = x
    assert torch.equal(fp8_block_linear(bx[:, 3:], wq, ws, out_dtype=dtype), want)
    wide_x = torch.zeros(M, K + 16, dtype=torch.bfloat16, device=cuda_device)
    wide_x[:, 8:K + 8] = x
    assert torch.equal(fp8_block_linear(wide_x[:, 8:K + 8], wq, ws, out_dtype=dtype), want)


@pytest.mark.parametrize("M", [5, 300])
def test_bad_numbers_stay_in_their_row(cuda_device, M):
    N, K = 256, 512
    x, wq, ws = make(cuda_device, M, N, K)
    xq, xs = per_token_group_quant_fp8(x)
    want = fp8_block_linear(xq, wq, ws, x_scale=xs)
    qw, sw = fp8_gate_up(xq, wq, ws, x_scale=xs)
    xq.view(torch.uint8)[2, 100] = 0x7F  # NaN
    xs[3, 1] = float("inf")
    got = fp8_block_linear(xq, wq, ws, x_scale=xs)
    q, s = fp8_gate_up(xq, wq, ws, x_scale=xs)
    assert got[2].isnan().all() and not got[3].isfinite().any()
    keep = [r for r in range(M) if r not in (2, 3)]
    assert torch.equal(got[keep], want[keep])
    assert torch.equal(q.view(torch.uint8)[keep], qw.view(torch.uint8)[keep]) and torch.equal(s[keep], sw[keep])


@pytest.mark.parametrize("M", [1, 48, 700])
def test_same_bits_every_time(cuda_device, M):
    x, w13, s13 = make(cuda_device, M, 1024, 1536)
    _, w2, s2 = make(cuda_device, 1, 1536, 512)
    first = fp8_mlp(x, w13, s13, w2, s2)
    for _ in range(5):
        assert torch.equal(fp8_mlp(x, w13, s13, w2, s2), first)


@pytest.mark.parametrize("M", [1, 64, 400])
def test_other_stream_and_graph(cuda_device, M):
    x, w13, s13 = make(cuda_device, M, 1024, 768)
    _, w2, s2 = make(cuda_device, 1, 768, 512)
    want = fp8_mlp(x, w13, s13, w2, s2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp8_mlp(x, w13, s13, w2, s2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs of the same shapes, replayed in turn on new inputs
    xs = [torch.zeros_like(x), torch.zeros_like(x)]
    graphs, outs = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fp8_mlp(xs[k], w13, s13, w2, s2))
        graphs.append(graph)
    xs[0].copy_(x)
    xs[1].copy_(-x)
    graphs[0].replay()
    graphs[1].replay()
    graphs[0].replay()
    assert torch.equal(outs[0], want)
    assert torch.equal(outs[1], fp8_mlp(-x, w13, s13, w2, s2))


def test_calls_at_once(cuda_device):
    """Every kind of product on six streams at the same time."""
    _, w13, s13 = make(cuda_device, 1, 2048, 2048)
    _, w2, s2 = make(cuda_device, 1, 2048, 1024)
    inputs = [make(cuda_device, M, 128, 2048, M)[0] for M in (1, 16, 64, 100, 400, 1500)]

    def work(x):
        y = fp8_mlp(x, w13, s13, w2, s2, residual=x)
        return y, fp8_block_linear(x, w13[:1000], s13[:8], residual=y[:, :1000])

    want = [work(x) for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[] for _ in inputs]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(work(inputs[k]))
    torch.cuda.synchronize()
    for k, outs in enumerate(got):
        for y, z in outs:
            assert torch.equal(y, want[k][0]) and torch.equal(z, want[k][1])
    for s in streams:
        with torch.cuda.stream(s):
            assert read_device_error(layer_error_word(cuda_device)) == 0


def test_ragged_weight_quantiser(cuda_device):
    for N in (1, 100, 128, 200, 300):
        w = torch.randn(N, 384, device=cuda_device).to(torch.bfloat16)
        full = torch.zeros(-(-N // 128) * 128, 384, dtype=torch.bfloat16, device=cuda_device)
        full[:N] = w
        q, s = per_block_quant_fp8(w)
        oq, os_ = orc.per_block_quant_fp8(full[None])
        assert torch.equal(s, os_[0]) and torch.equal(q.view(torch.uint8), oq[0, :N].view(torch.uint8))
    pair = torch.randn(2, 200, 256, device=cuda_device).to(torch.bfloat16)
    q, s = per_block_quant_fp8(pair)
    for e in range(2):
        q1, s1 = per_block_quant_fp8(pair[e])
        assert torch.equal(q[e].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[e], s1)


def test_row_quantiser_is_the_division(cuda_device):
    """Codes of groups of every size, zeros of both signs, subnormals, infinities
    and NaN: the bits of the IEEE quotient x / s, clamped and rounded."""
    g = torch.Generator(device=cuda_device).manual_seed(5)
    for k in range(6):
        x = torch.randn(8192, 1024, generator=g, device=cuda_device)
        if k > 0:  # spread inside a group, then groups from 2^-120 to 2^120
            x *= torch.exp2(torch.rand(8192, 1024, generator=g, device=cuda_device) * -8 * k)
            x *= torch.exp2(torch.randint(-120, 120, (8192, 1), generator=g, device=cuda_device).float())
        x = x.to(torch.bfloat16)
        x[0, ::3], x[1, ::2], x[2, :] = 0.0, -0.0, 0.0
        x[3, 7], x[4, 9] = float("inf"), float("nan")
        x[5] = torch.finfo(torch.bfloat16).max
        x[6] = torch.tensor(2.0 ** -130)
        x[7, ::2] = -x[7, ::2].abs() * 0.0
        q, s = per_token_group_quant_fp8(x)
        v = x.float().view(8192, 8, 128)
        amax = torch.nan_to_num(v.abs(), nan=0.0, posinf=float("inf")).amax(2)
        sw = (amax / torch.full_like(amax, 448.0)).clamp_min(1e-12)
        assert torch.equal(s, sw)
        quot = v / sw.unsqueeze(2)
        clamped = torch.where(quot.isnan(), torch.full_like(quot, -448.0), quot.clamp(-448.0, 448.0))
        want = clamped.to(FP8).view(8192, 1024)
        assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("M", [1, 2, 40, 200, 1300])
def test_in_place(cuda_device, M):
    """A residual stream updated in place; outputs beside the rows in one buffer."""
    H, I = 512, 1024
    x, w13, s13 = make(cuda_device, M, 2 * I, H, M)
    _, w2, s2 = make(cuda_device, 1, H, I, M + 1)
    want = fp8_mlp(x, w13, s13, w2, s2, residual=x)
    h = x.clone()
    assert fp8_mlp(h, w13, s13, w2, s2, residual=h, out=h) is h
    assert torch.equal(h, want)
    h = x.clone()
    assert torch.equal(fp8_mlp(h, w13, s13, w2, s2, out=h), fp8_mlp(x, w13, s13, w2, s2))
    _, wq, ws = make(cuda_device, 1, H, H, 5)
    buf = torch.cat([x, x, x], 1)
    fp8_block_linear(buf[:, :H], wq, ws, residual=buf[:, 2 * H:], out=buf[:, H:2 * H])
    assert torch.equal(buf, torch.cat([x, fp8_block_linear(x, wq, ws, residual=x), x], 1))
    for out, res in ((x, None), (buf[:, 1:H + 1], None if M > 1 else buf[:, :H]), (buf[:, 2:H + 2], buf[:, :H])):
        with pytest.raises(ValueError, match="overlap"):
            fp8_block_linear(buf[:, :H] if out is not x else x, wq, ws, residual=res, out=out)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 outputs, more than 2^32 bytes of rows: the last rows are the
    rows' own product."""
    M, N, K = 270_000, 8192, 128
    if torch.cuda.get_device_properties(cuda_device).total_memory < 40e9:
        pytest.skip("needs 40 GB")
    x, wq, ws = make(cuda_device, 1000, N, K)
    big = x.repeat(M // 1000, 1)
    want = fp8_block_linear(x, wq, ws, residual=None)
    out = fp8_block_linear(big, wq, ws)
    for first in (0, M // 2, M - 1000):
        assert torch.equal(out[first:first + 1000], want)
    assert torch.equal(fp8_block_linear(big, wq, ws, residual=out, out=out)[-1000:],
                       fp8_block_linear(x, wq, ws, residual=want))
    del out, big
    x, w13, s13 = make(cuda_device, 500, 256, 8192)
    q, s = fp8_gate_up(x.repeat(600, 1), w13, s13)
    assert torch.equal(q[-500:].view(torch.uint8), q[:500].view(torch.uint8)) and torch.equal(s[-500:], s[:500])


def test_refusals_on_device(cuda_device):
    x, wq, ws = make(cuda_device, 4, 200, 256)
    with pytest.raises(ValueError):
        fp8_block_linear(x, wq, ws[:1])
    with pytest.raises(ValueError):
        fp8_block_linear(x, wq, ws, out=torch.empty(4, 199, dtype=torch.bfloat16, device=cuda_device))
    with pytest.raises(NotImplementedError):
        fp8_block_linear(x, wq, ws, out_dtype=torch.float16)
    with pytest.raises(NotImplementedError):
        fp8_gate_up(x, wq, ws)  # 200 rows: I = 100
    with pytest.raises(NotImplementedError):  # weight rows that start misaligned
        buf = torch.zeros(200 * 256 + 8, dtype=torch.uint8, device=cuda_device)[8:].view(200, 256).view(FP8)
        fp8_block_linear(x, buf, ws)
    assert read_device_error(layer_error_word(cuda_device)) == 0
