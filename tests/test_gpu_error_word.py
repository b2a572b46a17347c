"""The error word of a (device, stream) through growth of the scratch, captures
and replays. A bit set in the word by hand stands for an error of an earlier
call: it stays until it is read."""
import pytest
import torch

from trials_b200 import (_lib, fp8_block_linear, fp8_mlp, layer_error_word, moe, per_block_quant_fp8,
                         read_device_error, synth)

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]


def weight(dev, N, K):
    return per_block_quant_fp8((torch.randn(N, K, device=dev) * K ** -0.5).to(torch.bfloat16))


def dense(dev):
    x = torch.randn(4, 256, device=dev).to(torch.bfloat16)
    w13, w2 = weight(dev, 512, 256), weight(dev, 256, 256)
    return lambda: fp8_mlp(x, *w13, *w2)


def layer(dev, M, H=512, seed=1, logits=False):
    E, k = 32, 4
    L = synth.make_layer(synth.LayerShape(M=M, H=H, I=256, E=E, topk=k), per_block_quant_fp8, seed=seed, device=dev)
    w = (L.w13, L.w13_scale, L.w2, L.w2_scale)
    if logits:
        x = torch.randn(M, E, device=dev)
        return lambda: moe.moe_layer_from_logits(L.hidden, x, *w, k, num_expert_group=4, topk_group=2)[0]
    ids = torch.randint(0, E, (M, k), device=dev).int()
    tw = torch.rand(M, k, device=dev)
    return lambda: moe.moe_decode_megakernel_full(L.hidden, *w, tw, ids)


def test_word_survives_larger_calls(cuda_device):
    stream = torch.cuda.Stream()
    calls = [dense(cuda_device), layer(cuda_device, 8), layer(cuda_device, 700), dense(cuda_device),
             layer(cuda_device, 1500, logits=True)]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        calls[0]()
        word = layer_error_word(cuda_device)
        word.fill_(_lib.DEVERR_TIMEOUT)
        for call in calls[1:]:
            call()
        assert layer_error_word(cuda_device).data_ptr() == word.data_ptr()
        assert read_device_error(layer_error_word(cuda_device)) == _lib.DEVERR_TIMEOUT
        assert read_device_error(word) == 0


def test_layer_reports_into_the_word(cuda_device):
    E, k, M = 32, 4, 8
    L = synth.make_layer(synth.LayerShape(M=M, H=512, I=256, E=E, topk=k), per_block_quant_fp8, seed=3,
                         device=cuda_device)
    ids = torch.randint(0, E, (M, k), device=cuda_device).int()
    ids[3, 1] = E + 5
    with torch.cuda.stream(torch.cuda.Stream()):
        word = layer_error_word(cuda_device)
        moe.moe_decode_megakernel_full(L.hidden, L.w13, L.w13_scale, L.w2, L.w2_scale,
                                       torch.ones(M, k, device=cuda_device), ids)
        assert read_device_error(word) == _lib.DEVERR_BAD_EXPERT_ID


@pytest.mark.parametrize("make", [dense, lambda dev: layer(dev, 8), lambda dev: layer(dev, 8, logits=True)])
def test_first_use_under_capture(cuda_device, make):
    """Two graphs captured on a stream that nothing ran on before, the second
    replayed first; no replay clears the word."""
    calls = [make(cuda_device), make(cuda_device)]
    want = [c() for c in calls]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(c())
        graphs.append(g)
    with torch.cuda.stream(stream):
        word = layer_error_word(cuda_device)
        assert read_device_error(word) == 0
        word.fill_(_lib.DEVERR_TIMEOUT)
        for k in (1, 0, 1):
            graphs[k].replay()
            assert torch.equal(outs[k], want[k])
        assert read_device_error(word) == _lib.DEVERR_TIMEOUT
    assert read_device_error(layer_error_word(cuda_device)) == 0  # the current stream's is another


@pytest.mark.parametrize("one_launch", [0, 1])
def test_graph_outlives_its_scratch(cuda_device, one_launch):
    """A graph captured with a small scratch, replayed after a larger call has
    replaced it: its results are right and memory allocated since is untouched."""
    prev = _lib.lib().b200moe_set_layer_launch(one_launch)
    try:
        small, large = layer(cuda_device, 8, seed=4), layer(cuda_device, 900, seed=5)
        want = small()
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            small()
            graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = small()
        with torch.cuda.stream(stream):
            large()
            bufs = [torch.full((2 ** n,), 7, dtype=torch.uint8, device=cuda_device) for n in range(16, 27)]
            for _ in range(3):
                out.zero_()
                graph.replay()
                assert torch.equal(out, want)
            for b in bufs:
                assert (b == 7).all()
            assert read_device_error(layer_error_word(cuda_device)) == 0
    finally:
        _lib.lib().b200moe_set_layer_launch(prev)


def test_word_under_capture(cuda_device):
    """The word of a stream can be asked for while it is captured."""
    x = torch.randn(4, 256, device=cuda_device).to(torch.bfloat16)
    w, ws = weight(cuda_device, 256, 256)
    want = fp8_block_linear(x, w, ws)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        word = layer_error_word(cuda_device)
        out = fp8_block_linear(x, w, ws)
    graph.replay()
    assert torch.equal(out, want)
    assert read_device_error(word) == 0


@pytest.mark.parametrize("bit,left", [(_lib.DEVERR_TIMEOUT, 0), (_lib.DEVERR_BAD_EXPERT_ID, 5)])
def test_counters_after_a_timeout(cuda_device, bit, left):
    """Reading a timeout puts the counters behind the word back to zero; they are
    nobody else's to touch, so other errors leave them alone."""
    with torch.cuda.stream(torch.cuda.Stream()):
        word = layer_error_word(cuda_device)
        header = torch.as_tensor(moe._DeviceInts(word.data_ptr(), 64), device=cuda_device)
        header[1:4] = 5
        word.fill_(bit)
        assert read_device_error(word, clear=False) == bit and (header[1:4] == 5).all()
        assert read_device_error(word) == bit
        assert header[0] == 0 and (header[1:4] == left).all()
        header.zero_()
        own = torch.full((8,), bit, dtype=torch.int32, device=cuda_device)  # a caller's own word
        assert read_device_error(own[:1]) == bit and (own[1:] == bit).all()
        call = layer(cuda_device, 8, logits=True)
        want = call()
        assert torch.equal(call(), want) and read_device_error(word) == 0
