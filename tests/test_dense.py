"""Refusals of the dense FP8 products (fp8_block_linear, fp8_gate_up, fp8_mlp):
checked on the host before anything is launched, so no GPU is needed."""
import struct
from pathlib import Path

import pytest
import torch

from trials_b200 import _lib, dense, fp8_block_linear, fp8_gate_up, fp8_mlp

P = 256  # a non-null, aligned address that no refused call touches
FP8 = torch.float8_e4m3fn


def call(name, *args):
    """A C entry whose arguments come packed (None = NULL)."""
    return getattr(_lib.lib(), name)(struct.pack(f"{len(args)}q", *(0 if a is None else a for a in args)))


def linear(x=P, xq=None, xs=None, ld_x=256, ld_xs=2, M=4, N=100, K=256, w=P, ld_w=256, ws=P, res=None, ld_res=0,
           out=P, ld_out=100, f32=0, work=P, nwork=1 << 20, err=P):
    return call("b200moe_linear", x, xq, xs, ld_x, ld_xs, M, N, K, w, ld_w, ws, res, ld_res, out, ld_out, f32, work,
                nwork, err, None)


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(N=0), dict(K=0), dict(w=None), dict(ws=None), dict(err=None), dict(ld_w=128), dict(x=None),
    dict(xq=P, xs=P), dict(x=None, xq=P), dict(x=None, xq=P, xs=P, ld_xs=1), dict(ld_x=128), dict(out=None),
    dict(ld_out=99), dict(res=P, ld_res=99)])
def test_linear_invalid_arguments(kw):
    assert linear(**kw) == _lib.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [
    dict(K=200, ld_x=256, ld_w=256), dict(w=P + 8), dict(ld_w=264), dict(x=P + 8), dict(ld_x=260),
    dict(x=None, xq=P, xs=P, ld_x=264), dict(out=P + 1), dict(f32=1, out=P + 2), dict(M=(1 << 30) + 1),
    dict(N=(1 << 24) + 1, ld_out=1 << 25)])
def test_linear_unsupported_layouts(kw):
    assert linear(**kw) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(M=3000, work=None), dict(M=3000, nwork=100), dict(M=3000, work=P + 16)])
def test_linear_workspace(kw):
    assert linear(**kw) == _lib.ERR_WORKSPACE


def test_output_over_an_input():
    """Refused where the product may still read what it stores over; columns side
    by side in one buffer are apart. (The base: P = M rows of K = N = 256.)"""
    base = dict(N=256, ld_out=256, w=1 << 30, ws=1 << 32, out=1 << 34)
    for kw in (dict(out=P), dict(out=P + 3 * 512 + 510, ld_out=300), dict(out=1 << 30), dict(out=1 << 32),
               dict(x=None, xq=P, xs=1 << 36, ld_xs=2, out=1 << 36), dict(x=None, xq=P, xs=1 << 36, out=P),
               dict(res=(1 << 34) + 2, ld_res=256), dict(res=1 << 34, ld_res=260),
               dict(res=1 << 34, ld_res=256, f32=1), dict(ld_out=1024, out=P + 256, ld_x=1024),
               dict(res=(1 << 34) + 768, ld_res=512, ld_out=512)):
        assert linear(**{**base, **kw}) == _lib.ERR_INVALID_ARG, kw
        assert b"overlap" in _lib.lib().b200moe_last_error_message()

    def mlp(out, res=None, ld_res=256):
        return call("b200moe_mlp", P, None, None, 256, 0, 4, 256, 128, 1 << 28, 1 << 29, 1 << 30, 1 << 32, res, ld_res,
                    out, 256, P, 1 << 20, P, None)

    for args in ((1 << 30,), (1 << 32,), (1 << 34, (1 << 34) + 4)):
        assert mlp(*args) == _lib.ERR_INVALID_ARG

    def gate_up(q, s):
        return call("b200moe_gate_up", P, None, None, 256, 0, 4, 256, 128, 1 << 30, 256, 1 << 32, q, 128, s, 1, P,
                    1 << 20, P, None)

    for args in ((P, 1 << 36), (1 << 34, P), (1 << 30, 1 << 36), (1 << 34, 1 << 32)):
        assert gate_up(*args) == _lib.ERR_INVALID_ARG


def test_empty_batches_launch_nothing():
    L = _lib.lib()
    assert linear(M=0, x=None, out=None, work=None, nwork=0) == _lib.OK
    assert call("b200moe_gate_up", None, None, None, 0, 0, 0, 256, 128, P, 256, P, None, 0, None, 0, None, 0, P,
                None) == _lib.OK
    assert call("b200moe_mlp", None, None, None, 0, 0, 0, 256, 128, P, P, P, P, None, 0, None, 0, None, 0, P,
                None) == _lib.OK
    for name in ("b200moe_linear", "b200moe_gate_up", "b200moe_mlp"):
        assert getattr(L, name)(None) == _lib.ERR_INVALID_ARG
    assert L.b200moe_linear_workspace_size(0, 256, 256, 1, 0) == 0
    assert L.b200moe_mlp_workspace_size(0, 256, 128, 1) == 0


def test_gate_up_and_mlp_host_checks():
    L = _lib.lib()

    def gate_up(I=128, q=P, ld_q=128, s=P, ld_s=1, H=256):
        return call("b200moe_gate_up", P, None, None, 256, 0, 4, H, I, P, 256, P, q, ld_q, s, ld_s, P, 1 << 20, P,
                    None)

    assert gate_up(I=0) == _lib.ERR_INVALID_ARG
    assert gate_up(q=None) == _lib.ERR_INVALID_ARG
    assert gate_up(ld_q=64) == _lib.ERR_INVALID_ARG
    assert gate_up(I=64, ld_q=64) == _lib.ERR_UNSUPPORTED
    assert gate_up(q=P + 8) == _lib.ERR_UNSUPPORTED
    assert gate_up(H=384) == _lib.ERR_INVALID_ARG  # row stride 256 is shorter than a row

    def mlp(I=128, w2=P, out=P, nwork=1 << 20, res=None):
        return call("b200moe_mlp", P, None, None, 256, 0, 4, 256, I, P, P, w2, P, res, 0, out, 256, P, nwork, P, None)

    assert mlp(I=0) == _lib.ERR_INVALID_ARG
    assert mlp(I=192) == _lib.ERR_UNSUPPORTED
    assert mlp(w2=None) == _lib.ERR_INVALID_ARG
    assert mlp(w2=P + 8) == _lib.ERR_UNSUPPORTED
    assert mlp(res=P) == _lib.ERR_INVALID_ARG  # residual without a stride
    assert mlp(nwork=L.b200moe_mlp_workspace_size(4, 256, 128, 1) - 1) == _lib.ERR_WORKSPACE


def test_workspace_sizes_cover_codes_and_scales():
    L = _lib.lib()
    # many bf16 rows are quantised into the workspace
    assert L.b200moe_linear_workspace_size(3000, 384, 384, 1, 0) >= 3000 * 384 + 3000 * 3 * 4
    assert L.b200moe_mlp_workspace_size(3, 384, 128, 0) >= 3 * 128 + 3 * 4
    assert L.b200moe_mlp_workspace_size(3000, 384, 128, 1) >= 3000 * (384 + 3 * 4) + 3000 * (128 + 4)
    for bad in ((-1, 1, 128), (1, 0, 128), (1, 1, 100)):
        assert L.b200moe_linear_workspace_size(*bad, 1, 0) == 0


def test_python_ops_refuse_cpu_tensors():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    w = torch.zeros(256, 256).to(FP8)
    s = torch.ones(2, 2)
    for call in (lambda: fp8_block_linear(x, w, s), lambda: fp8_gate_up(x, w, s), lambda: fp8_mlp(x, w, s, w, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


# The Python checks behind the device check, on CPU tensors.
def test_python_input_checks():
    bf, q, s = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 256).to(FP8), torch.ones(3, 2)
    assert dense._input(bf, None)[0] is bf and dense._input(q, s)[1] is s
    for bad in ((bf, s), (q, None), (q, s[:2]), (q, s[:, :1]), (bf[0], None)):
        with pytest.raises(ValueError):
            dense._input(*bad)
    for bad in ((bf.float(), None), (bf.half(), None), (q, s.double()), (bf[:, :200], None), (bf[:, :0], None)):
        with pytest.raises(NotImplementedError):
            dense._input(*bad)
    # layouts that the kernels cannot read are copied
    for odd in (bf.t().contiguous().t(), torch.zeros(3, 260, dtype=torch.bfloat16)[:, :256],
                torch.zeros(3 * 256 + 1, dtype=torch.bfloat16)[1:].view(3, 256), bf[:1].expand(3, 256)):
        got = dense._input(odd, None)[0]
        assert got is not odd and got.is_contiguous() and torch.equal(got, odd)
    strided = torch.zeros(3, 512, dtype=torch.bfloat16)[:, :256]
    assert dense._input(strided, None)[0] is strided


def test_python_weight_and_output_checks():
    w, s = torch.zeros(200, 256).to(FP8), torch.ones(2, 2)
    assert dense._weight(w, s, 256, "weight")[0] == 256
    for bad in ((w, s[:1]), (w[:, :128], s), (w[:0], s[:0]), (w.view(10, 20, 256), s)):
        with pytest.raises(ValueError):
            dense._weight(*bad, 256, "weight")
    with pytest.raises(ValueError):  # transposed storage
        dense._weight(torch.zeros(256, 256).to(FP8).t(), s, 256, "weight")
    for bad in ((w.float(), s), (w, s.double())):
        with pytest.raises(NotImplementedError):
            dense._weight(*bad, 256, "weight")
    out = torch.zeros(3, 5, dtype=torch.bfloat16)
    got = dense._output(out, out, 3, 5, torch.bfloat16, out.device)
    assert got[0] is out and got[1:] == (5, 5)
    for o, r in ((out[:2], None), (out.float(), None), (None, out[:, :4])):
        with pytest.raises(ValueError):
            dense._output(o, r, 3, 5, torch.bfloat16, out.device)
    with pytest.raises(NotImplementedError):
        dense._output(None, out.float(), 3, 5, torch.bfloat16, out.device)


class TwoDevices:
    """A stand-in for a process with two unlike GPUs, device 0 current and the
    tensors on device 1: what the library is asked, and on which device."""

    def __init__(self, monkeypatch):
        self.current, self.asked = 0, []
        outer = self

        class Guard:
            def __init__(self, index):
                self.index = index

            def __enter__(self):
                self.back, outer.current = outer.current, self.index

            def __exit__(self, *a):
                outer.current = self.back

        class Lib:
            b200moe_linear = b200moe_gate_up = b200moe_mlp = staticmethod(lambda packed: outer.note("call"))
            b200moe_linear_workspace_size = staticmethod(lambda *a: outer.note("size") or 256 * (outer.current + 1))
            b200moe_mlp_workspace_size = b200moe_linear_workspace_size

        monkeypatch.setattr(torch.cuda, "device", Guard)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
        monkeypatch.setattr(dense._lib, "lib", lambda: Lib)
        monkeypatch.setattr(dense, "_device_of", lambda *t: 1)
        monkeypatch.setattr(dense._workspaces, "header_ptr", lambda index, stream: P)
        dense._linear_bytes.cache_clear()
        dense._mlp_bytes.cache_clear()

    def note(self, what):
        self.asked.append((what, self.current))
        return 0


def test_everything_is_asked_on_the_tensors_device(monkeypatch):
    both = TwoDevices(monkeypatch)
    x = torch.zeros(3000, 256, dtype=torch.bfloat16)
    w, s = torch.zeros(512, 256).to(FP8), torch.ones(4, 2)
    w2, s2 = torch.zeros(256, 256).to(FP8), torch.ones(2, 2)
    fp8_block_linear(x, w, s)
    fp8_gate_up(x, w, s)
    fp8_mlp(x, w, s, w2, s2)
    assert both.asked == [("size", 1), ("call", 1)] * 3 and both.current == 0
    # and sizes kept for one device are not given to another
    both.current = 1
    assert dense._linear_bytes(1, 3000, 512, 256, 0) == 512
    dense._linear_bytes.cache_clear()
    dense._mlp_bytes.cache_clear()


@pytest.mark.parametrize("name", ["dense_common.cuh", "dense_split.cuh", "dense_tok.cuh", "dense_pair.cuh",
                                  "rowops.cuh"])
def test_inputs_are_not_read_through_the_read_only_path(name):
    """Kernels that start before the one ahead of them has ended (programmatic
    launch) may not read what it writes as memory nobody writes."""
    src = (Path(dense.__file__).parent / "csrc" / name).read_text()
    code = "\n".join(line.split("//")[0] for line in src.splitlines())
    assert "__ldg" not in code and "ld.global.nc" not in code and "__restrict__" not in code


@pytest.mark.parametrize("off", [1, 2])
def test_scales_and_words_must_be_aligned(off):
    """A float or word at an address that is no multiple of 4 would fault on the GPU."""
    assert linear(ws=P + off) == _lib.ERR_UNSUPPORTED
    assert linear(x=None, xq=P, xs=P + off) == _lib.ERR_UNSUPPORTED
    assert linear(err=P + off) == _lib.ERR_UNSUPPORTED

    def gate_up(x=P, xq=None, xs=None, ws=P, s=1 << 40, err=P):
        return call("b200moe_gate_up", x, xq, xs, 256, 2, 4, 256, 128, 1 << 30, 256, ws, 1 << 34, 128, s, 1, P,
                    1 << 20, err, None)

    def mlp(ws=P, w2s=P, err=P):
        return call("b200moe_mlp", P, None, None, 256, 0, 4, 256, 128, 1 << 28, ws, 1 << 30, w2s, None, 0, 1 << 34, 256,
                    P, 1 << 20, err, None)

    for got in (gate_up(ws=P + off), gate_up(x=None, xq=P, xs=P + off), gate_up(s=P + off), gate_up(err=P + off),
                mlp(ws=P + off), mlp(w2s=P + off), mlp(err=P + off)):
        assert got == _lib.ERR_UNSUPPORTED
