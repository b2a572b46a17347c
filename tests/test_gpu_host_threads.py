"""Calls from several host threads at once. A kernel's launch limits are the
process's, so they are set in a fresh process, whose first calls run side by
side with sizes that need different amounts of shared memory."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(600)]
ROOT = Path(__file__).resolve().parent.parent

DENSE = """
import threading
import torch
import trials_b200 as fw

dev = torch.device("cuda", 0)
torch.cuda.init()
calls = []
for M in (1, 20, 40, 64):          # 16, 32 and 64 tokens a tile, bf16 rows quantised in the product or ahead of it
    for K in (256, 512, 1024, 2048, 4096, 6144):
        x = torch.randn(M, K, device=dev).to(torch.bfloat16)
        calls.append((x, *fw.per_block_quant_fp8((torch.randn(512, K, device=dev) * K ** -0.5).to(torch.bfloat16))))
torch.cuda.synchronize()
threads = 12
gate = threading.Barrier(threads)
got, failed = [None] * threads, []


def work(k):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = calls[k:] + calls[:k]
            gate.wait()
            out = [fw.fp8_block_linear(*c) for c in mine]
            up = [fw.fp8_gate_up(*c) for c in mine]
            torch.cuda.current_stream().synchronize()
        n = len(calls)
        got[k] = [(out[(i - k) % n], *up[(i - k) % n]) for i in range(n)]
    except Exception as e:
        failed.append(e)


all_ = [threading.Thread(target=work, args=(k,)) for k in range(threads)]
for t in all_:
    t.start()
for t in all_:
    t.join()
assert not failed, failed
for i, c in enumerate(calls):      # and one after the other
    want = (fw.fp8_block_linear(*c), *fw.fp8_gate_up(*c))
    for k in range(threads):
        for a, b in zip(got[k][i], want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
print("fine")
"""


def run(script):
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", (r.stdout + r.stderr)[-3000:]


def test_first_products_of_several_threads(cuda_device):
    run(DENSE)


ROUTING = """
import threading
import torch
from trials_b200 import stages

dev = torch.device("cuda", 0)
calls = []
for E in (16, 64, 256, 512, 1024):
    for M in (4, 4096):            # one CTA, and several
        calls.append((torch.randn(M, E, device=dev), dict(num_expert_group=8, topk_group=4)))
        calls.append((calls[-1][0], {}))
torch.cuda.synchronize()


def call(x, groups):
    r, w, ids = stages.route_logits(x, 8, 32, "sigmoid", **groups)
    return r.sorted_ids, r.slot_pos, w, ids, stages.route(ids, x.shape[1], 32).slot_pos


threads = 10
gate = threading.Barrier(threads)
got, failed = [None] * threads, []


def work(k):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = list(range(len(calls)))
            mine = mine[2 * k:] + mine[:2 * k]
            gate.wait()
            for _ in range(20):
                out = {i: call(*calls[i]) for i in mine}
            torch.cuda.current_stream().synchronize()
        got[k] = out
    except Exception as e:
        failed.append(e)


all_ = [threading.Thread(target=work, args=(k,)) for k in range(threads)]
for t in all_:
    t.start()
for t in all_:
    t.join()
assert not failed, failed
for i, c in enumerate(calls):
    want = call(*c)
    for k in range(threads):
        for a, b in zip(got[k][i], want):
            assert torch.equal(a, b)
print("fine")
"""


def test_routing_of_several_threads(cuda_device):
    run(ROUTING)
