"""The first calls of attention in a process: from several host threads at once, each on a stream of its own, and while
a graph is captured. Each test runs a process of its own, so that nothing that a launch remembers is there yet."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent

CODE = """
import sys, threading
sys.path[:0] = [{repo!r}, {tests!r}]
import torch
from paged_oracle import Problem
from ako_b200 import paged_attention_cuda_sm100

dev = torch.device("cuda", 0)
todo = []
for i in range(8):
    new = 90 if i % 2 else 1
    p = Problem(torch.float16 if i & 2 else torch.bfloat16, bool(i & 4), 8, 2, 128, 16, [(new, 300), (new, 130)], True, i, dev)
    todo.append((p.q.to(dev), p.kv(), p.batch()))
torch.cuda.synchronize()
got, start = [None] * 8, threading.Barrier(8)

def work(i):
    stream = torch.cuda.Stream(dev)
    start.wait()
    with torch.cuda.stream(stream):
        got[i] = [paged_attention_cuda_sm100(*todo[i]) for _ in range(20)]
    stream.synchronize()

threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
for t in threads:
    t.start()
for t in threads:
    t.join()
for i in range(8):
    want = paged_attention_cuda_sm100(*todo[i])
    assert bool(torch.isfinite(want).all())
    assert all(torch.equal(x, want) for x in got[i]), i
print("equal")
"""


CAPTURED = """
import sys
sys.path[:0] = [{repo!r}, {tests!r}]
import torch
from paged_oracle import Problem, check_attention
from ako_b200 import paged_attention_cuda_sm100

dev = torch.device("cuda", 0)
for new in (90, 1):
    for quantised in (False, True):
        p = Problem(torch.bfloat16, quantised, 8, 2, 128, 16, [(new, 300), (new, 100)], False, 1, dev)
        q, cache, batch = p.q.to(dev), p.kv(), p.batch()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention_cuda_sm100(q, cache, batch)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(p, out)
print("equal")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("code", [CODE, CAPTURED], ids=["threads", "captured"])
def test_first_calls_of_a_process(cuda_device, code) -> None:
    got = subprocess.run([sys.executable, "-c", code.format(repo=str(REPO), tests=str(REPO / "tests"))],
                         capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "equal" in got.stdout, got.stderr[-3000:]
