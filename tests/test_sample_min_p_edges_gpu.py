"""Sampling with min-p, and the kernels of drafted trees, at the edges."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

EDGES = """
import ctypes
import torch
from easy_gpt.cpp_b200 import kernels
import test_tree_step_gpu as T

steps = [(T.Step(1, [8], [300], 14, 2, 64, 16), (16, 4, 1)), (T.Step(1, [8], [300], 14, 2, 64, 16), (128, 4, 1)), (T.Step(1, [8], [300], 4, 2, 64, 16, torch.float32), (0, 4, 1))]
n = lambda v, dtype=torch.float32: torch.full((2,), v, dtype=dtype, device="cuda")
args = (torch.randn((2, 5000), device="cuda"), n(0.8), n(20, torch.int32), n(0.9), n(0.1), n(0.5), n(0, torch.int32))
calls = [lambda: kernels.sample_min_p(*args)] + [lambda s=s, plan=plan: T.run_plan(s, plan) for s, plan in steps]
for call in calls:
    call()
torch.cuda.synchronize()
kinds = []
for call in calls:
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
        call()
    count = ctypes.c_size_t(4)
    nodes, others, data = (ctypes.c_void_p * 4)(), (ctypes.c_void_p * 4)(), (ctypes.c_ubyte * 32)()      # an edge's data: port, port, type, and zeros up to 8 bytes
    code = ctypes.CDLL("libcuda.so.1").cuGraphGetEdges_v2(ctypes.c_void_p(graph.raw_cuda_graph()), nodes, others, data, ctypes.byref(count))
    assert code == 0 and count.value == 1, (code, count)
    kinds.append(data[2])
print("edges", *kinds)
"""


@pytest.mark.gpu
@pytest.mark.parametrize("setting, kind", [(None, 1), ("2", 1), ("0", 0)])
def test_launches_are_programmatic_dependents_unless_told_otherwise(setting, kind):
    """EASY_GPT_PDL=0: no kernel starts before the one in front of it is done.  (The edge between two calls in a captured graph says it.)"""
    environment = {**os.environ, "PYTHONPATH": os.pathsep.join([str(ROOT), str(ROOT / "tests"), os.environ.get("PYTHONPATH", "")])}
    environment.pop("EASY_GPT_PDL", None)
    if setting is not None:
        environment["EASY_GPT_PDL"] = setting
    done = subprocess.run([sys.executable, "-c", EDGES], capture_output=True, text=True, env=environment, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
    assert done.stdout.split() == ["edges", *[str(kind)] * 4]
