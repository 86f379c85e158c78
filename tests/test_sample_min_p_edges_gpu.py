"""Sampling with min-p, and the kernels of drafted trees, at the edges."""
import math
import os
import subprocess
import sys
from decimal import Decimal, getcontext
from pathlib import Path

import numpy as np
import pytest
import torch

from test_tree_step_gpu import run_sample

ROOT = Path(__file__).resolve().parent.parent

# (logit, ones, others): exp(logit) lies above ones / others by 1.14 to 1.47 times 2^-43
BORDERS = [("-0x1.bee89ep-4", 492187, 548928), ("-0x1.5e909cp-6", 112589, 115024), ("-0x1.1fdca4p-2", 254872, 337605), ("-0x1.e9a53cp-3", 373766, 474715), ("-0x1.4bf1a6p-2", 345056, 477169),
           ("-0x1.910474p-3", 401512, 488357), ("-0x1.0c29a2p-4", 297768, 317915)]


@pytest.mark.gpu
@pytest.mark.parametrize("logit, ones, others", BORDERS)
def test_weights_are_off_by_hardly_more_than_half_a_unit(logit, ones, others):
    """`ones` tokens of weight 1, which is exact, then `others` of weight w = exp(logit), drawn with 1/2: the last of the ones if ones >= others * w, else the
    first of the others.  Whole numbers of 2^-42 round w by at most 2^-43, and the exponential is off by at most 2^-46 w (a series to z^5, with the sixth
    power spread over the second and fourth; 64-bit roundings beside it): 1.125 times 2^-43, less than what is between w and the border."""
    getcontext().prec = 50
    x = float.fromhex(logit)
    assert float(np.float32(x)) == x and ones + others <= 1 << 20
    above = (Decimal(x).exp() - Decimal(ones) / Decimal(others)) * 2 ** 43
    assert Decimal("1.14") < above < Decimal("1.5")
    row = torch.cat([torch.zeros(ones), torch.full((others,), x)])[None].cuda()
    assert run_sample(row, np.float32(1), 0, np.float32(1), np.float32(0), np.float32(0.5)).tolist() == [ones]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab, k, p, low", [(300, 20, 1.0, 0.0), (9000, 20, 0.9, 0.0), (9000, 400, 1.0, 0.0), (9000, 0, 1.0, 0.0), (151936, 0, 1.0, 0.0), (151936, 0, 0.5, 0.0), (151936, 0, 1.0, 0.1)])
def test_numbers_outside_of_zero_to_one(vocab, k, p, low):
    """What is below 0 or none draws the first token that is kept, 1 and more the last one."""
    x = np.random.default_rng(vocab + k).normal(0, 1, vocab).astype(np.float32)
    w = np.exp((x.astype(np.float64) - x.max()))
    order = np.argsort(-x, kind="stable")[:k if k else vocab]
    run = np.cumsum(w[order])
    kept = order[:1 + int((run[:-1] < float(np.float32(p)) * run[-1]).sum())] if p < 1 else order
    kept = kept[w[kept] >= low]
    numbers = [-math.inf, -1.0, 0.0, math.nan, 1.0, 2.0, 1e6, 1e7, 1e30, math.inf]
    logits = torch.from_numpy(np.broadcast_to(x, (len(numbers), vocab)).copy()).cuda()
    got = run_sample(logits, np.float32(1), k, np.float32(p), np.float32(low), np.array(numbers, np.float32)).tolist()
    assert got == [int(kept.min())] * 4 + [int(kept.max())] * 6


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
