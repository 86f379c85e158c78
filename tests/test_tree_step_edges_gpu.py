"""Attention over drafted trees where its kernels could differ from one another or from the formula."""
import math

import numpy as np
import pytest
import torch

from test_tree_step_gpu import Step, line_of, run_plan, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("parts", [1, 2, 4])
@pytest.mark.parametrize("row_tile", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)])
def test_the_likeliest_value_may_be_infinite(heads, row_tile, parts, bad):
    """An infinite value at the key that has all of every row's weight, in a tile behind the first: 1 * inf, whatever the scores in front of it were.  That
    key's score is 4096 dim^-1/2 (8 and 512 in the first column, zeros in the others), 360 and more above the others, whose weights are 0 in 32 bits."""
    step = Step([*heads, row_tile, parts], [18, 40], [200, 70], *heads, 16, kind="star")
    step.q.view(-1, heads[0], heads[2])[:, :, 0] = 8
    for r, c in enumerate(step.contexts):                             # node 0 is everybody's ancestor
        page, at = int(step.table[r, c // 16]), c % 16
        step.cache[page, 0, :, at] = 0
        step.cache[page, 0, :, at, 0] = 512
        step.cache[page, 1, :, at, :8] = bad
    got, want = run_plan(step, (row_tile, parts, 1)).view(-1, heads[0], heads[2]), step.plain().view(-1, heads[0], heads[2])
    assert int(step.status) == 0
    assert bool((got[:58, :, :8] == bad).all())
    got, want = got[:58, :, 8:].double().flatten(1), want[:58, :, 8:].flatten(1)
    assert float(((got - want).norm(dim=1) / want.norm(dim=1)).max()) <= tolerance(torch.bfloat16, heads[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(14, 2, 64), (4, 2, 32), (3, 1, 80)])
def test_keys_beyond_the_block_table_are_not_seen(heads, dtype):
    """A table of 48 places: an entry of 46 keys has all of them, one of 60 (its nodes behind the 50th among them) those that there are places for."""
    step = Step(4, [6, 10], [40, 50], *heads, 16, dtype)
    step.block_table = step.block_table[:, :3].contiguous()
    got, at, group = step.run().double(), 0, heads[0] // heads[1]
    assert int(step.status) == 2
    for r, (n, c) in enumerate(zip(step.nodes, step.contexts)):
        k, v = step.rows_of(r, 0), step.rows_of(r, 1)
        for i in range(n):
            seen = [x for x in [*range(c), *(c + a for a in line_of(step.parents[r], i))] if x < 48]
            q = step.q[at + i].double().view(heads[1], group, heads[2])
            w = (torch.einsum("ghd,gkd->ghk", q, k[:, seen]) * heads[2] ** -0.5).softmax(-1)
            want = torch.einsum("ghk,gkd->ghd", w, v[:, seen]).reshape(-1)
            assert float((got[at + i] - want).norm() / want.norm()) <= tolerance(dtype, heads[2]), (r, i)
        at += n


@pytest.mark.parametrize("dim", [64, 128])
def test_products_right_behind_it(dim):
    """The attention on tcgen05 and products that allocate tensor memory in front of their wait for it, in turn on one stream: the rows and sums that each
    gives alone, bit for bit."""
    from test_gemm_batch_gpu import RESID, library

    lib, rng, stream = library(), np.random.default_rng(dim), torch.cuda.current_stream().cuda_stream
    M, N, K = 64, 896, 896
    f32 = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    W, x, resid, gain = f32(N, K).bfloat16(), f32(M, K).bfloat16(), f32(M, N) * 30, f32(N)
    parts = lib.eg_gemm_batch_takes(RESID, N, K, 0)
    step = Step(dim, [24] * 16, [2000] * 16, 14, 2, dim, 64)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def product(r, xn, ss, mode):
        assert lib.eg_gemm_batch(stream, RESID, mode, W.data_ptr(), K, None, M, N, K, x.data_ptr(), K, 1e-6, None, 0, None, 0, 0, 0, 0, None, None, None, None, 1, 0, 0, 0, r.data_ptr(),
                                 gain.data_ptr(), xn.data_ptr(), ss.data_ptr(), None, 0, status.data_ptr()) == 0

    new = lambda: (resid.clone(), torch.empty(M, N, device="cuda", dtype=torch.bfloat16), torch.empty(M, parts, device="cuda"))  # noqa: E731
    alone, rows = new(), run_plan(step, (128, 4, 1)).clone()
    torch.cuda.synchronize()
    for _ in range(12):
        product(*alone, 0)
        torch.cuda.synchronize()
    for mode in (1, 2):
        together = new()
        step.out.fill_(7.0)
        for _ in range(12):
            run_plan(step, (128, 4, 1))
            product(*together, mode)
        torch.cuda.synchronize()
        assert int(status) == 0 and int(step.status) == 0 and torch.equal(step.out, rows)
        assert all(torch.equal(a, b) for a, b in zip(alone, together))


@pytest.mark.parametrize("row_tile", [0, 16, 128])
def test_the_most_nodes_of_an_entry(row_tile):
    """16,384 nodes: right, in the first rows and the last.  One more: a status, and that entry's rows are left; the other's are as ever."""
    step = Step(77, [16384, 5], [20, 40], 1, 1, 64, 64)
    got = run_plan(step, (row_tile, 1, 1)).double()
    assert int(step.status) == 0
    k, v = step.rows_of(0, 0)[0], step.rows_of(0, 1)[0]
    for i in (0, 1, 63, 64, 1000, 8191, 16320, 16383):
        seen = [*range(20), *(20 + a for a in line_of(step.parents[0], i))]
        want = ((k[seen] @ step.q[i].double()) * 0.125).softmax(0) @ v[seen]
        assert float((got[i] - want).norm() / want.norm()) <= tolerance(torch.bfloat16, 64), i
    other = got[16384:16389].clone()
    step.starts[1] += 1                                               # 16,385 and 4
    step.out.fill_(7.0)
    got = run_plan(step, (row_tile, 1, 1)).double()
    assert int(step.status) == 16 and bool((got[:16385] == 7).all()) and not bool((got[16385:16389] == 7).all(dim=1).any())
    step.starts[1] -= 1
    assert torch.equal(run_plan(step, (row_tile, 1, 1))[16384:16389].double(), other)
