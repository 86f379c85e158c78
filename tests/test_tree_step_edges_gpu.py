"""Attention over drafted trees where its kernels could differ from one another or from the formula."""
import math

import pytest
import torch

from test_tree_step_gpu import Step, run_plan, tolerance

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
