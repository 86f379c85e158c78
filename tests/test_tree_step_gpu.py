"""A step over trees of drafted tokens, its operators against plain loops in 64 bits: attention over a tree and the paged cache, sampling with
min-p, the walk to the accepted nodes, the move of their keys and values; and a run of them together."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def random_parents(rng, n, kind="random"):
    return [-1] + [i - 1 if kind == "chain" else 0 if kind == "star" else int(rng.integers(0, i)) for i in range(1, n)] if n else []


def line_of(parents, i):
    """Node i and its ancestors, itself first."""
    line = []
    while i >= 0:
        line.append(i)
        i = parents[i]
    return line


class Step:
    """Entries with trees over a paged cache, on the GPU and as lists."""

    def __init__(self, seed, nodes, contexts, heads, kv_heads, dim, page, dtype=torch.bfloat16, kind="random", pad=2, extra_pages=0):
        rng = np.random.default_rng(seed)
        self.nodes, self.contexts, self.heads, self.kv_heads, self.dim, self.page, self.dtype = nodes, contexts, heads, kv_heads, dim, page, dtype
        self.parents = [random_parents(rng, n, kind) for n in nodes]
        starts = np.cumsum([0, *nodes])
        total = int(starts[-1]) + pad
        need = [-(-(c + n) // page) for c, n in zip(contexts, nodes)]
        width = max(1, *need) + extra_pages
        order = rng.permutation(sum(need) + 1)
        self.table = np.full((len(nodes), width), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        g = torch.Generator("cuda").manual_seed(int(rng.integers(1 << 31)))
        new = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float32).to(dtype)  # noqa: E731
        self.qkv = new(total, (heads + 2 * kv_heads) * dim)
        self.q = self.qkv[:, :heads * dim]
        self.cache = new(sum(need) + 1, 2, kv_heads, page, dim)
        self.k, self.v = self.cache[:, 0], self.cache[:, 1]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.starts, self.context = i32(starts.tolist()), i32(contexts)
        self.flat = i32([p for tree in self.parents for p in tree] + [0] * pad)
        self.block_table = torch.from_numpy(self.table).cuda()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.out = torch.full((total, heads * dim), 7.0, device="cuda", dtype=dtype)

    def rows_of(self, r, which):
        """Entry r's keys (which 0) or values (1) in the order of their cache positions: float64 [kv_heads, tokens, dim]."""
        count = self.contexts[r] + self.nodes[r]
        pages = torch.from_numpy(self.table[r, :-(-count // self.page)]).long().clamp(min=0).cuda()
        return self.cache[pages, which].transpose(0, 1).reshape(self.kv_heads, -1, self.dim)[:, :count].double()

    def run(self, window=None, scale=None, **options):
        from easy_gpt.cpp_b200 import kernels

        kernels.attention_tree(self.q, self.k, self.v, self.block_table, self.starts, self.context, self.flat, self.out, self.heads, self.kv_heads, self.dim, window,
                               scale if scale is not None else self.dim ** -0.5, self.status, **options)
        return self.out

    def plain(self, window=None, scale=None):
        """Rows of the step in float64, from each node's visible keys alone."""
        scale = self.dim ** -0.5 if scale is None else scale
        want, at, group = torch.full(self.out.shape, 7.0, dtype=torch.float64, device="cuda"), 0, self.heads // self.kv_heads
        for r, (n, c) in enumerate(zip(self.nodes, self.contexts)):
            k, v = self.rows_of(r, 0), self.rows_of(r, 1)
            for i in range(n):
                line = line_of(self.parents[r], i)
                first = max(0, c + len(line) - 1 - window + 1) if window else 0
                seen = torch.tensor([*range(min(first, c), c), *(c + a for a in line[:window])], device="cuda")
                q = self.q[at + i].double().view(self.kv_heads, group, self.dim)
                w = (torch.einsum("ghd,gkd->ghk", q, k[:, seen]) * scale).softmax(-1)
                want[at + i] = torch.einsum("ghk,gkd->ghd", w, v[:, seen]).reshape(-1)
            at += n
        return want


def tolerance(dtype, dim):
    """Relative to a row's norm.  bfloat16: weights and the result are rounded, by at most 2^-8 each.  float32: a score is a sum of dim products,
    off by at most (dim + 2) 2^-24 of the sum of their sizes, which for normal numbers and a scale of dim^-1/2 is 0.64 dim^1/2; a weight is off by that
    and its sums by no more, the result by the two together; the exponent and the sums of the output add less than 64 roundings."""
    return 2.0 ** -7 + 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -24 * (2 * (dim + 2) * 0.64 * dim ** 0.5 + 64)


def check(step, window=None, scale=None, **options):
    got, want = step.run(window, scale, **options).double(), step.plain(window, scale)
    assert int(step.status) == 0
    total = sum(step.nodes)
    assert torch.equal(got[total:], want[total:])                     # rows behind the last entry's
    if total:
        off = (got[:total] - want[:total]).norm(dim=1) / want[:total].norm(dim=1)
        assert float(off.max()) <= tolerance(step.dtype, step.dim), (float(off.max()), int(off.argmax()))


HEADS = [(14, 2, 64), (4, 4, 40), (6, 2, 136), (12, 2, 128), (8, 8, 64), (6, 1, 32), (4, 2, 256), (3, 3, 80), (16, 1, 128), (2, 1, 18)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 64, 5])
def test_attention_tree(heads, page, dtype):
    """Contexts around the edges of key tiles and pages, none among them; trees of one node to a hundred, an entry without rows between others."""
    nodes = [1, 7, 0, 33, 16, 2, 100, 12, 64]
    contexts = [0, 1, 5, 63, 64, 65, 31, 200, 447]
    check(Step([*heads, page], nodes, contexts, *heads, page, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
@pytest.mark.parametrize("window", [1, 3, 40, 64, 1000])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (4, 4, 32)])
def test_attention_tree_window(heads, window, kind, dtype):
    """A window is over positions: a node's depth counts, not its row."""
    step = Step([*heads, window], [9, 70, 1, 24], [0, 130, 64, 517], *heads, 16, dtype, kind)
    for r, c in enumerate(step.contexts):                             # pages that no coming token can see have been given back
        step.table[r, :max(0, c - window + 1) // 16] = -1
    step.block_table = torch.from_numpy(step.table).cuda()
    check(step, window)


def run_plan(step, plan, window=None):
    """The call with a plan given: (rows of a CTA, parts, key tiles of a part)."""
    from easy_gpt.cpp_b200 import kernels

    k = step.k
    args = kernels._pack_attention_tree(step.q.data_ptr(), k.data_ptr(), step.v.data_ptr(), step.block_table.data_ptr(), step.starts.data_ptr(), step.context.data_ptr(), step.flat.data_ptr(),
                                        step.out.data_ptr(), step.status.data_ptr(), kernels.dtype_code(step.dtype), step.q.stride(0), step.out.stride(0), k.stride(0), k.stride(1),
                                        step.block_table.stride(0), step.block_table.shape[1], k.shape[0], step.flat.numel(), len(step.nodes), step.heads, step.kv_heads, step.dim, step.page,
                                        window or 0, 0, *plan, step.dim ** -0.5)
    assert kernels.library().eg_attention_tree(torch.cuda.current_stream().cuda_stream, args) == 0
    return step.out


@pytest.mark.parametrize("parts, part_tiles", [(1, 1), (2, 3), (8, 1), (16, 1)])
@pytest.mark.parametrize("row_tile", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("heads, window", [((14, 2, 64), None), ((14, 2, 64), 50), ((28, 4, 128), None), ((16, 1, 128), 200), ((3, 3, 64), 70), ((4, 2, 32), None), ((8, 1, 256), 33), ((6, 2, 80), None), ((4, 1, 200), 90), ((5, 5, 8), None)])
def test_attention_tree_every_kernel(heads, window, row_tile, parts, part_tiles):
    """Every kernel and cut by name, whatever the rule would choose: entries of less than a tile of rows, of one and of several; parts without keys."""
    if row_tile == 128 and heads[2] not in (64, 128) or parts == 16 and heads[2] == 256:
        pytest.skip("sizes that kernel does not take")
    step = Step([*heads, row_tile], [1, 18, 19, 0, 36, 37, 100], [0, 1000, 63, 7, 640, 1, 333], *heads, 32)
    got, want = run_plan(step, (row_tile, parts, part_tiles), window).double(), step.plain(window)
    total = sum(step.nodes)
    assert int(step.status) == 0 and torch.equal(got[total:], want[total:])
    assert float(((got[:total] - want[:total]).norm(dim=1) / want[:total].norm(dim=1)).max()) <= tolerance(step.dtype, step.dim)


@pytest.mark.parametrize("parts, part_tiles", [(1, 1), (2, 3), (4, 1), (8, 1), (16, 1)])
@pytest.mark.parametrize("heads, window", [((14, 2, 64), None), ((14, 2, 64), 50), ((12, 2, 128), None), ((16, 1, 128), 200), ((5, 5, 32), 90), ((6, 2, 30), None), ((8, 1, 256), 33), ((4, 2, 200), None)])
def test_attention_tree_float32_cuts(heads, window, parts, part_tiles):
    """The 32-bit kernel on float32: CTAs of 32 rows and of 64, whole 16-byte pieces (all but heads of 30) and not, every number of parts."""
    if parts == 16 and heads[2] > 128:
        pytest.skip("no room for clusters of 16")
    step = Step([*heads, parts], [1, 4, 5, 0, 18, 37, 70], [0, 1000, 31, 7, 640, 1, 333], *heads, 32, torch.float32)
    got, want = run_plan(step, (0, parts, part_tiles), window).double(), step.plain(window)
    total = sum(step.nodes)
    assert int(step.status) == 0 and torch.equal(got[total:], want[total:])
    assert float(((got[:total] - want[:total]).norm(dim=1) / want[:total].norm(dim=1)).max()) <= tolerance(step.dtype, step.dim)


@pytest.mark.parametrize("parts", [1, 4])
@pytest.mark.parametrize("row_tile", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128)])
def test_attention_tree_every_kernel_does_not_see_pages_that_are_none(heads, row_tile, parts):
    """Pages in the middle of a context, the tree's own and the table's end: their keys are left out, which is what the same cache without them gives."""
    step = Step([*heads, row_tile], [9, 12, 30], [700, 300, 500], *heads, 16)
    step.block_table[0, 20], step.block_table[0, 3], step.block_table[1, 18] = -1, step.cache.shape[0] + 5, -9
    step.block_table = step.block_table[:, :32].contiguous()          # entry 0 has 44 pages, entry 2 reaches into page 33
    got, at, group = run_plan(step, (row_tile, parts, 1)).double(), 0, heads[0] // heads[1]
    assert int(step.status) == 2
    for r, (n, c) in enumerate(zip(step.nodes, step.contexts)):
        gone = {0: {3, 20}, 1: {18}, 2: set()}[r]
        k, v = step.rows_of(r, 0), step.rows_of(r, 1)
        for i in range(n):
            seen = [x for x in [*range(c), *(c + a for a in line_of(step.parents[r], i))] if x // 16 not in gone and x // 16 < 32]
            q = step.q[at + i].double().view(heads[1], group, heads[2])
            w = (torch.einsum("ghd,gkd->ghk", q, k[:, seen]) * heads[2] ** -0.5).softmax(-1)
            want = torch.einsum("ghk,gkd->ghd", w, v[:, seen]).reshape(-1)
            assert float((got[at + i] - want).norm() / want.norm()) <= tolerance(step.dtype, step.dim), (r, i)
        at += n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_many_entries(dtype):
    """More entries than a warp looks at at once, some without rows, one of them with rows that cannot be in the middle."""
    rng = np.random.default_rng(3)
    nodes, contexts = [int(n) for n in rng.integers(0, 4, 150)], [int(c) for c in rng.integers(0, 40, 150)]
    step = Step(7, nodes, contexts, 4, 2, 64, 16, dtype)
    check(step)
    step.context[75] = -1
    want, got = step.plain(), step.run().double()
    first = sum(nodes[:75])
    keep = torch.ones(got.shape[0], dtype=torch.bool, device="cuda")
    keep[first:first + nodes[75]] = False
    assert int(step.status) == 16
    off = (got - want)[keep].norm(dim=1) / want[keep].norm(dim=1)
    assert float(off.max()) <= tolerance(dtype, 64)


def test_attention_tree_no_rows():
    step = Step(8, [0, 0], [5, 0], 4, 2, 64, 16, pad=3)
    before = step.out.clone()
    assert torch.equal(step.run(), before) and int(step.status) == 0
    step.flat = step.flat[:0]
    assert torch.equal(step.run(), before) and int(step.status) == 0


@pytest.mark.parametrize("row_tile", [0, 16, 64, 128])
def test_attention_tree_every_kernel_hides_what_is_not_a_number(row_tile):
    step = Step(6, [40, 20], [100, 700], 14, 2, 64, 16, kind="chain")
    step.cache[step.table[0, 3], :, :, 8] = math.nan                  # entry 0's key 56: seen with a window of 50 by nodes up to depth 5
    step.cache[step.table[1, 44], :, :, 15] = math.inf                # entry 1's node 19, the chain's last
    got, want = run_plan(step, (row_tile, 4, 1), 50).double(), step.plain(50)
    for i in range(60):
        hidden = i > 5 if i < 40 else i != 59
        assert bool(torch.isfinite(got[i]).all()) == hidden, i
        if hidden:
            assert float((got[i] - want[i]).norm() / want[i].norm()) <= tolerance(torch.bfloat16, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (8, 1, 256)])
@pytest.mark.parametrize("nodes", [1, 5, 64, 300])
def test_attention_tree_long(heads, nodes, dtype):
    """One entry with a long context beside a short one: keys in parts that are added up."""
    check(Step([*heads, nodes], [nodes, 3], [5000, 17], *heads, 64, dtype, extra_pages=3), max_context=5000 + nodes)


@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (4, 2, 32), (6, 2, 80)])
@pytest.mark.parametrize("n", [1024, 1100])
def test_attention_tree_wide(heads, n):
    check(Step([n, *heads], [n, 2], [70, 3], *heads, 32), max_context=n + 70)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 2, 128), (4, 2, 32), (4, 2, 256), (3, 1, 48)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_tree_hidden_places_may_hold_anything(heads, bad, dtype):
    """Keys and values of nodes that are nobody's ancestors, of the cache behind the last node and of the pool's other pages are not numbers."""
    step = Step([*heads, 3], [20, 40], [50, 100], *heads, 16, dtype)
    leaves = [[i for i in range(n) if i not in tree] for n, tree in zip(step.nodes, step.parents)]
    for r, (n, c) in enumerate(zip(step.nodes, step.contexts)):
        bad_leaves = leaves[r][::2]
        for i in bad_leaves:
            at = c + i
            step.cache[step.table[r, at // 16], :, :, at % 16] = bad
        end = c + n
        if end % 16:
            step.cache[step.table[r, end // 16], :, :, end % 16:] = bad
        leaves[r] = set(bad_leaves)
    used = set(step.table[step.table >= 0].tolist())
    for page in set(range(step.cache.shape[0])) - used:
        step.cache[page] = bad
    got, want, at = step.run().double(), step.plain(), 0
    for r, n in enumerate(step.nodes):
        for i in range(n):
            if i not in leaves[r]:
                assert float((got[at + i] - want[at + i]).norm() / want[at + i].norm()) <= tolerance(dtype, step.dim), (r, i)
            else:
                assert not bool(torch.isfinite(got[at + i]).all())
        at += n
    assert int(step.status) == 0


@pytest.mark.parametrize("parts", [1, 4])
@pytest.mark.parametrize("row_tile", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (64, 1, 64)])
def test_attention_tree_every_row_meets_what_is_not_a_number(heads, row_tile, parts):
    """Values that are not finite, in a tile that reaches into the tree: every row that sees them has them, whichever warps of a CTA the rows are in."""
    step = Step([*heads, row_tile], [40, 18], [70, 200], *heads, 16, kind="star")
    step.cache[step.table[0, 70 // 16], 1, :, 70 % 16, :8] = math.inf                 # node 0 of entry 0, every node's ancestor
    step.cache[step.table[1, 199 // 16], 1, :, 199 % 16, 3] = -math.inf               # entry 1's last cached key
    for _ in range(20):
        got = run_plan(step, (row_tile, parts, 1)).view(-1, heads[0], heads[2])
        assert int(step.status) == 0
        assert bool((got[:40, :, :8] == math.inf).all()) and bool(torch.isfinite(got[:40, :, 8:]).all())
        assert bool((got[40:58, :, 3] == -math.inf).all()) and bool(torch.isfinite(got[40:58, :, 4:]).all())


def test_attention_tree_window_hides_what_is_not_a_number():
    """Values that some rows' windows have left and others' have not."""
    step = Step(5, [40], [100], 14, 2, 64, 16, kind="chain")
    step.cache[step.table[0, 3], :, :, 8] = math.nan                  # key 56: seen with a window of 50 by nodes up to depth 5
    got, want = step.run(50).double(), step.plain(50)
    seen = [100 + i - 50 < 56 for i in range(40)]
    for i in range(40):
        assert bool(torch.isfinite(got[i]).all()) != seen[i]
        if not seen[i]:
            assert float((got[i] - want[i]).norm() / want[i].norm()) <= tolerance(torch.bfloat16, 64)


@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (4, 2, 32)])
def test_attention_tree_large_scores(heads):
    """Scores of some thousands: one key has all the weight, and the reference has to follow it."""
    step = Step([*heads, 9], [12, 33], [300, 65], *heads, 16)
    step.qkv *= 16
    step.cache[:, 0] *= 16
    check(step)


def test_attention_tree_strides():
    """q out of wider rows, out into wider ones, caches as slices of a pool of several layers, a block table out of a wider one."""
    step = Step(11, [10, 20], [70, 130], 14, 2, 64, 16)
    pool = torch.randn((3, *step.cache.shape), device="cuda").bfloat16()
    pool[1] = step.cache
    step.cache = pool[1]
    step.k, step.v = pool[1][:, 0], pool[1][:, 1]
    wide = torch.full((step.out.shape[0], step.out.shape[1] + 24), 7.0, device="cuda", dtype=torch.bfloat16)
    step.out = wide[:, 8:8 + step.heads * step.dim]
    table = torch.full((2, step.block_table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    table[:, 4:4 + step.block_table.shape[1]] = step.block_table
    step.block_table = table[:, 4:4 + step.block_table.shape[1]]
    check(step)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + step.heads * step.dim:] == 7).all())


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_attention_tree_unaligned(offset):
    """Rows of q and out and the caches that start at no multiple of 16 bytes."""
    step = Step(12, [10, 20], [70, 130], 6, 2, 64, 16)
    shift = lambda t: torch.empty(t.numel() + offset, device="cuda", dtype=t.dtype)[offset:].view(t.shape).copy_(t)  # noqa: E731
    step.q, step.out, step.cache = shift(step.q.contiguous()), shift(step.out), shift(step.cache)
    step.k, step.v = step.cache[:, 0], step.cache[:, 1]
    check(step)


@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 2, 128), (3, 1, 80)])
def test_attention_tree_bad_metadata_is_a_status(heads):
    """A parent that cannot be, a page that is none, rows that cannot be: a status bit each, and the other entries as ever."""
    step = Step([*heads, 2], [6, 10, 5], [40, 50, 60], *heads, 16)
    good = step.run().clone()
    step.flat[8] = 9                                                  # entry 1's node 2: a parent behind it
    step.parents[1][2] = -1
    want = step.plain()
    got = step.run().double()
    assert int(step.status) == 16
    assert float(((got[:21] - want[:21]).norm(dim=1) / want[:21].norm(dim=1)).max()) <= tolerance(torch.bfloat16, step.dim)
    step.status.zero_()
    step.flat[8] = step.flat[7]
    step.block_table[2, 1] = step.cache.shape[0]                      # a page beyond the pool
    got = step.run().clone()
    assert int(step.status) == 2 and torch.equal(got[:6], good[:6])
    step.status.zero_()
    step.block_table[2, 1] = -1
    again = step.run().clone()
    assert int(step.status) == 2 and torch.equal(got, again) and bool(torch.isfinite(again).all())
    step.status.zero_()
    step.block_table.copy_(torch.from_numpy(step.table))
    step.starts[3] = 1000                                             # entry 2's rows end behind the step's
    step.out.fill_(7.0)
    got = step.run()
    assert int(step.status) == 16 and torch.equal(got[:6], good[:6]) and bool((got[16:] == 7).all())
    step.status.zero_()
    step.starts[3] = 21
    step.context[0] = -5
    step.out.fill_(7.0)
    got = step.run()
    assert int(step.status) == 16 and bool((got[:6] == 7).all()) and torch.equal(got[16:21], good[16:21])


def test_attention_tree_keys_beyond_the_block_table():
    step = Step(4, [6, 10], [40, 50], 14, 2, 64, 16)
    step.block_table = step.block_table[:, :3].contiguous()           # 48 keys of 46 and 60
    got = step.run()
    assert int(step.status) == 2 and bool(torch.isfinite(got).all())
    off = (got[:6].double() - step.plain()[:6]).norm(dim=1)
    assert float(off.max()) < 1


@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("parts", [1, 4])
@pytest.mark.parametrize("row_tile", [0, 16, 32, 64, 128])
def test_attention_tree_contexts_far_beyond_the_block_table(row_tile, parts, window):
    """What no table has room for takes no time: the keys that there are places for are seen, behind a window none, the other entry as ever."""
    step = Step([row_tile, parts], [6, 10], [40, 50], 14, 2, 64, 16)
    table_keys = step.block_table.shape[1] * 16
    want = step.plain(window)
    for context in (1 << 20, (1 << 31) - 1 - 4096 - 6):
        step.context[0] = context
        step.status.zero_()
        step.out.fill_(7.0)
        got = run_plan(step, (row_tile, parts, 1), window).double()
        assert int(step.status) == 2
        assert float(((got[6:16] - want[6:16]).norm(dim=1) / want[6:16].norm(dim=1)).max()) <= tolerance(step.dtype, 64)
        if window:
            assert not bool(got[:6].any())
        else:
            step.contexts[0], nodes, step.nodes[0] = int((step.table[0] >= 0).sum()) * 16, step.nodes[0], 0
            k, v = step.rows_of(0, 0), step.rows_of(0, 1)
            step.contexts[0], step.nodes[0] = 40, nodes
            q = step.q[:6].double().view(6, 2, 7, 64)
            w = (torch.einsum("nghd,gkd->nghk", q, k[:, :table_keys]) * 0.125).softmax(-1)
            sure = torch.einsum("nghk,gkd->nghd", w, v[:, :table_keys]).reshape(6, -1)
            assert float(((got[:6] - sure).norm(dim=1) / sure.norm(dim=1)).max()) <= tolerance(step.dtype, 64)
    step.context[0] = (1 << 31) - 1 - 4096 - 5                          # of this one nothing can be
    step.status.zero_()
    step.out.fill_(7.0)
    got = run_plan(step, (row_tile, parts, 1), window)
    assert int(step.status) == 16 and bool((got[:6] == 7).all())


def test_attention_tree_replayed_and_on_another_stream():
    """A captured call, replayed with other trees, contexts and values, while an eager one runs on another stream."""
    a, b = Step(21, [12, 30], [3000, 700], 14, 2, 64, 64), Step(22, [12, 30], [2999, 705], 14, 2, 64, 64)
    a.run(max_context=3100)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        a.run(max_context=3100)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second, stream=side):
        b.run(max_context=3100)
    want_a, want_b = a.plain(), b.plain()
    torch.cuda.synchronize()
    for _ in range(3):
        a.out.zero_()
        b.out.zero_()
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        graph.replay()
        with torch.cuda.stream(other):
            second.replay()
        torch.cuda.synchronize()
        for step, want in ((a, want_a), (b, want_b)):
            assert float(((step.out[:42].double() - want[:42]).norm(dim=1) / want[:42].norm(dim=1)).max()) <= tolerance(torch.bfloat16, 64)
    a.context.copy_(b.context)
    a.flat.copy_(b.flat)
    a.qkv.copy_(b.qkv)
    a.starts.copy_(b.starts)
    a.cache.copy_(b.cache)
    a.block_table.copy_(b.block_table)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.out[:42], b.out[:42])


def test_attention_tree_same_result_every_time():
    step = Step(23, [12, 30, 64], [3000, 700, 1500], 14, 2, 64, 64)
    first = step.run().clone()
    for _ in range(5):
        assert torch.equal(step.run(), first)


# ---- sampling -------------------------------------------------------------------------------------------------------
def plain_sample(x, t, k, p, low, u):
    """The rule in 64 bits: (token, the distance of u from the borders of its share)."""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if not t > 0:
        return (int(np.argmax(x)) if top > -np.inf else 0), 1.0
    if top == -np.inf:
        return 0, 1.0
    with np.errstate(over="ignore", invalid="ignore"):
        w = (x == np.inf).astype(np.float64) if top == np.inf else np.exp((x - top) / t)
    w[x == -np.inf] = 0.0
    order = np.argsort(-x, kind="stable")
    n = k if 0 < k < len(x) else len(x)
    if 0 < p < 1:
        run = np.cumsum(w[order[:n]])
        n = min(n, 1 + int((run[:-1] < p * run[-1]).sum()))
    kept = np.zeros(len(x))
    kept[order[:n]] = w[order[:n]]
    if low > 0:
        kept[kept < min(low, 1.0)] = 0.0
    run = np.cumsum(kept)
    token = int(np.searchsorted(run, u * run[-1], side="right"))
    token = min(token, int(np.flatnonzero(kept)[-1]))
    before = run[token] - kept[token]
    return token, min(abs(u * run[-1] - before), abs(run[token] - u * run[-1])) / run[-1]


def run_sample(logits, t, k, p, low, u, out=None):
    from easy_gpt.cpp_b200 import kernels

    rows = logits.shape[0]
    f = lambda v, dtype=torch.float32: torch.as_tensor(v, device="cuda").to(dtype).expand(rows).contiguous()  # noqa: E731
    out = torch.full((rows,), -9, dtype=torch.int32, device="cuda") if out is None else out
    kernels.sample_min_p(logits, f(t), f(k, torch.int32), f(p), f(low), f(u), out)
    return out


SETTINGS = [(0.8, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.02), (0.3, 20, 0.95, 0.0), (1.5, 5, 1.0, 0.3), (0.8, 0, 0.9, 0.0), (2.0, 1, 1.0, 0.0), (1.0, 50, 0.5, 0.05), (0.7, 1000000, 0.3, 1e-4),
            (1.2, 700, 0.99, 0.0), (0.0, 20, 0.9, 0.1), (1.0, 0, 0.999, 1.0), (5.0, 0, 0.95, 0.0), (1.0, 2000, 1.0, 0.0)]


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("spread", [0.5, 3.0])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4097, 32001, 151936])
def test_sample_min_p(vocab, spread, rounded):
    """Every setting, logits with ties (those of a product in bfloat16) and without.  Sums of weights are off by less than 2^-43 a token, so a token
    may differ only where u is nearer to a border of its share than 2^-43 times the vocabulary."""
    rng = np.random.default_rng([vocab, int(10 * spread), rounded])
    rows = 4 * len(SETTINGS)
    x = rng.normal(0, spread, size=(rows, vocab)).astype(np.float32)
    if rounded:
        x = torch.from_numpy(x).bfloat16().float().numpy()
    u = rng.random(rows).astype(np.float32)
    t, k, p, low = (np.array([SETTINGS[r % len(SETTINGS)][i] for r in range(rows)]) for i in range(4))
    t, p, low = (a.astype(np.float32) for a in (t, p, low))
    got = run_sample(torch.from_numpy(x).cuda(), t, k, p, low, u).tolist()
    for r in range(rows):
        want, room = plain_sample(x[r], float(t[r]), int(k[r]), float(p[r]), float(low[r]), float(u[r]))
        assert got[r] == want or room < vocab * 2.0 ** -43, (r, SETTINGS[r % len(SETTINGS)], got[r], want, room)


def test_sample_min_p_odd_values():
    """Infinities, NaN, masks of the type's lowest value, equal logits, zeros of both signs, settings out of their ranges."""
    inf, nan, lowest = math.inf, math.nan, torch.finfo(torch.float32).min
    rows = [[nan] * 8, [-inf] * 8, [nan, -inf, 1.0, nan, 0.5, -inf, nan, 1.0], [lowest] * 8, [lowest, 2.0, lowest, 1.0] * 2, [1.0, inf, 3.0, inf, -inf, nan, 2.0, 0.0], [0.5] * 8,
            [0.0, -0.0] * 4, [-0.0, 0.0] * 4, [3e38, -3e38, 3e38, 0.0, 1e38, 2e38, -inf, 3e38], [-inf] * 7 + [-5.0], [1e-40, 0.0, -1e-40, 2e-40] * 2]
    x = np.array(rows, np.float32)
    settings = [(1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.9), (0.0, 0, 1.0, 0.0), (-1.0, 2, 0.5, 0.5), (nan, 0, 1.0, 0.0), (1e-30, 0, 0.9, 0.0), (inf, 0, 1.0, 0.0),
                (1.0, -7, 1.0, 0.0), (1.0, 8, 0.0, -1.0), (1.0, 2**31 - 1, 2.0, 7.0), (1.0, 5, 0.75, 1.0), (1.0, 0, nan, 0.0)]
    for s, (t, k, p, low) in enumerate(settings):
        for u in (0.0, 0.3, 0.5, 0.99999994):
            got = run_sample(torch.from_numpy(x).cuda(), np.float32(t), k, np.float32(p), np.float32(low), np.float32(u)).tolist()
            for r in range(len(rows)):
                want, _ = plain_sample(x[r], float(np.float32(t)), k, float(np.float32(p)), float(np.float32(low)), float(np.float32(u)))
                assert got[r] == want, (s, u, r, got[r], want)


@pytest.mark.parametrize("vocab", [100, 40000, 151936])
def test_sample_min_p_ties(vocab):
    """Rows of few values: cuts that fall among equal logits take the first ones."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(0, 3, size=(40, vocab)).astype(np.float32)
    x[:, 5] = 2.0
    ks = [0, 1, 2, 10, vocab // 2, vocab - 1, vocab, vocab + 1]
    u = (rng.random(40) * 0.98 + 0.01).astype(np.float32)
    t = np.full(40, 0.7, np.float32)
    k = np.array([ks[r % 8] for r in range(40)])
    p = np.array([[1.0, 0.37, 0.9][r % 3] for r in range(40)], np.float32)
    got = run_sample(torch.from_numpy(x).cuda(), t, k, p, np.float32(0), u).tolist()
    for r in range(40):
        want, room = plain_sample(x[r], float(t[r]), int(k[r]), float(p[r]), 0.0, float(u[r]))
        assert got[r] == want or room < vocab * 2.0 ** -43, (r, got[r], want, room)


def test_sample_min_p_strides_and_rows():
    """Rows out of wider ones that start at no multiple of 16 bytes; no rows; more outputs than rows."""
    rng = np.random.default_rng(1)
    wide = torch.from_numpy(rng.normal(0, 2, size=(9, 5003)).astype(np.float32)).cuda()
    x = wide[:, 3:4004]
    u = rng.random(9).astype(np.float32)
    out = torch.full((12,), -9, dtype=torch.int32, device="cuda")
    got = run_sample(x, np.float32(0.9), 100, np.float32(0.9), np.float32(0.01), u, out).tolist()
    assert got[:9] == [plain_sample(x[r].cpu().numpy(), float(np.float32(0.9)), 100, float(np.float32(0.9)), float(np.float32(0.01)), float(u[r]))[0] for r in range(9)]
    assert got[9:] == [-9] * 3
    run_sample(wide[:0], 1.0, 0, 1.0, 0.0, 0.5)


@pytest.mark.parametrize("vocab", [262147, 600001, 800000, 1048576])
def test_sample_min_p_large_vocabularies(vocab):
    """Slices of every size, and rows that 16 CTAs do not hold."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 2, size=(len(SETTINGS), vocab)).astype(np.float32)
    u = rng.random(len(SETTINGS)).astype(np.float32)
    t, k, p, low = (np.array([s[i] for s in SETTINGS]) for i in range(4))
    t, p, low = (a.astype(np.float32) for a in (t, p, low))
    got = run_sample(torch.from_numpy(x).cuda(), t, k, p, low, u).tolist()
    for r in range(len(SETTINGS)):
        want, room = plain_sample(x[r], float(t[r]), int(k[r]), float(p[r]), float(low[r]), float(u[r]))
        assert got[r] == want or room < vocab * 2.0 ** -43, (r, SETTINGS[r], got[r], want, room)


def test_sample_min_p_on_two_streams_at_once():
    """Calls that share the GPU, as sizes and settings of each ask for other clusters, draw what they draw alone."""
    from easy_gpt.cpp_b200 import kernels

    calls = []
    for seed, (rows, vocab) in enumerate([(24, 151936), (60, 32001), (3, 1000), (40, 70001)]):
        rng, g = np.random.default_rng(seed), torch.Generator("cuda").manual_seed(seed)
        x = torch.randn((rows, vocab), generator=g, device="cuda") * 2
        f32 = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
        top_k = torch.tensor(rng.choice([0, 1, 20, 700], rows), dtype=torch.int32, device="cuda")
        calls.append((x, f32(rng.choice([0.0, 0.7, 1.3], rows)), top_k, f32(rng.choice([1.0, 0.9], rows)), f32(rng.choice([0.0, 0.01], rows)), f32(rng.random(rows))))
    alone = []
    for call in calls:
        out = torch.empty(call[0].shape[0], dtype=torch.int32, device="cuda")
        kernels.sample_min_p(*call, out)
        alone.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        outs = [torch.full_like(out, -1) for out in alone]
        torch.cuda.synchronize()
        for call, out, stream in zip(calls, outs, streams):
            with torch.cuda.stream(stream):
                kernels.sample_min_p(*call, out)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, outs))


def test_sample_min_p_agrees_with_sample():
    """Without min-p the rule is ``sample``'s."""
    from easy_gpt.cpp_b200 import kernels

    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.normal(0, 2.5, size=(64, 151936)).astype(np.float32)).cuda()
    u = rng.random(64).astype(np.float32)
    out = torch.empty(64, dtype=torch.int32, device="cuda")
    f = lambda v, dtype=torch.float32: torch.full((64,), v, dtype=dtype, device="cuda")  # noqa: E731
    kernels.sample(x, f(0.8), f(50, torch.int32), f(0.95), torch.from_numpy(u).cuda(), out)
    assert run_sample(x, np.float32(0.8), 50, np.float32(0.95), np.float32(0), u).tolist() == out.tolist()


# ---- the walk and the move ------------------------------------------------------------------------------------------
def plain_accept(tokens, targets, parents, longest):
    path, at = [], 0
    while at is not None and len(path) < longest and tokens:
        path.append(at)
        at = next((i for i in range(len(tokens)) if parents[i] == at and tokens[i] == targets[at]), None)
    return path


def run_accept(tokens, targets, parents, longest):
    from easy_gpt.cpp_b200 import kernels

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = np.cumsum([0, *map(len, tokens)]).tolist()
    path = torch.full((len(tokens), longest), -9, dtype=torch.int32, device="cuda")
    emitted, accepted, status = path.clone(), i32([-9] * (len(tokens) + 2)), i32([0])
    flat = lambda lists: i32([v for x in lists for v in x])  # noqa: E731
    kernels.tree_accept(flat(tokens), flat(targets), i32(starts), flat(parents), path, accepted, emitted, status)
    return path.tolist(), accepted.tolist(), emitted.tolist(), int(status)


@pytest.mark.parametrize("longest", [1, 3, 64])
@pytest.mark.parametrize("kind", ["random", "chain", "star"])
def test_tree_accept(kind, longest):
    """Trees of none to two hundred nodes, few different tokens, so that siblings share theirs and walks are long."""
    rng = np.random.default_rng([longest, len(kind)])
    sizes = [1, 0, 2, 31, 32, 33, 64, 65, 100, 200, 7]
    parents = [random_parents(rng, n, kind) for n in sizes]
    words = 1 if kind == "chain" else 4
    tokens, targets = ([rng.integers(0, words, n).tolist() for n in sizes] for _ in range(2))
    if kind == "chain":
        targets = [[int(i != 50) - 1 for i in range(n)] for n in sizes]
    path, accepted, emitted, status = run_accept(tokens, targets, parents, longest)
    assert status == 0 and accepted[len(sizes):] == [-9, -9]
    for r in range(len(sizes)):
        want = plain_accept(tokens[r], targets[r], parents[r], longest)
        assert accepted[r] == len(want) and path[r] == want + [-1] * (longest - len(want))
        assert emitted[r] == [targets[r][i] for i in want] + [-1] * (longest - len(want))


def test_tree_accept_bad_metadata_is_a_status():
    path, accepted, emitted, status = run_accept([[1, 2, 3], [4, 5]], [[2, 3, 9], [5, 6]], [[-1, 0, 1], [-1, 0]], 4)
    assert (accepted[:2], status) == ([3, 2], 0) and emitted == [[2, 3, 9, -1], [5, 6, -1, -1]]
    path, accepted, emitted, status = run_accept([[1, 2, 3], [4, 5]], [[2, 3, 9], [5, 6]], [[-1, 0, 2], [-1, 0]], 4)
    assert (accepted[:2], status) == ([2, 2], 16)
    path, accepted, emitted, status = run_accept([[1, 2, 3], [4, 5]], [[2, 3, 9], [5, 6]], [[-1, 0, 1], [-1, -2]], 4)
    assert (accepted[:2], status) == ([3, 1], 16)


@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 64), (torch.bfloat16, 20), (torch.bfloat16, 18), (torch.bfloat16, 5), (torch.float32, 128), (torch.float32, 3)])
@pytest.mark.parametrize("page", [16, 5])
def test_cache_keep(dtype, dim, page):
    rng = np.random.default_rng([dim, page])
    contexts, longest = [0, 1, 15, 16, 70, 33, 9], 70
    paths = [[0, 2, 3, 7], [], [0], [1, 2, 5], list(range(5)), [0, *range(3, 72)], [0, 1, 4, 5, 6, 20]]
    need = [-(-(c + 80) // page) for c in contexts]
    order, table, at = rng.permutation(sum(need)), np.full((7, max(need)), -1, np.int32), 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    kv = torch.randn((3, at, 2, 2, page, dim), device="cuda").to(dtype)
    want = kv.clone()
    for r, path in enumerate(paths):
        for j, node in enumerate(path):
            a, b = contexts[r] + node, contexts[r] + j
            want[:, table[r, b // page], :, :, b % page] = want[:, table[r, a // page], :, :, a % page]
    run_keep(kv, table, contexts, paths, longest, 0)
    assert torch.equal(kv, want)


def run_keep(kv, table, contexts, paths, longest, status_wanted, accepted=None):
    from easy_gpt.cpp_b200 import kernels

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    status = i32([0])
    path = i32([p + [-1] * (longest - len(p)) for p in paths])
    kernels.cache_keep(kv, torch.from_numpy(table).cuda(), i32(contexts), path, i32(accepted or [len(p) for p in paths]), status)
    assert int(status) == status_wanted


def test_cache_keep_strides():
    """A pool cut out of a larger one: some layers, and heads whose rows lie apart."""
    big = torch.randn((5, 20, 2, 4, 16, 64), device="cuda").bfloat16()
    before = big.clone()
    kv = big[1:4, :, :, 1:3]
    table = np.arange(20, dtype=np.int32).reshape(2, 10)
    want = before.clone()
    for r, c, path in ((0, 30, [0, 3, 9]), (1, 100, [0, 2])):
        for j, node in enumerate(path):
            a, b = c + node, c + j
            want[1:4, table[r, b // 16], :, 1:3, b % 16] = want[1:4, table[r, a // 16], :, 1:3, a % 16]
    run_keep(kv, table, [30, 100], [[0, 3, 9], [0, 2]], 5, 0)
    assert torch.equal(big, want)


def test_cache_keep_refuses_what_cannot_be():
    """A path that does not ascend or reaches back, more accepted than it has places: nothing of that request moves; a page that is none: not that row."""
    kv = torch.randn((2, 12, 2, 2, 16, 64), device="cuda").bfloat16()
    table = np.arange(12, dtype=np.int32).reshape(2, 6)
    good = kv.clone()
    good[:, table[1, 1], :, :, 5] = good[:, table[1, 1], :, :, 8]     # request 1: context 20, path 0, 4 -> 1
    for bad in ([0, 3, 3], [0, 5, 4], [0, -1], [1, 0]):
        mine = kv.clone()
        run_keep(mine, table, [10, 20], [bad, [0, 4]], 4, 16)
        assert torch.equal(mine, good)
    for accepted in ([5, 2], [-1, 2]):
        mine = kv.clone()
        run_keep(mine, table, [10, 20], [[0, 2], [0, 4]], 4, 16, accepted)
        assert torch.equal(mine, good)
    for page in (-1, 12):
        mine, other = kv.clone(), table.copy()
        other[0, 1] = page                                            # request 0: positions 16 .. 31 have no page
        run_keep(mine, other, [10, 20], [[0, 2, 8], [0, 4]], 4, 2)
        want = good.clone()
        want[:, table[0, 0], :, :, 11] = want[:, table[0, 0], :, :, 12]
        assert torch.equal(mine, want)


# ---- together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_of_all_of_them(dtype):
    """Attention over the trees, a product for logits, samples, the walk and the move, captured once and replayed: what the tokens and the cache are then is
    what the plain forms say, and the next token's attention over the moved keys is that of a tree which was the accepted chain from the start."""
    from easy_gpt.cpp_b200 import kernels

    step = Step(31, [16, 24, 9], [100, 37, 0], 14, 2, 64, 16, dtype)
    total, vocab, longest, rng = 49, 500, 6, np.random.default_rng(31)
    head = torch.randn((vocab, 14 * 64), device="cuda").to(dtype)
    f = lambda v: torch.full((total,), v, device="cuda")  # noqa: E731
    top_k, uniform = torch.full((total,), 50, dtype=torch.int32, device="cuda"), torch.from_numpy(rng.random(total).astype(np.float32)).cuda()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    tokens, targets, path, emitted, accepted = i32(total), i32(total), i32(3, longest), i32(3, longest), i32(3)
    kv = step.cache.unsqueeze(0)
    before = step.cache.clone()

    def run():
        step.run(max_context=128)
        logits = (step.out[:total] @ head.T).float()
        kernels.sample_min_p(logits, f(0.8), top_k, f(0.9), f(0.05), uniform, targets)
        kernels.tree_accept(tokens, targets, step.starts, step.flat, path, accepted, emitted, step.status)
        kernels.cache_keep(kv, step.block_table, step.context, path, accepted, step.status)
        return logits

    run()                                                             # what the model answers does not hang on the drafts' tokens here
    at, drafted = 0, targets.tolist()
    for r, n in enumerate(step.nodes):                                # drafts that the model agrees with, down some path of every tree
        for i in range(1, n):
            if rng.random() < 0.7:
                tokens[at + i] = drafted[at + step.parents[r][i]]
            else:
                tokens[at + i] = -1
        at += n
    step.cache.copy_(before)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        logits = run()
    for _ in range(2):
        step.cache.copy_(before)
        graph.replay()
    torch.cuda.synchronize()
    assert int(step.status) == 0
    x, answers, drafts, at = logits.cpu().numpy(), targets.tolist(), tokens.tolist(), 0
    assert answers == [plain_sample(x[i], float(np.float32(0.8)), 50, float(np.float32(0.9)), float(np.float32(0.05)), float(uniform[i]))[0] for i in range(total)]
    want = before.clone()
    for r, n in enumerate(step.nodes):
        walk = plain_accept(drafts[at:at + n], answers[at:at + n], step.parents[r], longest)
        assert path[r].tolist() == walk + [-1] * (longest - len(walk)) and int(accepted[r]) == len(walk)
        assert emitted[r].tolist() == [answers[at + i] for i in walk] + [-1] * (longest - len(walk))
        for j, node in enumerate(walk):
            a, b = step.contexts[r] + node, step.contexts[r] + j
            want[step.table[r, b // 16], :, :, b % 16] = before[step.table[r, a // 16], :, :, a % 16]
        at += n
    assert torch.equal(step.cache, want) and max(accepted.tolist()) > 2
    # one more token of every request over what was kept
    more = Step(32, [1, 1, 1], [c + a for c, a in zip(step.contexts, accepted.tolist())], 14, 2, 64, 16, dtype)
    more.cache, more.table, more.block_table = step.cache, step.table, step.block_table
    more.k, more.v = step.cache[:, 0], step.cache[:, 1]
    check(more)
