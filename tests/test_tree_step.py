"""What the operators of a step over drafted trees refuse before anything is launched (no GPU): by their Python faces, and by the launchers alone."""
import ctypes
import math

import pytest
import torch

from easy_gpt.cpp_b200 import kernels


class Reached(Exception):
    pass


@pytest.fixture
def on_the_host(monkeypatch):
    """Tensors of the host pass for tensors of a device, and a launch is an exception of its own."""
    def reached():
        raise Reached

    monkeypatch.setattr(kernels, "_device_of", lambda *tensors: 0)
    monkeypatch.setattr(kernels, "_current_device", lambda: 0)
    monkeypatch.setattr(kernels, "library", reached)
    monkeypatch.setattr(kernels, "_stream_of", lambda device: 0)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


CACHE = torch.zeros((4, 2, 2, 16, 64), dtype=torch.bfloat16)
ROWS = torch.zeros((10, 256), dtype=torch.bfloat16)
ATTENTION = dict(q=ROWS, k_cache=CACHE[:, 0], v_cache=CACHE[:, 1], block_table=i32(2, 3), entry_starts=i32(3), context=i32(2), parents=i32(10), out=ROWS.clone(), num_heads=4, num_kv_heads=2,
                 head_dim=64, window=None, scale=0.125, status=i32(1))
NUMBERS = torch.zeros(2)
SAMPLE = dict(logits=torch.zeros((2, 8)), temperature=NUMBERS, top_k=i32(2), top_p=NUMBERS, min_p=NUMBERS, uniform=NUMBERS, out=i32(2))
ACCEPT = dict(tokens=i32(2), targets=i32(2), entry_starts=i32(3), parents=i32(2), path=i32(2, 3), accepted=i32(2), emitted=i32(2, 3), status=i32(1))
KV = torch.zeros((1, 4, 2, 2, 16, 64))
KEEP = dict(kv=KV, block_table=i32(2, 2), context=i32(2), path=i32(2, 3), accepted=i32(2), status=i32(1))
REFUSED = [
    *(("attention_tree", ATTENTION, w) for w in (
        dict(q=ROWS.float()), dict(q=ROWS.half(), out=ROWS.half(), k_cache=CACHE[:, 0].half(), v_cache=CACHE[:, 1].half()), dict(num_heads=3), dict(num_kv_heads=0), dict(num_heads=0), dict(head_dim=32),
        dict(head_dim=300), dict(block_table=i32(2, 3).long()), dict(block_table=i32(3, 2).t()), dict(block_table=i32(6)), dict(entry_starts=i32(2)), dict(context=i32(1)), dict(context=i32(4)[::2]),
        dict(parents=i32(11)), dict(parents=i32(20)[::2]), dict(out=ROWS[:4]), dict(out=ROWS[:, :255]), dict(v_cache=CACHE[:1, 1]), dict(k_cache=CACHE[:, 0].transpose(2, 3)), dict(k_cache=CACHE[0, 0]),
        dict(status=i32(1).long()), dict(q=ROWS[:, :64]), dict(q=ROWS[0]), dict(window=-3), dict(window=0), dict(scale=0.0), dict(scale=-0.1), dict(scale=math.nan), dict(scale=math.inf), dict(v_cache=CACHE[:, 1].float()))),
    *(("sample_min_p", SAMPLE, w) for w in (
        dict(logits=torch.zeros((2, 8), dtype=torch.float64)), dict(logits=torch.zeros((8, 2)).t()), dict(logits=torch.zeros(8)), dict(temperature=NUMBERS.double()), dict(top_k=NUMBERS),
        dict(min_p=NUMBERS[:1]), dict(out=i32(2).long()), dict(logits=torch.zeros((2, 0))), dict(logits=torch.zeros((1, 1)).expand(2, (1 << 20) + 1)), dict(top_p=torch.zeros(4)[::2]))),
    *(("tree_accept", ACCEPT, w) for w in (
        dict(tokens=i32(2).long()), dict(targets=i32(1)), dict(parents=i32(1)), dict(path=i32(1, 3)), dict(emitted=i32(2, 2)), dict(accepted=i32(1)), dict(path=i32(2, 0), emitted=i32(2, 0)),
        dict(path=i32(3, 2).t()), dict(path=i32(6)), dict(entry_starts=i32(0)))),
    *(("cache_keep", KEEP, w) for w in (
        dict(kv=KV[0]), dict(kv=KV.double()), dict(kv=KV[:, :, :1]), dict(kv=KV.transpose(4, 5)), dict(kv=KV[..., ::2]), dict(block_table=i32(1, 2)), dict(block_table=i32(4)), dict(context=i32(1)),
        dict(path=i32(2, 3).long()), dict(accepted=i32(1)), dict(path=i32(3)), dict(path=i32(2, 0)), dict(path=i32(2, 6)[:, ::2]))),
]


@pytest.mark.parametrize("name, base, wrong", REFUSED)
def test_refused_before_a_launch(name, base, wrong, on_the_host):
    with pytest.raises(kernels.KernelError):
        getattr(kernels, name)(**{**base, **wrong})


@pytest.mark.parametrize("name, base", [("attention_tree", ATTENTION), ("sample_min_p", SAMPLE), ("tree_accept", ACCEPT), ("cache_keep", KEEP)])
def test_taken(name, base, on_the_host):
    with pytest.raises(Reached):
        getattr(kernels, name)(**base)


@pytest.mark.parametrize("name, base", [("attention_tree", ATTENTION), ("sample_min_p", SAMPLE), ("tree_accept", ACCEPT), ("cache_keep", KEEP)])
def test_there_is_no_cpu_path(name, base):
    with pytest.raises(kernels.KernelError, match="no CPU path"):
        getattr(kernels, name)(**base)


def test_launchers_refuse_sizes_they_do_not_take():
    """The C entry points by themselves: cudaErrorInvalidValue (1) for what their callers could get wrong, 0 for nothing to do; nothing is launched."""
    lib, at = kernels.library(), 0x1000
    sample = lambda rows, vocab: lib.eg_sample_min_p(None, at, vocab, rows, vocab, at, at, at, at, at, at)  # noqa: E731
    assert [sample(0, 8), sample(1, 0), sample(1, (1 << 20) + 1)] == [0, 1, 1]
    accept = lambda entries, rows, longest, status=at: lib.eg_tree_accept(None, kernels._pack_tree_accept(at, at, at, at, at, at, at, status, entries, rows, longest))  # noqa: E731
    assert [accept(0, 0, 1), accept(1, -1, 1), accept(1, 1, 0), accept(1, 1, 1, 0), accept(1, 1 << 31, 1), accept(1 << 31, 1, 1), lib.eg_tree_accept(None, None)] == [0, 1, 1, 1, 1, 1, 1]

    def keep(kv=at, size=2, layers=1, pages=4, heads=2, page=16, dim=64, entries=1, longest=3, status=at):
        return lib.eg_cache_keep(None, kernels._pack_cache_keep(kv, at, at, at, at, status, size, layers, pages, heads, page, dim, 0, 2 * heads * page * dim, heads * page * dim, page * dim, 2, 2,
                                                                entries, longest))

    assert [keep(entries=0), keep(layers=0)] == [0, 0]
    assert [keep(size=1), keep(size=8), keep(pages=0), keep(heads=0), keep(page=0), keep(dim=0), keep(longest=0), keep(status=0), keep(entries=65536), keep(kv=at + 1),
            keep(layers=1 << 30), keep(layers=1 << 40), lib.eg_cache_keep(None, None)] == [1] * 13

    def attend(dtype=kernels.BF16, rows=4, entries=1, heads=4, kv_heads=2, dim=64, page=16, pages=4, parts=1, tiles=1, status=at, q=at, ldq=256, row_tile=0, scale=0.125,
               window=0, table_pages=3, cache=at):
        return lib.eg_attention_tree(None, kernels._pack_attention_tree(q, cache, cache, at, at, at, at, at, status, dtype, ldq, 256, 4096, 1024, 3, table_pages, pages, rows, entries, heads,
                                                                        kv_heads, dim, page, window, 100, row_tile, parts, tiles, scale))

    assert [attend(rows=0), attend(entries=0)] == [0, 0]
    assert lib.eg_attention_tree(None, None) == 1
    for wrong in (dict(dtype=2), dict(heads=3), dict(kv_heads=0), dict(dim=0), dict(dim=257), dict(page=0), dict(pages=0), dict(parts=0), dict(tiles=0), dict(parts=3), dict(parts=32), dict(status=0),
                  dict(entries=65536), dict(rows=1 << 30), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1), dict(table_pages=-1), dict(row_tile=8),
                  dict(row_tile=16, dtype=kernels.F32), dict(row_tile=16, dim=84), dict(row_tile=64, page=24), dict(row_tile=32, q=at + 2), dict(row_tile=16, ldq=257),
                  dict(row_tile=16, cache=at + 8), dict(row_tile=128, dim=32), dict(row_tile=128, q=at + 8), dict(row_tile=128, dim=128, ldq=260), dict(row_tile=128, heads=258), dict(row_tile=256)):
        assert attend(**wrong) == 1, wrong


def test_plans():
    """From sizes alone: what the tensor-core kernels do not take on the 32-bit one, short contexts of few units on the warp-level one, the rest of heads of 64
    and 128 on tcgen05; never more parts than CTAs find room, and more of them the fewer units there are."""
    plan = kernels.attention_tree_plan
    assert plan(kernels.F32, 2, 8, 1, 14, 2, 64, 16, 500)[0] == plan(kernels.BF16, 2, 8, 1, 14, 2, 68, 16, 500)[0] == plan(kernels.BF16, 2, 8, 1, 14, 2, 64, 24, 500)[0] == 0
    assert plan(kernels.BF16, 0, 8, 1, 14, 2, 64, 16, 500)[0] == 0
    assert [plan(kernels.BF16, 2, 8, 1, 14, 2, 64, 16, keys)[0] for keys in (500, 1024, 1025, 30000)] == [16, 16, 128, 128]
    assert plan(kernels.BF16, 2, 1024, 64, 12, 2, 128, 64, 700)[0] == 128
    assert [plan(kernels.BF16, aligned, 64 * n, 64, 14, 2, dim, 16, 5000)[0] for aligned, dim in ((1, 64), (2, 32), (2, 80), (2, 256)) for n in (1, 4, 64)] == [16, 32, 64] * 4
    for aligned in (0, 1, 2):
        for nodes in (1, 9, 64, 300):
            parts = [plan(kernels.BF16, aligned, nodes * entries, entries, 28, 4, 128, 64, 4000)[1] for entries in (1, 4, 16, 64, 256)]
            assert parts == sorted(parts, reverse=True) and all(p in (1, 2, 4, 8, 16) for p in parts) and parts[-1] == 1, parts


def test_plans_of_float32():
    """Rows in whole 16-byte pieces go in CTAs of 32, two an SM, in up to 16 parts where the keys are many; others, and heads of more than 128, in 8 at most."""
    def parts(aligned, *sizes):
        plan = (ctypes.c_int * 3)()
        assert kernels.library().eg_attention_tree_plan(kernels.F32, aligned, *sizes, 148, plan) == 0 and plan[0] == 0
        return plan[1]

    assert [parts(2, 1, 1, 12, 12, 128, 16, keys) for keys in (100, 1000, 4000)] == [2, 8, 16]
    assert [parts(0, 1, 1, 12, 12, 128, 16, keys) for keys in (100, 1000, 4000)] == [2, 8, 8]
    assert parts(2, 1, 1, 12, 12, 256, 16, 4000) == 8
    assert [parts(2, 13 * n, n, 12, 2, 128, 16, 1000) for n in (4, 16, 64)] == [8, 2, 1]
