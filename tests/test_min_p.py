"""Min-p as an option of a request: its checks, the command line's (no GPU), and the engines' (GPU)."""
import subprocess

import numpy as np
import pytest

import tiny_configs
from easy_gpt.cpp_b200 import cli
from easy_gpt.cpp_b200.sampling import SamplingParams


def test_option():
    assert SamplingParams().min_p == 0.0 and SamplingParams(min_p=1.0).min_p == 1.0
    for wrong in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="Min-p"):
            SamplingParams(min_p=wrong)


def test_command_line():
    options, error = cli.parse_args(["--min-p", "0.05", "hello"])
    assert error == "" and options.min_p == 0.05 and cli.parse_args(["hello"])[0].min_p == 0.0
    for argv, text in ((["--min-p", "1.5"], "Min-p must be in [0, 1]"), (["--min-p", "-1"], "Min-p must be in [0, 1]"), (["--min-p", "x"], "Invalid number for min-p: x"),
                       (["--min-p"], "Missing number after --min-p")):
        assert cli.parse_args(argv) == (None, text)


def test_native_command_line():
    """The C++ program's own parsing (it stops at the error, before any device is touched)."""
    from easy_gpt.cpp_b200.csrc.build import engine_paths

    program = str(engine_paths()[1])
    for argv, text in ((["--min-p", "1.5", "a"], "Min-p must be in [0, 1]"), (["--min-p", "x", "a"], "Invalid number for min-p: x"), (["--min-p"], "Missing number after --min-p")):
        done = subprocess.run([program, *argv], capture_output=True, text=True)
        assert done.returncode != 0 and text in done.stdout + done.stderr
    assert "--min-p" in subprocess.run([program, "--help"], capture_output=True, text=True).stdout


def plain_token(logits, p, u):
    """The rule in 64 bits, over one row."""
    x = logits.astype(np.float64)
    w = np.exp((x - x.max()) / float(np.float32(p.temperature)))
    order = np.argsort(-x, kind="stable")
    n = p.top_k if 0 < p.top_k < len(x) else len(x)
    if 0 < p.top_p < 1:
        run = np.cumsum(w[order[:n]])
        n = min(n, 1 + int((run[:-1] < float(np.float32(p.top_p)) * run[-1]).sum()))
    kept = np.zeros(len(x))
    kept[order[:n]] = w[order[:n]]
    kept[kept < float(np.float32(p.min_p))] = 0.0
    run = np.cumsum(kept)
    return int(np.searchsorted(run, np.float32(u) * run[-1], side="right"))


@pytest.mark.gpu
def test_sampler_takes_rows_with_and_without_min_p():
    """Rows of both kinds and greedy ones between each other: those with min-p follow the rule, the others get the tokens that they get alone."""
    import torch

    from easy_gpt.cpp_b200.sampling import GREEDY, Sampler
    from easy_gpt.cpp_b200.sampling.rng import uniform

    logits = torch.from_numpy(np.random.default_rng(4).normal(0, 2, size=(40, 5000)).astype(np.float32)).cuda()
    kinds = [SamplingParams(), SamplingParams(min_p=0.1, top_k=0, top_p=1.0), GREEDY, SamplingParams(min_p=0.3, temperature=1.5, top_k=50), SamplingParams(top_k=0, top_p=1.0, min_p=1.0)]
    params = [kinds[(r * r) % 5] for r in range(40)]
    tokens = Sampler("cuda").sample(logits, params, list(range(40)), [3] * 40).tolist()
    for r, p in enumerate(params):
        if p.min_p:
            assert tokens[r] == plain_token(logits[r].cpu().numpy(), p, uniform(p.seed, r, 3)), r
        else:
            assert tokens[r] == Sampler("cuda").sample(logits[r:r + 1], [p], [r], [3]).tolist()[0], r


@pytest.mark.gpu
def test_engines_take_min_p(tmp_path):
    """Min-p of 1 leaves the likeliest token alone, which is greedy; requests with and without it in one batch get what they get alone; both engines agree."""
    from easy_gpt.cpp_b200.engine import GptEngine
    from easy_gpt.cpp_b200.native import NativeEngine, NativeError  # noqa: F401
    from easy_gpt.cpp_b200.sampling import GREEDY

    folder = tiny_configs.write_tiny("A", tmp_path / "model")
    options = dict(dtype="float32", page_size=4, cache_tokens=512, max_active=6, chunk_size=16, max_batch_tokens=64)
    prompts = [tiny_configs.random_tokens(256, n, n) for n in (5, 17, 9, 12, 7, 3)]
    first = SamplingParams(min_p=1.0, top_k=0, top_p=1.0)
    kinds = [first, SamplingParams(seed=7), SamplingParams(min_p=0.02, seed=3), GREEDY, SamplingParams(min_p=0.2, top_k=0, temperature=1.3), SamplingParams(top_k=0, top_p=1.0, seed=1)]

    def outputs(engine, kinds):
        ids = [engine.add_request(p, k, max_new_tokens=10) for p, k in zip(prompts, kinds)]
        engine.run_to_completion()
        return [engine.output(i) if hasattr(engine, "output") else list(i.output) for i in ids]

    native, torch_face = NativeEngine(folder, **options), GptEngine(folder, **options)
    together = outputs(native, kinds)
    assert together == outputs(torch_face, kinds)
    assert outputs(NativeEngine(folder, **options), [first] * 6) == outputs(NativeEngine(folder, **options), [GREEDY] * 6)
    without = outputs(NativeEngine(folder, **options), [k if not k.min_p else GREEDY for k in kinds])
    assert [t for t, k in zip(together, kinds) if not k.min_p] == [t for t, k in zip(without, kinds) if not k.min_p]
    assert together[0] == without[0]
    with pytest.raises(ValueError, match="Min-p"):
        native.add_request(prompts[0], SamplingParams(min_p=2.0), max_new_tokens=1)
