"""Batches of requests with and without min-p: launches that a step takes, vocabularies that the kernel of min-p does not take."""
import numpy as np
import pytest

import tiny_configs
from easy_gpt.cpp_b200.sampling import GREEDY, SamplingParams


def test_largest_vocabulary():
    """What the engines go by is what the launcher takes."""
    from easy_gpt.cpp_b200 import kernels

    assert kernels.library().eg_sample_min_p_most_tokens() == kernels.SAMPLE_MAX_VOCAB


@pytest.mark.gpu
def test_a_vocabulary_beyond_the_kernel_is_refused_with_the_request(tmp_path):
    """Min-p takes vocabularies of up to 2^20 tokens.  A request that asks for it over a larger one is refused when it is added, and the others run."""
    from easy_gpt.cpp_b200 import kernels
    from easy_gpt.cpp_b200.engine import GptEngine
    from easy_gpt.cpp_b200.native import NativeEngine
    from easy_gpt.cpp_b200.weights.random_init import write_random_model

    vocab = kernels.SAMPLE_MAX_VOCAB + 1
    small = {"vocab_size": vocab, "hidden_size": 16, "num_attention_heads": 1, "num_key_value_heads": 1}
    folder = write_random_model(tmp_path / "model", {**tiny_configs.CONFIG_A, **small}, **tiny_configs.RANDOM_A)
    options = dict(dtype="float32", page_size=4, cache_tokens=512, max_active=6, chunk_size=16, max_batch_tokens=64)
    outputs = []
    for engine in (NativeEngine(folder, **options), GptEngine(folder, **options)):
        good = [engine.add_request([5, 17, vocab - 1], p, max_new_tokens=3) for p in (GREEDY, SamplingParams(seed=3), SamplingParams(greedy=True, min_p=0.5))]
        with pytest.raises(ValueError, match="Min-p needs a vocabulary"):
            engine.add_request([5, 17], SamplingParams(min_p=0.1), max_new_tokens=3)
        engine.run_to_completion()
        outputs.append([engine.output(r) if hasattr(engine, "output") else list(r.output) for r in good])
    assert [len(o) for o in outputs[0]] == [3] * 3 and outputs[0] == outputs[1]


KINDS = [SamplingParams(), SamplingParams(min_p=0.1, top_k=0, top_p=1.0), GREEDY, SamplingParams(min_p=0.3, temperature=1.5, top_k=50)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 64, 300])
def test_a_mixed_batch_takes_two_launches(rows):
    """However its requests lie: with and without min-p in turn, greedy ones between them.  Every request gets the token that it gets alone."""
    import torch

    from easy_gpt.cpp_b200 import kernels
    from easy_gpt.cpp_b200.sampling import Sampler

    logits = torch.from_numpy(np.random.default_rng(rows).normal(0, 2, size=(rows, 5000)).astype(np.float32)).cuda()
    params = [KINDS[r % 4] for r in range(rows)]
    sampler, single = Sampler("cuda"), Sampler("cuda")
    want = [int(single.sample(logits[r:r + 1], [p], [r], [7])[0]) for r, p in enumerate(params)]
    for _ in range(3):
        before = kernels.launch_count
        got = sampler.sample(logits, params, list(range(rows)), [7] * rows)
        assert kernels.launch_count - before == min(rows, 2)
        assert got.tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["sample", "sample_min_p"])
def test_rows_by_number(name):
    """Some rows of a batch, in any order: those alone are sampled, as in a call over all of them; the others' places are left, and so is what no row has."""
    import torch

    from easy_gpt.cpp_b200 import kernels

    rng = np.random.default_rng(5)
    logits = torch.from_numpy(rng.normal(0, 2, size=(20, 3001)).astype(np.float32)).cuda()
    f = lambda *s: torch.tensor(rng.choice(s, 20).astype(np.float32), device="cuda")  # noqa: E731
    top_k = torch.tensor(rng.choice([0, 20, 700], 20).astype(np.int32), device="cuda")
    settings = [f(0.0, 0.8, 1.3), top_k, f(1.0, 0.9)] + ([f(0.0, 0.05)] if name == "sample_min_p" else []) + [torch.from_numpy(rng.random(20).astype(np.float32)).cuda()]
    whole, some = (torch.full((20,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    getattr(kernels, name)(logits, *settings, whole)
    picked = [3, 19, 0, 7, 8]
    numbers = torch.tensor([*picked, -1, 20, 2**31 - 1, -2**31], dtype=torch.int32, device="cuda")
    getattr(kernels, name)(logits, *settings, some, which=numbers)
    assert some.tolist() == [t if r in picked else -9 for r, t in enumerate(whole.tolist())]
    getattr(kernels, name)(logits, *settings, some, which=numbers[:0])
    for wrong in (numbers.long(), numbers[::2], numbers.cpu(), numbers.view(3, 3)):
        with pytest.raises(kernels.KernelError):
            getattr(kernels, name)(logits, *settings, some, which=wrong)
