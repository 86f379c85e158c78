"""Batches of requests with and without min-p: launches that a step takes, vocabularies that the kernel of min-p does not take."""
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
