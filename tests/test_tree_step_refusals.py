"""What the operators of a step over drafted trees refuse before anything is launched (no GPU), beside the sizes and types."""
import pytest

from easy_gpt.cpp_b200 import kernels
from test_tree_step import ATTENTION, Reached, on_the_host  # noqa: F401


@pytest.mark.parametrize("scale", [1e-50, 2e38, 3e38])
def test_scales_that_32_bits_do_not_hold(scale, on_the_host):  # noqa: F811
    """A scale that is 0 in 32 bits, or infinite once the exponents' base is in it: 0 times the -inf of a hidden score is NaN, and so is infinity times a score of 0."""
    with pytest.raises(kernels.KernelError, match="scale"):
        kernels.attention_tree(**{**ATTENTION, "scale": scale})


@pytest.mark.parametrize("scale", [1e-44, 1e-30, 1e30, 1.9e38])
def test_scales_that_32_bits_hold(scale, on_the_host):  # noqa: F811
    with pytest.raises(Reached):
        kernels.attention_tree(**{**ATTENTION, "scale": scale})


def test_the_launcher_refuses_such_scales():
    lib, at = kernels.library(), 0x1000
    attend = lambda scale: lib.eg_attention_tree(None, kernels._pack_attention_tree(at, at, at, at, at, at, at, at, at, kernels.BF16, 256, 256, 4096, 1024, 3, 3, 4, 4, 1, 4, 2, 64, 16, 0, 100, 0, 1,  # noqa: E731
                                                                                    1, scale))
    assert [attend(scale) for scale in (1e-50, 1e-46, 2e38, 3e38)] == [1] * 4
