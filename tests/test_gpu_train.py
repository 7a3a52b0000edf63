"""detllm_amd.train on torch tensors, in a process of its own: torch has a HIP runtime
of its own, which the library shares only where torch is loaded first."""
import pytest

from test_gpu_adjust import run_apart


@pytest.mark.gpu
def test_embeddings():
    run_apart("torch_embedding.py")


@pytest.mark.gpu
def test_gradient_norms_and_clipping():
    run_apart("torch_clip.py")


@pytest.mark.gpu
def test_the_operators_together():
    run_apart("torch_together.py")


@pytest.mark.gpu
def test_other_modes():
    run_apart("torch_more_modes.py")


def test_other_modes_without_a_gpu():
    run_apart("torch_more_modes.py", "-m", "not gpu")
