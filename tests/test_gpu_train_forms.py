"""detllm_amd.train over the ranges of its arguments, on torch tensors, in processes of
their own: torch has a HIP runtime of its own, which the library shares only where
torch is loaded first."""
import pytest

from test_gpu_adjust import run_apart


@pytest.mark.gpu
def test_constants():
    run_apart("torch_constants.py")


@pytest.mark.gpu
def test_lists_without_elements():
    run_apart("torch_no_gradients.py")


@pytest.mark.gpu
def test_long_runs_of_a_token():
    run_apart("torch_embedding_runs.py")


@pytest.mark.gpu
def test_large_lists_and_norms():
    run_apart("torch_clip_large.py")
