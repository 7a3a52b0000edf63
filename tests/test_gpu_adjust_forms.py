"""adjust_logits over the ranges of its arguments, on torch tensors, in processes of
their own: torch has a HIP runtime of its own, which the library shares only where
torch is loaded first."""
import pytest

from test_gpu_adjust import run_apart


@pytest.mark.gpu
def test_prompts():
    run_apart("torch_adjust_prompts.py")


def test_prompts_without_a_gpu():
    run_apart("torch_adjust_prompts.py", "-m", "not gpu")


@pytest.mark.gpu
def test_every_kernel():
    run_apart("torch_adjust_kernels.py")


@pytest.mark.gpu
def test_ids():
    run_apart("torch_ids.py")
