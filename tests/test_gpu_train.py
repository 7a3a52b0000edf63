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
