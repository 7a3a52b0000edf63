"""torch_scores_modes.py and torch_scores_large.py in processes of their own, where
torch is loaded first."""
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def run(which, name="torch_scores_modes.py"):
    subprocess.run([sys.executable, "-u", "-m", "pytest", str(HERE / name), "-v", "-m", which, "-p",
                    "no:cacheprovider", "--timeout", "60", "--timeout-method", "thread"], cwd=HERE.parent, check=True,
                   timeout=300)


def test_without_a_gpu():
    run("not gpu")


@pytest.mark.gpu
def test_on_the_gpu():
    run("gpu")


@pytest.mark.gpu
def test_past_the_cache():
    run("gpu", "torch_scores_large.py")
