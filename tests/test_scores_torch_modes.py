"""torch_scores_modes.py in a process of its own, where torch is loaded first."""
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def run(which):
    subprocess.run([sys.executable, "-u", "-m", "pytest", str(HERE / "torch_scores_modes.py"), "-v", "-m", which, "-p",
                    "no:cacheprovider", "--timeout", "60", "--timeout-method", "thread"], cwd=HERE.parent, check=True,
                   timeout=300)


def test_without_a_gpu():
    run("not gpu")


@pytest.mark.gpu
def test_on_the_gpu():
    run("gpu")
