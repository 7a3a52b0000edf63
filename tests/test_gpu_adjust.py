"""detllm_amd.scores.adjust_logits on torch tensors, in a process of its own: torch
has a HIP runtime of its own, which the library shares only where torch is loaded
first."""
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def run_apart(name, *which):
    p = subprocess.Popen([sys.executable, "-u", "-m", "pytest", str(HERE / name), *which, "-x", "-v", "-p", "no:cacheprovider",
                          "--timeout", "60", "--timeout-method", "thread"], cwd=HERE.parent, stdout=subprocess.PIPE,
                         stderr=subprocess.STDOUT, text=True)
    lines = []
    try:
        for line in p.stdout:  # passed on as they come
            print(line, end="", flush=True)
            lines.append(line)
        assert p.wait(timeout=60) == 0, "".join(lines[-40:])
    finally:
        if p.poll() is None:
            p.kill()
            p.wait()


@pytest.mark.gpu
def test_adjusted_logits_of_torch_tensors():
    run_apart("torch_adjust.py")
