"""detllm_amd.scores on torch tensors, in a process of its own: torch has a HIP
runtime of its own, which the library shares only where torch is loaded first."""
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


@pytest.mark.gpu
def test_scores_on_torch_tensors():
    p = subprocess.Popen([sys.executable, "-u", "-m", "pytest", str(HERE / "torch_scores.py"), "-x", "-v", "-p",
                          "no:cacheprovider", "--timeout", "60", "--timeout-method", "thread"], cwd=HERE.parent,
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
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


def test_two_hip_runtimes_are_refused():
    code = ("import detllm_amd._lib\n"
            "try:\n    import detllm_amd.scores\n"
            "except ImportError as e:\n    assert 'import torch before' in str(e)\n"
            "else:\n    raise SystemExit('not refused')\n")
    subprocess.run([sys.executable, "-c", code], cwd=HERE.parent, check=True, timeout=300)
