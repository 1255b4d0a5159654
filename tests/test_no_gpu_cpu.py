"""Where there is no GPU the tests that need one are skipped, whichever file they stand in."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
@pytest.mark.parametrize("file", ["test_gpu_text_cache.py", "test_gpu_parity.py"])
def test_gpu_tests_are_skipped(file):
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", os.path.join("tests", file)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "failed" not in run.stdout and "skipped" in run.stdout, run.stdout[-2000:]
