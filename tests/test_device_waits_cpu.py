"""Words in shared memory that a kernel's bounded waits look at: a barrier of the block stands between their clearing and the first wait.

Without it a warp that starts early may find what an earlier block left there and give up. That shows on no GPU on demand, so the order of
the statements is checked where they stand."""
import os
import re

import pytest

from owoinfer_b200 import build

KERNELS = [(f, m.start()) for f in build.SOURCES for m in re.finditer(r"__shared__ int s_abort\b", open(os.path.join(build.CSRC, f)).read())]


def test_kernels_were_found():
    assert len(KERNELS) >= 4


@pytest.mark.parametrize("file,at", KERNELS, ids=[f for f, _ in KERNELS])
def test_abort_words_are_cleared_before_any_wait(file, at):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(build.CSRC, file)).read()[at:])
    cleared = re.search(r"\bs_abort = 0\b", text).end()
    waits = re.search(r"\b(?:warp_)?wait(?:_bar(?:_relaxed)?)?(?:<\w+>)?\(", text[cleared:])
    assert waits is not None and "__syncthreads();" in text[cleared:cleared + waits.start()]
