"""Kernels that start before the kernel ahead of them has ended (programmatic dependents) may find its output still being
written: they read it by coherent loads only.  A non-coherent one (ld.global.nc, __ldg) asks for data that nobody writes while
the kernel lives.  Read off the sources: no run could be relied on to show it."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "accel_b200" / "csrc"


@pytest.mark.parametrize("name", ["window.cuh", "window_attention.cu", "window_prefill.cu", "logprobs.cu", "cache_pages.cu"])
def test_programmatic_dependents_load_coherently(name):
    code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    found = re.findall(r"__ldg\w*|ld\.global[\w.:]*\.nc[\w.:]*|__restrict__", code)
    assert not found, f"{name}: {found}"
