"""Read off the sources: a kernel that gives up a wait for the copy engine (the waits are bounded) lets the copies that it has under way land
before its shared memory goes to other uses or to the next CTA."""
import re
from pathlib import Path

import pytest

import ml_framework_b200

CSRC = Path(ml_framework_b200.__file__).parent / "csrc"
SOURCES = sorted(p for p in CSRC.rglob("*.cu") if re.search(r"\bmbar_wait\w*\(", p.read_text()) and re.search(r"\btma_load\w*\(", p.read_text()))


def test_there_are_such_kernels():
    assert {"paged_attn_q8.cu", "flash_fwd.cu", "gemm_tcgen05.cu"} <= {p.name for p in SOURCES}


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_copies_land_after_an_expired_wait(path):
    """Behind the last wait stands: if the abort flag is up, a bounded pause and a barrier."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    pause = r"if \([^;{}]*(?:abort_flag|s_abort)\) \{\s*const long long t0 = clock64\(\);\s*while \(clock64\(\) - t0 < \d+LL\) __nanosleep\(\d+\);\s*__syncthreads\(\);"
    found = [m.start() for m in re.finditer(pause, text)]
    assert found, f"{path.name}: no pause behind an expired wait"
    assert found[-1] > max(m.start() for m in re.finditer(r"\bmbar_wait\w*\([^;]*abort", text))
