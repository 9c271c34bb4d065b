"""The polynomial that stands for tanh(x) / x near 0 in the attention kernels with capped
scores (csrc/chunk_rows.h), in extended precision on the host: its error is what the header
states (no GPU needed)."""
import re
from pathlib import Path

import numpy as np

HEADER = Path(__file__).resolve().parent.parent / "voom_amd" / "csrc" / "chunk_rows.h"


def test_the_polynomials_error_is_the_stated_one():
    text = HEADER.read_text()
    near = float(re.search(r"kNear = ([\d.]+)f;", text)[1])
    found = re.search(r"kTanh\[4\] = \{([^}]*)\}", text)[1].replace("f", "").split(",")
    stated = float(re.search(r"off by ([\d.e-]+) at most", text)[1])
    k = [np.longdouble(np.float32(c)) for c in found]
    x = np.linspace(1e-6, near, 1_000_001, dtype=np.longdouble)
    s = x * x
    ratio = ((k[3] * s + k[2]) * s + k[1]) * s + k[0]
    worst = np.abs(ratio * x / np.tanh(x) - 1).max()
    assert 0.95 * stated <= worst <= stated
