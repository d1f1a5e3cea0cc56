"""What needs no torch works where there is none: the host loop with numpy alone,
and the build of the library and the server for callers in C."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

NO_TORCH = "import sys; sys.modules['torch'] = None\n"


def run(code):
    done = subprocess.run([sys.executable, "-c", NO_TORCH + code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    return done


def test_the_host_loop_needs_numpy_alone():
    run("""
import numpy as np
from cruise_b200.host_loop import first_max, host_loop_epoch, row_slot
assert first_max(np.array([0.0, 2.0, 2.0], dtype=np.float32)) == 1
""")
