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


def test_the_build_leaves_the_python_calls_out(tmp_path):
    done = run(f"""
from pathlib import Path
from cruise_b200 import build
build.BINDING = Path({str(tmp_path)!r}) / "_decoder_bind.so"
build._fresh = lambda target, sources: target.exists()   # the library and the server are there
compiled = []
build.build_server = lambda: compiled.append("server")
assert build.up_to_date()
assert build.build() == build.LIBRARY and not compiled
build.up_to_date = lambda: False
assert build.build() == build.LIBRARY and compiled == ["server"] and not build.BINDING.exists()
""")
    assert "_decoder_bind.so not built" in done.stderr


def test_the_build_has_the_python_calls_where_torch_is():
    from cruise_b200 import build

    assert build.binding_possible()
