"""CPU: what the operators over drafted tokens ask for as workspace."""
import os
import subprocess
import sys

from sili__new_amd import device as dev
from tests.test_draft_ops_host import attend, changed, linear

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

EMPTY_LINEAR = [dict(tokens=0), dict(w__n_out=0), dict(w__n_in=0), dict(tokens=0, w__n_out=0), dict(tokens=0, w__n_in=0), dict(tokens=20, w__n_out=0),
                dict(tokens=20, w__n_in=0)]
EMPTY_TREES = [dict(tokens=0), dict(requests=0), dict(max_new=0), dict(max_len=0), dict(table_width=0), dict(cache__n_pages=0)]


def test_an_empty_call_needs_none():
    """In a process of its own: a division by zero would end it."""
    code = ("from tests.test_draft_ops_workspace import *\n"
            "for kw in EMPTY_LINEAR:\n"
            "    for dtype in (dev.F32, dev.BF16, dev.F16): assert dev.fp4_linear_workspace(changed(linear, dtype=dtype, **kw)) == 0, kw\n"
            "for kw in EMPTY_TREES:\n"
            "    for dtype in (dev.F32, dev.BF16, dev.F16): assert dev.kv4_attend_tree_workspace(changed(attend, dtype=dtype, **kw)) == 0, kw\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)
