"""A workspace that is short by a byte, not aligned or missing is refused (no GPU)."""
import pytest

from sili__new_amd import device as dev
from tests.test_block_ops_host import P, attend, changed


@pytest.mark.parametrize("dtype", [dev.F32, dev.BF16, dev.F16])
def test_refused(dtype):
    a = changed(attend, dtype=dtype, max_len=1 << 20, table_width=1 << 16)
    need = dev.kv4_attend_workspace(a)
    assert need > 0
    for at, size in ((P, need - 1), (P + 8, need), (None, need)):
        a.workspace, a.workspace_bytes = at, size
        with pytest.raises(ValueError, match="kv4_attend: workspace"):
            dev.kv4_attend(a)
