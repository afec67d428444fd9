"""The largest max_new is a bound that bounds nothing, whatever the group of query heads (no GPU)."""
import pytest

from sili__new_amd import device as dev
from tests.test_block_ops_host import attend, changed


@pytest.mark.parametrize("q_heads", [2, 4, 10, 80])
@pytest.mark.parametrize("dtype", [dev.F32, dev.BF16])
def test_no_more_workspace_than_the_batch_needs(q_heads, dtype):
    long = dict(q_heads=q_heads, dtype=dtype, cache__n_pages=9000, table_width=4096, max_len=1 << 16)
    tight = dev.kv4_attend_workspace(changed(attend, max_new=2, **long))
    assert tight > 0
    for most in (1 << 30, (1 << 31) - 1):
        assert dev.kv4_attend_workspace(changed(attend, max_new=most, **long)) == tight
