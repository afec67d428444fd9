"""Windows that hide nothing, as the host plans them (no GPU): the workspace grows
with the splits of the axis, so it shows whether a call looks at all its keys."""
import pytest

from sili__new_amd import device as dev
from tests.test_block_ops_host import attend, changed

# lengths are int32: a window of 2^31 - 1 and more is none
WIDE = [(1 << 31) - 1, 1 << 31, (1 << 32) + 5, (1 << 63) - 64, (1 << 63) - 1]


@pytest.mark.parametrize("window", [131071, (1 << 31) - 2] + WIDE)
@pytest.mark.parametrize("dtype", [dev.F32, dev.BF16, dev.F16])
def test_a_wide_window_splits_the_axis_as_none_does(window, dtype):
    one = dict(requests=1, tokens=1, q_heads=4, cache__n_pages=9000, table_width=8192, max_len=131071, dtype=dtype)
    none = dev.kv4_attend_workspace(changed(attend, **one))
    assert none > 0
    assert dev.kv4_attend_workspace(changed(attend, window=window, **one)) == none


@pytest.mark.parametrize("window", WIDE)
def test_a_wide_window_still_needs_the_causal_mask(window):
    with pytest.raises(ValueError, match="kv4_attend"):
        dev.kv4_attend(changed(attend, window=window, causal=0))
