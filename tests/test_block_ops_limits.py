"""Refusals of sizes whose products pass 64 or 32 bits, and of grids that no
launch could have (no GPU)."""
import pytest

from sili__new_amd import device as dev
from tests.test_block_ops_host import attend, changed, kv_rows, rotary

HUGE = [dict(cache__n_pages=1 << 60), dict(cache__n_pages=(1 << 62) + 1), dict(cache__n_pages=(1 << 27) + 1)]


@pytest.mark.parametrize("bad", HUGE + [dict(tokens=1 << 31), dict(tokens=(1 << 31) - 1)])
def test_kv4_rows_refuse(bad):
    for call in (dev.kv4_append, dev.kv4_read):
        with pytest.raises(ValueError, match="kv4"):
            call(changed(kv_rows, **bad))


@pytest.mark.parametrize("bad", HUGE + [dict(max_new=1 << 62), dict(max_len=1 << 62), dict(table_width=1 << 60), dict(tokens=1 << 31),
                                        dict(tokens=1 << 29, max_new=1 << 29)])
def test_kv4_attend_refuses(bad):
    with pytest.raises(ValueError, match="kv4_attend"):
        dev.kv4_attend(changed(attend, **bad))


@pytest.mark.parametrize("bad", [dict(tokens=1 << 60), dict(tokens=(1 << 31) - 1, rot_dim=64), dict(q_heads=(1 << 63) - 1)])
def test_rotary_refuses(bad):
    with pytest.raises(ValueError, match="rotary"):
        dev.rotary(changed(rotary, **bad))


def test_bounds_beyond_the_table_ask_for_no_more_workspace():
    """max_len and max_new bound the work; a table and a batch that hold less bound it too."""
    tight = changed(attend, max_len=32, max_new=2)
    loose = changed(attend, max_len=(1 << 31) - 1, max_new=(1 << 30) - 1)
    assert dev.kv4_attend_workspace(loose) == dev.kv4_attend_workspace(tight)
