"""request_slots refuses outputs on its inputs or on each other (raised before any device call)."""
import pytest

from sili__new_amd import device as dev

SIZES = dict(cached_lens=8, new_lens=8, free_pages=5, block_table=8 * 4, q_start=9, kv_lens=8, positions=20, slots=20, status=2)
READ = ("cached_lens", "new_lens", "free_pages")


def apart():
    at = {name: (1 << 20) + (i << 12) for i, name in enumerate(SIZES)}
    return dev.RequestSlots(requests=8, page_size=16, n_free=5, table_width=4, max_tokens=20, **at)


@pytest.mark.parametrize("a", SIZES)
@pytest.mark.parametrize("b", SIZES)
def test_overlap_is_refused(a, b):
    if a == b or (a in READ and b in READ):
        return
    s = apart()
    for at in (getattr(s, b), getattr(s, b) - 4 * SIZES[a] + 4, getattr(s, b) + 4 * SIZES[b] - 4):
        setattr(s, a, at)
        with pytest.raises(ValueError, match="request_slots: .*overlap"):
            dev.request_slots(s)


def test_a_table_of_any_width_is_measured():
    s = apart()
    s.table_width = (1 << 63) - 1
    with pytest.raises(ValueError, match="request_slots: .*overlap"):
        dev.request_slots(s)
