"""GPU: steps whose kv_lens are the next step's cached_lens, in buffers that lie
side by side and are swapped."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 700, 5000])
def test_two_buffers_swapped(hip, n):
    rng = np.random.default_rng(n)
    page, width, steps = 16, 6, 4
    free = rng.permutation(n * width)
    table = np.full((n, width), -1)
    lens, taken = np.zeros(n, np.int64), 0
    total = 3 * n
    one = torch.zeros(2 * n + n + 1 + 2 * total + 2, dtype=torch.int32, device="cuda")
    parts = dict(zip(("a", "b", "q_start", "positions", "slots", "status"), torch.split(one, [n, n, n + 1, total, total, 2])))
    t, f = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (table, free))
    now, then = parts["a"], parts["b"]
    for _ in range(steps):
        new = rng.integers(0, 4, n)
        fresh = torch.from_numpy(new.astype(np.int32)).cuda()
        rest = f[taken:].clone()
        torch.cuda.synchronize()
        dev.request_slots(dev.RequestSlots(
            cached_lens=now.data_ptr(), new_lens=fresh.data_ptr(), requests=n, page_size=page, free_pages=rest.data_ptr(), n_free=len(rest),
            block_table=t.data_ptr(), table_width=width, max_tokens=total, kv_lens=then.data_ptr(),
            **{k: parts[k].data_ptr() for k in ("q_start", "positions", "slots", "status")}))
        torch.cuda.synchronize()
        want = ref.request_slots(lens, new, page, free[taken:], table, total)
        for name, w in want.items():
            got = {"block_table": t, "kv_lens": then}.get(name, parts.get(name))
            assert np.array_equal(got.cpu().numpy(), w), name
        lens, table, taken = lens + new, want["block_table"], taken + int(want["status"][0])
        now, then = then, now
