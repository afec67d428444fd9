"""GPU: attention under windows that hide nothing, equal to no window at all."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv4 import attend, check, filled, queries, starts
from tests.test_kv4_window import WIDE

pytestmark = pytest.mark.gpu


def same_as_none(host, gpu, q, new, lens, table, windows=WIDE):
    none = attend(gpu, q, starts(new), lens, table)
    check(host, none, starts(new), lens, table)
    for window in windows:
        s = attend(gpu, q, starts(new), lens, table, window=window)
        assert torch.equal(s["out"], none["out"]) and torch.equal(s["lse"], none["lse"]), window


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_long_axis(hip, dtype):
    lens = np.array([5000, 3])
    host, gpu, table = filled(lens, 2, 16, 64, 1)
    same_as_none(host, gpu, queries(2, 4, 64, dtype, 5), [1, 1], lens, table)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_new_tokens_than_keys(hip, dtype):
    """Rows before the first key share a tile with rows that see some."""
    new, lens = np.array([9, 3, 30]), np.array([4, 0, 29])
    host, gpu, table = filled(lens, 1, 16, 128, 1)
    same_as_none(host, gpu, queries(42, 2, 128, dtype, 2), new, lens, table)
    # the largest window that is kept as one
    wide = attend(gpu, queries(42, 2, 128, dtype, 2), starts(new), lens, table, window=(1 << 31) - 2)
    check(host, wide, starts(new), lens, table)


def test_blocks_of_many_rows(hip):
    new, lens = np.array([300, 290, 257, 320]), np.array([290, 411, 257, 700])
    host, gpu, table = filled(lens, 64, 16, 128, 3)
    q = queries(int(new.sum()), 64, 128, torch.bfloat16, 4)
    none = attend(gpu, q, starts(new), lens, table)
    for window in WIDE + [(1 << 31) - 2]:
        s = attend(gpu, q, starts(new), lens, table, window=window)
        assert torch.equal(s["out"], none["out"]) and torch.equal(s["lse"], none["lse"]), window
