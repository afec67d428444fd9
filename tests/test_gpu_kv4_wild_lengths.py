"""GPU: attention over lengths and starts that no step would write: negative,
descending, past what a table or 31 bits hold.  They hide keys or queries; every
other request keeps its results."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv4 import attend, check, filled, new_cache, queries

pytestmark = pytest.mark.gpu
MOST, LEAST = 2 ** 31 - 1, -2 ** 31


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal,window", [(1, 0), (0, 0), (1, 5), (1, 64), (1, 2 ** 31 - 2)])
def test_lengths(hip, dtype, causal, window):
    lens, new = np.array([70, 40, 50, 60, 33, 64]), np.array([2, 1, 3, 1, 2, 1])
    host, gpu, table = filled(lens, 2, 16, 64, 3, fill=0)  # what is past a length is seen here
    wild = np.array([70, LEAST, MOST, -1, MOST - 64, 64])
    start = np.concatenate([[0], np.cumsum(new)])
    q = queries(int(new.sum()), 4, 64, dtype, 5)
    for max_len in (100, MOST):
        s = attend(gpu, q, start, wild, table, causal, window, max_len=max_len)
        check(host, s, start, wild, table, causal, window, max_len=max_len)


@pytest.mark.parametrize("window", [0, 5])
def test_lengths_of_long_chunks(hip, window):
    new = np.array([300, 300, 300, 300])
    lens = np.array([300, 411, 300, 700])
    host, gpu, table = filled(lens, 48, 16, 128, 3, fill=0)
    wild = np.array([300, LEAST, MOST, 700])
    start = np.concatenate([[0], np.cumsum(new)])
    q = queries(1200, 48, 128, torch.bfloat16, 4)
    check(host, attend(gpu, q, start, wild, table, 1, window, max_len=704), start, wild, table, 1, window, max_len=704)


@pytest.mark.parametrize("group", [1, 3])
@pytest.mark.parametrize("start,left", [([0, 2, -5, 3, 3], [2, 3]), ([LEAST, 0, 2, 4, MOST], []), ([0, -10 ** 9, MOST, LEAST, 4], [0, 1, 2, 3]),
                                        ([4, 4, MOST, 0, 1], [1, 2, 3])])
def test_starts(hip, start, left, group):
    lens = np.array([30, 20, 40, 17])
    host, gpu, table = filled(lens, 1, 16, 64, 3)
    q = queries(4, group, 64, torch.float32, 5)
    s = attend(gpu, q, np.array(start), lens, table, max_new=MOST // 4)
    for t in range(4):
        untouched = float((s["out"][t] - 7.0).abs().max()) == 0 and float((s["lse"][t] - 7.0).abs().max()) == 0
        assert untouched == (t in left), t


def test_a_cache_without_pages(hip):
    """Nothing to see, and nothing is looked at."""
    _, gpu = new_cache(0, 2, 16, 64)
    q = queries(3, 2, 64, torch.bfloat16, 5)
    for window in (0, 5):
        s = attend(gpu, q, np.arange(4), np.array([LEAST, 9, MOST]), np.zeros((3, 2), int), window=window, max_len=MOST)
        assert float(s["out"].float().abs().max()) == 0 and np.isneginf(s["lse"].cpu().numpy()).all()
