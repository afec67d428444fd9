"""GPU: request slots of lengths far past the table: said in the status, and done
in the time of the table's entries, not of the pages the lengths ask for."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests.test_gpu_slots import build, same

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("requests", [3, 600, 4096, 5000])
def test_lengths_past_the_table(hip, requests):
    old, new = np.zeros(requests, np.int64), np.full(requests, MOST)
    old[1], new[1], new[-1] = 3, MOST - 3, 5
    free, width = np.arange(100, 110), 4
    table = np.full((requests, width), 7)
    got = build(old, new, 1, free, table, 9)
    want = np.full((requests, width), -1)
    want[0] = free[:4]
    want[1] = [7, 7, 7, -1]
    same(got, dict(block_table=want, status=[10, dev.SLOTS_NO_PAGE | dev.SLOTS_TABLE_FULL | dev.SLOTS_TOKENS_FULL],
                   kv_lens=old + new, positions=np.arange(9), slots=[100, 101, 102, 103] + [-1] * 5,
                   q_start=np.minimum(np.concatenate([[0], np.cumsum(new)]), MOST)))
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    dev.request_slots(got["again"], torch.cuda.current_stream().cuda_stream)
    end.record()
    torch.cuda.synchronize()
    # 2^31 pages at one a clock of every CU are 3 ms; a walk over them takes far longer
    assert begin.elapsed_time(end) < 10.0
