"""GPU: attention where what the device holds passes what the host said: the
tokens inside the batch get what they would get, nothing else is written."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests.test_gpu_kv4 import attend, check, filled, queries, starts
from tests.test_gpu_slots import build

pytestmark = pytest.mark.gpu


def short_batch(host, gpu, q, start, lens, table, tokens, **kw):
    """The call on the first `tokens` tokens of q, with the q_start of all of them."""
    full = attend(gpu, q, start, lens, table, **kw)
    check(host, full, start, lens, table)
    out = torch.full((len(q) + 2,) + q.shape[1:], 5.0, device="cuda").to(q.dtype)
    s = attend(gpu, q[:tokens], start, lens, table, max_new=int(np.max(np.diff(start))), out=out[:tokens], **kw)
    check(host, dict(s, q=q, out=torch.cat([s["out"], full["out"][tokens:]]), lse=torch.cat([s["lse"], full["lse"][tokens:]])), start, lens, table)
    assert float((out[tokens:].float() - 5.0).abs().max()) == 0


@pytest.mark.parametrize("dtype,group,new,tokens", [
    (torch.bfloat16, 5, [2], 1), (torch.bfloat16, 1, [9], 3), (torch.bfloat16, 1, [4, 30], 5), (torch.float32, 1, [5], 3), (torch.float32, 1, [7], 1),
    (torch.float16, 3, [1, 40, 2], 8), (torch.float32, 2, [3, 3, 3], 3), (torch.bfloat16, 16, [2, 2], 1)])
@pytest.mark.parametrize("n", [50, 3000])
def test_q_start_past_the_batch(hip, n, dtype, group, new, tokens):
    lens = np.array([n + 13 * r for r in range(len(new))])
    host, gpu, table = filled(lens, 2, 16, 128, n + group)
    short_batch(host, gpu, queries(sum(new), 2 * group, 128, dtype, 3), starts(new), lens, table, tokens)


def test_q_start_past_a_batch_of_long_chunks(hip):
    new, lens = np.array([300, 270, 320, 290]), np.array([300, 411, 700, 290])
    host, gpu, table = filled(lens, 48, 16, 128, 3)
    short_batch(host, gpu, queries(int(new.sum()), 48, 128, torch.bfloat16, 4), starts(new), lens, table, 1000)


def test_slots_that_leave_tokens_out_then_attention(hip):
    """request_slots leaves q_start at the total where max_tokens is less; the step goes on without a host wait."""
    old, new, page = np.array([40, 100, 7]), np.array([3, 6, 5]), 16
    host, gpu, table = filled(old + new, 1, page, 128, 8)
    step = build(old, new, page, np.zeros(0, np.int32), table, 7)
    assert step["status"].cpu().tolist() == [0, dev.SLOTS_TOKENS_FULL]
    assert step["q_start"].cpu().tolist() == [0, 3, 9, 14]
    q = queries(14, 5, 128, torch.bfloat16, 4)
    short_batch(host, gpu, q, step["q_start"].cpu().numpy(), old + new, table, 7)


@pytest.mark.parametrize("group", [2, 5])
def test_the_largest_max_new(hip, group):
    new, lens = np.array([2, 1, 3]), np.array([70, 900, 3])
    host, gpu, table = filled(lens, 2, 16, 64, 3)
    q = queries(6, 2 * group, 64, torch.float32, 5)
    s = attend(gpu, q, starts(new), lens, table, max_new=(1 << 31) - 1)
    check(host, s, starts(new), lens, table)
