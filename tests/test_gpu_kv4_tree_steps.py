"""GPU: attention of drafted tokens in a server's steps, with buffers kept from one to the next."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests.test_gpu_kv4 import filled, queries, starts
from tests.test_gpu_kv4_tree import attend, check, tree_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,group,d", [(torch.float32, 1, 128), (torch.bfloat16, 5, 128), (torch.float16, 2, 64)])
def test_one_workspace_for_every_step(hip, dtype, group, d):
    """Asked for once, for the most requests, tokens and keys: fewer are split further."""
    rng = np.random.default_rng(group)
    most, longest, requests = 20, 3000, 24
    new = np.full(requests, most)
    lens = rng.integers(most, 200, requests)
    lens[:3] = longest, 2000, 700
    host, gpu, table = filled(lens, 2, 16, d, 5)
    s = attend(gpu, queries(int(new.sum()), 2 * group, d, dtype, 3), tree_masks(rng, new), starts(new), lens, table, max_new=most, max_len=longest)
    work, size = s["work"], s["args"].workspace_bytes
    assert size > 0
    for n, upto, keys in ((1, 1, longest), (1, 20, longest), (2, 3, longest), (3, 7, 1500), (24, 2, longest), (5, 20, 300), (23, 19, longest)):
        count = rng.integers(1, upto + 1, n)
        count[0] = upto
        have = np.minimum(lens[:n], keys)
        masks = tree_masks(rng, count)
        q = queries(int(count.sum()), 2 * group, d, dtype, 4)
        s = attend(gpu, q, masks, starts(count), have, table[:n], max_new=upto, max_len=keys)
        want, a = s["out"].clone(), s["args"]
        work.fill_(255)
        s["out"].fill_(7)
        a.workspace, a.workspace_bytes = work.data_ptr(), size
        torch.cuda.synchronize()
        dev.kv4_attend_tree(a, s["masks"].data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(s["out"], want) and bool((work[size:] == 255).all())
        check(host, s, masks, starts(count), have, table[:n])


def test_a_call_that_is_not_split_needs_none(hip):
    """Enough blocks to fill the GPU: no workspace, though smaller steps would need one."""
    rng = np.random.default_rng(1)
    new, lens = np.full(70, 3), rng.integers(200, 400, 70)
    host, gpu, table = filled(lens, 8, 16, 64, 5)
    masks = tree_masks(rng, new)
    s = attend(gpu, queries(210, 8, 64, torch.bfloat16, 3), masks, starts(new), lens, table)
    a, want = s["args"], s["out"].clone()
    assert a.workspace_bytes > 0
    a.workspace, a.workspace_bytes = None, 0
    s["out"].fill_(7)
    torch.cuda.synchronize()
    dev.kv4_attend_tree(a, s["masks"].data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(s["out"], want)
