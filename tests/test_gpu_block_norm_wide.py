"""GPU: norms of more than 8192 channels over more rows than the backward pass has
blocks, so that its sums over tokens go on from row to row."""
import pytest
import torch

from tests.test_gpu_block_norm import backward, check_backward, check_forward, forward, kept, scene

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,n,dtype,gate", [(257, 8193, torch.float32, "channel"), (600, 8200, torch.bfloat16, "channel"),
                                            (300, 12288, torch.float16, "token"), (513, 9001, torch.bfloat16, "none")])
@pytest.mark.parametrize("dy,dh", [(True, True), (False, True), (True, False)])
def test_many_wide_rows(hip, t, n, dtype, gate, dy, dh):
    s = scene(t, n, dtype, gate, True, True, True, n)
    check_forward(s, forward(s))
    k = kept(s)
    o = backward(s, *k, dy=dy, dh=dh)
    check_backward(s, o, *k, dy=dy, dh=dh)
    again = backward(s, *k, dy=dy, dh=dh)
    for name in ("du", "dx", "dw_post", "dw_pre"):
        assert torch.equal(o[name], again[name]), name
