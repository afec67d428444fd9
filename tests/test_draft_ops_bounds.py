"""CPU: bounds of the operators over drafted tokens, refused before any device call."""
import pytest

from sili__new_amd import device as dev
from tests.test_draft_ops_host import P, changed, linear, logits


@pytest.mark.parametrize("vocab", [1, 100])
@pytest.mark.parametrize("rows", [(1 << 31) - 8192, (1 << 31) - 1024, (1 << 31) - 1])
def test_logits_constrain_refuses_rows_that_an_int32_cannot_step_past(rows, vocab):
    """A block's next row lies up to 1024 past its last one."""
    with pytest.raises(ValueError, match="rows out of range"):
        dev.logits_constrain(changed(logits, rows=rows, vocab=vocab, requests=1))


@pytest.mark.parametrize("stride", [99, 1, 0, -1, -99])
def test_logits_constrain_refuses_rows_of_out_that_overlap(stride):
    for kw in (dict(), dict(out=P, logits_stride=stride)):
        with pytest.raises(ValueError, match="logits_constrain: rows of out overlap"):
            dev.logits_constrain(changed(logits, out_stride=stride, **kw))


@pytest.mark.parametrize("stride", [47, 1, 0, -1, -47])
@pytest.mark.parametrize("tokens", [2, 3, 16, 17, 300])
def test_fp4_linear_refuses_rows_of_y_that_overlap(tokens, stride):
    a = changed(linear, tokens=tokens, y=1 << 30, y_stride=stride, workspace=1 << 31, workspace_bytes=1 << 30)
    with pytest.raises(ValueError, match="fp4_linear: rows of y overlap"):
        dev.fp4_linear(a)
