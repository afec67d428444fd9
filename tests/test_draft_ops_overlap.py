"""CPU: outputs that lie on an input or on each other are refused, before any device call."""
import pytest

from sili__new_amd import device as dev
from tests.test_draft_ops_host import P, changed, logits


@pytest.mark.parametrize("bad", [dict(out=P + 4), dict(out=P - 4), dict(out=P + 400), dict(out=P + 1596), dict(out=P - 1596), dict(out=P + 4, logits_stride=120),
                                 dict(out=P + 300, out_stride=120, logits_stride=120), dict(out=P + 1596, out_stride=-100)]
                         + [{k: 2 * P + 1596} for k in ("q_start", "history", "history_lens", "counted_from", "tokens", "ancestors", "repetition", "presence",
                                                        "frequency", "bias", "allow", "allow_row")]
                         + [dict(history=2 * P - 79), dict(tokens=2 * P - 12), dict(ancestors=2 * P - 28), dict(bias=2 * P - 796), dict(allow=2 * P - 28),
                            dict(bias=2 * P - 396, bias_stride=0)])
def test_logits_constrain(bad):
    with pytest.raises(ValueError, match="logits_constrain: out overlaps an input"):
        dev.logits_constrain(changed(logits, **bad))
