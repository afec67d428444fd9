"""CPU: outputs that lie on an input or on each other are refused, before any device call."""
import pytest

from sili__new_amd import device as dev
from tests.test_draft_ops_host import P, attend, changed, linear, logits, pack


@pytest.mark.parametrize("bad", [dict(out=P + 4), dict(out=P - 4), dict(out=P + 400), dict(out=P + 1596), dict(out=P - 1596), dict(out=P + 4, logits_stride=120),
                                 dict(out=P + 300, out_stride=120, logits_stride=120), dict(out=P + 1596, out_stride=-100)]
                         + [{k: 2 * P + 1596} for k in ("q_start", "history", "history_lens", "counted_from", "tokens", "ancestors", "repetition", "presence",
                                                        "frequency", "bias", "allow", "allow_row")]
                         + [dict(history=2 * P - 79), dict(tokens=2 * P - 12), dict(ancestors=2 * P - 28), dict(bias=2 * P - 796), dict(allow=2 * P - 28),
                            dict(bias=2 * P - 396, bias_stride=0)])
def test_logits_constrain(bad):
    with pytest.raises(ValueError, match="logits_constrain: out overlaps an input"):
        dev.logits_constrain(changed(logits, **bad))


def product(**kw):
    """A call that needs a workspace, its buffers apart."""
    a = changed(linear, w__n_in=1 << 16, w__codes_stride=1 << 15, w__scales_stride=1 << 11, w__codes=P << 4, w__scales=P << 5, x=P << 6, x_stride=1 << 16,
                y=P << 7, workspace=P << 8)
    a.workspace_bytes = dev.fp4_linear_workspace(a)
    return changed(lambda: a, **kw)


@pytest.mark.parametrize("bad", [dict(y=(P << 6) + 4), dict(y=(P << 6) - 572), dict(y=(P << 6) + (3 << 18) - 4), dict(y=(P << 6) + (1 << 18), tokens=2),
                                 dict(y=(P << 6) + 1024, y_stride=1 << 16), dict(y=(P << 4) + (48 << 15) - 4), dict(y=(P << 5) - 4), dict(y=(P << 5) + (48 << 13) - 4),
                                 dict(workspace=P << 6), dict(workspace=(P << 4) + 16), dict(workspace=(P << 5) - 16), dict(y=(P << 6) + (3 << 18) + 188, y_stride=-48)])
def test_fp4_linear(bad):
    with pytest.raises(ValueError, match="fp4_linear: y or the workspace overlaps an input"):
        dev.fp4_linear(product(**bad))


@pytest.mark.parametrize("at", [-572, 0, 4, 1 << 10])
def test_fp4_linear_on_its_workspace(at):
    with pytest.raises(ValueError, match="fp4_linear: y overlaps the workspace"):
        dev.fp4_linear(product(y=(P << 8) + at))


@pytest.mark.parametrize("bad", [dict(w__codes=(P << 6) + 48 * 1024 - 16), dict(w__codes=P << 6), dict(w__codes=(P << 6) - 48 * 128 + 16), dict(w__scales=P << 6),
                                 dict(w__scales=(P << 6) + 48 * 1024 - 4), dict(w__scales=(P << 6) - 48 * 32 + 4), dict(w__scales=P), dict(w__scales=P + 48 * 128 - 4),
                                 dict(w__scales=P - 48 * 32 + 4), dict(w__codes=(P << 6) + 512, w__codes_stride=1024), dict(w__scales=P + 124, w__codes_stride=160, w__scales_stride=40)])
def test_fp4_pack(bad):
    apart = changed(pack, rows=P << 6, w__scales=P << 5)
    with pytest.raises(ValueError, match="fp4_pack: outputs overlap the rows or each other"):
        dev.fp4_pack(changed(lambda: apart, **bad))


def trees(**kw):
    """A call that needs a workspace, its buffers apart."""
    a = changed(attend, max_len=1 << 20, table_width=1 << 16, cache__k=1 << 40, cache__v=2 << 40, cache__k_scale=3 << 40, cache__v_scale=4 << 40,
                q=5 << 40, out=6 << 40, lse=7 << 40, q_start=8 << 40, kv_lens=9 << 40, block_table=10 << 40, workspace=11 << 40, tokens=6, max_new=3)
    a.workspace_bytes = dev.kv4_attend_tree_workspace(a)
    return changed(lambda: a, **kw)


PAGES, SCALES, MASKS = 4 * 2 * 16 * 64, 4 * 2 * 16 * 4, 12 << 40


@pytest.mark.parametrize("written,bytes_", [("out", 6 * 4 * 128 * 4), ("lse", 6 * 4 * 4), ("workspace", 4096)])
@pytest.mark.parametrize("at,n", [(1 << 40, PAGES), (2 << 40, PAGES), (3 << 40, SCALES), (4 << 40, SCALES), (5 << 40, 6 * 4 * 128 * 4), (8 << 40, 12), (9 << 40, 8),
                                  (10 << 40, 2 << 18), (MASKS, 48)])
def test_kv4_attend_tree(written, bytes_, at, n):
    for address in (at + n - (16 if n > 16 else 0), at - bytes_ + 16, at + (16 if n > 16 else 0)):
        if n <= 16 and address >= at + n:
            address = at
        with pytest.raises(ValueError, match="kv4_attend_tree: out, lse or the workspace overlaps an input"):
            dev.kv4_attend_tree(trees(**{written: address}), MASKS)


@pytest.mark.parametrize("bad", [dict(lse=6 << 40), dict(lse=(6 << 40) + 6 * 512 * 4 - 4), dict(out=(11 << 40) - 16), dict(lse=(11 << 40) + 16),
                                 dict(out=(6 << 40) - 4, lse=(6 << 40) - 4), dict(out_token_stride=128, out_head_stride=1024, lse=(6 << 40) + 512),
                                 dict(out_token_stride=-512, lse=(6 << 40) - 2048)])
def test_kv4_attend_tree_outputs_on_each_other(bad):
    with pytest.raises(ValueError, match="kv4_attend_tree: out, lse and the workspace overlap"):
        dev.kv4_attend_tree(trees(**bad), MASKS)


@pytest.mark.parametrize("bad", [dict(out=(5 << 40) + 16), dict(out=5 << 40, out_token_stride=1024), dict(out=5 << 40, q_head_stride=132),
                                 dict(out=(5 << 40) + 1024, out_token_stride=1024, q_token_stride=1024), dict(out=(5 << 40) + 512, out_head_stride=768, q_head_stride=768, out_token_stride=128, q_token_stride=128)])
def test_kv4_attend_tree_on_q_at_another_place(bad):
    with pytest.raises(ValueError, match="kv4_attend_tree: out, lse or the workspace overlaps an input"):
        dev.kv4_attend_tree(trees(**bad), MASKS)
