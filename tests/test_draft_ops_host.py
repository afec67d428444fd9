"""CPU: the argument structs of the operators over drafted tokens against the
header, and their refusals (raised before any device call)."""
import ctypes as C
import os
import subprocess

import pytest

from sili__new_amd import device as dev

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"sili_draft_tree_args": dev.DraftTree, "sili_fp4_weights": dev.Fp4Weights, "sili_fp4_pack_args": dev.Fp4Pack,
           "sili_fp4_linear_args": dev.Fp4Linear, "sili_logits_constrain_args": dev.LogitsConstrain}

# addresses that no refused call reads
P = 1 << 20


def test_structs_have_the_headers_layout(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "sili_hip.h"\nint main(void) {' + "\n".join(lines)
                   + 'printf("most %d\\n", SILI_TREE_MOST); return 0; }\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            what, n = line.split()
            name, _, field = what.partition(".")
            got = dev.TREE_MOST if name == "most" else getattr(STRUCTS[name], field).offset if field else C.sizeof(STRUCTS[name])
            assert got == int(n), what


def changed(make, **kw):
    a = make()
    for k, v in kw.items():
        o = a
        *path, last = k.split("__")
        for p in path:
            o = getattr(o, p)
        setattr(o, last, v)
    return a


def tree():
    return dev.DraftTree(parents=P, q_start=2 * P, cached_lens=3 * P, requests=2, tokens=8, max_new=4, ancestors=4 * P, positions=5 * P)


@pytest.mark.parametrize("bad", [dict(requests=-1), dict(requests=1 << 26), dict(tokens=-1), dict(tokens=1 << 31), dict(max_new=-1),
                                 dict(max_new=65), dict(parents=None), dict(q_start=None), dict(cached_lens=None), dict(ancestors=None),
                                 dict(positions=None)])
def test_draft_tree_refuses(bad):
    with pytest.raises(ValueError, match="draft_tree"):
        dev.draft_tree(changed(tree, **bad))


@pytest.mark.parametrize("bad", [dict(positions=P), dict(positions=P + 28), dict(positions=2 * P + 8), dict(ancestors=P - 60), dict(ancestors=3 * P),
                                 dict(positions=4 * P + 60), dict(ancestors=5 * P - 56)])
def test_draft_tree_refuses_what_overlaps(bad):
    with pytest.raises(ValueError, match="overlap"):
        dev.draft_tree(changed(tree, **bad))


def attend():
    cache = dev.Kv4Cache(k=P, v=P, k_scale=P, v_scale=P, n_pages=4, kv_heads=2, head_dim=128, page_size=16)
    return dev.Kv4Attend(cache=cache, dtype=dev.F32, causal=1, requests=2, tokens=2, q_heads=4, q_start=P, kv_lens=P, block_table=P,
                         table_width=2, max_new=1, max_len=32, scale=1.0, q=P, out=P, q_token_stride=512, q_head_stride=128,
                         out_token_stride=512, out_head_stride=128, workspace=P, workspace_bytes=1 << 40)


@pytest.mark.parametrize("bad", [dict(cache__head_dim=96), dict(cache__page_size=8), dict(cache__k=None), dict(cache__v=P + 4), dict(dtype=3),
                                 dict(requests=65536), dict(tokens=-1), dict(q_heads=3), dict(max_new=65), dict(max_new=-1), dict(causal=0),
                                 dict(max_len=1 << 31), dict(window=-1), dict(q=None), dict(out=None), dict(q_start=None), dict(kv_lens=None),
                                 dict(block_table=None)])
def test_kv4_attend_tree_refuses(bad):
    with pytest.raises(ValueError, match="kv4_attend"):
        dev.kv4_attend_tree(changed(attend, **bad), P)


def test_kv4_attend_tree_refuses_no_masks_and_a_short_workspace():
    with pytest.raises(ValueError, match="ancestors"):
        dev.kv4_attend_tree(attend(), None)
    a = changed(attend, max_len=1 << 20, table_width=1 << 16)
    need = dev.kv4_attend_tree_workspace(a)
    assert need > 0
    for kw in (dict(workspace_bytes=need - 1), dict(workspace_bytes=need, workspace=P + 8)):
        with pytest.raises(ValueError, match="workspace"):
            dev.kv4_attend_tree(changed(lambda: a, **kw), P)
    with pytest.raises(ValueError, match="kv4_attend_tree"):
        dev.kv4_attend_tree_workspace(changed(attend, max_new=65))


def weights():
    return dev.Fp4Weights(codes=P, scales=P, n_out=48, n_in=256, group=32, codes_stride=128, scales_stride=8, scale_dtype=dev.F32)


def linear():
    return dev.Fp4Linear(w=weights(), dtype=dev.F32, out_dtype=dev.F32, tokens=3, x=P, x_stride=256, y=P, y_stride=48)


def pack():
    return dev.Fp4Pack(w=weights(), dtype=dev.F32, rows=P, row_stride=256)


WEIGHTS_BAD = [dict(w__codes=None), dict(w__scales=None), dict(w__codes=P + 8), dict(w__codes_stride=120), dict(w__codes_stride=112), dict(w__scales_stride=7), dict(w__group=16), dict(w__group=0),
               dict(w__group=256), dict(w__n_in=240), dict(w__n_in=-32), dict(w__n_in=1 << 31), dict(w__n_out=-1), dict(w__n_out=1 << 31),
               dict(w__scale_dtype=3)]


@pytest.mark.parametrize("bad", WEIGHTS_BAD + [dict(dtype=3), dict(rows=None)])
def test_fp4_pack_refuses(bad):
    with pytest.raises(ValueError, match="fp4_pack"):
        dev.fp4_pack(changed(pack, **bad))


@pytest.mark.parametrize("bad", WEIGHTS_BAD + [dict(dtype=-1), dict(out_dtype=3), dict(tokens=-1), dict(tokens=1 << 31), dict(x=None), dict(y=None)])
def test_fp4_linear_refuses(bad):
    with pytest.raises(ValueError, match="fp4_linear"):
        dev.fp4_linear(changed(linear, **bad))


def test_fp4_linear_refuses_what_no_grid_holds():
    a = changed(linear, w__n_in=1 << 30, w__codes_stride=1 << 29, w__scales_stride=1 << 25, w__n_out=1, tokens=16, workspace=P, workspace_bytes=1 << 60)
    with pytest.raises(ValueError, match="too many"):
        dev.fp4_linear(a)
    with pytest.raises(ValueError, match="too many"):
        dev.fp4_linear(changed(linear, tokens=(1 << 31) - 1, w__n_out=(1 << 31) - 1, workspace=P, workspace_bytes=1 << 62))


def test_fp4_linear_refuses_a_short_workspace():
    a = changed(linear, w__n_in=1 << 16, w__codes_stride=1 << 15, w__scales_stride=1 << 11)
    need = dev.fp4_linear_workspace(a)
    assert need > 0
    for kw in (dict(workspace=None, workspace_bytes=need), dict(workspace=P, workspace_bytes=need - 1), dict(workspace=P + 8, workspace_bytes=need)):
        with pytest.raises(ValueError, match="workspace"):
            dev.fp4_linear(changed(lambda: a, **kw))


def logits():
    return dev.LogitsConstrain(dtype=dev.F32, rows=4, vocab=100, requests=2, logits=P, logits_stride=100, out=2 * P, out_stride=100, q_start=P,
                               history=P, history_lens=P, history_stride=10, tokens=P, ancestors=P, bias=P, bias_stride=100, allow=P,
                               allow_stride=4, n_allow=2)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(rows=-1), dict(rows=1 << 31), dict(vocab=-1), dict(vocab=1 << 31), dict(requests=-1),
                                 dict(requests=1 << 31), dict(history_stride=-1), dict(history_lens=None), dict(tokens=None), dict(ancestors=None),
                                 dict(bias_stride=99), dict(bias_stride=-1), dict(allow_stride=3), dict(n_allow=-1), dict(logits=None),
                                 dict(out=None), dict(out=P, out_stride=101)])
def test_logits_constrain_refuses(bad):
    with pytest.raises(ValueError, match="logits_constrain"):
        dev.logits_constrain(changed(logits, **bad))


@pytest.mark.parametrize("bad", [dict(vocab=(1 << 31) - 8192, bias=None, allow=None), dict(history_stride=(1 << 31) - 8192)])
def test_logits_constrain_refuses_what_an_int32_cannot_step_past(bad):
    """A thread's next token or entry lies up to 8192 past the last one."""
    with pytest.raises(ValueError, match="out of range"):
        dev.logits_constrain(changed(logits, **bad))


def test_empty_calls_do_nothing():
    """No tokens, rows or outputs: nothing is launched, so nothing needs a GPU or a buffer."""
    for kw in (dict(requests=0), dict(tokens=0), dict(max_new=0)):
        dev.draft_tree(changed(tree, **kw))
    for kw in (dict(tokens=0), dict(requests=0), dict(max_new=0)):
        dev.kv4_attend_tree(changed(attend, **kw), None)
    for kw in (dict(tokens=0), dict(w__n_out=0)):
        dev.fp4_linear(changed(linear, **kw))
    for kw in (dict(w__n_in=0), dict(w__n_out=0)):
        dev.fp4_pack(changed(pack, **kw))
    for kw in (dict(rows=0), dict(vocab=0), dict(requests=0)):
        dev.logits_constrain(changed(logits, **kw))


def test_null_arguments_are_refused():
    for call in (dev.draft_tree, dev.fp4_pack, dev.fp4_linear, dev.logits_constrain):
        with pytest.raises(ValueError, match="NULL arguments"):
            call(None)
    with pytest.raises(ValueError, match="NULL arguments"):
        dev.kv4_attend_tree(None, P)
