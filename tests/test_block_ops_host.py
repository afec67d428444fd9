"""CPU: the argument structs of sili__new_amd.device against the header, the
refusals of the operators between the layers (raised before any device call),
and the rotary phase steps."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from sili__new_amd import device as dev

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"sili_request_slots_args": dev.RequestSlots, "sili_rotary_args": dev.Rotary, "sili_block_norm_args": dev.BlockNorm,
           "sili_block_norm_grads": dev.BlockNormGrad, "sili_kv4_cache": dev.Kv4Cache, "sili_kv4_rows_args": dev.Kv4Rows,
           "sili_kv4_attend_args": dev.Kv4Attend}


def test_structs_have_the_headers_layout(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "sili_hip.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", f"-I{ROOT}/include", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            what, n = line.split()
            name, _, field = what.partition(".")
            got = getattr(STRUCTS[name], field).offset if field else C.sizeof(STRUCTS[name])
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


# addresses that no refused call reads
P = 1 << 20


def slots():
    return dev.RequestSlots(cached_lens=P, new_lens=P, requests=2, page_size=16, free_pages=P, n_free=4, block_table=P, table_width=4,
                            max_tokens=8, q_start=P, kv_lens=P, positions=P, slots=P, status=P)


@pytest.mark.parametrize("bad", [dict(requests=-1), dict(page_size=0), dict(page_size=1 << 31), dict(n_free=-1), dict(table_width=-1),
                                 dict(max_tokens=-1), dict(max_tokens=(1 << 31) - 1), dict(cached_lens=None), dict(new_lens=None),
                                 dict(kv_lens=None), dict(block_table=None), dict(free_pages=None), dict(positions=None),
                                 dict(slots=None), dict(q_start=None), dict(status=None)])
def test_request_slots_refuses(bad):
    with pytest.raises(ValueError, match="request_slots"):
        dev.request_slots(changed(slots, **bad))


def rotary():
    return dev.Rotary(dtype=dev.F32, tokens=2, head_dim=64, rot_dim=32, q_heads=2, k_heads=1, positions=P, phase_steps=P, scale=1.0,
                      q=P, k=P, q_out=P, k_out=P, q_token_stride=128, q_head_stride=64, k_token_stride=64, k_head_stride=64,
                      q_out_token_stride=128, q_out_head_stride=64, k_out_token_stride=64, k_out_head_stride=64)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(layout=2), dict(tokens=-1), dict(head_dim=0), dict(head_dim=1 << 20), dict(rot_dim=33),
                                 dict(rot_dim=66), dict(rot_dim=-2), dict(q_heads=-1), dict(k_heads=-1), dict(q_heads=65536),
                                 dict(positions=None), dict(phase_steps=None), dict(q=None), dict(k=None), dict(q_out=None),
                                 dict(k_out=None)])
def test_rotary_refuses(bad):
    with pytest.raises(ValueError, match="rotary"):
        dev.rotary(changed(rotary, **bad))


def norm():
    return dev.BlockNorm(dtype=dev.BF16, tokens=2, width=64, u=P, x=P, y=P, h=P, w_post=P, w_pre=P, gate=P, rstd_post=P, rstd_pre=P,
                         u_stride=64, x_stride=64, y_stride=64, h_stride=64, eps=1e-5, u_scale=1.0, x_scale=1.0)


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(width=0), dict(width=32769), dict(u=None),
                                 dict(y=None), dict(h=None)])
def test_block_norm_refuses(bad):
    with pytest.raises(ValueError, match="block_norm_forward"):
        dev.block_norm_forward(changed(norm, **bad))


def grads():
    return dev.BlockNormGrad(dy=P, dh=P, dy_stride=64, dh_stride=64, du=P, dx=P, du_stride=64, dx_stride=64, dgate=P, dw_post=P, dw_pre=P,
                             workspace=P, workspace_bytes=1 << 30)


@pytest.mark.parametrize("bad_args,bad_grads", [
    (dict(dtype=7), {}), (dict(width=0), {}), (dict(u=None), {}), (dict(y=None), {}), (dict(rstd_post=None), {}), (dict(rstd_pre=None), {}),
    (dict(w_pre=None), {}), (dict(gate=None), {}), (dict(gate_stride=64), {}), (dict(), dict(dgate_stride=64)),
    (dict(w_post=None), {}), (dict(), dict(workspace=None)), (dict(), dict(workspace_bytes=8))])
def test_block_norm_backward_refuses(bad_args, bad_grads):
    with pytest.raises(ValueError, match="block_norm_backward"):
        dev.block_norm_backward(changed(norm, **bad_args), changed(grads, **bad_grads))


def cache():
    return dev.Kv4Cache(k=P, v=P, k_scale=P, v_scale=P, n_pages=4, kv_heads=2, head_dim=128, page_size=16)


def kv_rows():
    return dev.Kv4Rows(cache=cache(), dtype=dev.F16, tokens=3, slots=P, k=P, v=P)


CACHE_BAD = [dict(cache__head_dim=96), dict(cache__head_dim=0), dict(cache__page_size=8), dict(cache__page_size=24), dict(cache__kv_heads=0),
             dict(cache__n_pages=-1), dict(cache__n_pages=1 << 28), dict(cache__k=None), dict(cache__v=None), dict(cache__k_scale=None),
             dict(cache__v_scale=None), dict(cache__k=P + 8), dict(cache__v=P + 4), dict(cache__v_scale=P + 4)]


@pytest.mark.parametrize("bad", CACHE_BAD + [dict(dtype=5), dict(tokens=-1), dict(slots=None), dict(k=None), dict(v=None)])
def test_kv4_rows_refuse(bad):
    for call in (dev.kv4_append, dev.kv4_read):
        with pytest.raises(ValueError, match="kv4"):
            call(changed(kv_rows, **bad))


def attend():
    return dev.Kv4Attend(cache=cache(), dtype=dev.F32, causal=1, requests=2, tokens=2, q_heads=4, q_start=P, kv_lens=P, block_table=P,
                         table_width=2, max_new=1, max_len=32, scale=1.0, q=P, out=P, q_token_stride=512, q_head_stride=128,
                         out_token_stride=512, out_head_stride=128, workspace=P, workspace_bytes=1 << 40)


@pytest.mark.parametrize("bad", CACHE_BAD + [dict(dtype=3), dict(requests=-1), dict(requests=65536), dict(tokens=-1), dict(q_heads=3),
                                             dict(q_heads=0), dict(table_width=-1), dict(max_new=-1), dict(max_len=-1), dict(max_len=1 << 31),
                                             dict(window=-1), dict(window=4, causal=0), dict(q=None), dict(out=None), dict(q_start=None),
                                             dict(kv_lens=None), dict(block_table=None)])
def test_kv4_attend_refuses(bad):
    with pytest.raises(ValueError, match="kv4_attend"):
        dev.kv4_attend(changed(attend, **bad))


def test_a_short_workspace_is_refused():
    a = changed(attend, max_len=1 << 20, table_width=1 << 16)
    need = dev.kv4_attend_workspace(a)
    if need:
        a.workspace_bytes = need - 1
        with pytest.raises(ValueError, match="workspace"):
            dev.kv4_attend(a)
        a.workspace_bytes, a.workspace = need, P + 8
        with pytest.raises(ValueError, match="workspace"):
            dev.kv4_attend(a)


def test_empty_calls_do_nothing():
    """No tokens: nothing is launched, so nothing needs a GPU or a buffer."""
    dev.rotary(dev.Rotary(head_dim=64, rot_dim=64))
    dev.block_norm_forward(dev.BlockNorm(width=8))
    dev.block_norm_backward(dev.BlockNorm(width=8), dev.BlockNormGrad())
    dev.kv4_append(changed(kv_rows, tokens=0))
    dev.kv4_attend(changed(attend, tokens=0))
    dev.kv4_attend(changed(attend, requests=0))


def test_null_arguments_are_refused():
    for call in (dev.request_slots, dev.rotary, dev.block_norm_forward, dev.kv4_append, dev.kv4_read, dev.kv4_attend):
        with pytest.raises(ValueError, match="NULL arguments"):
            call(None)


@pytest.mark.parametrize("rot", [2, 64, 128])
@pytest.mark.parametrize("scaling,factor", [(dev.ROTARY_PLAIN, 1.0), (dev.ROTARY_LINEAR, 4.0), (dev.ROTARY_BANDS, 8.0), (dev.ROTARY_BASE, 2.0)])
def test_rotary_steps(rot, scaling, factor):
    if scaling == dev.ROTARY_BASE and rot == 2:
        with pytest.raises(ValueError):
            dev.rotary_steps(rot, 10000.0, scaling, factor)
        return
    steps, scale = dev.rotary_steps(rot, 10000.0, scaling, factor, 8192.0, 1.0, 32.0)
    base = 10000.0 * factor ** (rot / (rot - 2)) if scaling == dev.ROTARY_BASE else 10000.0
    turns = base ** (-np.arange(0, rot, 2) / rot) / (2 * np.pi)
    if scaling == dev.ROTARY_LINEAR:
        turns = turns / factor
    if scaling == dev.ROTARY_BANDS:
        keep = np.clip((8192 * turns - 1) / 31, 0, 1)
        turns = turns * ((1 - keep) / factor + keep)
    # pow of two libraries: a few units of 2^-52
    assert np.allclose(steps.astype(np.float64) / 2.0 ** 64, turns, rtol=1e-13, atol=2.0 ** -64)
    assert scale == pytest.approx(0.1 * np.log(factor) + 1 if scaling == dev.ROTARY_BANDS else 1.0, rel=1e-6)


@pytest.mark.parametrize("bad", [dict(rot_dim=3), dict(rot_dim=-2), dict(base=1.0), dict(base=float("inf")), dict(scaling=4),
                                 dict(scaling=1, factor=0.5), dict(scaling=1, factor=float("nan")), dict(scaling=2, factor=2.0),
                                 dict(scaling=2, factor=2.0, original_len=4096.0, low=3.0, high=3.0)])
def test_rotary_steps_refuses(bad):
    with pytest.raises(ValueError, match="rotary_steps"):
        dev.rotary_steps(**{"rot_dim": 8, **bad})
