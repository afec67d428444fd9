"""The operators between the layers, on device buffers.

Each function here is one entry point of include/sili_hip.h; each class is its
argument struct, with the header's field names (pointers as integers, e.g.
`tensor.data_ptr()`; unnamed fields are zero).  The header documents them:

    from sili__new_amd import device as dev
    args = dev.Rotary(dtype=dev.F32, tokens=8, ...)
    dev.rotary(args)                      # HIP's default stream
    dev.rotary(args, stream.cuda_stream)  # or another

The calls are asynchronous on their stream.  Errors raise the exceptions that
SparseLinearLayer's methods raise: ValueError, MemoryError, IndexError,
RuntimeError.  An argument struct may be kept and called again.  A program that
also uses torch imports torch before this package (torch brings a HIP runtime
of its own and finds no device next to another one).
"""
from __future__ import annotations

import ctypes as C

from . import LIB_PATH

F32, BF16, F16 = 0, 1, 2
DTYPES = {"float32": F32, "bfloat16": BF16, "float16": F16}
ROTARY_HALF, ROTARY_INTERLEAVED = 0, 1
TREE_MOST = 64
ROTARY_PLAIN, ROTARY_LINEAR, ROTARY_BANDS, ROTARY_BASE = 0, 1, 2, 3
SLOTS_NO_PAGE, SLOTS_TABLE_FULL, SLOTS_TOKENS_FULL, SLOTS_BAD_LENGTH, SLOTS_BAD_PAGE = 1, 2, 4, 8, 16

_ptr, _i32, _i64, _f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float


def _fields(text):
    """`type: name, name; type: ...` as ctypes fields."""
    kinds = {"ptr": _ptr, "i32": _i32, "i64": _i64, "f32": _f32, "size": C.c_size_t}
    out = []
    for part in text.split(";"):
        kind, names = part.split(":")
        out += [(n.strip(), kinds[kind.strip()]) for n in names.split(",")]
    return out


class RequestSlots(C.Structure):
    _fields_ = _fields("ptr: cached_lens, new_lens; i64: requests, page_size; ptr: free_pages; i64: n_free; ptr: block_table;"
                       "i64: table_width, max_tokens; ptr: q_start, kv_lens, positions, slots, status")


class Rotary(C.Structure):
    _fields_ = _fields("i32: dtype, layout, inverse; f32: scale; i64: tokens, head_dim, rot_dim, q_heads, k_heads;"
                       "ptr: positions, phase_steps, q, k; i64: q_token_stride, q_head_stride, k_token_stride, k_head_stride;"
                       "ptr: q_out, k_out; i64: q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride")


class BlockNorm(C.Structure):
    _fields_ = _fields("i32: dtype; f32: u_scale, x_scale, eps; i64: tokens, width; ptr: u, x, gate;"
                       "i64: u_stride, x_stride, gate_stride; ptr: w_post, w_pre, y, h; i64: y_stride, h_stride;"
                       "ptr: rstd_post, rstd_pre")


class BlockNormGrad(C.Structure):
    _fields_ = _fields("ptr: dy, dh; i64: dy_stride, dh_stride; ptr: du, dx, dgate; i64: du_stride, dx_stride, dgate_stride;"
                       "ptr: dw_post, dw_pre, workspace; size: workspace_bytes")


class Kv4Cache(C.Structure):
    _fields_ = _fields("ptr: k, v, k_scale, v_scale; i64: n_pages, kv_heads, head_dim, page_size")


class Kv4Rows(C.Structure):
    _fields_ = [("cache", Kv4Cache)] + _fields("i32: dtype; i64: tokens; ptr: slots, k, v;"
                                               "i64: k_token_stride, k_head_stride, v_token_stride, v_head_stride")


class Kv4Attend(C.Structure):
    _fields_ = [("cache", Kv4Cache)] + _fields("i32: dtype, causal; i64: requests, tokens, q_heads;"
                                               "ptr: q_start, kv_lens, block_table; i64: table_width, max_new, max_len, window;"
                                               "f32: scale; ptr: q; i64: q_token_stride, q_head_stride;"
                                               "ptr: out; i64: out_token_stride, out_head_stride; ptr: lse, workspace;"
                                               "size: workspace_bytes")


class DraftTree(C.Structure):
    _fields_ = _fields("ptr: parents, q_start, cached_lens; i64: requests, tokens, max_new; ptr: ancestors, positions")


class Fp4Weights(C.Structure):
    _fields_ = _fields("ptr: codes, scales; i64: n_out, n_in, group, codes_stride, scales_stride; i32: scale_dtype")


class Fp4Pack(C.Structure):
    _fields_ = [("w", Fp4Weights)] + _fields("i32: dtype; ptr: rows; i64: row_stride")


class Fp4Linear(C.Structure):
    _fields_ = [("w", Fp4Weights)] + _fields("i32: dtype, out_dtype; i64: tokens; ptr: x; i64: x_stride; ptr: y; i64: y_stride;"
                                             "ptr: workspace; size: workspace_bytes")


class LogitsConstrain(C.Structure):
    _fields_ = _fields("i32: dtype; i64: rows, vocab, requests; ptr: logits; i64: logits_stride; ptr: out; i64: out_stride;"
                       "ptr: q_start, history, history_lens; i64: history_stride; ptr: counted_from, tokens, ancestors;"
                       "ptr: repetition, presence, frequency, bias; i64: bias_stride; ptr: allow, allow_row; i64: allow_stride, n_allow")


_lib = C.CDLL(LIB_PATH)
_lib.sili_last_error.restype = C.c_char_p
_RAISES = {1: ValueError, 2: MemoryError, 4: IndexError}


def _raise(rc):
    raise _RAISES.get(rc, RuntimeError)(_lib.sili_last_error().decode())


def _call(name, *structs):
    fn = getattr(_lib, name)
    fn.argtypes = [C.POINTER(s) for s in structs] + [_ptr]

    def one(args, stream=None):
        rc = fn(args, stream)
        if rc:
            _raise(rc)

    def two(args, grads, stream=None):
        rc = fn(args, grads, stream)
        if rc:
            _raise(rc)

    call = one if len(structs) == 1 else two
    call.__name__ = call.__qualname__ = name[len("sili_"):]
    call.__doc__ = f"{name} of include/sili_hip.h, on `stream` (an address; None: HIP's default stream)."
    return call


def _bytes(name, struct):
    fn = getattr(_lib, name)
    fn.argtypes = [C.POINTER(struct), C.POINTER(C.c_size_t)]

    def call(args):
        n = C.c_size_t()
        rc = fn(args, n)
        if rc:
            _raise(rc)
        return n.value

    call.__name__ = call.__qualname__ = name[len("sili_"):]
    call.__doc__ = f"{name} of include/sili_hip.h: bytes of device workspace a call with these arguments needs."
    return call


request_slots = _call("sili_request_slots", RequestSlots)
rotary = _call("sili_rotary", Rotary)
block_norm_forward = _call("sili_block_norm_forward", BlockNorm)
block_norm_backward = _call("sili_block_norm_backward", BlockNorm, BlockNormGrad)
block_norm_workspace = _bytes("sili_block_norm_workspace", BlockNorm)
kv4_append = _call("sili_kv4_append", Kv4Rows)
kv4_read = _call("sili_kv4_read", Kv4Rows)
kv4_attend = _call("sili_kv4_attend", Kv4Attend)
kv4_attend_workspace = _bytes("sili_kv4_attend_workspace", Kv4Attend)
draft_tree = _call("sili_draft_tree", DraftTree)
kv4_attend_tree_workspace = _bytes("sili_kv4_attend_tree_workspace", Kv4Attend)
fp4_pack = _call("sili_fp4_pack", Fp4Pack)
fp4_linear = _call("sili_fp4_linear", Fp4Linear)
fp4_linear_workspace = _bytes("sili_fp4_linear_workspace", Fp4Linear)
logits_constrain = _call("sili_logits_constrain", LogitsConstrain)

_lib.sili_kv4_attend_tree.argtypes = [C.POINTER(Kv4Attend), _ptr, _ptr]


def kv4_attend_tree(args, ancestors, stream=None):
    """sili_kv4_attend_tree of include/sili_hip.h: `ancestors` the address of the tokens' masks, on `stream`."""
    rc = _lib.sili_kv4_attend_tree(args, ancestors, stream)
    if rc:
        _raise(rc)


_lib.sili_rotary_steps.argtypes = [_i64, C.c_double, C.c_int] + [C.c_double] * 4 + [_ptr, C.POINTER(_f32)]


def rotary_steps(rot_dim, base=10000.0, scaling=ROTARY_PLAIN, factor=1.0, original_len=0.0, low=1.0, high=32.0):
    """sili_rotary_steps: (phase steps as a numpy uint64 array, scale)."""
    import numpy as np

    steps, scale = np.zeros(max(0, int(rot_dim)) // 2, np.uint64), _f32()
    rc = _lib.sili_rotary_steps(int(rot_dim), base, scaling, factor, original_len, low, high, steps.ctypes.data, scale)
    if rc:
        _raise(rc)
    return steps, scale.value
