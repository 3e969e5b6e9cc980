"""One Python function per C-ABI compute entry point, on DeviceArray operands.

Names follow the reference's operators.  Nothing here computes: each function allocates the result
buffer and forwards to libctorch_b200.so.
"""
import ctypes
import math

import numpy as np

from ._lib import lib, check
from .device import DeviceArray, _sh

OP = dict(Add=0, Sub=1, Neg=2, Mul=3, Div=4, MatMul=5, Dot=6, Cos=7, Sin=8, ReLU=11, Tanh=12, Sigmoid=13,
          Softmax=14, MSE=17, MAE=18, CE=19, Sum=21)
B_SAME, B_SCALAR, B_ROW, A_SCALAR = 0, 1, 2, 3
MODE_3XTF32, MODE_TF32, MODE_FP32_SIMT = 0, 1, 2
MODES = {"3xtf32": 0, "tf32": 1, "fp32_simt": 2}

_i64 = ctypes.c_int64
_f = ctypes.c_float


def binary(op, a, b, layout=B_SAME, out=None, stream=None):
    big = b if layout == A_SCALAR else a
    out = out or DeviceArray(big.shape)
    inner = b.size if layout == B_ROW else 1
    check(lib.ctk_binary_f32(OP[op], a.p, b.p, out.p, _i64(big.size), layout, _i64(inner), _sh(stream)))
    return out


def unary(op, a, out=None, stream=None):
    out = out or DeviceArray(a.shape)
    check(lib.ctk_unary_f32(OP[op], a.p, out.p, _i64(a.size), _sh(stream)))
    return out


def scalar(kind, a, s, out=None, stream=None):
    out = out or DeviceArray(a.shape)
    check(lib.ctk_scalar_f32(kind, a.p, _f(s), out.p, _i64(a.size), _sh(stream)))
    return out


def fill(a, value, stream=None):
    check(lib.ctk_fill_f32(a.p, _f(value), None, _i64(a.size), _sh(stream)))
    return a


def tile(src, n, stream=None):
    out = DeviceArray((n,))
    check(lib.ctk_tile_f32(src.p, _i64(src.size), out.p, _i64(n), _sh(stream)))
    return out


def unary_backward(op, x, g, stream=None):
    dx = DeviceArray(g.shape)
    check(lib.ctk_unary_backward_f32(OP[op], x.p if x is not None else None, g.p, dx.p, _i64(g.size), _sh(stream)))
    return dx


def binary_backward(op, a, b, g, layout=B_SAME, want_da=True, want_db=True, stream=None):
    da = DeviceArray(a.shape) if want_da else None
    db = DeviceArray(b.shape) if want_db else None
    inner = b.size if layout == B_ROW else 1
    check(lib.ctk_binary_backward_f32(OP[op], a.p, b.p, g.p, da.p if da else None, db.p if db else None, _i64(g.size),
                                      layout, _i64(inner), _sh(stream)))
    return da, db


def accumulate(dst, src, stream=None):
    check(lib.ctk_accumulate_f32(dst.p, src.p, _i64(dst.size), _sh(stream)))
    return dst


def sgd_update(p, g, lr, stream=None):
    check(lib.ctk_sgd_update_f32(p.p, g.p, _f(lr), _i64(p.size), _sh(stream)))
    return p


def _scalar_out():
    return DeviceArray(())


def sum(a, scratch=None, stream=None):  # noqa: A001 (mirrors Tensor::sum)
    out = _scalar_out()
    check(lib.ctk_sum_f32(a.p, _i64(a.size), out.p, scratch.p if scratch else None, _sh(stream)))
    return out


def dot(a, b, stream=None):
    out = _scalar_out()
    check(lib.ctk_dot_f32(a.p, b.p, _i64(a.size), out.p, None, _sh(stream)))
    return out


def mse(a, b, stream=None):
    out = _scalar_out()
    check(lib.ctk_mse_f32(a.p, b.p, _i64(a.size), out.p, None, _sh(stream)))
    return out


def mae(a, b, stream=None):
    out = _scalar_out()
    check(lib.ctk_mae_f32(a.p, b.p, _i64(a.size), out.p, None, _sh(stream)))
    return out


def mse_backward(p, t, g=None, stream=None):
    dp = DeviceArray(p.shape)
    check(lib.ctk_mse_backward_f32(p.p, t.p, g.p if g else None, dp.p, _i64(p.size), _sh(stream)))
    return dp


def mae_backward(p, t, g=None, stream=None):
    dp = DeviceArray(p.shape)
    check(lib.ctk_mae_backward_f32(p.p, t.p, g.p if g else None, dp.p, _i64(p.size), _sh(stream)))
    return dp


def _rc(a):
    return (1, a.shape[0]) if len(a.shape) == 1 else (a.shape[0], a.shape[1])


def softmax(x, out=None, stream=None):
    r, c = _rc(x)
    out = out or DeviceArray(x.shape)
    check(lib.ctk_softmax_rows_f32(x.p, out.p, _i64(r), _i64(c), _sh(stream)))
    return out


def softmax_backward(y, g, stream=None):
    r, c = _rc(y)
    dx = DeviceArray(y.shape)
    check(lib.ctk_softmax_backward_rows_f32(y.p, g.p, dx.p, _i64(r), _i64(c), _sh(stream)))
    return dx


def cross_entropy(logits, target, stream=None, bad_flag=None):
    """target: one-hot of logits' shape, or [rows] class indices stored as floats."""
    r, c = _rc(logits)
    out = _scalar_out()
    if target.shape == logits.shape:
        check(lib.ctk_ce_onehot_f32(logits.p, target.p, _i64(r), _i64(c), out.p, None, _sh(stream)))
    else:
        check(lib.ctk_ce_index_f32(logits.p, target.p, _i64(r), _i64(c), out.p, bad_flag.p if bad_flag else None, None, _sh(stream)))
    return out


def cross_entropy_backward(logits, onehot, g=None, stream=None):
    r, c = _rc(logits)
    d = DeviceArray(logits.shape)
    check(lib.ctk_ce_backward_f32(logits.p, onehot.p, g.p if g else None, d.p, _i64(r), _i64(c), _sh(stream)))
    return d


def cross_entropy_fused(logits, labels, stream=None, bad_flag=None):
    r, c = _rc(logits)
    out = _scalar_out()
    d = DeviceArray(logits.shape)
    check(lib.ctk_ce_fused_index_f32(logits.p, labels.p, _i64(r), _i64(c), out.p, d.p, bad_flag.p if bad_flag else None, None, _sh(stream)))
    return out, d


def matmul(a, b, ta=False, tb=False, mode=-1, out=None, workspace=None, stream=None):
    """a stored [m,k] (or [k,m] viewed through t() if ta); b stored [k,n] (or [n,k] if tb)."""
    mode = MODES.get(mode, mode)
    m, k = (a.shape[1], a.shape[0]) if ta else a.shape
    n = b.shape[0] if tb else b.shape[1]
    sa = (1, m) if ta else (k, 1)
    sb = (1, k) if tb else (n, 1)
    out = out or DeviceArray((m, n))
    check(lib.ctk_matmul_f32(a.p, b.p, out.p, _i64(m), _i64(n), _i64(k), _i64(sa[0]), _i64(sa[1]), _i64(sb[0]),
                             _i64(sb[1]), mode, workspace.p if workspace else None, _sh(stream)))
    return out


_fused_cache = {}


def matmul_fused(a, b, bias=None, relu=False, mask=None, want_split=False, ta=False, tb=False, stream=None, keep_split=False):
    """[relu](a.b + bias) * (mask > 0), the epilogue forms of the 3xTF32 product in one launch.
    Returns (c, hi, rest) when want_split (the split the epilogue wrote, decoded by _decode_split), else c.
    keep_split: write the split too, into buffers (and c) reused from call to call, and do not read it back."""
    m, k = (a.shape[1], a.shape[0]) if ta else a.shape
    n = b.shape[0] if tb else b.shape[1]
    sa = (1, m) if ta else (k, 1)
    sb = (1, k) if tb else (n, 1)
    split = None
    if keep_split:
        if (m, n) not in _fused_cache:
            _fused_cache[(m, n)] = (DeviceArray((m, n)), DeviceArray((int(lib.ctk_matmul_split_bytes(m, n)) // 4,)))
        out, split = _fused_cache[(m, n)]
    else:
        out = DeviceArray((m, n))
        if want_split:
            split = DeviceArray((int(lib.ctk_matmul_split_bytes(m, n)) // 4,))
    check(lib.ctk_matmul_3xtf32_fused_f32(a.p, b.p, out.p, _i64(m), _i64(n), _i64(k), _i64(sa[0]), _i64(sa[1]), _i64(sb[0]), _i64(sb[1]),
                                          None, None, None, None, bias.p if bias else None, int(bool(relu)), mask.p if mask else None,
                                          split.p if split else None, None, _sh(stream)))
    if not want_split:
        return out
    hi, rest = _decode_split(split, m, n, out)
    return out, hi, rest


def _decode_split(split, outer, inner, source):
    """The arrays of a split buffer as numpy: (hi, lo) as float32 [outer, inner] when the correction terms
    run on the TF32 path, (hi, bits) with bits a uint16 [2, outer, inner] array holding the bf16 patterns
    of h16 and l16 when they run on the bf16 path (see ctk_set_matmul_correction).  source: the contiguous
    [outer, inner] device array the split belongs to; where it serves as the split's hi part itself (see
    ctk_matmul_split_tag_for) hi is returned as the tensor core reads it: the low 13 mantissa bits cleared."""
    pitch = (inner + 7) // 8 * 8
    pad = (-split.ptr) % 256 // 4          # the library aligns the buffer to 256 bytes
    flat = split.numpy()
    if lib.ctk_matmul_split_tag_for(source.p, _i64(inner), _i64(inner)) >= 3:
        hi = (np.ascontiguousarray(source.numpy(), np.float32).reshape(outer, inner).view(np.uint32) & np.uint32(0xFFFFE000)).view(np.float32)
    else:
        hi = flat[pad:pad + outer * pitch].reshape(outer, pitch)[:, :inner]
    if lib.ctk_get_matmul_correction() == 0:
        return hi, flat[pad + outer * pitch:pad + 2 * outer * pitch].reshape(outer, pitch)[:, :inner]
    u16 = flat.view(np.uint16)
    o = 2 * (pad + outer * pitch)
    h16 = u16[o:o + outer * pitch].reshape(outer, pitch)[:, :inner]
    l16 = u16[o + outer * pitch:o + 2 * outer * pitch].reshape(outer, pitch)[:, :inner]
    return hi, np.stack([h16, l16])


def sgd_update_split(p, g, lr, stream=None):
    """p -= g*lr on a 2-D array and the split of the new p in the same pass; returns it as _decode_split does."""
    outer, inner = p.shape
    split = DeviceArray((int(lib.ctk_matmul_split_bytes(inner, outer)) // 4,))
    check(lib.ctk_sgd_update_split_f32(p.p, g.p, _f(lr), _i64(outer), _i64(inner), _i64(inner), split.p, _sh(stream)))
    return _decode_split(split, outer, inner, p)


# ---- orthogonalised updates and 4-bit weights -----------------------------------------------------------
# (These calls take microseconds on the device, so their way there is short: argument types are declared once, in
# _lib, and pointers and sizes go over as plain ints.)
_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(lib, name)
    return f


def _s(stream):
    return None if stream is None else _sh(stream)


_F32 = np.dtype(np.float32)
_workspaces = {}


def _matrix(a, what):
    if len(a.shape) != 2:
        raise ValueError(f"{what}: a 2-D array expected, got shape {a.shape}")
    if a.dtype != _F32:
        raise ValueError(f"{what}: a float32 array expected, got {a.dtype}")
    return a.shape


def _workspace(a, shape, what):
    if a is None:
        return None
    need = _workspaces.get(shape)
    if need is None:
        need = _workspaces[shape] = int(lib.ctk_orthogonalize_workspace_bytes(_i64(shape[0]), _i64(shape[1])))
    if a.nbytes < need:
        raise ValueError(f"{what}: a workspace of {a.nbytes} bytes, {need} needed")
    return a.ptr


def orthogonalize(g, steps=5, eps=1e-7, out=None, workspace=None, stream=None):
    """NS(g): g's singular vectors with singular values near 1 (Newton-Schulz steps)."""
    rows, cols = _matrix(g, "orthogonalize")
    if out is None:
        out = DeviceArray(g.shape)
    elif out.shape != g.shape or out.dtype != _F32:
        raise ValueError(f"orthogonalize: out has shape {out.shape} and type {out.dtype}, g {g.shape}")
    ld = cols or 1
    st = _fn("ctk_orthogonalize_f32")(g.ptr, ld, out.ptr, ld, rows, cols, steps, eps, _workspace(workspace, g.shape, "orthogonalize"), _s(stream))
    if st:
        check(st)
    return out


def orthogonalize_workspace(shape):
    """A workspace for orthogonalize / muon_update of a matrix of this shape, to be kept between calls."""
    return DeviceArray((int(lib.ctk_orthogonalize_workspace_bytes(_i64(shape[0]), _i64(shape[1]))),), np.uint8)


def muon_update(p, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=None, steps=5, eps=1e-7, workspace=None, stream=None):
    """One orthogonalised step of the weights p [in, out], in place, with its momentum m (updated in place too).
    scale: None for sqrt(max(1, out / in)), which keeps the step's effect on the layer's output alike for every shape."""
    rows, cols = _matrix(p, "muon_update")
    if g.shape != p.shape or m.shape != p.shape:
        raise ValueError(f"muon_update: shapes {p.shape}, {g.shape}, {m.shape} of weights, gradient and momentum differ")
    if g.dtype != _F32 or m.dtype != _F32:
        raise ValueError(f"muon_update: float32 arrays expected, got {g.dtype} and {m.dtype}")
    if scale is None:
        scale = math.sqrt(max(1.0, cols / max(rows, 1)))
    ld = cols or 1
    st = _fn("ctk_muon_update_f32")(p.ptr, ld, g.ptr, ld, m.ptr, ld, rows, cols, lr, momentum, 1 if nesterov else 0, weight_decay, scale, steps, eps,
                                    _workspace(workspace, p.shape, "muon_update"), _s(stream))
    if st:
        check(st)
    return p


def orthogonalize_status():
    s = ctypes.c_int()
    check(lib.ctk_orthogonalize_status(ctypes.byref(s)))
    return s.value


class W4Weight:
    """A [k, n] weight in 4 bits: packed [n, kw] uint32, scales [n, groups], zeros [n, groups] uint8 or None."""
    __slots__ = ("packed", "scales", "zeros", "k", "n", "group")

    def __init__(self, packed, scales, zeros, k, n, group):
        if group not in (32, 64, 128):
            raise ValueError("W4Weight: group must be 32, 64 or 128")
        groups = -(-k // group)
        if packed.shape != (n, groups * group // 8) or scales.shape != (n, groups) or (zeros is not None and zeros.shape != (n, groups)):
            raise ValueError("W4Weight: packed, scales and zeros do not fit k, n and group")
        if packed.dtype not in (np.uint32, np.int32) or scales.dtype != _F32 or (zeros is not None and zeros.dtype != np.uint8):
            raise ValueError("W4Weight: packed is uint32, scales float32, zeros uint8")
        self.packed, self.scales, self.zeros, self.k, self.n, self.group = packed, scales, zeros, k, n, group

    @staticmethod
    def empty(k, n, group=128, symmetric=True):
        if group not in (32, 64, 128):
            raise ValueError("W4Weight: group must be 32, 64 or 128")
        groups = -(-k // group)
        return W4Weight(DeviceArray((n, groups * group // 8), np.uint32), DeviceArray((n, groups)),
                        None if symmetric else DeviceArray((n, groups), np.uint8), k, n, group)


def w4_quantize(w, group=128, symmetric=True, out=None, stream=None):
    """The 4-bit form of w [k, n] (see ctorch_b200.h for the rounding)."""
    k, n = _matrix(w, "w4_quantize")
    if out is None:
        out = W4Weight.empty(k, n, group, symmetric)
    elif (out.k, out.n) != (k, n) or out.group != group or (out.zeros is None) != bool(symmetric):
        raise ValueError("w4_quantize: out is not a weight of this shape and form")
    st = _fn("ctk_w4_quantize_f32")(w.ptr, n or 1, k, n, group, out.packed.ptr, out.scales.ptr, None if out.zeros is None else out.zeros.ptr, _s(stream))
    if st:
        check(st)
    return out


def w4_dequantize(w4, out=None, stream=None):
    """The [k, n] values a 4-bit weight stands for."""
    if out is None:
        out = DeviceArray((w4.k, w4.n))
    elif out.shape != (w4.k, w4.n) or out.dtype != _F32:
        raise ValueError(f"w4_dequantize: out has shape {out.shape} and type {out.dtype}, the weight {(w4.k, w4.n)}")
    st = _fn("ctk_w4_dequantize_f32")(w4.packed.ptr, w4.scales.ptr, None if w4.zeros is None else w4.zeros.ptr, w4.k, w4.n, w4.group, out.ptr, w4.n or 1, _s(stream))
    if st:
        check(st)
    return out


def matmul_w4(x, w4, bias=None, relu=False, out=None, stream=None):
    """[relu](x . W + bias) for x [m, k] (or [k]) and W in 4 bits."""
    k, n, shape = w4.k, w4.n, x.shape
    if not 1 <= len(shape) <= 2 or shape[-1] != k:
        raise ValueError(f"matmul_w4: x has shape {shape}, the weight {(k, n)}")
    if x.dtype != _F32:
        raise ValueError(f"matmul_w4: float32 x expected, got {x.dtype}")
    if bias is not None and (bias.size != n or bias.dtype != _F32):
        raise ValueError(f"matmul_w4: bias of {bias.size} elements ({bias.dtype}), {n} columns")
    m = shape[0] if len(shape) == 2 else 1
    shape = shape[:-1] + (n,)
    if out is None:
        out = DeviceArray(shape)
    elif out.shape != shape or out.dtype != _F32:
        raise ValueError(f"matmul_w4: out has shape {out.shape} and type {out.dtype}, expected {shape}")
    st = _fn("ctk_w4_matmul_f32")(x.ptr, k or 1, w4.packed.ptr, w4.scales.ptr, None if w4.zeros is None else w4.zeros.ptr, None if bias is None else bias.ptr,
                                  1 if relu else 0, out.ptr, n or 1, m, k, n, w4.group, _s(stream))
    if st:
        check(st)
    return out


def w4_status():
    s = ctypes.c_int()
    check(lib.ctk_w4_status(ctypes.byref(s)))
    return s.value


CMP = {"gt": 0, "lt": 1, "eq": 2, "ge": 3, "le": 4, "ne": 5}
CMP_TENSOR, CMP_SCALAR_RIGHT, CMP_SCALAR_LEFT = 0, 1, 2
DTYPES = {0: np.float32, 1: np.float64, 2: np.int32, 3: np.int64, 4: np.uint8}   # DType values; bool as bytes


def compare(cmp, a, other, scalar_left=False, stream=None):
    """a cmp other (other a DeviceArray or a float), or other cmp a when scalar_left; bytes 0/1."""
    out = DeviceArray(a.shape, np.uint8)
    if isinstance(other, DeviceArray):
        check(lib.ctk_compare_f32(CMP[cmp], CMP_TENSOR, a.p, other.p, _f(0.0), out.p, _i64(a.size), _sh(stream)))
    else:
        form = CMP_SCALAR_LEFT if scalar_left else CMP_SCALAR_RIGHT
        check(lib.ctk_compare_f32(CMP[cmp], form, a.p, None, _f(other), out.p, _i64(a.size), _sh(stream)))
    return out


def cast(a, dtype_code, stream=None):
    out = DeviceArray(a.shape, DTYPES[dtype_code])
    check(lib.ctk_cast_f32(int(dtype_code), a.p, out.p, _i64(a.size), _sh(stream)))
    return out


def fill_dtype(out, dtype_code, value, stream=None):
    check(lib.ctk_fill_dtype(int(dtype_code), out.p, ctypes.c_double(value), _i64(out.size), _sh(stream)))
    return out


def rand_uniform(shape, seed, offset=0, out=None, stream=None):
    out = out or DeviceArray(shape)
    check(lib.ctk_rand_uniform_f32(out.p, _i64(out.size), ctypes.c_uint64(seed), ctypes.c_uint64(offset), _sh(stream)))
    return out


def matmul_path(a, b, ta=False, tb=False, mode=-1):
    mode = MODES.get(mode, mode)
    m, k = (a.shape[1], a.shape[0]) if ta else a.shape
    n = b.shape[0] if tb else b.shape[1]
    sa = (1, m) if ta else (k, 1)
    sb = (1, k) if tb else (n, 1)
    return lib.ctk_matmul_path(a.p, b.p, _i64(m), _i64(n), _i64(k), _i64(sa[0]), _i64(sa[1]), _i64(sb[0]), _i64(sb[1]), mode)


def u8_to_f32(src_u8, divisor, out=None):
    """src_u8: a DeviceArray of dtype uint8; returns float(src) / divisor."""
    out = out or DeviceArray(src_u8.shape)
    check(lib.ctk_u8_to_f32(src_u8.p, _i64(src_u8.size), ctypes.c_float(divisor), out.p, None))
    return out


def argmax_rows(x, init=float("-inf")):
    r, c = _rc(x)
    out = DeviceArray((r,))
    check(lib.ctk_argmax_rows_f32(x.p, _i64(r), _i64(c), ctypes.c_float(init), out.p, None))
    return out


def colsum(x):
    r, c = _rc(x)
    out = DeviceArray((c,))
    check(lib.ctk_colsum_f32(x.p, _i64(r), _i64(c), out.p, None))
    return out


def count_matches(a, b):
    out = _scalar_out()
    check(lib.ctk_count_matches_f32(a.p, b.p, _i64(a.size), out.p, None, None))
    return out


def rowwise_status():
    s = ctypes.c_int()
    check(lib.ctk_rowwise_status(ctypes.byref(s)))
    return s.value


def set_matmul_pairing(pairing):
    """0: 256 x 256 tiles on CTA pairs where the shape allows (default); 1: single-CTA kernel only."""
    check(lib.ctk_set_matmul_pairing(int(pairing)))


def set_matmul_correction(bf16):
    """Correction terms of the fp32-accurate mode: 0 on the TF32 path (3xTF32), 1 on the bf16 path."""
    check(lib.ctk_set_matmul_correction(int(bf16)))


def set_matmul_tail_split(on):
    check(lib.ctk_set_matmul_tail_split(int(on)))


def matmul_status():
    s = ctypes.c_int()
    check(lib.ctk_matmul_status(ctypes.byref(s)))
    return s.value
