"""Expert layers in front of an index, and rows packed in 8 bits.

The products of a layer whose rows are routed in ragged groups, each group with
a matrix of its own, their gradients, the same product over rows packed in 8
bits, and activations whose input is kept packed for their backward pass. No
reference counterpart: these are the layers whose outputs an index stores.

All functions take torch tensors on the GPU, run on torch's current stream and
return without waiting; outputs are new tensors unless `out` is given. Rows may
be strided; a row's columns are contiguous. `offsets` is an int64 tensor of
groups + 1 values: group g is the rows offsets[g] to offsets[g + 1], and rows
of no group get zeros.
"""
import ctypes as C
import sys
from collections import namedtuple

from ._capi import lib as _lib

__all__ = [
    "Block8", "block8_pack", "block8_unpack", "block8_matmul", "grouped_matmul", "grouped_matmul_grad_input",
    "grouped_matmul_grad_weight", "activation_pack", "activation_grad",
]

ACTIVATIONS = {"silu": 0, "gelu": 1}


class Block8(namedtuple("Block8", ["codes", "scales", "cols"])):
    """Rows packed in 8 bits: e4m3 codes (uint8 [rows, cols rounded up to 128])
    and one power-of-two scale per block of 128 columns (uint8 [rows, blocks
    rounded up to 4]), as block8_pack lays them out."""

    __slots__ = ()

    @property
    def rows(self):
        return self.codes.shape[0]

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def _torch():
    return sys.modules["torch"]  # a caller with tensors has imported it


def _type(t, name, f32=True):
    torch = _torch()
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(t)
    if kind is None or (kind == 0 and not f32):
        raise ValueError(f"{name} must be {'float32, ' if f32 else ''}float16 or bfloat16, got {t}")
    return kind


def _matrix(t, name, dims=2):
    if not hasattr(t, "data_ptr") or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {t.dim()}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous rows")
    return t


def _same(actual, expected, what):
    from . import DimensionMismatch
    if actual != expected:
        raise DimensionMismatch(f"dimension mismatch: {what} is {actual}, expected {expected}", expected, actual)


def _packed(p, name):
    if not isinstance(p, Block8):
        raise ValueError(f"{name} must be a Block8")
    for t, what, wide in ((p.codes, "codes", _lib.pxg_block8_code_stride(p.cols)),
                          (p.scales, "scales", _lib.pxg_block8_scale_stride(p.cols))):
        if not t.is_cuda or t.dtype != _torch().uint8 or not t.is_contiguous():
            raise ValueError(f"{name}.{what} must be a contiguous uint8 GPU tensor")
        _same(tuple(t.shape), (p.codes.shape[0], wide), f"{name}.{what}'s shape")
    return p


def _groups(offsets, device):
    """(pointer or None, number of groups)"""
    if offsets is None:
        return None, 1
    if not offsets.is_cuda or offsets.dtype != _torch().int64 or offsets.dim() != 1 or not offsets.is_contiguous():
        raise ValueError("offsets must be a contiguous one-dimensional int64 GPU tensor")
    if offsets.numel() < 2:
        raise ValueError("offsets must hold at least two values")
    if offsets.device != device:
        raise ValueError("offsets must be on the operands' device")
    return offsets.data_ptr(), offsets.numel() - 1


def _out(out, shape, dtype, like, name="out"):
    if out is None:
        return like.new_empty(shape, dtype=dtype)
    _matrix(out, name, len(shape))
    _same(tuple(out.shape), tuple(shape), f"{name}'s shape")
    if out.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {out.dtype}")
    if out.device != like.device:
        raise ValueError(f"{name} must be on the operands' device")
    return out


def _stride(t):
    """Elements from row to row; a single row has none of its own."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def _call(fn, like, *others):
    """Checks that the operands share a device; a caller of fn(..., stream) on torch's current stream there."""
    from . import _check
    cuda = _torch().cuda
    device = like.device
    for t in others:
        if t.device != device:
            raise ValueError("operands must be on one device")

    def call(*args):
        if cuda.current_device() == device.index:
            _check(fn(*args, cuda.current_stream(device).cuda_stream))
        else:
            with cuda.device(device):
                _check(fn(*args, cuda.current_stream(device).cuda_stream))
    return call


def _new_packed(like, rows, cols):
    torch = _torch()
    return Block8(like.new_empty((rows, _lib.pxg_block8_code_stride(cols)), dtype=torch.uint8),
                  like.new_empty((rows, _lib.pxg_block8_scale_stride(cols)), dtype=torch.uint8), cols)


def block8_pack(x, out=None):
    """x [rows, cols] (f32, f16 or bf16) packed in 8 bits: a Block8, `out` if given."""
    _matrix(x, "x")
    kind = _type(x.dtype, "x")
    rows, cols = x.shape
    if out is None:
        out = _new_packed(x, rows, cols)
    else:
        _packed(out, "out")
        _same((out.rows, out.cols), (rows, cols), "out's shape")
    _call(_lib.pxg_block8_pack_device, x, out.codes, out.scales)(
        kind, x.data_ptr(), rows, cols, _stride(x), out.codes.data_ptr(), out.scales.data_ptr())
    return out


def block8_unpack(packed, dtype=None, out=None):
    """The values of packed rows as [rows, cols] of `dtype` (bf16 by default; exact there and in f32)."""
    _packed(packed, "packed")
    dtype = dtype or (out.dtype if out is not None else _torch().bfloat16)
    kind = _type(dtype, "dtype")
    out = _out(out, (packed.rows, packed.cols), dtype, packed.codes)
    _call(_lib.pxg_block8_unpack_device, packed.codes, packed.scales, out)(
        kind, packed.codes.data_ptr(), packed.scales.data_ptr(), packed.rows, packed.cols, out.data_ptr(),
        _stride(out))
    return out


def block8_matmul(x, w, offsets=None, out_dtype=None, out=None):
    """y[t] = x[t] w_g^T for t in group g: x a Block8 of [rows, k], w a Block8 of
    [groups * n, k] (the groups' matrices one after the other), y [rows, n] of
    out_dtype (bf16 by default, f16 or f32). Without offsets, one group."""
    _packed(x, "x")
    _packed(w, "w")
    _same(w.cols, x.cols, "w's columns")
    ptr, groups = _groups(offsets, x.codes.device)
    if w.rows % groups:
        from . import DimensionMismatch
        raise DimensionMismatch(f"dimension mismatch: w's {w.rows} rows are not a multiple of {groups} groups", groups,
                                w.rows)
    n = w.rows // groups
    dtype = out_dtype or (out.dtype if out is not None else _torch().bfloat16)
    kind = _type(dtype, "out_dtype")
    out = _out(out, (x.rows, n), dtype, x.codes)
    _call(_lib.pxg_block8_matmul_device, x.codes, x.scales, w.codes, w.scales, out)(
        x.codes.data_ptr(), x.scales.data_ptr(), x.rows, x.cols, w.codes.data_ptr(), w.scales.data_ptr(), groups, n,
        ptr, kind, out.data_ptr(), _stride(out))
    return out


def _weights(w, offsets, like):
    """(w as [groups, n, k], offsets' pointer, groups)"""
    if offsets is None and w.dim() == 2:
        w = w.unsqueeze(0)
    _matrix(w, "w", 3)
    if w.dtype != like.dtype:
        raise ValueError(f"w must be {like.dtype}, got {w.dtype}")
    ptr, groups = _groups(offsets, like.device)
    _same(w.shape[0], groups, "w's groups")
    return w, ptr, groups


def grouped_matmul(x, w, offsets=None, out_dtype=None, out=None):
    """y[t] = x[t] w[g]^T for t in group g: x [rows, k] and w [groups, n, k] in
    f16 or bf16, y [rows, n] in x's type or f32. Without offsets, one group (w
    may then be [n, k])."""
    _matrix(x, "x")
    kind = _type(x.dtype, "x", False)
    w, ptr, groups = _weights(w, offsets, x)
    _, n, k = w.shape
    _same(x.shape[1], k, "x's columns")
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    out = _out(out, (x.shape[0], n), dtype, x)
    _call(_lib.pxg_grouped_matmul_device, x, w, out)(
        kind, x.data_ptr(), x.shape[0], k, _stride(x), w.data_ptr(), groups, n, _stride(w), w.stride(0), ptr,
        _type(dtype, "out_dtype"), out.data_ptr(), _stride(out))
    return out


def grouped_matmul_grad_input(grad, w, offsets=None, out_dtype=None, out=None):
    """grouped_matmul's gradient by x: dx[t] = grad[t] w[g], grad [rows, n]."""
    _matrix(grad, "grad")
    kind = _type(grad.dtype, "grad", False)
    w, ptr, groups = _weights(w, offsets, grad)
    _, n, k = w.shape
    _same(grad.shape[1], n, "grad's columns")
    dtype = out_dtype or (out.dtype if out is not None else grad.dtype)
    out = _out(out, (grad.shape[0], k), dtype, grad)
    _call(_lib.pxg_grouped_matmul_grad_input_device, grad, w, out)(
        kind, grad.data_ptr(), grad.shape[0], n, _stride(grad), w.data_ptr(), groups, k, _stride(w), w.stride(0), ptr,
        _type(dtype, "out_dtype"), out.data_ptr(), _stride(out))
    return out


def grouped_matmul_grad_weight(grad, x, offsets, out_dtype=None, out=None):
    """grouped_matmul's gradient by w: dw[g] = the sum over t in group g of
    grad[t]^T x[t], [groups, n, k], zeros for an empty group. x is [rows, k] of
    grad's type, or a Block8 (grad is then bf16)."""
    _matrix(grad, "grad")
    kind = _type(grad.dtype, "grad", False)
    rows, n = grad.shape
    ptr, groups = _groups(offsets, grad.device)
    if ptr is None:
        raise ValueError("offsets must be given")
    dtype = out_dtype or (out.dtype if out is not None else grad.dtype)
    if isinstance(x, Block8):
        _packed(x, "x")
        _same(x.rows, rows, "x's rows")
        if grad.dtype != _torch().bfloat16:
            raise ValueError("grad must be bfloat16 with a packed x")
        k = x.cols
        out = _out(out, (groups, n, k), dtype, grad)
        _call(_lib.pxg_grouped_matmul_grad_weight_block8_device, grad, x.codes, x.scales, out)(
            grad.data_ptr(), rows, n, _stride(grad), x.codes.data_ptr(), x.scales.data_ptr(), k, ptr, groups,
            _type(dtype, "out_dtype"), out.data_ptr(), _stride(out), out.stride(0))
        return out
    _matrix(x, "x")
    if x.dtype != grad.dtype:
        raise ValueError(f"x must be {grad.dtype}, got {x.dtype}")
    _same(x.shape[0], rows, "x's rows")
    k = x.shape[1]
    out = _out(out, (groups, n, k), dtype, grad)
    _call(_lib.pxg_grouped_matmul_grad_weight_device, grad, x, out)(
        kind, grad.data_ptr(), rows, n, _stride(grad), x.data_ptr(), k, _stride(x), ptr, groups,
        _type(dtype, "out_dtype"), out.data_ptr(), _stride(out), out.stride(0))
    return out


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(sorted(ACTIVATIONS))}, got {name!r}")
    return ACTIVATIONS[name]


def activation_pack(h, activation, out=None):
    """(a, packed): a = f(h), computed from h itself, f "silu" or "gelu" (the erf
    form), and h packed in 8 bits for activation_grad."""
    which = _activation(activation)
    _matrix(h, "h")
    kind = _type(h.dtype, "h")
    rows, cols = h.shape
    out = _out(out, (rows, cols), h.dtype, h)
    packed = _new_packed(h, rows, cols)
    _call(_lib.pxg_activation_pack_device, h, out)(
        which, kind, h.data_ptr(), rows, cols, _stride(h), out.data_ptr(), _stride(out), packed.codes.data_ptr(),
        packed.scales.data_ptr())
    return out, packed


def activation_grad(grad, packed, activation, out=None):
    """dh = grad * f'(h), h the values of `packed` as activation_pack returned it."""
    which = _activation(activation)
    _matrix(grad, "grad")
    kind = _type(grad.dtype, "grad")
    _packed(packed, "packed")
    rows, cols = grad.shape
    _same((packed.rows, packed.cols), (rows, cols), "packed's shape")
    out = _out(out, (rows, cols), grad.dtype, grad)
    _call(_lib.pxg_activation_grad_device, grad, packed.codes, packed.scales, out)(
        which, kind, grad.data_ptr(), rows, cols, _stride(grad), packed.codes.data_ptr(), packed.scales.data_ptr(),
        out.data_ptr(), _stride(out))
    return out
