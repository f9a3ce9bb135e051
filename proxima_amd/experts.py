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

None of them records history for autograd: the gradients are functions of their
own. An operand that requires grad is refused while grad mode is on, so that no
gradient is lost unseen; inside torch.no_grad() and a torch.autograd.Function
it is off.
"""
import sys

from . import DimensionMismatch, _check
from ._capi import lib as _lib

__all__ = [
    "Block8", "block8_pack", "block8_unpack", "block8_matmul", "grouped_matmul", "grouped_matmul_grad_input",
    "grouped_matmul_grad_weight", "activation_pack", "activation_grad",
]

ACTIVATIONS = {"silu": 0, "gelu": 1}


class Block8:
    """Rows packed in 8 bits, as block8_pack lays them out: e4m3 codes (uint8
    [rows, cols rounded up to 128], contiguous) and one power-of-two scale per
    block of 128 columns (uint8 [rows, blocks rounded up to 4])."""

    __slots__ = ("_codes", "_scales", "_cols")

    def __init__(self, codes, scales, cols):
        if _torch is None:
            _setup()
        for t, what in ((codes, "codes"), (scales, "scales")):
            if not t.is_cuda or t.dtype is not _torch.uint8 or not t.is_contiguous():
                raise ValueError(f"{what} must be a contiguous uint8 GPU tensor")
        if cols < 1:
            raise ValueError("cols must be at least 1")
        wide, few = _strides(cols)
        rows = codes.shape[0]
        if codes.shape != (rows, wide):
            _mismatch(tuple(codes.shape), (rows, wide), "codes' shape")
        if scales.shape != (rows, few):
            _mismatch(tuple(scales.shape), (rows, few), "scales' shape")
        self._codes, self._scales, self._cols = codes, scales, cols

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    cols = property(lambda self: self._cols)
    rows = property(lambda self: self._codes.shape[0])

    def nbytes(self):
        return self._codes.numel() + self._scales.numel()

    def __repr__(self):
        return f"Block8({self.rows} x {self.cols})"


# torch is the caller's: this package does not import it by itself. Filled on the first call with a tensor.
_KINDS = {}  # torch dtype -> pxg_type
_torch = _current_device = _current_stream = None


def _setup():
    global _torch, _current_device, _current_stream
    _torch = sys.modules["torch"]
    _current_device, _current_stream = _torch._C._cuda_getDevice, _torch._C._cuda_getCurrentRawStream
    _KINDS.update({_torch.float32: 0, _torch.float16: 1, _torch.bfloat16: 2})


def _type(dtype, name, f32=True):
    if _torch is None:
        _setup()
    kind = _KINDS.get(dtype)
    if kind is None or (kind == 0 and not f32):
        raise ValueError(f"{name} must be {'float32, ' if f32 else ''}float16 or bfloat16, got {dtype}")
    return kind


def _matrix(t, name, dims=2):
    """Checks a GPU tensor of contiguous rows; its shape."""
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{name} must be a GPU tensor")
    shape = t.shape
    if len(shape) != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {len(shape)}")
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous rows")
    return shape


def _mismatch(actual, expected, what):
    raise DimensionMismatch(f"dimension mismatch: {what} is {actual}, expected {expected}", expected, actual)


def _strides(cols):
    """Bytes from row to row of a Block8's codes and scales."""
    blocks = (cols + 127) >> 7
    return blocks << 7, (blocks + 3) & ~3


def _packed(p, name):
    """(codes, scales, rows, cols) of a Block8."""
    if type(p) is not Block8:
        raise ValueError(f"{name} must be a Block8")
    codes = p._codes
    return codes, p._scales, codes.shape[0], p._cols


def _groups(offsets):
    """(pointer or None, number of groups)"""
    if offsets is None:
        return None, 1
    if _torch is None:
        _setup()
    if not offsets.is_cuda or offsets.dtype is not _torch.int64 or offsets.dim() != 1 or not offsets.is_contiguous():
        raise ValueError("offsets must be a contiguous one-dimensional int64 GPU tensor")
    n = offsets.shape[0]
    if n < 2:
        raise ValueError("offsets must hold at least two values")
    return offsets.data_ptr(), n - 1


def _out(out, shape, dtype, like):
    """(tensor, elements from row to row)"""
    if out is None:
        return like.new_empty(shape, dtype=dtype), shape[-1]
    if _matrix(out, "out", len(shape)) != shape:
        _mismatch(tuple(out.shape), tuple(shape), "out's shape")
    if out.dtype is not dtype:
        raise ValueError(f"out must be {dtype}, got {out.dtype}")
    return out, _stride(out)


def _stride(t):
    """Elements from row to row; a single row has none of its own."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def _run(fn, tensors, *args):
    """fn(*args, stream) on torch's current stream of the device that all tensors share."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None:
            if t.get_device() != device:
                raise ValueError("operands must be on one device")
            if t.requires_grad and _torch.is_grad_enabled():
                raise ValueError("an operand requires grad, but no history is recorded here: call the gradients' own "
                                 "functions, under torch.no_grad() or from a torch.autograd.Function")
    if _current_device() == device:
        status = fn(*args, _current_stream(device))
    else:
        with _torch.cuda.device(device):
            status = fn(*args, _current_stream(device))
    if status:
        _check(status)


def _new_packed(like, rows, cols):
    wide, few = _strides(cols)
    p = Block8.__new__(Block8)
    p._codes = like.new_empty((rows, wide), dtype=_torch.uint8)
    p._scales = like.new_empty((rows, few), dtype=_torch.uint8)
    p._cols = cols
    return p


def block8_pack(x, out=None):
    """x [rows, cols] (f32, f16 or bf16) packed in 8 bits: a Block8, `out` if given."""
    rows, cols = _matrix(x, "x")
    kind = _type(x.dtype, "x")
    if out is None:
        out = _new_packed(x, rows, cols)
    codes, scales, prows, pcols = _packed(out, "out")
    if prows != rows or pcols != cols:
        _mismatch((prows, pcols), (rows, cols), "out's shape")
    _run(_lib.pxg_block8_pack_device, (x, codes, scales), kind, x.data_ptr(), rows, cols, _stride(x),
         codes.data_ptr(), scales.data_ptr())
    return out


def block8_unpack(packed, dtype=None, out=None):
    """The values of packed rows as [rows, cols] of `dtype` (bf16 by default; exact there and in f32)."""
    codes, scales, rows, cols = _packed(packed, "packed")
    dtype = dtype or (out.dtype if out is not None else _torch.bfloat16)
    kind = _type(dtype, "dtype")
    out, stride = _out(out, (rows, cols), dtype, codes)
    _run(_lib.pxg_block8_unpack_device, (codes, scales, out), kind, codes.data_ptr(), scales.data_ptr(), rows, cols,
         out.data_ptr(), stride)
    return out


def block8_matmul(x, w, offsets=None, out_dtype=None, out=None):
    """y[t] = x[t] w_g^T for t in group g: x a Block8 of [rows, k], w a Block8 of
    [groups * n, k] (the groups' matrices one after the other), y [rows, n] of
    out_dtype (bf16 by default, f16 or f32). Without offsets, one group.

    f32 results are exact products summed in f32. Those of 16 bits are
    multiplied in 8 bits on the matrix cores where that is faster; these cut
    each product of eight neighbouring columns below 2^-13 of the eight's
    largest power of two and sum the eights in f32. That costs 1.5e-5 to 8e-5 of
    the result as a whole, where rounding costs 2e-4 (f16) or 1.7e-3 (bf16); a
    sum that cancels may be off by more of itself."""
    codes, scales, rows, k = _packed(x, "x")
    wcodes, wscales, wrows, wk = _packed(w, "w")
    if wk != k:
        _mismatch(wk, k, "w's columns")
    ptr, groups = _groups(offsets)
    n, left = divmod(wrows, groups)
    if left:
        raise DimensionMismatch(f"dimension mismatch: w's {wrows} rows are not a multiple of {groups} groups", groups,
                                wrows)
    dtype = out_dtype or (out.dtype if out is not None else _torch.bfloat16)
    kind = _type(dtype, "out_dtype")
    out, stride = _out(out, (rows, n), dtype, codes)
    _run(_lib.pxg_block8_matmul_device, (codes, scales, wcodes, wscales, offsets, out), codes.data_ptr(),
         scales.data_ptr(), rows, k, wcodes.data_ptr(), wscales.data_ptr(), groups, n, ptr, kind, out.data_ptr(),
         stride)
    return out


def _weights(w, offsets, like):
    """(w as [groups, n, k], offsets' pointer, groups, n, k)"""
    if offsets is None and w.dim() == 2:
        w = w.unsqueeze(0)
    g, n, k = _matrix(w, "w", 3)
    if w.dtype is not like.dtype:
        raise ValueError(f"w must be {like.dtype}, got {w.dtype}")
    ptr, groups = _groups(offsets)
    if g != groups:
        _mismatch(g, groups, "w's groups")
    return w, ptr, groups, n, k


def grouped_matmul(x, w, offsets=None, out_dtype=None, out=None):
    """y[t] = x[t] w[g]^T for t in group g: x [rows, k] and w [groups, n, k] in
    f16 or bf16, y [rows, n] in x's type or f32. Without offsets, one group (w
    may then be [n, k])."""
    rows, xk = _matrix(x, "x")
    kind = _type(x.dtype, "x", False)
    w, ptr, groups, n, k = _weights(w, offsets, x)
    if xk != k:
        _mismatch(xk, k, "x's columns")
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    out, stride = _out(out, (rows, n), dtype, x)
    _run(_lib.pxg_grouped_matmul_device, (x, w, offsets, out), kind, x.data_ptr(), rows, k, _stride(x), w.data_ptr(),
         groups, n, _stride(w), w.stride(0), ptr, _type(dtype, "out_dtype"), out.data_ptr(), stride)
    return out


def grouped_matmul_grad_input(grad, w, offsets=None, out_dtype=None, out=None):
    """grouped_matmul's gradient by x: dx[t] = grad[t] w[g], grad [rows, n]."""
    rows, gn = _matrix(grad, "grad")
    kind = _type(grad.dtype, "grad", False)
    w, ptr, groups, n, k = _weights(w, offsets, grad)
    if gn != n:
        _mismatch(gn, n, "grad's columns")
    dtype = out_dtype or (out.dtype if out is not None else grad.dtype)
    out, stride = _out(out, (rows, k), dtype, grad)
    _run(_lib.pxg_grouped_matmul_grad_input_device, (grad, w, offsets, out), kind, grad.data_ptr(), rows, n,
         _stride(grad), w.data_ptr(), groups, k, _stride(w), w.stride(0), ptr, _type(dtype, "out_dtype"),
         out.data_ptr(), stride)
    return out


def grouped_matmul_grad_weight(grad, x, offsets, out_dtype=None, out=None):
    """grouped_matmul's gradient by w: dw[g] = the sum over t in group g of
    grad[t]^T x[t], [groups, n, k], zeros for an empty group. x is [rows, k] of
    grad's type, or a Block8 (grad is then bf16)."""
    rows, n = _matrix(grad, "grad")
    kind = _type(grad.dtype, "grad", False)
    ptr, groups = _groups(offsets)
    if ptr is None:
        raise ValueError("offsets must be given")
    dtype = out_dtype or (out.dtype if out is not None else grad.dtype)
    out_kind = _type(dtype, "out_dtype")
    if isinstance(x, Block8):
        codes, scales, xrows, k = _packed(x, "x")
        if kind != 2:
            raise ValueError("grad must be bfloat16 with a packed x")
    else:
        xrows, k = _matrix(x, "x")
        if x.dtype is not grad.dtype:
            raise ValueError(f"x must be {grad.dtype}, got {x.dtype}")
    if xrows != rows:
        _mismatch(xrows, rows, "x's rows")
    out, stride = _out(out, (groups, n, k), dtype, grad)
    size = _lib.pxg_grouped_matmul_grad_weight_workspace(rows, n, k, groups)
    space = grad.new_empty(size, dtype=_torch.uint8) if size else None
    at = space.data_ptr() if size else None
    if isinstance(x, Block8):
        _run(_lib.pxg_grouped_matmul_grad_weight_block8_device, (grad, codes, scales, offsets, out), grad.data_ptr(),
             rows, n, _stride(grad), codes.data_ptr(), scales.data_ptr(), k, ptr, groups, out_kind, out.data_ptr(),
             stride, out.stride(0), at, size)
    else:
        _run(_lib.pxg_grouped_matmul_grad_weight_device, (grad, x, offsets, out), kind, grad.data_ptr(), rows, n,
             _stride(grad), x.data_ptr(), k, _stride(x), ptr, groups, out_kind, out.data_ptr(), stride, out.stride(0),
             at, size)
    return out


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(sorted(ACTIVATIONS))}, got {name!r}")
    return ACTIVATIONS[name]


def activation_pack(h, activation, out=None):
    """(a, packed): a = f(h), computed from h itself, f "silu" or "gelu" (the erf
    form), and h packed in 8 bits for activation_grad."""
    which = _activation(activation)
    rows, cols = _matrix(h, "h")
    kind = _type(h.dtype, "h")
    out, stride = _out(out, (rows, cols), h.dtype, h)
    packed = _new_packed(h, rows, cols)
    codes, scales = packed._codes, packed._scales
    _run(_lib.pxg_activation_pack_device, (h, out), which, kind, h.data_ptr(), rows, cols, _stride(h), out.data_ptr(),
         stride, codes.data_ptr(), scales.data_ptr())
    return out, packed


def activation_grad(grad, packed, activation, out=None):
    """dh = grad * f'(h), h the values of `packed` as activation_pack returned it."""
    which = _activation(activation)
    rows, cols = _matrix(grad, "grad")
    kind = _type(grad.dtype, "grad")
    codes, scales, prows, pcols = _packed(packed, "packed")
    if prows != rows or pcols != cols:
        _mismatch((prows, pcols), (rows, cols), "packed's shape")
    out, stride = _out(out, (rows, cols), grad.dtype, grad)
    _run(_lib.pxg_activation_grad_device, (grad, codes, scales, out), which, kind, grad.data_ptr(), rows, cols,
         _stride(grad), codes.data_ptr(), scales.data_ptr(), out.data_ptr(), stride)
    return out
