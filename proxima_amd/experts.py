"""Expert layers in front of an index, and rows packed in 8 bits.

The products of a layer whose rows are routed in ragged groups, each group with
a matrix of its own, their gradients, the same product over rows packed in 8
bits, and activations whose input is kept packed for their backward pass;
layers with their bias, activation and residual, and their backward pass; whole
layers for a few tokens; and the loss of an encoder that learns to rank as an
index' answers do. No reference counterpart: these are the layers whose outputs
an index stores.

All functions take torch tensors on the GPU, run on torch's current stream and
return without waiting; outputs are new tensors unless `out` is given. Rows may
be strided; a row's columns are contiguous. `offsets` is an int64 tensor of
groups + 1 values: group g is the rows offsets[g] to offsets[g + 1], and rows
of no group get zeros (a layer's: its residual).

None of them records history for autograd: the gradients are functions of their
own. An operand that requires grad is refused while grad mode is on, so that no
gradient is lost unseen; inside torch.no_grad() and a torch.autograd.Function
it is off.
"""
import sys
from functools import lru_cache as _lru_cache
from struct import Struct as _Struct

from . import DimensionMismatch, _check
from ._capi import lib as _lib

__all__ = [
    "Block8", "block8_pack", "block8_unpack", "block8_matmul", "grouped_matmul", "grouped_matmul_grad_input",
    "grouped_matmul_grad_weight", "grouped_linear", "block8_linear", "grouped_linear_grad", "expert_layer",
    "activation_pack", "activation_grad", "distill_loss", "distill_loss_grad",
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


# torch is the caller's: this package does not import it by itself. Filled by what looks at a call's first operand
# (_matrix, _device, _packed, and Block8's constructor), _torch last: another thread takes it as the sign that all is.
_KINDS = {}  # torch dtype -> pxg_type
_torch = _current_device = _current_stream = None


def _setup():
    global _torch, _current_device, _current_stream
    torch = sys.modules["torch"]
    _current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    _KINDS.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    _torch = torch


def _type(dtype, name, f32=True):
    kind = _KINDS.get(dtype)
    if kind is None or (kind == 0 and not f32):
        raise ValueError(f"{name} must be {'float32, ' if f32 else ''}float16 or bfloat16, got {dtype}")
    return kind


def _matrix(t, name, dims=2):
    """Checks a GPU tensor of contiguous rows; its shape."""
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{name} must be a GPU tensor")
    if _torch is None:
        _setup()
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
    if _torch is None:
        _setup()
    codes = p._codes
    return codes, p._scales, codes.shape[0], p._cols


def _groups(offsets):
    """(pointer or None, number of groups)"""
    if offsets is None:
        return None, 1
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


_NO_HISTORY = ("an operand requires grad, but no history is recorded here: call the gradients' own functions, under "
               "torch.no_grad() or from a torch.autograd.Function")


def _run(fn, tensors, *args):
    """fn(*args, stream) on torch's current stream of the device that all tensors share."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None:
            if t.get_device() != device:
                raise ValueError("operands must be on one device")
            if t.requires_grad and _torch.is_grad_enabled():
                raise ValueError(_NO_HISTORY)
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


def _packed_weights(w, offsets, k):
    """(codes, scales, groups, n, offsets' pointer) of packed [groups * n, k] matrices"""
    wcodes, wscales, wrows, wk = _packed(w, "w")
    if wk != k:
        _mismatch(wk, k, "w's columns")
    ptr, groups = _groups(offsets)
    n, left = divmod(wrows, groups)
    if left:
        raise DimensionMismatch(f"dimension mismatch: w's {wrows} rows are not a multiple of {groups} groups", groups,
                                wrows)
    return wcodes, wscales, groups, n, ptr


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
    wcodes, wscales, groups, n, ptr = _packed_weights(w, offsets, k)
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


# The C structs' arguments, 8 bytes each: packing them as bytes takes a third of the time of 20 converted one by one.
_LINEAR, _LINEAR_GRAD, _EXPERT_LAYER, _DISTILL = map(_Struct, ("4q20Q", "3q14Q", "5q34Q", "q10Qd6Q"))


def _device(t, name):
    """The index of the GPU that a call's first operand is on, and so all others."""
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{name} must be a GPU tensor")
    if _torch is None:
        _setup()
    return t.get_device()


def _rows(t, name, device, dims=2):
    """Checks a tensor of contiguous rows on that GPU; (shape, elements from row to row)."""
    try:
        on, shape, strides = t.get_device(), t.shape, t.stride()
    except AttributeError:
        on = -1
    if on != device:
        raise ValueError(f"{name} must be a GPU tensor" if on < 0 else "operands must be on one device")
    if t.requires_grad and _torch.is_grad_enabled():
        raise ValueError(_NO_HISTORY)
    if len(strides) != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {len(strides)}")
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must have contiguous rows")
    return shape, strides[-2] if shape[-2] > 1 else shape[-1]


def _here(device, *tensors):
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError("operands must be on one device")


def _call(fn, device, args):
    """fn(struct, stream) on torch's current stream of a device."""
    if _current_device() == device:
        status = fn(args, _current_stream(device))
    else:
        with _torch.cuda.device(device):
            status = fn(args, _current_stream(device))
    if status:
        _check(status)


def _bias(bias, name, rows, n, dtype, device):
    """(pointer, pxg_type, elements from row to row) of a bias [rows, n] of `dtype` or f32, [n] where rows is None."""
    if bias is None:
        return 0, 0, 0
    if rows is None:
        rows = 1
        if bias.dim() == 1:
            bias = bias.unsqueeze(0)
    shape, stride = _rows(bias, name, device)
    if shape != (rows, n):
        _mismatch(tuple(shape), (rows, n), f"{name}'s shape")
    kind = bias.dtype
    if kind is not dtype and kind is not _torch.float32:
        raise ValueError(f"{name} must be {dtype} or float32, got {kind}")
    return bias.data_ptr(), _KINDS[kind], stride


def _residual(residual, shape, dtype, device):
    """(pointer, elements from row to row)"""
    if residual is None:
        return 0, 0
    got, stride = _rows(residual, "residual", device)
    if got != shape:
        _mismatch(tuple(got), shape, "residual's shape")
    if residual.dtype is not dtype:
        raise ValueError(f"residual must be {dtype}, got {residual.dtype}")
    return residual.data_ptr(), stride


def _result(out, shape, dtype, like, device):
    """(tensor, elements from row to row)"""
    if out is None:
        return like.new_empty(shape, dtype=dtype), shape[-1]
    got, stride = _rows(out, "out", device, len(shape))
    if got != shape:
        _mismatch(tuple(got), shape, "out's shape")
    if out.dtype is not dtype:
        raise ValueError(f"out must be {dtype}, got {out.dtype}")
    return out, stride


def _optional(activation):
    return -1 if activation is None else _activation(activation)


def grouped_linear(x, w, offsets=None, bias=None, activation=None, residual=None, out_dtype=None, out=None, keep=False):
    """y[t] = f(h[t]) + residual[t], h[t] = x[t] w[g]^T + bias[g] for t in group g: x and w as grouped_matmul takes
    them, bias [groups, n] (or [n] without offsets) in x's type or f32, f "silu", "gelu" or None, residual [rows, n]
    in y's type. `out` may be the residual itself, unless that is x: it shares no memory with x. With keep, (y, h), h in
    y's type for grouped_linear_grad. y is rounded once, from the unrounded h. Rows of no group: y is the residual, or
    zeros, and h zeros."""
    device = _device(x, "x")
    (rows, xk), x_stride = _rows(x, "x", device)
    xtype = x.dtype
    kind = _type(xtype, "x", False)
    w, ptr, groups, n, k = _weights(w, offsets, x)
    _, w_stride = _rows(w, "w", device, 3)
    if xk != k:
        _mismatch(xk, k, "x's columns")
    _here(device, offsets)
    dtype = out_dtype or (out.dtype if out is not None else xtype)
    out_kind, which = _type(dtype, "out_dtype"), _optional(activation)
    bias_ptr, bias_kind, bias_stride = _bias(bias, "bias", None if offsets is None else groups, n, xtype, device)
    r, r_stride = _residual(residual, (rows, n), dtype, device)
    out, stride = _result(out, (rows, n), dtype, x, device)
    h = x.new_empty((rows, n), dtype=dtype) if keep else None
    _call(_lib.pxg_grouped_linear_device, device,
          _LINEAR.pack(kind, out_kind, bias_kind, which, rows, k, groups, n, x.data_ptr(), x_stride, w.data_ptr(),
                       w_stride, w.stride(0), ptr or 0, bias_ptr, bias_stride, r, r_stride,
                       h.data_ptr() if keep else 0, n, out.data_ptr(), stride, 0, 0))
    return (out, h) if keep else out


def block8_linear(x, w, offsets=None, bias=None, activation=None, residual=None, out_dtype=None, out=None):
    """y[t] = f(x[t] w_g^T + bias[g]) + residual[t] for t in group g: x and w Block8, multiplied as block8_matmul
    does (into 16 bits with products cut, before the bias, activation and residual; into f32 exactly), bias bf16 or f32,
    the rest as grouped_linear, of packed x."""
    codes, scales, rows, k = _packed(x, "x")
    wcodes, wscales, groups, n, ptr = _packed_weights(w, offsets, k)
    device = codes.get_device()
    _here(device, scales, wcodes, wscales, offsets)
    dtype = out_dtype or (out.dtype if out is not None else _torch.bfloat16)
    out_kind, which = _type(dtype, "out_dtype"), _optional(activation)
    bias_ptr, bias_kind, bias_stride = _bias(bias, "bias", None if offsets is None else groups, n, _torch.bfloat16, device)
    r, r_stride = _residual(residual, (rows, n), dtype, device)
    out, stride = _result(out, (rows, n), dtype, codes, device)
    _call(_lib.pxg_block8_linear_device, device,
          _LINEAR.pack(0, out_kind, bias_kind, which, rows, k, groups, n, codes.data_ptr(), 0, wcodes.data_ptr(), 0, 0,
                       ptr or 0, bias_ptr, bias_stride, r, r_stride, 0, 0, out.data_ptr(), stride, scales.data_ptr(),
                       wscales.data_ptr()))
    return out


_grad_space = _lru_cache(1024)(_lib.pxg_grouped_linear_grad_workspace)  # bytes, by sizes


def grouped_linear_grad(grad, h=None, activation=None, offsets=None, bias_dtype=None, out=None):
    """(dh, dbias): grouped_linear's backward pass up to the products. dh = grad * f'(h), h as grouped_linear kept it
    and of grad's type, zeros for rows of no group; dbias[g] is the sum of group g's dh before its rounding,
    [groups, n] (or [n] without offsets) of bias_dtype (f32 by default, or grad's type). Without an activation dh is
    grad itself. `out` may be grad or h itself. dx and dw are grouped_matmul_grad_input's and
    grouped_matmul_grad_weight's of dh, and the residual's gradient is grad."""
    device = _device(grad, "grad")
    (rows, n), grad_stride = _rows(grad, "grad", device)
    dtype = grad.dtype
    kind = _type(dtype, "grad")
    ptr, groups = _groups(offsets)
    _here(device, offsets)
    which = _optional(activation)
    if which < 0:
        if h is not None or out is not None:
            raise ValueError("h and out are for an activation")
        dh, h_ptr, h_stride, stride = grad, 0, 0, 0
    else:
        if h is None:
            raise ValueError("h must be given with an activation")
        shape, h_stride = _rows(h, "h", device)
        if shape != (rows, n):
            _mismatch(tuple(shape), (rows, n), "h's shape")
        if h.dtype is not dtype:
            raise ValueError(f"h must be {dtype}, got {h.dtype}")
        h_ptr = h.data_ptr()
        dh, stride = _result(out, (rows, n), dtype, grad, device)
    bias_dtype = bias_dtype or _torch.float32
    if bias_dtype is not dtype and bias_dtype is not _torch.float32:
        raise ValueError(f"bias_dtype must be {dtype} or float32, got {bias_dtype}")
    dbias = grad.new_empty((groups, n) if offsets is not None else (n,), dtype=bias_dtype)
    size = _grad_space(rows, n, groups)
    space = grad.new_empty(size, dtype=_torch.uint8) if size else None
    _call(_lib.pxg_grouped_linear_grad_device, device,
          _LINEAR_GRAD.pack(kind, _KINDS[bias_dtype], which, rows, n, groups, grad.data_ptr(), grad_stride, h_ptr, h_stride,
                            ptr or 0, dh.data_ptr(), stride, dbias.data_ptr(), n, space.data_ptr() if size else 0, size))
    return dh, dbias


def _expert_matrix(w, name, experts, height, width, dtype, device):
    """(data, stride, group stride, scales) of [experts, height, width] matrices, or of a Block8 of [experts * height,
    width] where dtype is None."""
    if dtype is None:
        codes, scales, rows, cols = _packed(w, name)
        if rows != experts * height or cols != width:
            _mismatch((rows, cols), (experts * height, width), f"{name}'s shape")
        _here(device, codes, scales)
        return codes.data_ptr(), 0, 0, scales.data_ptr()
    shape, stride = _rows(w, name, device, 3)
    if shape != (experts, height, width):
        _mismatch(tuple(shape), (experts, height, width), f"{name}'s shape")
    if w.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {w.dtype}")
    return w.data_ptr(), stride, w.stride(0), 0


def _picks(t, name, dtype, expected, device):
    """Checks a tensor [rows, some] of `dtype`; (its columns, elements from row to row)."""
    shape, stride = _rows(t, name, device)
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    rows, cols = expected
    if shape[0] != rows or (cols is not None and shape[1] != cols):
        _mismatch(tuple(shape), expected, f"{name}'s shape")
    return shape[1], stride


_layer_space = _lru_cache(1024)(_lib.pxg_expert_layer_workspace)


def expert_layer(x, experts, w1, w2, gates, activation=None, up=None, bias1=None, bias2=None, residual=None,
                 out_dtype=None, out=None):
    """A whole expert layer for a few tokens, in the rows' own order:
    y[t] = residual[t] + sum over j of gates[t, j] * (w2[e] (f(w1[e] x[t] + bias1[e]) * up[e] x[t]) + bias2[e]),
    e = experts[t, j].

    x [rows, k] f16 or bf16; experts [rows, picks] int64 and gates [rows, picks] f32, picks at most 16 (an id that is
    no expert's is left out, one that a token has twice counts with both gates); w1 and up (optional) [experts, hidden,
    k] and w2 [experts, n, hidden] of x's type, or each a Block8 of the experts' rows one after the other (x is then
    bf16); biases [experts, .] of x's type or f32; residual and y [rows, n] of x's type or f32. `out` may be the
    residual itself, also where that is x. Nothing between the two products is rounded to x's type: for f32 results it
    is f32, for 16-bit ones it is held to 2^-16, 2^-8 of what their rounding costs in bf16 and 2^-5 in f16. The matrices
    of the experts in use are read once for each 64 rows: for batches use grouped_linear."""
    device = _device(x, "x")
    (rows, k), x_stride = _rows(x, "x", device)
    xtype = x.dtype
    kind = _type(xtype, "x", False)
    picks, ids_stride = _picks(experts, "experts", _torch.int64, (rows, None), device)
    _, gates_stride = _picks(gates, "gates", _torch.float32, (rows, picks), device)
    packed = type(w1) is Block8
    if packed:
        if xtype is not _torch.bfloat16:
            raise ValueError(f"x must be bfloat16 with packed matrices, got {xtype}")
        _, _, rows2, hidden = _packed(w2, "w2")
        number, left = divmod(w1.rows, hidden)
        if left or not number:
            raise DimensionMismatch(f"dimension mismatch: w1's {w1.rows} rows are not a multiple of w2's {hidden} columns",
                                    hidden, w1.rows)
        n, left = divmod(rows2, number)
        if left or not n:
            raise DimensionMismatch(f"dimension mismatch: w2's {rows2} rows are not a multiple of {number} experts",
                                    number, rows2)
        of = None
    else:
        number, hidden, _ = _matrix(w1, "w1", 3)
        n = _matrix(w2, "w2", 3)[1]
        of = xtype
    m1 = _expert_matrix(w1, "w1", number, hidden, k, of, device)
    m3 = _expert_matrix(up, "up", number, hidden, k, of, device) if up is not None else (0, 0, 0, 0)
    m2 = _expert_matrix(w2, "w2", number, n, hidden, of, device)
    if bias1 is not None and bias2 is not None and bias1.dtype is not bias2.dtype:
        raise ValueError(f"biases must be of one type, got {bias1.dtype} and {bias2.dtype}")
    b1, kind1, stride1 = _bias(bias1, "bias1", number, hidden, xtype, device)
    b2, kind2, stride2 = _bias(bias2, "bias2", number, n, xtype, device)
    dtype = out_dtype or (out.dtype if out is not None else xtype)
    out_kind = _type(dtype, "out_dtype")
    which = _optional(activation)
    r, r_stride = _residual(residual, (rows, n), dtype, device)
    out, stride = _result(out, (rows, n), dtype, x, device)
    size = _layer_space(rows, picks, number, hidden, n, out_kind)
    space = x.new_empty(size, dtype=_torch.uint8) if size else None
    _call(_lib.pxg_expert_layer_device, device,
          _EXPERT_LAYER.pack(kind, out_kind, kind1 if b1 else kind2, which, packed, rows, k, picks, number, hidden, n,
                             x.data_ptr(), x_stride, experts.data_ptr(), ids_stride, gates.data_ptr(), gates_stride, *m1,
                             *m3, *m2, b1, stride1, b2, stride2, r, r_stride, out.data_ptr(), stride,
                             space.data_ptr() if size else 0, size))
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


def _vector(t, name, rows, dtype, device):
    """Checks a contiguous tensor of `rows` values on a GPU."""
    if _device(t, name) != device:
        raise ValueError("operands must be on one device")
    if t.requires_grad and _torch.is_grad_enabled():
        raise ValueError(_NO_HISTORY)
    if t.dim() != 1 or not t.is_contiguous() or t.dtype is not dtype:
        raise ValueError(f"{name} must be a contiguous one-dimensional {dtype} tensor")
    if t.shape[0] != rows:
        _mismatch(t.shape[0], rows, f"{name}'s length")
    return t.data_ptr()


_distill_space = _lru_cache(1024)(_lib.pxg_distill_workspace)


def _distill(fn, weight, logits, ids, scores, counts, temperature, grad, out):
    device = _device(logits, "logits")
    (rows, cols), stride = _rows(logits, "logits", device)
    dtype = logits.dtype
    kind = _type(dtype, "logits")
    top, ids_stride = _picks(ids, "ids", _torch.int64, (rows, None), device)
    _, scores_stride = _picks(scores, "scores", _torch.float32, (rows, top), device)
    counts_ptr = _vector(counts, "counts", rows, _torch.int32, device)
    weight_ptr = out_ptr = out_stride = 0
    if grad:
        weight_ptr = _vector(weight, "weight", rows, _torch.float32, device)
        out, out_stride = _result(out, (rows, cols), dtype, logits, device)
        out_ptr = out.data_ptr()
    loss = logits.new_empty((rows,), dtype=_torch.float32)
    size = _distill_space(kind, rows, cols, top)
    space = logits.new_empty(size, dtype=_torch.uint8) if size else None
    _call(fn, device,
          _DISTILL.pack(kind, rows, cols, top, logits.data_ptr(), stride, ids.data_ptr(), ids_stride, scores.data_ptr(),
                        scores_stride, counts_ptr, float(temperature), loss.data_ptr(), weight_ptr, out_ptr, out_stride,
                        space.data_ptr() if size else 0, size))
    return loss, out


def distill_loss(logits, ids, scores, counts, temperature=1.0):
    """The loss [rows] (f32) of a model that is to rank as a teacher does, as search_device gives the teacher's best:
    sum over entries of p (log p - log q[id]), p the softmax of scores / temperature over a row's first counts[t]
    entries, q that of its logits / temperature.

    logits [rows, cols] f32, f16 or bf16; ids [rows, top] int64 and scores [rows, top] f32 (larger is nearer: of
    distances their negatives), top at most 4096; counts [rows] int32. Entries whose id is outside [0, cols) are left
    out. A row without entries, or whose scores are all -inf, has loss 0; an entry of p = 0 adds nothing; a logit of
    -inf has q = 0, so that p > 0 there costs infinity. temperature is a number between 1e-6 and 1e6. Sums are held
    in f32."""
    return _distill(_lib.pxg_distill_loss_device, None, logits, ids, scores, counts, temperature, False, None)[0]


def distill_loss_grad(weight, logits, ids, scores, counts, temperature=1.0, out=None):
    """(loss, dx): distill_loss and the logits' gradient, weight[t] / temperature (q - p), of the logits' type and
    rounded once; weight [rows] f32 is the loss' own gradient (1 / rows for the mean). Rows without a teacher have zeros.
    `out` may be the logits themselves. Of 16-bit logits the exponentials in dx are off by at most 2^-16 of themselves,
    2^-8 of what dx' rounding costs in bf16 and 2^-5 in f16. The time grows with the square of `top`, from some 100
    entries on."""
    return _distill(_lib.pxg_distill_loss_grad_device, weight, logits, ids, scores, counts, temperature, True, out)
