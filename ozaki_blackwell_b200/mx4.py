"""Microscaled 4-bit operands (E2M1 codes, one power of two for every 32 of them) and their products, over torch tensors.

    quantize(x, dim=-1, rule="floor", routing=None)   rows (dim=-1) or columns (dim=-2) of x -> Mx4
    dequantize(q, dtype)                              the values that an Mx4 stands for
    matmul(x, w, dtype)                               Y = X W^T
    grouped_matmul(x, w, offsets, dtype)              rows offsets[g] .. offsets[g + 1] of X with W[g]
    segment_matmul(a, b, offsets, dtype)              Y[g] = A[:, segment g] B[:, segment g]^T
    status(device=None)                               raises what products so far could not tell when they were called

The format and the exact meaning of each are in include/ozb.h (ozb_mx4_*). Every call is asynchronous on the current stream of the
operands' device and may be captured into a CUDA graph; results are new tensors unless out= is given. So a call returns before its
kernels have run, and a wait that expires in one of them (its result is then not valid) is only heard of from status().

The backward pass of a product is two products: from y = matmul(quantize(x), quantize(w)) with a gradient dy,
dx = matmul(quantize(dy), quantize(w, dim=-2)) and dw = matmul(quantize(dy, dim=-2), quantize(x, dim=-2)). The calls take no part in
autograd, and warn where an operand requires a gradient.
"""
import warnings
from typing import NamedTuple

import torch

from . import OzakiError
from ._lib import lib as _lib

_current_device = torch._C._cuda_getDevice         # torch.cuda.current_device where CUDA is in use already, as it is behind a tensor on a GPU
_raw_stream = torch._C._cuda_getCurrentRawStream   # the number behind torch.cuda.current_stream(index), without making the object

__all__ = ["Mx4", "quantize", "dequantize", "matmul", "grouped_matmul", "segment_matmul", "status"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_RULES = {"floor": 0, "ceil": 1}
_INT32 = torch.int32
_MOST = 2 ** 31 - 1   # of rows, columns, vectors, values: the library counts in 32 bits (where memory is large enough for more)


class Mx4(NamedTuple):
    """Vectors of `length` values: codes [..., n, pitch] and scales [..., n, pitch], both uint8, one row to a vector."""
    codes: torch.Tensor
    scales: torch.Tensor
    length: int


def _type(dtype):
    try:
        return _TYPES[dtype]
    except KeyError:
        raise TypeError(f"float32, bfloat16 or float16 are supported, not {dtype}") from None


def _call(index, entry, *args):
    """One call of the library on the current stream of device `index`."""
    if index == _current_device():
        status = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _raw_stream(index))
    if status:
        raise OzakiError(status)


def _cut(name):
    """An operand requires a gradient that the result will not carry."""
    if torch.is_grad_enabled():
        warnings.warn(f"{name} takes no part in autograd and an operand requires a gradient, which ends here: call it from the forward of a "
                      "torch.autograd.Function whose backward makes the gradients' calls, or under torch.no_grad()", UserWarning, stacklevel=3)


def _few(role, sizes):
    if max(sizes) > _MOST:
        raise ValueError(f"{role} of sizes {tuple(sizes)}: none may pass {_MOST}")


def _pitch(x, role, dims=2):
    """Checks that x is a matrix (or a stack of them) on a GPU whose rows are contiguous; elements from one row to the next (a single row
    has any stride)."""
    shape, stride = x.shape, x.stride()
    if len(shape) != dims:
        raise ValueError(f"{role} must have {dims} dimensions, not {len(shape)}")
    if not x.is_cuda:
        raise TypeError(f"{role} must be on a GPU")
    if stride[-1] != 1 and shape[-1] != 1:
        raise ValueError(f"the rows of {role} must be contiguous; make it contiguous first")
    if shape[0] > _MOST or shape[-2] > _MOST or shape[-1] > _MOST:
        _few(role, shape)
    return stride[-2] if shape[-2] > 1 else max(stride[-2], shape[-1])


def _codes(q, role, dims, index):
    """Pointers and pitches of an Mx4 on device `index`: codes, ldq, scales, lds."""
    codes, scales, length = q
    blocks = (length + 31) >> 5
    have, bytes_, at, steps = codes.shape, scales.shape, codes.stride(), scales.stride()
    if (codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and len(have) == dims and have[:-1] == bytes_[:-1] and at[-1] == 1 and steps[-1] == 1
            and have[-1] >= 16 * blocks and bytes_[-1] >= (blocks + 15) & ~15 and codes.get_device() == index == scales.get_device() and index >= 0):
        if length > _MOST or codes.numel() > _MOST:
            _few(role, (*have[:-1], length))
        if have[-2] > 1:
            return codes.data_ptr(), at[-2], scales.data_ptr(), steps[-2]
        return codes.data_ptr(), max(at[-2], have[-1]), scales.data_ptr(), max(steps[-2], bytes_[-1])   # one vector has any pitch
    # something is wrong: say what
    _pitch(codes, role, dims)
    _pitch(scales, role, dims)
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise TypeError(f"{role}: codes and scales are uint8, not {codes.dtype} and {scales.dtype}")
    if have[:-1] != bytes_[:-1]:
        raise ValueError(f"{role}: codes {tuple(have)} and scales {tuple(bytes_)} are of different vectors")
    if have[-1] < 16 * blocks or bytes_[-1] < (blocks + 15) & ~15:
        raise ValueError(f"{role}: rows of {have[-1]} and {bytes_[-1]} bytes do not hold {length} values")
    raise ValueError(f"{role} must be on cuda:{index} with the other operands")


def _result(like, out, shape, dtype, dims=2):
    """out, checked, or a new tensor on the device of `like`; and the pitch of its rows."""
    if out is None:
        return like.new_empty(*shape, dtype=dtype), shape[-1]
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != like.device:
        raise ValueError(f"out= must be {tuple(shape)} of {dtype} on {like.device}")
    return out, _pitch(out, "out", dims)


def _offsets(offsets, index):
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or not offsets.is_contiguous() or offsets.shape[0] < 2:
        raise ValueError("offsets must be a contiguous int32 vector of at least two numbers")
    if offsets.get_device() != index:
        raise ValueError(f"offsets must be on cuda:{index}, not {offsets.device}")
    return offsets.shape[0] - 1


def _routed(r, index):
    """Checks the maps of a Routing (of experts.sort) on device `index`; (tokens, top)."""
    _, rows, slots, _ = r
    if not (rows.dtype is _INT32 is slots.dtype and rows.is_contiguous() and slots.is_contiguous() and rows.get_device() == index == slots.get_device()
            and rows.numel() <= _MOST and slots.numel() <= _MOST):
        for name, t in (("rows", rows), ("slots", slots)):
            if t.dtype is not _INT32 or not t.is_contiguous() or t.get_device() != index:
                raise ValueError(f"routing.{name} must be contiguous int32 on cuda:{index}")
            _few(f"routing.{name}", (t.numel(),))
    shape = rows.shape
    if len(shape) != 2:
        raise ValueError("routing.rows has a row for each token")
    return shape


def quantize(x, dim=-1, rule="floor", routing=None):
    """x (float32, bfloat16 or float16; a matrix or a stack of matrices) in blocks of 32 along `dim` (-1 or -2). With dim=-2 the
    columns come out as the vectors. rule "floor" lets the largest of a block saturate at 6 times its scale, "ceil" does not.
    `routing` (of experts.sort) takes the rows of a matrix x in the order of their experts first, zeros where there is none."""
    if dim not in (-1, -2) or rule not in _RULES:
        raise ValueError(f"dim is -1 or -2 and rule one of {sorted(_RULES)}")
    kind, shape = _type(x.dtype), x.shape
    dims = len(shape)
    if dims not in (2, 3):
        raise ValueError(f"x must be a matrix or a stack of matrices, not {dims}-dimensional")
    ldx, index = _pitch(x, "x", dims), x.get_device()
    if x.requires_grad:
        _cut("quantize")
    rows, cols = shape[-2:]
    maps = None, None, 0, 0
    if routing is not None:
        if dims != 2 or rows != routing.rows.shape[0]:
            raise ValueError("routing= takes a matrix with a row for each token")
        tokens, top = _routed(routing, index)
        maps, rows = (routing.rows.data_ptr(), routing.slots.data_ptr(), top, tokens), routing.slots.shape[0]
    vectors, length = (rows, cols) if dim == -1 else (cols, rows)
    blocks = (length + 31) >> 5
    ldq, lds = 16 * blocks, (blocks + 15) & ~15
    if dims == 2:
        codes, scales = x.new_empty(vectors, ldq, dtype=torch.uint8), x.new_empty(vectors, lds, dtype=torch.uint8)
        planes = 1, 0, 0, 0
    else:
        codes, scales = x.new_empty(shape[0], vectors, ldq, dtype=torch.uint8), x.new_empty(shape[0], vectors, lds, dtype=torch.uint8)
        planes = shape[0], x.stride(0), vectors * ldq, vectors * lds
    _call(index, _lib.ozb_mx4_quantize, x.data_ptr(), kind, vectors, length, ldx, dim == -1, _RULES[rule], *maps, planes[0], planes[1],
          codes.data_ptr(), ldq, planes[2], scales.data_ptr(), lds, planes[3])
    return Mx4(codes, scales, length)


def dequantize(q, dtype=torch.float32, out=None):
    """The values of an Mx4 of vectors, [n, length] of `dtype` (exact in float32 and bfloat16)."""
    like = q.codes
    index = like.get_device()
    codes, ldq, scales, lds = _codes(q, "q", 2, index)
    n, length = like.shape[0], q.length
    y, ldy = _result(like, out, (n, length), dtype)
    _call(index, _lib.ozb_mx4_dequantize, codes, ldq, scales, lds, n, length, y.data_ptr(), _type(dtype), ldy)
    return y


def status(device=None):
    """Waits for `device` (default: the current one) and raises OzakiError if, since the last call, a bounded wait of a product on it
    expired, whose result is then not valid, or a product along the vectors refused its segments, whose results are NaN."""
    if device is None:
        code = _lib.ozb_status()
    else:
        with torch.cuda.device(device):
            code = _lib.ozb_status()
    if code:
        raise OzakiError(code)


def _common_length(a, b):
    if a.length != b.length:
        raise ValueError(f"cannot multiply vectors of {a.length} by vectors of {b.length}")
    return a.length


def matmul(x, w, dtype=torch.bfloat16, out=None):
    """Y = X W^T, [rows of x, rows of w] of `dtype`: summed in FP32, rounded once."""
    k, like = _common_length(x, w), x.codes
    index = like.get_device()
    left, right = _codes(x, "x", 2, index), _codes(w, "w", 2, index)
    m, n = like.shape[0], w.codes.shape[0]
    kind = _type(dtype)
    y, ldy = _result(like, out, (m, n), dtype)
    _call(index, _lib.ozb_mx4_gemm, m, n, k, *left, *right, y.data_ptr(), kind, ldy)
    return y


def grouped_matmul(x, w, offsets, dtype=torch.bfloat16, out=None):
    """Rows offsets[g] .. offsets[g + 1] - 1 of X times W[g]^T for each g; w is a stack [groups, n, ...], offsets int32 on the device
    (groups + 1 numbers that do not decrease). Rows outside of the segments are not written."""
    k, like = _common_length(x, w), x.codes
    index = like.get_device()
    left, (wc, ldw, ws, ldws) = _codes(x, "x", 2, index), _codes(w, "w", 3, index)
    groups, n = w.codes.shape[:2]
    if _offsets(offsets, index) != groups:
        raise ValueError(f"{groups} groups need {groups + 1} offsets")
    kind = _type(dtype)
    y, ldy = _result(like, out, (like.shape[0], n), dtype)
    _call(index, _lib.ozb_mx4_gemm_grouped, groups, like.shape[0], n, k, offsets.data_ptr(), *left, wc, ldw, w.codes.stride(0), ws, ldws, w.scales.stride(0),
          y.data_ptr(), kind, ldy)
    return y


def segment_matmul(a, b, offsets, dtype=torch.bfloat16, out=None):
    """Y[g] = A[:, offsets[g] : offsets[g + 1]] B[:, the same]^T, [groups, rows of a, rows of b]; the offsets are multiples of 64 (an end
    may also be the vectors' length). Y[g] of a segment that is not so is NaN."""
    r, like = _common_length(a, b), a.codes
    index = like.get_device()
    groups = _offsets(offsets, index)
    left, right = _codes(a, "a", 2, index), _codes(b, "b", 2, index)
    m, n = like.shape[0], b.codes.shape[0]
    kind = _type(dtype)
    y, ldy = _result(like, out, (groups, m, n), dtype, 3)
    _call(index, _lib.ozb_mx4_gemm_segments, groups, m, n, r, offsets.data_ptr(), *left, *right, y.data_ptr(), kind, ldy, y.stride(0))
    return y
