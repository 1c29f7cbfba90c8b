"""Microscaled 4-bit operands (E2M1 codes, one power of two for every 32 of them) and their products, over torch tensors.

    quantize(x, dim=-1, rule="floor", routing=None)   rows (dim=-1) or columns (dim=-2) of x -> Mx4
    dequantize(q, dtype)                              the values that an Mx4 stands for
    matmul(x, w, dtype)                               Y = X W^T
    grouped_matmul(x, w, offsets, dtype)              rows offsets[g] .. offsets[g + 1] of X with W[g]
    segment_matmul(a, b, offsets, dtype)              Y[g] = A[:, segment g] B[:, segment g]^T

The format and the exact meaning of each are in include/ozb.h (ozb_mx4_*). Every call is asynchronous on the current stream of the
operands' device and may be captured into a CUDA graph; results are new tensors unless out= is given. The backward pass of a
product is two products: from y = matmul(quantize(x), quantize(w)) with a gradient dy,
dx = matmul(quantize(dy), quantize(w, dim=-2)) and dw = matmul(quantize(dy, dim=-2), quantize(x, dim=-2)).
"""
from typing import NamedTuple

import torch

from . import OzakiError
from ._lib import lib as _lib

__all__ = ["Mx4", "quantize", "dequantize", "matmul", "grouped_matmul", "segment_matmul"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_RULES = {"floor": 0, "ceil": 1}


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


def _call(device, entry, *args):
    """One call of the library on the current stream of `device`."""
    if device.index == torch.cuda.current_device():
        status = entry(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            status = entry(*args, torch.cuda.current_stream().cuda_stream)
    if status:
        raise OzakiError(status)


def _dense(x, role, dims=2):
    """Checks that x is a matrix (or a stack of them) on a GPU whose rows are contiguous."""
    if not x.is_cuda:
        raise TypeError(f"{role} must be on a GPU")
    if x.dim() != dims:
        raise ValueError(f"{role} must have {dims} dimensions, not {x.dim()}")
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        raise ValueError(f"the rows of {role} must be contiguous; make it contiguous first")
    return x


def _pitch(x):
    """Elements from one row to the next (a single row has any stride)."""
    return x.stride(-2) if x.shape[-2] > 1 else max(x.stride(-2), x.shape[-1])


def _codes(q, role, dims, device=None):
    for t in (q.codes, q.scales):
        if t.dtype != torch.uint8:
            raise TypeError(f"{role}: codes and scales are uint8, not {t.dtype}")
        _dense(t, role, dims)
    if q.codes.shape[:-1] != q.scales.shape[:-1]:
        raise ValueError(f"{role}: codes {tuple(q.codes.shape)} and scales {tuple(q.scales.shape)} are of different vectors")
    blocks = -(-q.length // 32)
    if q.codes.shape[-1] < 16 * blocks or q.scales.shape[-1] < -(-blocks // 16) * 16:
        raise ValueError(f"{role}: rows of {q.codes.shape[-1]} and {q.scales.shape[-1]} bytes do not hold {q.length} values")
    if q.scales.device != q.codes.device or (device is not None and q.codes.device != device):
        raise ValueError(f"{role} must be on one device with the other operands")
    return q.codes.data_ptr(), _pitch(q.codes), q.scales.data_ptr(), _pitch(q.scales)


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}, not {t.device}")


def _result(out, shape, dtype, device):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"out= must be {tuple(shape)} of {dtype} on {device}")
    return _dense(out, "out", len(shape))


def _offsets(offsets, device):
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or not offsets.is_contiguous() or offsets.numel() < 2:
        raise ValueError("offsets must be a contiguous int32 vector of at least two numbers")
    _same_device(device, offsets=offsets)
    return offsets.numel() - 1


def quantize(x, dim=-1, rule="floor", routing=None):
    """x (float32, bfloat16 or float16; a matrix or a stack of matrices) in blocks of 32 along `dim` (-1 or -2). With dim=-2 the
    columns come out as the vectors. rule "floor" lets the largest of a block saturate at 6 times its scale, "ceil" does not.
    `routing` (of experts.sort) takes the rows of a matrix x in the order of their experts first, zeros where there is none."""
    if dim not in (-1, -2) or rule not in _RULES:
        raise ValueError(f"dim is -1 or -2 and rule one of {sorted(_RULES)}")
    kind = _type(x.dtype)
    if x.dim() not in (2, 3):
        raise ValueError(f"x must be a matrix or a stack of matrices, not {x.dim()}-dimensional")
    _dense(x, "x", x.dim())
    rows, cols = x.shape[-2:]
    slots = per = None
    if routing is not None:
        if x.dim() != 2 or rows != routing.rows.shape[0]:
            raise ValueError("routing= takes a matrix with a row for each token")
        _same_device(x.device, routing=routing.slots)
        slots, per, rows = routing.slots.data_ptr(), routing.rows.shape[1], routing.slots.numel()
    vectors, length = (rows, cols) if dim == -1 else (cols, rows)
    blocks = -(-length // 32)
    lead = tuple(x.shape[:-2])
    codes = torch.empty((*lead, vectors, 16 * blocks), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*lead, vectors, -(-blocks // 16) * 16), dtype=torch.uint8, device=x.device)
    planes = x.shape[0] if lead else 1
    _call(x.device, _lib.ozb_mx4_quantize, x.data_ptr(), kind, vectors, length, _pitch(x), 1 if dim == -1 else 0, _RULES[rule], slots, per or 0,
          x.shape[-2], planes, x.stride(0) if lead else 0, codes.data_ptr(), codes.shape[-1], codes.stride(0), scales.data_ptr(), scales.shape[-1],
          scales.stride(0))
    return Mx4(codes, scales, length)


def dequantize(q, dtype=torch.float32, out=None):
    """The values of an Mx4 of vectors, [n, length] of `dtype` (exact in float32 and bfloat16)."""
    codes, ldq, scales, lds = _codes(q, "q", 2)
    y = _result(out, (q.codes.shape[0], q.length), dtype, q.codes.device)
    _call(y.device, _lib.ozb_mx4_dequantize, codes, ldq, scales, lds, y.shape[0], q.length, y.data_ptr(), _type(dtype), _pitch(y))
    return y


def _common_length(a, b):
    if a.length != b.length:
        raise ValueError(f"cannot multiply vectors of {a.length} by vectors of {b.length}")
    return a.length


def matmul(x, w, dtype=torch.bfloat16, out=None):
    """Y = X W^T, [rows of x, rows of w] of `dtype`: summed in FP32, rounded once."""
    k, device = _common_length(x, w), x.codes.device
    left, right = _codes(x, "x", 2), _codes(w, "w", 2, device)
    y = _result(out, (x.codes.shape[0], w.codes.shape[0]), dtype, device)
    _call(device, _lib.ozb_mx4_gemm, y.shape[0], y.shape[1], k, *left, *right, y.data_ptr(), _type(dtype), _pitch(y))
    return y


def grouped_matmul(x, w, offsets, dtype=torch.bfloat16, out=None):
    """Rows offsets[g] .. offsets[g + 1] - 1 of X times W[g]^T for each g; w is a stack [groups, n, ...], offsets int32 on the device
    (groups + 1 numbers that do not decrease). Rows outside of the segments are not written."""
    k, device, groups = _common_length(x, w), x.codes.device, w.codes.shape[0]
    if _offsets(offsets, device) != groups:
        raise ValueError(f"{groups} groups need {groups + 1} offsets")
    left, (wc, ldw, ws, ldws) = _codes(x, "x", 2), _codes(w, "w", 3, device)
    y = _result(out, (x.codes.shape[0], w.codes.shape[1]), dtype, device)
    _call(device, _lib.ozb_mx4_gemm_grouped, groups, y.shape[0], y.shape[1], k, offsets.data_ptr(), *left, wc, ldw, w.codes.stride(0), ws, ldws,
          w.scales.stride(0), y.data_ptr(), _type(dtype), _pitch(y))
    return y


def segment_matmul(a, b, offsets, dtype=torch.bfloat16, out=None):
    """Y[g] = A[:, offsets[g] : offsets[g + 1]] B[:, the same]^T, [groups, rows of a, rows of b]; the offsets are multiples of 64."""
    r, device = _common_length(a, b), a.codes.device
    groups = _offsets(offsets, device)
    left, right = _codes(a, "a", 2), _codes(b, "b", 2, device)
    y = _result(out, (groups, a.codes.shape[0], b.codes.shape[0]), dtype, device)
    _call(device, _lib.ozb_mx4_gemm_segments, groups, y.shape[1], y.shape[2], r, offsets.data_ptr(), *left, *right, y.data_ptr(), _type(dtype), _pitch(y),
          y.stride(0))
    return y
