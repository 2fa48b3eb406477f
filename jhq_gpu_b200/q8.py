"""8-bit rows (jhq_q8_* of include/jhq.h): the RMS norm that ends an encoder layer and writes 8-bit rows, their
product with an 8-bit projection, and a cache that rows are written to in 8 bits and read back from.

    rows = Q8Rows.of(q, scale)                       # q: (n, d) int8, scale: (n,) float32, both on the GPU
    q8_rms_norm(View.of(x), rows, weight=View.of(w), residual=View.of(r), residual_out=View.of(r))
    q8_matmul(rows, Q8Rows.of(wq, w_scale), View.of(out))

A View or Q8Rows describes device memory and does not keep it alive; `of` takes any 2-D tensor with data_ptr(),
shape, stride() and dtype, such as torch's. Calls are asynchronous on `stream` (a raw CUDA stream, as
torch.cuda.current_stream().cuda_stream) on the current device; errors are those of the package. Memory that `of` found
elsewhere (on the host, on another GPU) is refused by the call that is given it.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import jhq_gpu_b200 as _J

F32, F16, BF16 = range(3)
_TYPES = {"float32": F32, "float16": F16, "bfloat16": BF16,
          "torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}
_VIEW, _Q8_ROWS = struct.Struct("Pqqqii").pack, struct.Struct("PPqqqii").pack   # the structures' bytes: made in less time than field by field
_PAIRS = set()                                            # dtypes of values and scales that were found right


def _kind(dtype) -> int:
    kind = _TYPES.get(str(dtype))
    if kind is None:
        raise ValueError(f"View: float32, float16 or bfloat16 is needed, got {dtype}")
    _TYPES[dtype] = kind                                  # the next look finds the dtype itself
    return kind


def _shape(shape, stride, what: str):
    """rows, columns and row stride of a 2-D (or, as one row, 1-D) tensor."""
    if len(shape) == 2:
        rows, cols = shape
        ld, step = stride
    elif len(shape) == 1:
        rows, cols, ld, step = 1, shape[0], 0, stride[0]
    else:
        raise ValueError(f"{what}: a 2-D tensor is needed, got {len(shape)} dimensions")
    if step != 1 and cols > 1:
        raise ValueError(f"{what}: the values of a row must follow one another (stride {step})")
    return rows, cols, ld if rows > 1 else cols


# A description's `place` says where `of` found its memory: the GPU's ordinal + 2, 1 for host memory, 0 if the tensor doesn't
# say. It lies in the C structure's padding, which C does not look at.
def _check_places(L, fn, *operands) -> None:
    """Refuses operands, in fn's order, whose memory is known not to be the current device's."""
    here = L.jhq_current_device() + 2
    try:
        for o in operands:
            if o is not None and o.place != here and o.place:
                break
        else:
            return
    except AttributeError:                                # not a description: refused by ctypes as such
        return
    kinds = [k._type_ for k in fn.argtypes if k._type_ in (View, Q8Rows)]
    if all(b is None or isinstance(b, k) for b, k in zip(operands, kinds)):   # else the same
        raise ValueError(f"{fn.__name__[4:]}: an operand lies in " + ("host memory" if o.place == 1 else f"the memory of GPU {o.place - 2}")
                         + (f"; the current device is GPU {here - 2}" if here >= 2 else "; there is no current device"))


def _slots(L, slots, v):
    """The address that C takes: of a tensor, once it is known to be an int64 of the current device for each row of v; else as given."""
    if not hasattr(slots, "data_ptr"):
        return slots
    rows = v.rows
    if str(slots.dtype) not in ("torch.int64", "int64"):
        raise ValueError(f"slots: int64s are needed, got {slots.dtype}")
    if tuple(slots.shape) != (rows,) or (rows > 1 and slots.stride()[0] != 1):
        raise ValueError(f"slots: {rows} values that follow one another are needed, got a shape of {tuple(slots.shape)}"
                         f" with strides {tuple(slots.stride())}")
    here = L.jhq_current_device()
    if hasattr(slots, "get_device") and slots.get_device() != here:
        raise ValueError("slots: not in the memory of " + (f"the current device, GPU {here}" if here >= 0 else "a current device"))
    return slots.data_ptr()


class View(C.Structure):
    """jhq_view: a matrix of floating-point rows in device memory."""
    _fields_ = [("data", C.c_void_p), ("rows", C.c_int64), ("cols", C.c_int64), ("ld", C.c_int64),
                ("type", C.c_int), ("place", C.c_int)]

    @classmethod
    def of(cls, t) -> "View":
        kind = _TYPES.get(t.dtype)
        shape, stride = t.shape, t.stride()
        if len(shape) == 2 and stride[1] == 1:            # the common matrix
            rows, cols = shape
            ld = stride[0] if rows > 1 else cols
        else:
            rows, cols, ld = _shape(shape, stride, "View")
        try:
            place = t.get_device() + 2
        except AttributeError:
            place = 0
        return cls.from_buffer_copy(_VIEW(t.data_ptr(), rows, cols, ld, _kind(t.dtype) if kind is None else kind, place))


class Q8Rows(C.Structure):
    """jhq_q8_rows: a matrix of 8-bit rows in device memory, one float32 scale for each group of a row."""
    _fields_ = [("q", C.c_void_p), ("scale", C.c_void_p), ("rows", C.c_int64), ("dim", C.c_int64),
                ("ld", C.c_int64), ("groups", C.c_int), ("place", C.c_int)]

    @classmethod
    def of(cls, q, scale, groups: int = 1) -> "Q8Rows":
        """q: (rows, dim) int8; scale: rows * groups float32, packed."""
        if (q.dtype, scale.dtype) not in _PAIRS:
            if str(q.dtype) not in ("torch.int8", "int8") or str(scale.dtype) not in ("torch.float32", "float32"):
                raise ValueError(f"Q8Rows: int8 values and float32 scales are needed, got {q.dtype} and {scale.dtype}")
            _PAIRS.add((q.dtype, scale.dtype))
        shape, stride = q.shape, q.stride()
        if len(shape) == 2 and stride[1] == 1:            # the common matrix
            rows, dim = shape
            ld = stride[0] if rows > 1 else dim
        else:
            rows, dim, ld = _shape(shape, stride, "Q8Rows")
        if scale.numel() != rows * groups or not scale.is_contiguous():
            raise ValueError(f"Q8Rows: {rows} x {groups} packed scales are needed")
        try:
            place = q.get_device() + 2
            if scale.get_device() + 2 != place:
                raise ValueError("Q8Rows: values and scales must be on one device")
        except AttributeError:
            place = 0
        return cls.from_buffer_copy(_Q8_ROWS(q.data_ptr(), scale.data_ptr(), rows, dim, ld, groups, place))


def _declare(L: C.CDLL) -> None:
    v, r, p = C.POINTER(View), C.POINTER(Q8Rows), C.c_void_p
    L.jhq_q8_rms_norm.argtypes = [v, v, v, C.c_float, v, r, p]
    L.jhq_q8_matmul.argtypes = [r, r, v, v, p]
    L.jhq_q8_write.argtypes = [v, p, r, p]
    L.jhq_q8_read.argtypes = [r, p, v, p]
    L.jhq_q8_status.argtypes = []
    L.jhq_current_device = C.PyDLL(L._name).jhq_current_device   # too quick to hand the interpreter's lock back
    L.jhq_current_device.argtypes = []


def q8_rms_norm(x: View, out: Q8Rows, weight: Optional[View] = None, residual: Optional[View] = None,
                residual_out: Optional[View] = None, eps: float = 1e-6, stream: int = 0) -> None:
    """out = 8-bit rows of h * weight / sqrt(mean(h^2) + eps), h = x + residual; residual_out = h."""
    L = _J._lib or _J.load_library()
    _check_places(L, L.jhq_q8_rms_norm, x, residual, weight, residual_out, out)
    rc = L.jhq_q8_rms_norm(x, residual, weight, eps, residual_out, out, stream)
    if rc:
        _J._check(rc)


def q8_matmul(x: Q8Rows, w: Q8Rows, out: View, bias: Optional[View] = None, stream: int = 0) -> None:
    """out[t][n] = (sum_k x.q[t][k] w.q[n][k]) * x.scale[t] * w.scale[n] + bias[n], the sum exact."""
    L = _J._lib or _J.load_library()
    _check_places(L, L.jhq_q8_matmul, x, w, bias, out)
    rc = L.jhq_q8_matmul(x, w, bias, out, stream)
    if rc:
        _J._check(rc)


def q8_write(x: View, cache: Q8Rows, slots=None, stream: int = 0) -> None:
    """Row i of x, quantised, to row slots[i] of the cache (None: row i). slots is a tensor of as many int64s as x has
    rows, or their device address, which is taken unseen; slots outside the cache (-1) are skipped."""
    L = _J._lib or _J.load_library()
    _check_places(L, L.jhq_q8_write, x, cache)
    rc = L.jhq_q8_write(x, slots if slots is None or type(slots) is int else _slots(L, slots, x), cache, stream)
    if rc:
        _J._check(rc)


def q8_read(cache: Q8Rows, out: View, slots=None, stream: int = 0) -> None:
    """Row slots[i] of the cache into row i of out, as scale * q (slots as q8_write takes them, one for each row of out);
    slots outside the cache read as zeros."""
    L = _J._lib or _J.load_library()
    _check_places(L, L.jhq_q8_read, cache, out)
    rc = L.jhq_q8_read(cache, slots if slots is None or type(slots) is int else _slots(L, slots, out), out, stream)
    if rc:
        _J._check(rc)


def q8_check_status() -> None:
    """Raises JHQError (JHQ_ETIMEDOUT) if a device wait of these operators gave up; synchronises."""
    _J._check(_J.load_library().jhq_q8_status())
