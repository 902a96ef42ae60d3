"""Microscaled 4-bit floating point (MXFP4): matrices held in it, and products with them.

Along K a matrix is cut into blocks of 32 elements of 4 bits (a sign and the magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or
6) that share a scale 2^(s - 127) with a byte s: 4.25 bits a value.  A model's matrices in this form (`Model.load(...,
weights="mxfp4")`) are 3.8 times fewer bytes than in bfloat16, and reading them is what a decode step takes its time for.
The reference has 4-bit weights as integers with float scales (fastllm_py/kernels/marlin.py); this form needs no zero
points, its scales are exact, and the tensor cores of sm_100a multiply it as it is.

    q = mxfp4.Matrix.empty(rows, k, device)   # or Matrix(data, rows, k) over a packed tensor
    mxfp4.quantize(x, q)                      # x float32 or bfloat16
    mxfp4.dequantize(q, out)
    mxfp4.linear(x, q, out)                   # out = x q^T, x bfloat16 as it is
    mxfp4.linear_gated(x, q, out)             # out = act(x gate^T) * (x up^T), q = [gate; up]
    mxfp4.product(a, q, out)                  # out = a q^T, both in 4 bits
    mxfp4.check(device)                       # raises if a product gave up

Everything launches on the current stream of the current device and allocates nothing.  No output may overlap an operand.

A tensor-core kernel whose wait gives up records that in the device's status word, which the engine's other tensor-core kernels share; its
output is not valid, and those of the products after it are not written until the word has been looked at: by `check`, or between an
engine's steps by the engine itself.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_long, c_void_p

import torch

from . import ops
from .ops import KernelError

ROWS, CHUNK_K, CHUNK_BYTES = 128, 128, 8704      # a tile's rows, a chunk's elements along K and its bytes (csrc/mxfp4.cuh)
MOST_ROWS, MOST_K = 2**31 - 1024, 2**26 - 1024   # rows are counted in 32 bits, to the end of their tile; a grid holds 65535 x 8 chunks
LIBRARIES = ["mxfp4", "mxfp4_tc", "gemm_tcgen05"]


class Matrix:
    """A matrix [rows, k] in the packed form: uint8 [ceil(rows / 128), ceil(k / 128), 8704] (csrc/mxfp4.cuh says how a chunk
    lies).  Codes behind k are zero, and so are the scales of whole blocks there; rows behind the last are not read for any
    result."""

    __slots__ = ("data", "rows", "k", "shape")

    def __init__(self, data: torch.Tensor, rows: int, k: int):
        if not (1 <= rows <= MOST_ROWS and 1 <= k <= MOST_K):
            raise KernelError(f"mxfp4: a matrix has 1 to {MOST_ROWS} rows and 1 to {MOST_K} columns, got {rows} x {k}")
        if data.dtype is not torch.uint8 or data.shape != (-(-rows // ROWS), -(-k // CHUNK_K), CHUNK_BYTES) or not data.is_contiguous():
            raise KernelError(f"mxfp4: [{rows}, {k}] packed is a contiguous uint8 tensor "
                              f"{(-(-rows // ROWS), -(-k // CHUNK_K), CHUNK_BYTES)}, got {data.dtype} {tuple(data.shape)}")
        if data.data_ptr() % 16:
            raise KernelError("mxfp4: a packed matrix begins on 16 bytes")
        self.data, self.rows, self.k, self.shape = data, rows, k, (rows, k)

    @classmethod
    def empty(cls, rows: int, k: int, device) -> "Matrix":
        return cls(torch.empty((-(-rows // ROWS), -(-k // CHUNK_K), CHUNK_BYTES), dtype=torch.uint8, device=device), rows, k)

    @classmethod
    def of(cls, x: torch.Tensor) -> "Matrix":
        """x [rows, k] rounded to the format."""
        if x.dim() != 2:
            raise KernelError(f"mxfp4: x is a matrix, got shape {tuple(x.shape)}")
        q = cls.empty(x.shape[0], x.shape[1], x.device)
        quantize(x, q)
        return q

    @property
    def device(self):
        return self.data.device


_device = torch._C._cuda_getDevice               # the current device's index
_raw_stream = ops._raw_stream


def _stream_of(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor | None = None) -> int:
    """The current stream of the device that all are on, which has to be the current one."""
    index = a.get_device()
    if index < 0 or b.get_device() != index or (c is not None and c.get_device() != index):
        tensors = [t for t in (a, b, c) if t is not None]
        if all(t.is_cuda for t in tensors):
            raise KernelError(f"mxfp4: operands on {', '.join(str(t.device) for t in tensors)}")
        raise KernelError("the engine's kernels run on a CUDA device only; got a CPU tensor")
    if index != _device():
        raise KernelError(f"mxfp4: operands on {a.device}, the current device is cuda:{_device()}")
    return _raw_stream(index)


def _rows_of(t: torch.Tensor, what: str) -> int:
    """Elements between the rows of a 2-D tensor whose rows are dense and do not overlap."""
    stride = t.stride()
    if len(stride) == 2 and stride[1] == 1 and stride[0] >= t.shape[1]:
        return stride[0]
    if len(stride) != 2:
        raise KernelError(f"mxfp4: {what} is a matrix, got shape {tuple(t.shape)}")
    rows, cols = t.shape
    if stride[1] != 1 and cols > 1:
        raise KernelError(f"mxfp4: the rows of {what} must be contiguous")
    if stride[0] < cols and rows > 1:
        raise KernelError(f"mxfp4: the rows of {what} overlap")
    return max(stride[0], cols)


def _activations(x: torch.Tensor) -> int:
    pitch = _rows_of(x, "x")
    if x.dtype is not torch.bfloat16:
        raise KernelError(f"mxfp4: activations are bfloat16, got {x.dtype}")
    if pitch % 8 and x.shape[0] == 1:
        pitch = -(-pitch // 8) * 8                               # (a single row has no pitch)
    if pitch % 8 or x.data_ptr() % 16:
        raise KernelError("mxfp4: activations must be 16-byte aligned with a row pitch that is a multiple of 8 elements")
    return pitch


_fns: dict = {}                                  # launchers, and status words by device: looked up once
_QUANTIZE = ("mxfp4", "fl_mx_quantize", [c_void_p, c_int, c_long, c_void_p, c_int, c_int, c_void_p])
_DEQUANTIZE = ("mxfp4", "fl_mx_dequantize", [c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_void_p])
_FEW = ("mxfp4", "fl_mx_few", [c_void_p, c_long, c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_int, c_int, c_int, c_float, c_float,
                               c_int, c_int, c_void_p])
_MANY = ("mxfp4_tc", "fl_mxt_product", [c_void_p, c_long, c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_int, c_int, c_int, c_float,
                                        c_float, c_int, c_int, c_int, c_void_p, c_void_p])
_BOTH = ("mxfp4_tc", "fl_mxq_product", [c_void_p, c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p])


def _fn(which):
    fn = _fns.get(which[1])
    if fn is None:
        fn = _fns[which[1]] = ops._fn(*which)
    return fn


def _known(t: torch.Tensor):
    """(address of the word in which kernels record that they gave up, gemm_tc.status_word, and number of SMs) of t's device."""
    found = _fns.get(t.get_device())
    if found is None:
        from . import gemm_tc
        if torch.cuda.is_current_stream_capturing():
            raise KernelError("mxfp4: run the product once eagerly (or call mxfp4.reserve) before capturing it")
        found = _fns[t.get_device()] = (gemm_tc.status_word(t.device).data_ptr(), ops.sm_count(t.device))
    return found


def reserve(device) -> None:
    """Make what products on `device` share, once, before one is captured into a graph."""
    _known(torch.empty(0, device=device))


def check(device) -> None:
    """Wait for `device` and raise KernelError if a kernel has recorded a fault since the last look: what products have written
    since then is not valid, and may not have been written at all.  The record is cleared, so that products run again."""
    device = torch.device(device)
    if device.type != "cuda":
        raise KernelError(f"the engine's kernels run on a CUDA device only; got {device}")
    if torch.cuda.is_current_stream_capturing():
        raise KernelError("mxfp4.check waits for the device, which a stream that is being captured cannot")
    from . import gemm_tc
    torch.cuda.synchronize(device)
    word = gemm_tc.status_word(device)
    code = int(word.item())
    if code:
        word.zero_()
        raise KernelError(f"mxfp4: a kernel reported error code {code} (a wait that gave up): products since the last check are not valid")


def quantize(x: torch.Tensor, out: Matrix) -> None:
    """out = x [rows, k] (float32 or bfloat16) rounded to nearest, ties to even codes; a block's scale is the power of two that
    puts its largest magnitude into [4, 8) (the codes end at 6), a block that holds a NaN or an infinity becomes NaN."""
    pitch, data = _rows_of(x, "x"), out.data
    if x.shape != out.shape:
        raise KernelError(f"mxfp4.quantize: {tuple(x.shape)} into {out.shape}")
    code, stream = ops.dtype_code(x), _stream_of(x, data)
    rc = (_fns.get("fl_mx_quantize") or _fn(_QUANTIZE))(x.data_ptr(), code, pitch, data.data_ptr(), out.rows, out.k, stream)
    ops._check(rc, "mxfp4.quantize")


def dequantize(q: Matrix, out: torch.Tensor) -> None:
    """out [rows, k] (float32 or bfloat16) = the values that q stands for, exact in both types."""
    pitch, data = _rows_of(out, "out"), q.data
    if out.shape != q.shape:
        raise KernelError(f"mxfp4.dequantize: {q.shape} into {tuple(out.shape)}")
    code, stream = ops.dtype_code(out), _stream_of(data, out)
    rc = (_fns.get("fl_mx_dequantize") or _fn(_DEQUANTIZE))(data.data_ptr(), out.data_ptr(), code, pitch, q.rows, q.k, stream)
    ops._check(rc, "mxfp4.dequantize")


# The kernel for few rows takes up to 8 of them, and no more time than those on the tensor cores with matrices of up to 2^26 values
# (one row, 4096 -> 12288: 10.1 and 13.9 us); with larger ones their launcher says which does (LESS: fl_mx_few, csrc/mxfp4_tc.cu).
FEW_ROWS, FEW_VALUES, LESS = 8, 1 << 26, -1


def _times_weights(name, x, w: Matrix, out, gated, n, activation, params, constant_w, kernel) -> None:
    pitch, out_pitch, data = _activations(x), _rows_of(out, "out"), w.data
    m, k = x.shape
    if w.k != k or out.shape != (m, n) or (gated and w.rows % 2):
        raise KernelError(f"mxfp4.{name}: {tuple(x.shape)} x {w.shape}^T -> {tuple(out.shape)}")
    if kernel and kernel not in (1, 2):
        raise KernelError(f"mxfp4.{name}: there is no kernel {kernel}")
    if m > MOST_ROWS:
        raise KernelError(f"mxfp4.{name}: {m} rows, at most {MOST_ROWS}")
    from_x, to = x.data_ptr(), out.data_ptr()
    if from_x == to and m > 0:
        raise KernelError(f"mxfp4.{name}: out lies on x, which the kernels read while they write")
    if activation is None and not gated:
        act = -1
    else:
        act = ops.activation_code(activation)                    # (a gated product without a unit would leave its up half out)
    code, stream = ops.dtype_code(out), _stream_of(x, data, out)
    if m == 0:
        return
    status, sms = _known(x)
    rc = LESS
    if kernel or m > FEW_ROWS or w.rows * k > FEW_VALUES:
        rc = _fn(_MANY)(from_x, pitch, data.data_ptr(), to, code, out_pitch, m, n, k, gated, act, params[0], params[1], constant_w, kernel,
                        sms, status, stream)
    if rc == LESS:
        rc = _fn(_FEW)(from_x, pitch, data.data_ptr(), to, code, out_pitch, m, n, k, gated, act, params[0], params[1], constant_w, sms, stream)
    ops._check(rc, name)


def linear(x: torch.Tensor, w: Matrix, out: torch.Tensor, activation: str | None = None, params=(0.0, 0.0),
           constant_w: bool = False, kernel: int = 0) -> None:
    """out[m, n] (bfloat16 or float32) = x[m, k] @ w[n, k]^T; x bfloat16 (16-byte aligned, its row pitch a multiple of 8
    elements), products and sums in float.  `activation` (`ops.ACTIVATIONS`, f(v, 1)) is applied on the way out.  `constant_w`
    says that nothing that may still be running writes w (a model's matrix, written long since), so that its first bytes may be
    read while the kernels before this one in the stream run.  `kernel`: 0 the one that suits the sizes, 1 the tensor-core kernel on
    tiles, 2 the one on pairs of CTAs."""
    _times_weights("linear", x, w, out, 0, w.rows, activation, params, constant_w, kernel)


def linear_gated(x: torch.Tensor, w: Matrix, out: torch.Tensor, activation: str = "silu", params=(0.0, 0.0),
                 constant_w: bool = False, kernel: int = 0) -> None:
    """out[m, i] = act(x @ gate^T) * (x @ up^T) for w = [gate; up] stacked as [2 i, k] (any i: the halves' border may lie
    inside a row tile); both products stay in float until the unit (`ops.ACTIVATIONS`, with its `params`) has been applied.
    `constant_w` and `kernel` as in `linear`."""
    _times_weights("linear_gated", x, w, out, 1, w.rows // 2, activation, params, constant_w, kernel)


def product(a: Matrix, b: Matrix, out: torch.Tensor, kernel: int = 0) -> None:
    """out[m, n] (bfloat16 or float32) = a[m, k] @ b[n, k]^T, both in 4 bits; sums in float.  `kernel`: 0 the one that suits the
    sizes, 1 the one on tiles, 2 the one on pairs of CTAs."""
    out_pitch = _rows_of(out, "out")
    if b.k != a.k or out.shape != (a.rows, b.rows):
        raise KernelError(f"mxfp4.product: {a.shape} x {b.shape}^T -> {tuple(out.shape)}")
    if kernel not in (0, 1, 2):
        raise KernelError(f"mxfp4.product: there is no kernel {kernel}")
    code, x, w = ops.dtype_code(out), a.data, b.data
    stream = _stream_of(x, w, out)
    status, sms = _known(x)
    ops._check(_fn(_BOTH)(x.data_ptr(), w.data_ptr(), out.data_ptr(), code, out_pitch, a.rows, b.rows, a.k, kernel, sms, status, stream),
               "mxfp4.product")
