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

Everything launches on the current stream of the current device and allocates nothing.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_long, c_void_p

import torch

from . import ops
from .ops import KernelError

ROWS, CHUNK_K, CHUNK_BYTES = 128, 128, 8704      # a tile's rows, a chunk's elements along K and its bytes (csrc/mxfp4.cu)
LIBRARIES = ["mxfp4"]


class Matrix:
    """A matrix [rows, k] in the packed form: uint8 [ceil(rows / 128), ceil(k / 128), 8704] (csrc/mxfp4.cu says how a chunk
    lies).  Codes behind k are zero; rows behind the last are not read for any result."""

    __slots__ = ("data", "rows", "k")

    def __init__(self, data: torch.Tensor, rows: int, k: int):
        if rows < 1 or k < 1:
            raise KernelError(f"mxfp4: a matrix has rows and columns, got {rows} x {k}")
        if data.dtype is not torch.uint8 or data.shape != (-(-rows // ROWS), -(-k // CHUNK_K), CHUNK_BYTES) or not data.is_contiguous():
            raise KernelError(f"mxfp4: [{rows}, {k}] packed is a contiguous uint8 tensor "
                              f"{(-(-rows // ROWS), -(-k // CHUNK_K), CHUNK_BYTES)}, got {data.dtype} {tuple(data.shape)}")
        if data.data_ptr() % 16:
            raise KernelError("mxfp4: a packed matrix begins on 16 bytes")
        self.data, self.rows, self.k = data, rows, k

    @classmethod
    def empty(cls, rows: int, k: int, device) -> "Matrix":
        return cls(torch.empty((-(-rows // ROWS), -(-k // CHUNK_K), CHUNK_BYTES), dtype=torch.uint8, device=device), rows, k)

    @classmethod
    def of(cls, x: torch.Tensor) -> "Matrix":
        """x [rows, k] rounded to the format."""
        q = cls.empty(x.shape[0], x.shape[1], x.device)
        quantize(x, q)
        return q

    @property
    def shape(self):
        return (self.rows, self.k)

    @property
    def device(self):
        return self.data.device


def _launch_stream(*tensors) -> int:
    """The current stream of the device that all tensors are on, which has to be the current one."""
    device = tensors[0].device
    if device.type != "cuda":
        raise KernelError("the engine's kernels run on a CUDA device only; got a CPU tensor")
    for t in tensors[1:]:
        if t.device != device:
            raise KernelError(f"mxfp4: operands on {device} and {t.device}")
    if device.index != torch.cuda.current_device():
        raise KernelError(f"mxfp4: operands on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return ops._raw_stream(device.index)


def _rows_of(t: torch.Tensor, what: str) -> int:
    """Elements between the rows of a 2-D tensor whose rows are dense and do not overlap."""
    if t.dim() != 2:
        raise KernelError(f"mxfp4: {what} is a matrix, got shape {tuple(t.shape)}")
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise KernelError(f"mxfp4: the rows of {what} must be contiguous")
    if rows > 1 and t.stride(0) < cols:
        raise KernelError(f"mxfp4: the rows of {what} overlap")
    return t.stride(0) if rows > 1 else max(t.stride(0), cols)


def quantize(x: torch.Tensor, out: Matrix) -> None:
    """out = x [rows, k] (float32 or bfloat16) rounded to nearest, ties to even codes; a block's scale is the power of two that
    puts its largest magnitude into [4, 8) (the codes end at 6), a block that holds a NaN or an infinity becomes NaN."""
    ld = _rows_of(x, "x")
    if tuple(x.shape) != out.shape:
        raise KernelError(f"mxfp4.quantize: {tuple(x.shape)} into {out.shape}")
    code, stream = ops.dtype_code(x), _launch_stream(x, out.data)
    fn = ops._fn("mxfp4", "fl_mx_quantize", [c_void_p, c_int, c_long, c_void_p, c_int, c_int, c_void_p])
    ops._check(fn(x.data_ptr(), code, ld, out.data.data_ptr(), out.rows, out.k, stream), "mxfp4.quantize")


def dequantize(q: Matrix, out: torch.Tensor) -> None:
    """out [rows, k] (float32 or bfloat16) = the values that q stands for, exact in both types."""
    ld = _rows_of(out, "out")
    if tuple(out.shape) != q.shape:
        raise KernelError(f"mxfp4.dequantize: {q.shape} into {tuple(out.shape)}")
    code, stream = ops.dtype_code(out), _launch_stream(q.data, out)
    fn = ops._fn("mxfp4", "fl_mx_dequantize", [c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_void_p])
    ops._check(fn(q.data.data_ptr(), out.data_ptr(), code, ld, q.rows, q.k, stream), "mxfp4.dequantize")


def _product(name, x, x_ptr, ldx, m, k, w: Matrix, out, gated, activation, params) -> None:
    n = w.rows // 2 if gated else w.rows
    ldo = _rows_of(out, "out")
    if w.k != k or tuple(out.shape) != (m, n) or (gated and w.rows % 2):
        raise KernelError(f"mxfp4.{name}: [{m}, {k}] x {w.shape}^T -> {tuple(out.shape)}")
    act = -1 if activation is None else ops.activation_code(activation)
    code = ops.dtype_code(out)
    stream = _launch_stream(out, x, w.data)
    fn = ops._fn("mxfp4", "fl_mx_product", [c_void_p, c_long, c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_int, c_int, c_int,
                                            c_float, c_float, c_void_p])
    if m == 0:
        return
    if ldx:
        fn = ops._fn("mxfp4_tc", "fl_mxt_product", [c_void_p, c_long, c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_int, c_int, c_int,
                                                    c_float, c_float, c_int, c_void_p, c_void_p])
        from . import gemm_tc
        rc = fn(x_ptr, ldx, w.data.data_ptr(), out.data_ptr(), code, ldo, m, n, k, int(gated), act, params[0], params[1],
                ops.sm_count(out.device), gemm_tc.status_word(out.device).data_ptr(), stream)
        if rc != -1:
            ops._check(rc, f"mxfp4.{name}")
            return
    else:
        fn2 = ops._fn("mxfp4_tc", "fl_mxq_product", [c_void_p, c_void_p, c_void_p, c_int, c_long, c_int, c_int, c_int, c_int, c_void_p, c_void_p])
        from . import gemm_tc
        rc = fn2(x_ptr, w.data.data_ptr(), out.data_ptr(), code, ldo, m, n, k, ops.sm_count(out.device),
                 gemm_tc.status_word(out.device).data_ptr(), stream)
        if rc != -1:
            ops._check(rc, f"mxfp4.{name}")
            return
    ops._check(fn(x_ptr, ldx, w.data.data_ptr(), out.data_ptr(), code, ldo, m, n, k, int(gated), act,
                  float(params[0]), float(params[1]), stream), f"mxfp4.{name}")


def _activations(x: torch.Tensor) -> int:
    ld = _rows_of(x, "x")
    if x.dtype is not torch.bfloat16:
        raise KernelError(f"mxfp4: activations are bfloat16, got {x.dtype}")
    if x.shape[0] == 1:
        ld = -(-ld // 8) * 8                                     # (a single row has no pitch)
    if ld % 8 or x.data_ptr() % 16:
        raise KernelError("mxfp4: activations must be 16-byte aligned with a row pitch that is a multiple of 8 elements")
    return ld


def linear(x: torch.Tensor, w: Matrix, out: torch.Tensor, activation: str | None = None, params=(0.0, 0.0)) -> None:
    """out[m, n] (bfloat16 or float32) = x[m, k] @ w[n, k]^T; x bfloat16 (16-byte aligned, its row pitch a multiple of 8
    elements), products and sums in float.  `activation` (`ops.ACTIVATIONS`, f(v, 1)) is applied on the way out."""
    ld = _activations(x)
    _product("linear", x, x.data_ptr(), ld, x.shape[0], x.shape[1], w, out, False, activation, params)


def linear_gated(x: torch.Tensor, w: Matrix, out: torch.Tensor, activation: str = "silu", params=(0.0, 0.0)) -> None:
    """out[m, i] = act(x @ gate^T) * (x @ up^T) for w = [gate; up] stacked as [2 i, k] (any i: the halves' border may lie
    inside a row tile); both products stay in float until the unit (`ops.ACTIVATIONS`, with its `params`) has been applied."""
    ld = _activations(x)
    _product("linear_gated", x, x.data_ptr(), ld, x.shape[0], x.shape[1], w, out, True, activation, params)


def product(a: Matrix, b: Matrix, out: torch.Tensor) -> None:
    """out[m, n] (bfloat16 or float32) = a[m, k] @ b[n, k]^T, both in 4 bits; sums in float."""
    _product("product", a.data, a.data.data_ptr(), 0, a.rows, a.k, b, out, False, None, (0.0, 0.0))
