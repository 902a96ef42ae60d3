"""The microscaled 4-bit format on the host: what the wrappers refuse, and the plain implementation against itself."""
import numpy as np
import pytest
import torch

import plain_mxfp4 as plain
from fastllm_py_b200.native import mxfp4
from fastllm_py_b200.native.ops import KernelError


def empty(rows, k):
    return mxfp4.Matrix.empty(rows, k, "cpu")


@pytest.mark.parametrize("rows, k", [(1, 1), (128, 128), (129, 129), (300, 4097)])
def test_a_matrix_takes_its_packed_shape_only(rows, k):
    q = empty(rows, k)
    assert q.shape == (rows, k) and q.data.shape == (-(-rows // 128), -(-k // 128), 8704)
    mxfp4.Matrix(q.data, rows, k)
    wide = torch.empty(*q.data.shape[:2], 8720, dtype=torch.uint8)[:, :, :8704]
    for data in (q.data[:, :, :8703], q.data.to(torch.int16), torch.cat([q.data, q.data]), wide[0]) + ((wide,) if q.data.shape != (1, 1, 8704) else ()):
        with pytest.raises(KernelError):
            mxfp4.Matrix(data, rows, k)
    shifted = torch.empty(q.data.numel() + 16, dtype=torch.uint8)
    at = 1 - shifted.data_ptr() % 16 + 16 if shifted.data_ptr() % 16 else 1
    with pytest.raises(KernelError):
        mxfp4.Matrix(shifted[at:at + q.data.numel()].view(q.data.shape), rows, k)
    for r, c in ((0, k), (rows, 0), (-1, k)):
        with pytest.raises(KernelError):
            mxfp4.Matrix(q.data, r, c)


def test_sizes_that_the_kernels_cannot_count_are_refused():
    for rows, k in ((2**31 - 1023, 1), (1, 2**26 - 1023), (2**32 + 1, 128)):
        with pytest.raises(KernelError, match="1 to"):
            mxfp4.Matrix(torch.empty(1, dtype=torch.uint8).expand(-(-rows // 128), -(-k // 128), 8704), rows, k)
    long = torch.empty(2**31 - 1023, 8, dtype=torch.bfloat16, device="meta")
    with pytest.raises(KernelError, match="rows, at most"):
        mxfp4.linear(long, empty(8, 8), torch.empty(2**31 - 1023, 8, dtype=torch.bfloat16, device="meta"))


def test_a_matrix_of_something_else_than_rows_is_refused():
    for x in (torch.zeros(96), torch.zeros(2, 3, 96)):
        with pytest.raises(KernelError, match="is a matrix"):
            mxfp4.Matrix.of(x)


def test_kernels_that_do_not_exist_and_outputs_on_an_operand_are_refused():
    x, w, a = torch.zeros(5, 64, dtype=torch.bfloat16), empty(64, 64), empty(5, 64)
    for kernel in (-1, 3):
        for call in (lambda: mxfp4.linear(x, w, torch.zeros(5, 64), kernel=kernel), lambda: mxfp4.linear_gated(x, w, torch.zeros(5, 32), kernel=kernel),
                     lambda: mxfp4.product(a, w, torch.zeros(5, 64), kernel=kernel)):
            with pytest.raises(KernelError, match="there is no kernel"):
                call()
    for call in (lambda: mxfp4.linear(x, w, x), lambda: mxfp4.linear_gated(x, w, x[:, :32])):
        with pytest.raises(KernelError, match="out lies on x"):
            call()


def test_wrappers_refuse_what_the_kernels_do_not_take():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    w, a = empty(64, 96), empty(5, 96)
    ok = bf(5, 96)
    for x, q, out in ((bf(5, 95), w, bf(5, 64)), (ok, w, bf(5, 63)), (ok, w, bf(4, 64)), (ok.float(), w, bf(5, 64)), (bf(96, 5).t(), w, bf(5, 64)),
                      (bf(5, 97)[:, :96], w, bf(5, 64)), (bf(5, 104)[:, 1:97], w, bf(5, 64)), (bf(480), w, bf(5, 64)), (ok, w, bf(64, 5).t()),
                      (ok, w, bf(1, 64).expand(5, 64)), (bf(1, 96).expand(5, 96), w, bf(5, 64))):
        with pytest.raises(KernelError):
            mxfp4.linear(x, q, out)
    with pytest.raises(KernelError):
        mxfp4.linear(ok, w, bf(5, 64), activation="tanh")
    with pytest.raises(KernelError):
        mxfp4.linear(ok, w, torch.zeros(5, 64, dtype=torch.float16))
    with pytest.raises(KernelError):
        mxfp4.linear_gated(ok, empty(63, 96), bf(5, 31))
    with pytest.raises(KernelError):
        mxfp4.linear_gated(ok, w, bf(5, 64))
    with pytest.raises(KernelError):
        mxfp4.product(a, empty(64, 97), bf(5, 64))
    with pytest.raises(KernelError):
        mxfp4.product(a, w, bf(6, 64))
    for x in (bf(5, 95), bf(5, 96).half(), bf(96, 5).t(), bf(1, 96).expand(5, 96)):
        with pytest.raises(KernelError):
            mxfp4.quantize(x, a)
    for out in (bf(5, 95), bf(5, 96).half(), bf(96, 5).t(), bf(1, 96).expand(5, 96)):
        with pytest.raises(KernelError):
            mxfp4.dequantize(a, out)


def test_wrappers_refuse_the_host():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    for call in (lambda: mxfp4.quantize(bf(5, 96), empty(5, 96)), lambda: mxfp4.dequantize(empty(5, 96), bf(5, 96)),
                 lambda: mxfp4.linear(bf(5, 96), empty(64, 96), bf(5, 64)), lambda: mxfp4.linear_gated(bf(5, 96), empty(64, 96), bf(5, 32)),
                 lambda: mxfp4.product(empty(5, 96), empty(64, 96), bf(5, 64))):
        with pytest.raises(KernelError, match="CUDA device only"):
            call()


def test_plain_packing_and_its_values_agree():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((131, 200)) * 2.0 ** rng.integers(-20, 20, (131, 1))).astype(np.float32)
    s, codes = plain.scales_and_codes(x)
    want = plain.GRID[codes & 7] * np.where(codes & 8, -1, 1) * np.repeat(2.0 ** (s - 127.0), 32, axis=1)[:, :200]
    assert np.array_equal(plain.values(plain.pack(x), 131, 200), want)
    # half a step of the grid at most, the step being 2 at the top, and what saturates: magnitudes in (7, 8) units fall to 6
    unit = np.repeat(2.0 ** (s - 127.0), 32, axis=1)[:, :200]
    assert np.all(np.abs(want - x) <= 2 * unit)
    assert np.all(np.abs(want - x)[np.abs(x) <= 6 * unit] <= unit[np.abs(x) <= 6 * unit])


def test_engine_options():
    from fastllm_py_b200.config import EngineConfig

    assert EngineConfig().weights == "stored" and EngineConfig(weights="mxfp4").dtype == "bfloat16"
    with pytest.raises(ValueError, match="bfloat16"):
        EngineConfig(dtype="float32", weights="mxfp4")
    with pytest.raises(ValueError, match="weights must be"):
        EngineConfig(weights="int4")
