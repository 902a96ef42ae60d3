"""Calls of the 4-bit operators that the documentation allows: what they record, capture and count, and every kernel with the values that
it can go wrong at.  Tolerances are those that tests/test_mxfp4_gpu.py derives."""
import numpy as np
import pytest
import torch

import plain_mxfp4 as plain
from test_mxfp4_gpu import DEV, bf16, check_gated, check_sum, matrix, operands, rows_in

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", [1, 2])
def test_check_raises_a_recorded_fault_and_products_run_again(kernel):
    """Products after a fault leave their outputs as they were, without an error: `check` tells, once."""
    from fastllm_py_b200.native import gemm_tc, mxfp4
    from fastllm_py_b200.native.ops import KernelError

    m, n, k = 40, 300, 264
    x, data, w = operands(m, n, k, 1)
    xs, q, out = rows_in(x, torch.bfloat16), matrix(data, n, k), torch.full((m, n), 7.0, dtype=torch.bfloat16, device=DEV)
    mxfp4.check(DEV)
    word = gemm_tc.status_word(torch.device(DEV))
    try:
        word.fill_(121)
        mxfp4.linear(xs, q, out, kernel=kernel)
        with pytest.raises(KernelError, match="121"):
            mxfp4.check(DEV)
    finally:
        word.zero_()
    assert bool((out == 7.0).all())
    mxfp4.linear(xs, q, out, kernel=kernel)
    mxfp4.check("cuda")
    check_sum(out, x @ w.T, np.abs(x) @ np.abs(w).T, k, torch.bfloat16)
