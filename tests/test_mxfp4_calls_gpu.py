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


# ------------------------------------------------------------------------------------------------ captured and replayed

@pytest.mark.parametrize("m", [1, 5, 12, 90, 400])
def test_a_replayed_feed_forward_takes_the_activations_of_the_moment(m):
    """A captured layer replayed with other activations in the same place gives what the eager calls give for those, bit for bit."""
    from fastllm_py_b200.native import mxfp4

    hidden, inter = 264, 712
    rng = np.random.default_rng(m)
    q1 = mxfp4.Matrix.of(torch.from_numpy((rng.standard_normal((2 * inter, hidden)) / np.sqrt(hidden)).astype(np.float32)).to(DEV))
    q2 = mxfp4.Matrix.of(torch.from_numpy((rng.standard_normal((hidden, inter)) / np.sqrt(inter)).astype(np.float32)).to(DEV))
    inputs = [rows_in(bf16(rng.standard_normal((m, hidden))), torch.bfloat16) for _ in range(3)]
    xs, act = torch.empty_like(inputs[0]), torch.empty(m, inter, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(m, hidden, dtype=torch.bfloat16, device=DEV)

    def run():
        mxfp4.linear_gated(xs, q1, act)
        mxfp4.linear(act, q2, out)

    want = []
    for x in inputs:
        xs.copy_(x)
        run()
        want.append((act.clone(), out.clone()))
    assert not torch.equal(want[0][1], want[1][1]) and not torch.equal(want[1][1], want[2][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in (1, 2, 0, 1):
        xs.copy_(inputs[i])
        act.fill_(0), out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(act, want[i][0]) and torch.equal(out, want[i][1]), i
    w1 = plain.values(q1.data.cpu().numpy(), q1.rows, q1.k)
    check_gated(want[1][0], inputs[1].double().cpu().numpy(), w1, "silu", (0, 0), hidden, torch.bfloat16)


FIRST_CAPTURE = '''
import torch
from fastllm_py_b200.native import mxfp4
dev = "cuda:0"
g = torch.Generator(device=dev).manual_seed(1)
xs = [torch.randn(m, 264, generator=g, device=dev).to(torch.bfloat16) for m in (3, 40, 700)]
x32 = torch.randn(1424, 264, generator=g, device=dev)
q, back = mxfp4.Matrix.empty(1424, 264, dev), torch.empty(1424, 264, device=dev)
a = mxfp4.Matrix.empty(700, 264, dev)
def outputs():
    return [torch.zeros(x.shape[0], n, dtype=torch.bfloat16, device=dev) for x in xs for n in (1424, 712)] + [
        torch.zeros(700, 1424, dtype=torch.bfloat16, device=dev) for _ in range(2)]
def run(outs):
    mxfp4.quantize(x32, q)
    mxfp4.dequantize(q, back)
    mxfp4.quantize(xs[2], a)
    for i, x in enumerate(xs):
        for kernel in ((0,) if i == 0 else (1, 2)):
            mxfp4.linear(x, q, outs[2 * i], kernel=kernel)
            mxfp4.linear_gated(x, q, outs[2 * i + 1], kernel=kernel)
    mxfp4.product(a, q, outs[6], kernel=1)
    mxfp4.product(a, q, outs[7], kernel=2)
mxfp4.reserve(dev)
captured = outputs()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run(captured)
graph.replay()
torch.cuda.synchronize()
got = [o.clone() for o in captured] + [back.clone()]
eager = outputs()
run(eager)
mxfp4.check(dev)
assert all(torch.equal(a, b) for a, b in zip(got, eager + [back]))
assert all(bool(o.any()) for o in got)
print("same")
'''


def test_the_first_calls_of_a_process_may_be_captured():
    """After `reserve` nothing has to run eagerly before it is captured: a process whose first products are in a graph."""
    import subprocess
    import sys
    from pathlib import Path

    done = subprocess.run([sys.executable, "-c", FIRST_CAPTURE], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0 and "same" in done.stdout, done.stdout + done.stderr


# ------------------------------------------------------------------------------------------------ extreme and other values, on every kernel

KERNELS = [(0, 5), (1, 1), (1, 20), (1, 70), (1, 200), (2, 3), (2, 200), (2, 300)]


@pytest.mark.parametrize("kernel, m", KERNELS)
def test_extreme_scales_in_every_kernel(kernel, m):
    """Weights with scales from 2^-123 to 2^118 (a row of blocks whose factor takes two steps beside ordinary ones), the smallest and
    the largest scale, blocks that are NaN; K of one chunk and a half, features that end inside a tile."""
    from fastllm_py_b200.native import mxfp4

    n, k = 300, 192
    rng = np.random.default_rng(10 * m + kernel)
    e = rng.integers(-120, 121, n)
    data = plain.pack((rng.standard_normal((n, k)) * 2.0 ** e[:, None]).astype(np.float32))
    code, shift, scale = plain.addresses(n, k)
    flat = data.reshape(-1)
    flat[scale[3]], flat[scale[4]], flat[scale[5, 64:96]], flat[scale[299, :32]] = 0, 252, 255, 255
    w = plain.values(data, n, k)
    x = bf16(rng.standard_normal((m, k)) * 2.0 ** -20)
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.linear(rows_in(x, torch.bfloat16), matrix(data, n, k), out, kernel=kernel)
    mxfp4.check(DEV)
    nan = [5, 299]
    assert bool(torch.isnan(out[:, nan]).all())
    ok = [j for j in range(n) if j not in nan]
    check_sum(out[:, ok], x @ w[ok].T, np.abs(x) @ np.abs(w[ok]).T, k, torch.float32)


@pytest.mark.parametrize("kernel, m", KERNELS)
def test_gated_units_with_extreme_scales_in_every_kernel(kernel, m):
    """Gate and up rows with scales from 2^-63 to 2^48 that meet in one unit; with silu, a block that is NaN in a gate row and in an
    up row makes those features NaN and no other."""
    from fastllm_py_b200.native import mxfp4

    n, k = 150, 192
    rng = np.random.default_rng(10 * m + kernel)
    x = bf16(rng.standard_normal((m, k)))
    xs = rows_in(x, torch.bfloat16)
    e = rng.integers(-60, 51, 2 * n)
    data = plain.pack((rng.standard_normal((2 * n, k)) * 2.0 ** e[:, None]).astype(np.float32))
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.linear_gated(xs, matrix(data, 2 * n, k), out, "relu", kernel=kernel)
    check_gated(out, x, plain.values(data, 2 * n, k), "relu", (0, 0), k, torch.float32)
    data = plain.pack((rng.standard_normal((2 * n, k)) / np.sqrt(k)).astype(np.float32))
    _, _, scale = plain.addresses(2 * n, k)
    data.reshape(-1)[scale[7, 32:64]] = data.reshape(-1)[scale[n + 140, 160:]] = 255
    mxfp4.linear_gated(xs, matrix(data, 2 * n, k), out, kernel=kernel)
    mxfp4.check(DEV)
    assert bool(torch.isnan(out[:, [7, 140]]).all())
    ok = [j for j in range(n) if j not in (7, 140)]
    w = plain.values(data, 2 * n, k)
    check_gated(out[:, ok], x, w[ok + [n + j for j in ok]], "silu", (0, 0), k, torch.float32)


@pytest.mark.parametrize("kernel, m", KERNELS)
def test_a_token_that_is_not_finite_in_every_kernel(kernel, m):
    """An infinity and a NaN in tokens of their own concern those tokens; what lies between the rows and behind the last is not read."""
    from fastllm_py_b200.native import mxfp4

    n, k = 280, 200
    x, data, w = operands(m, n, k, m)
    x[m // 2, 7] = np.inf
    if m > 4:
        x[m - 1, 150] = np.nan
    bad = {m // 2, m - 1} if m > 4 else {m // 2}
    buf = torch.full((m + 3, 208), float("nan"), dtype=torch.bfloat16, device=DEV)
    buf[:m, :k] = torch.from_numpy(x).to(DEV).to(torch.bfloat16)
    q = matrix(data, n, k)
    out = torch.full((m + 3, n), -5.0, dtype=torch.bfloat16, device=DEV)
    unit = torch.full((m + 3, n // 2), -5.0, dtype=torch.bfloat16, device=DEV)
    mxfp4.linear(buf[:m, :k], q, out[:m], kernel=kernel)
    mxfp4.linear_gated(buf[:m, :k], q, unit[:m], kernel=kernel)
    mxfp4.check(DEV)
    assert bool((out[m:] == -5.0).all()) and bool((unit[m:] == -5.0).all())
    assert not bool(torch.isfinite(out[sorted(bad)]).any())
    keep = [t for t in range(m) if t not in bad]
    if keep:
        check_sum(out[keep], x[keep] @ w.T, np.abs(x[keep]) @ np.abs(w).T, k, torch.bfloat16)
        check_gated(unit[keep], x[keep], w, "silu", (0, 0), k, torch.bfloat16)


@pytest.mark.parametrize("act", ["silu", "relu", "gelu_tanh", "clamped_swish", "relu_squared"])
@pytest.mark.parametrize("kernel, m", [(1, 3), (1, 70), (2, 3), (2, 70), (2, 300)])
def test_every_activation_in_every_kernel(kernel, m, act):
    """In units and of one argument; the bounds are those of test_mxfp4_gpu.test_every_activation."""
    from fastllm_py_b200.native import mxfp4

    n, k = 200, 300
    params = (1.25, 1.5) if act == "clamped_swish" else (0.0, 0.0)
    x, data, w = operands(m, 2 * n, k, m)
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.linear_gated(rows_in(x, torch.bfloat16), matrix(data, 2 * n, k), out, act, params, kernel=kernel)
    check_gated(out, x, w, act, params, k, torch.float32)
    one = torch.empty(m, 2 * n, dtype=torch.float32, device=DEV)
    mxfp4.linear(rows_in(x, torch.bfloat16), matrix(data, 2 * n, k), one, activation=act, params=params, kernel=kernel)
    y = x @ w.T
    e = (k / 16 + 64) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    want = plain.unit(act, y, np.ones_like(y), params)
    bound = 1.5 * np.maximum(*(np.abs(plain.unit(act, y + s * e, np.ones_like(y), params) - want) for s in (-1, 1))) + 2.0 ** -18 * np.abs(want) + 2.0 ** -22 * np.abs(y) + 2.0 ** -24
    off = np.abs(one.double().cpu().numpy() - want)
    assert np.all(off <= bound), float((off / bound).max())


# ------------------------------------------------------------------------------------------------ both operands in 4 bits

def with_scales(rows, k, scales, seed):
    """Random codes (of both signs, zeros among them) with scale byte scales[r, block] of each row's blocks."""
    rng = np.random.default_rng(seed)
    data = np.zeros((-(-rows // 128), -(-k // 128), plain.CHUNK), dtype=np.uint8)
    code, shift, scale = plain.addresses(rows, k)
    flat = data.reshape(-1)
    np.bitwise_or.at(flat, code, (rng.integers(0, 16, (rows, k)) << shift).astype(np.uint8))
    flat[scale] = np.repeat(scales, 32, axis=1)[:, :k].astype(np.uint8)
    return data


@pytest.mark.parametrize("kernel, m", [(0, 5), (1, 1), (1, 70), (1, 200), (2, 3), (2, 300)])
def test_product_with_scales_that_meet_in_range(kernel, m):
    """Scale bytes over their whole range in a, the opposite ones in b, so that every product of two scales lies within float's normal
    numbers and the sums are exact up to their rounding: 0 against 252, 252 against 0, and all between."""
    from fastllm_py_b200.native import mxfp4

    n, k = 300, 328
    blocks = -(-k // 32)
    rng = np.random.default_rng(m + kernel)
    per_block = rng.permutation(np.r_[0, 252, 2, 250, rng.integers(20, 230, blocks - 4)])
    sa = np.broadcast_to(per_block, (m, blocks))
    sb = np.broadcast_to(252 - per_block, (n, blocks)) + rng.integers(-4, 5, (n, blocks))
    sb = np.clip(sb, 0, 252)
    a_data, b_data = with_scales(m, k, sa, 1), with_scales(n, k, sb, 2)
    a, b = plain.values(a_data, m, k), plain.values(b_data, n, k)
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.product(matrix(a_data, m, k), matrix(b_data, n, k), out, kernel=kernel)
    mxfp4.check(DEV)
    check_sum(out, a @ b.T, np.abs(a) @ np.abs(b).T, k, torch.float32)


@pytest.mark.parametrize("kernel, m", [(0, 5), (1, 1), (1, 70), (1, 200), (2, 3), (2, 300)])
def test_product_beyond_the_range_of_float(kernel, m):
    """Row kinds of a against row kinds of b: scales so small that every product underflows, so large that it overflows, blocks of zeros
    against the largest scales, and blocks that are NaN.  What float cannot hold is an infinity, what is below it zero or nearly; a
    zero times a number is zero whatever their scales, and a row that is NaN leaves the others alone."""
    from fastllm_py_b200.native import mxfp4

    n, k = 260, 160
    blocks = k // 32
    rng = np.random.default_rng(3)
    kinds = {"plain": 107, "tiny": 0, "huge": 252, "zero": 252, "nan": 107}
    names = list(kinds)

    def make(rows, seed):
        kind = np.arange(rows) % len(names)
        scales = np.array([kinds[names[i]] for i in kind])[:, None] + np.zeros((1, blocks), dtype=np.int64)
        data = with_scales(rows, k, scales, seed)
        code, shift, scale = plain.addresses(rows, k)
        flat = data.reshape(-1)
        for r in range(rows):
            if names[kind[r]] == "huge":             # all of one sign and none zero: sums overflow in any order, to one infinity
                np.bitwise_and.at(flat, code[r], (~(0xF << shift[r])).astype(np.uint8))
                np.bitwise_or.at(flat, code[r], (rng.integers(1, 8, k) << shift[r]).astype(np.uint8))
            elif names[kind[r]] == "zero":
                np.bitwise_and.at(flat, code[r], (~(0xF << shift[r])).astype(np.uint8))
            elif names[kind[r]] == "nan":
                flat[scale[r, 64:96]] = 255
        return data, kind

    a_data, ka = make(m, 4)
    b_data, kb = make(n, 5)
    a, b = plain.values(a_data, m, k), plain.values(b_data, n, k)
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.product(matrix(a_data, m, k), matrix(b_data, n, k), out, kernel=kernel)
    mxfp4.check(DEV)
    got = out.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want, absolute = a @ b.T, np.abs(a) @ np.abs(b).T
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    huge = ~nan & (np.abs(want) > 2.0 ** 130)
    # (a row of one sign against one of both may pass through either infinity; against one of its own kind it has a sign)
    both = (ka == names.index("huge"))[:, None] & (kb == names.index("huge"))[None, :]
    assert np.all(got[both] == np.inf) and both.sum() == huge.sum()
    rest = ~nan & ~huge
    bound = (k / 16 + 64) * 2.0 ** -23 * absolute + 2 * k * 2.0 ** -149
    bound = bound + 2.0 ** -24 * (np.abs(want) + bound)
    assert np.all(np.abs(got - want)[rest] <= bound[rest]), [(names[ka[i]], names[kb[j]], got[i, j], want[i, j]) for i, j in np.argwhere(rest & ~(np.abs(got - want) <= bound))[:6]]
