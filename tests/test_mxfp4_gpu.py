"""The kernels of the microscaled 4-bit format against plain implementations in 64 bits (tests/plain_mxfp4.py).

Tolerances.  Rounding to the format is exact arithmetic: bytes are equal.  A product's operands are exact, every product of two
elements is exact in float, and the sum of k of them is off by at most `steps` 2^-23 sum |a| |b| where no partial sum takes
part in more than `steps` additions, each off by no more than a whole step of float (an addition that truncates): 64 more than
k / 16 covers one accumulation per 16 elements, the sums within a matrix instruction and the joining of parts.  Below 2^-126
float's step is 2^-149 whatever the value: k products and k sums add at most 2 k 2^-149.  The result is then rounded once: half
a step of its type."""
import numpy as np
import pytest
import torch

import plain_mxfp4 as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def matrix(data, rows, k):
    from fastllm_py_b200.native import mxfp4

    return mxfp4.Matrix(torch.from_numpy(np.ascontiguousarray(data)).to(DEV), rows, k)


def rows_in(x, dtype, pad=0):
    """x as a device tensor of rows with `pad` elements of 7 and a multiple of 8 between them."""
    m, k = x.shape
    buf = torch.full((m, -(-k // 8) * 8 + pad), 7.0, dtype=dtype, device=DEV)
    buf[:, :k] = torch.from_numpy(np.ascontiguousarray(x)).to(DEV).to(dtype)
    return buf[:, :k]


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).double().numpy()


def check_sum(got, want, absolute, k, dtype):
    """|got - want| within the bound above; where `want` is not finite the same kind of value."""
    got = got.double().cpu().numpy()
    bound = (k / 16 + 64) * 2.0 ** -23 * absolute + 2 * k * 2.0 ** -149
    bound = bound + half_step(dtype) * (np.abs(want) + bound)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(got - want)[fine]
    assert np.all(off <= bound[fine]), float((off / np.maximum(bound[fine], 1e-300)).max())


# ------------------------------------------------------------------------------------------------------------- rounding

def awkward(rows, k, dtype, seed):
    """Values of every size, ties of the grid, zeros of both signs, subnormals, blocks of zeros."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-12, 12, (rows, k))
    x[rng.random((rows, k)) < 0.05] = 0.0
    x[rng.random((rows, k)) < 0.02] = -0.0
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5, 0.2490234375, 5.03125])
    for r in range(0, rows, 3):
        e = 2.0 ** rng.integers(-100, 100)
        x[r] = rng.choice(ties, k) * rng.choice([-1, 1], k) * e
    if rows > 4:
        x[4] = rng.standard_normal(k) * 1e-39
        x[1, : min(k, 64)] = 0.0
    if rows > 5:
        x[5] = rng.standard_normal(k) * 1e38
    return torch.from_numpy(x).float().to(dtype).float().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, k, pad", [(1, 1, 0), (1, 128, 0), (7, 31, 0), (8, 33, 3), (9, 200, 8), (127, 127, 1), (130, 260, 0),
                                          (300, 1000, 5), (5, 4096, 0)])
def test_rounding_is_exact(rows, k, pad, dtype):
    from fastllm_py_b200.native import mxfp4

    x = awkward(rows, k, dtype, rows + k)
    buf = torch.full((rows, k + pad), 3.0, dtype=dtype, device=DEV)
    buf[:, :k] = torch.from_numpy(x).to(DEV).to(dtype)
    q = mxfp4.Matrix.empty(rows, k, DEV)
    q.data.fill_(0xA5)
    mxfp4.quantize(buf[:, :k], q)
    out = torch.full((rows, k + pad), -5.0, dtype=dtype, device=DEV)
    mxfp4.dequantize(q, out[:, :k])
    torch.cuda.synchronize()
    assert np.array_equal(q.data.cpu().numpy(), plain.pack(x))              # codes behind k and rows behind the last are zero too
    want = plain.values(plain.pack(x), rows, k)
    assert np.array_equal(out[:, :k].double().cpu().numpy(), want)
    assert bool((out[:, k:] == -5.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rounding_of_a_shifted_view(dtype):
    """Rows that begin on no 16-byte boundary."""
    from fastllm_py_b200.native import mxfp4

    x = awkward(20, 300, dtype, 3)
    buf = torch.zeros((20, 303), dtype=dtype, device=DEV)
    buf[:, 1:301] = torch.from_numpy(x).to(DEV).to(dtype)
    q = mxfp4.Matrix.of(buf[:, 1:301])
    out = torch.zeros((20, 303), dtype=dtype, device=DEV)
    mxfp4.dequantize(q, out[:, 1:301])
    assert np.array_equal(q.data.cpu().numpy(), plain.pack(x))
    assert np.array_equal(out[:, 1:301].double().cpu().numpy(), plain.values(plain.pack(x), 20, 300))
    assert bool((out[:, 0] == 0).all()) and bool((out[:, 301:] == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_block_with_a_value_that_is_not_finite_is_nan(bad):
    from fastllm_py_b200.native import mxfp4

    x = awkward(10, 100, torch.float32, 5)
    x[2, 40], x[9, 99] = bad, bad
    q = mxfp4.Matrix.of(torch.from_numpy(x).to(DEV))
    out = torch.empty(10, 100, device=DEV)
    mxfp4.dequantize(q, out)
    assert np.array_equal(q.data.cpu().numpy(), plain.pack(x))
    want = np.zeros((10, 100), dtype=bool)
    want[2, 32:64] = want[9, 96:] = True
    assert np.array_equal(torch.isnan(out).cpu().numpy(), want)


def test_every_code_and_scale():
    """All 256 scales with all 16 codes, into float32 and (as far as it reaches) bfloat16."""
    from fastllm_py_b200.native import mxfp4

    rows, k = 256, 32
    data = np.zeros((2, 1, plain.CHUNK), dtype=np.uint8)
    code, shift, scale = plain.addresses(rows, k)
    flat = data.reshape(-1)
    np.bitwise_or.at(flat, code, ((np.arange(k)[None, :] % 16) << shift).astype(np.uint8))
    flat[scale] = np.arange(256, dtype=np.uint8)[:, None]
    want = plain.values(data, rows, k)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.empty(rows, k, dtype=dtype, device=DEV)
        mxfp4.dequantize(matrix(data, rows, k), out)
        with np.errstate(over="ignore"):
            expect = want.astype(np.float32).astype(np.float64)            # 4 and 6 times 2^127 and the like overflow
        assert np.array_equal(out.double().cpu().numpy(), expect, equal_nan=True)


# ------------------------------------------------------------------------------------------------------------- products

# (tokens, features, k): single tokens, few, every tile's borders and one more, odd everything, K of one block and of many
SIZES = [(1, 1, 1), (1, 16, 32), (1, 515, 200), (2, 130, 129), (3, 96, 4096), (7, 33, 40), (8, 256, 1000), (9, 300, 257), (16, 320, 264),
         (17, 515, 200), (31, 129, 384), (33, 130, 72), (40, 257, 2056), (64, 256, 1024), (65, 384, 328), (100, 640, 512), (128, 128, 128),
         (129, 200, 1100), (256, 129, 300), (257, 513, 136), (300, 257, 1160), (520, 1000, 392)]


def operands(m, n, k, seed):
    rng = np.random.default_rng(seed)
    x = bf16(rng.standard_normal((m, k)) * np.exp(0.5 * rng.standard_normal(k)))
    w = plain.pack((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32))
    return x, w, plain.values(w, n, k)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_linear(m, n, k, out_dtype):
    from fastllm_py_b200.native import mxfp4

    x, data, w = operands(m, n, k, m + n + k)
    out = torch.full((m, n + 3), -5.0, dtype=out_dtype, device=DEV)
    mxfp4.linear(rows_in(x, torch.bfloat16, 8 * (m % 2)), matrix(data, n, k), out[:, :n])
    torch.cuda.synchronize()
    assert bool((out[:, n:] == -5.0).all()), "wrote outside the output columns"
    check_sum(out[:, :n], x @ w.T, np.abs(x) @ np.abs(w).T, k, out_dtype)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 300, 129), (5, 64, 4096), (16, 257, 40), (33, 130, 300), (97, 513, 72), (128, 256, 128), (129, 384, 1000),
                                     (192, 700, 256), (193, 129, 520), (385, 2300, 136), (600, 1000, 1928)])
def test_linear_and_gated_on_every_tensor_core_kernel(m, n, k, kernel):
    """Each of the two kernels for many rows whatever the rule would choose: tiles of tokens that end early, features that end inside
    a tile, in a pair's second CTA and before it, a gated unit's halves that meet inside a tile, K of one and of many chunks."""
    from fastllm_py_b200.native import gemm_tc, mxfp4

    x, data, w = operands(m, 2 * n, k, m + n + k)
    xs = rows_in(x, torch.bfloat16)
    for out_dtype, wide in ((torch.bfloat16, 3), (torch.float32, 8)):
        out = torch.full((m, 2 * n + wide), -5.0, dtype=out_dtype, device=DEV)
        mxfp4.linear(xs, matrix(data, 2 * n, k), out[:, :2 * n], kernel=kernel)
        act = torch.full((m, n + wide), -5.0, dtype=out_dtype, device=DEV)
        mxfp4.linear_gated(xs, matrix(data, 2 * n, k), act[:, :n], kernel=kernel)
        torch.cuda.synchronize()
        assert int(gemm_tc.status_word(torch.device(DEV)).item()) == 0
        assert bool((out[:, 2 * n:] == -5.0).all()) and bool((act[:, n:] == -5.0).all())
        check_sum(out[:, :2 * n], x @ w.T, np.abs(x) @ np.abs(w).T, k, out_dtype)
        check_gated(act[:, :n], x, w, "silu", (0, 0), k, out_dtype)


@pytest.mark.parametrize("kernel", [1, 2])
def test_products_after_a_recorded_fault_leave_at_once(kernel):
    """With a fault in the status word every role gives up at its first look: the launches return and write nothing, and the next
    launch without it works again."""
    from fastllm_py_b200.native import gemm_tc, mxfp4

    m, n, k = 300, 700, 520
    x, data, w = operands(m, n, k, 1)
    xs, q = rows_in(x, torch.bfloat16), matrix(data, n, k)
    a = mxfp4.Matrix.of(xs.float())
    word = gemm_tc.status_word(torch.device(DEV))
    outs = [torch.full((m, c), 7.0, dtype=torch.bfloat16, device=DEV) for c in (n, n // 2, n)]
    try:
        word.fill_(101)
        mxfp4.linear(xs, q, outs[0], kernel=kernel)
        mxfp4.linear_gated(xs, q, outs[1], kernel=kernel)
        mxfp4.product(a, q, outs[2])
        torch.cuda.synchronize()
        assert int(word.item()) == 101 and all(bool((o == 7.0).all()) for o in outs)
    finally:
        word.zero_()
    mxfp4.linear(xs, q, outs[0], kernel=kernel)
    check_sum(outs[0], x @ w.T, np.abs(x) @ np.abs(w).T, k, torch.bfloat16)


def test_a_first_product_inside_a_capture():
    """What is made once per device is not made inside a capture: the product is refused there, and works after `reserve`."""
    from fastllm_py_b200.native import mxfp4
    from fastllm_py_b200.native.ops import KernelError

    x, data, w = operands(20, 64, 96, 1)
    xs, q, out = rows_in(x, torch.bfloat16), matrix(data, 64, 96), torch.empty(20, 64, dtype=torch.bfloat16, device=DEV)
    kept = mxfp4._fns.pop(0, None)
    graph = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(graph):
        xs.add_(0.0)
        try:
            mxfp4.linear(xs, q, out)
        except KernelError:
            refused = True
    mxfp4.reserve(DEV)
    assert refused and mxfp4._fns[0] == (kept or mxfp4._fns[0])
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        mxfp4.linear(xs, q, out)


@pytest.mark.parametrize("m, n, k", [s for s in SIZES if s[1] > 1])
def test_product_of_two_packed_matrices(m, n, k):
    from fastllm_py_b200.native import mxfp4

    rng = np.random.default_rng(m * n + k)
    a_data = plain.pack((rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k))).astype(np.float32))
    _, data, w = operands(1, n, k, m + n)
    a = plain.values(a_data, m, k)
    for out_dtype, kernel in ((torch.bfloat16, 0), (torch.float32, 1), (torch.bfloat16, 2), (torch.float32, 2)):
        out = torch.full((m, n + 8), -5.0, dtype=out_dtype, device=DEV)
        mxfp4.product(matrix(a_data, m, k), matrix(data, n, k), out[:, :n], kernel=kernel)
        torch.cuda.synchronize()
        assert bool((out[:, n:] == -5.0).all())
        check_sum(out[:, :n], a @ w.T, np.abs(a) @ np.abs(w).T, k, out_dtype)


def check_gated(got, x, w, act, params, k, dtype):
    """The unit's derivatives bound what the two sums' errors become; its own evaluation in float is within 2^-18 of its value
    (fast exponential and quotient: a few steps each, and the argument's rounding times the argument, up to 30 here), and where
    its two terms cancel within 2^-22 |g u|: gelu is g u (1 + tanh z) / 2, tanh is within two steps of float below 1, 2^-23,
    the sum's rounding is 2^-24, and z's error of 4 steps, |z| 2^-22, moves tanh by at most |z| sech(z)^2 2^-22 <= 0.45 2^-22:
    together |g u| (2^-23 + 2^-24 + 0.9 2^-23) / 2 = 1.2 2^-23 |g u|."""
    n = w.shape[0] // 2
    g, u = x @ w[:n].T, x @ w[n:].T
    eg, eu = ((k / 16 + 64) * 2.0 ** -23 * (np.abs(x) @ np.abs(part).T) for part in (w[:n], w[n:]))
    want = plain.unit(act, g, u, params)
    corners = [np.abs(plain.unit(act, g + a * eg, u + b * eu, params) - want) for a in (-1, 1) for b in (-1, 1)]
    bound = 1.5 * np.max(corners, axis=0) + 2.0 ** -18 * np.abs(want) + np.abs(u) * (2.0 ** -22 * np.abs(g) + 2.0 ** -24) + half_step(dtype) * np.abs(want) * 1.01
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound + 1e-30), float((off / (bound + 1e-30)).max())


@pytest.mark.parametrize("m, n, k", [s for s in SIZES if s[1] > 1] + [(5, 64, 100), (70, 64, 260)])
def test_gated(m, n, k):
    from fastllm_py_b200.native import mxfp4

    x, data, w = operands(m, 2 * n, k, m + n + k)
    for act, params, out_dtype in (("silu", (0.0, 0.0), torch.bfloat16), ("clamped_swish", (1.5, 1.702), torch.float32)):
        out = torch.full((m, n + 8), -5.0, dtype=out_dtype, device=DEV)
        mxfp4.linear_gated(rows_in(x, torch.bfloat16), matrix(data, 2 * n, k), out[:, :n], act, params)
        torch.cuda.synchronize()
        assert bool((out[:, n:] == -5.0).all())
        check_gated(out[:, :n], x, w, act, params, k, out_dtype)


@pytest.mark.parametrize("act", ["silu", "relu", "gelu_tanh", "clamped_swish", "relu_squared"])
@pytest.mark.parametrize("m", [3, 70, 300])
def test_every_activation(m, act):
    from fastllm_py_b200.native import mxfp4

    n, k = 200, 300
    params = (1.25, 1.5) if act == "clamped_swish" else (0.0, 0.0)
    x, data, w = operands(m, 2 * n, k, m)
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.linear_gated(rows_in(x, torch.bfloat16), matrix(data, 2 * n, k), out, act, params)
    check_gated(out, x, w, act, params, k, torch.float32)
    one = torch.empty(m, 2 * n, dtype=torch.float32, device=DEV)
    mxfp4.linear(rows_in(x, torch.bfloat16), matrix(data, 2 * n, k), one, activation=act, params=params)
    y = x @ w.T
    e = (k / 16 + 64) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    want = plain.unit(act, y, np.ones_like(y), params)
    bound = 1.5 * np.maximum(*(np.abs(plain.unit(act, y + s * e, np.ones_like(y), params) - want) for s in (-1, 1))) + 2.0 ** -18 * np.abs(want) + 2.0 ** -22 * np.abs(y) + 2.0 ** -24
    off = np.abs(one.double().cpu().numpy() - want)                          # (the bound of check_gated, u = 1)
    assert np.all(off <= bound), float((off / bound).max())


@pytest.mark.parametrize("m", [1, 5, 20, 70, 300])
def test_products_with_extreme_scales(m):
    """Weights with scales from 2^-127 to 2^126 against activations that bring the sums back into range, and blocks that are NaN."""
    from fastllm_py_b200.native import mxfp4

    n, k = 150, 192
    rng = np.random.default_rng(m)
    e = rng.integers(-120, 121, n)
    base = rng.standard_normal((n, k))
    w32 = (base * 2.0 ** e[:, None]).astype(np.float32)
    data = plain.pack(w32)
    w = plain.values(data, n, k)
    x = bf16(rng.standard_normal((m, k)))
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.linear(rows_in(x, torch.bfloat16), matrix(data, n, k), out)
    check_sum(out, x @ w.T, np.abs(x) @ np.abs(w).T, k, torch.float32)
    # the smallest and the largest scale, and a NaN block, in rows of their own
    code, shift, scale = plain.addresses(n, k)
    flat = data.reshape(-1)
    flat[scale[3]], flat[scale[4]], flat[scale[5, 64:96]] = 0, 252, 255
    w = plain.values(data, n, k)
    small = bf16(x * 2.0 ** -20)
    out = torch.empty(m, n, dtype=torch.float32, device=DEV)
    mxfp4.linear(rows_in(small, torch.bfloat16), matrix(data, n, k), out)
    got = out.double().cpu().numpy()
    assert np.isnan(got[:, 5]).all() and np.isfinite(np.delete(got, 5, axis=1)).all()
    ok = [j for j in range(n) if j not in (3, 5)]
    check_sum(out[:, ok], small @ w[ok].T, np.abs(small) @ np.abs(w[ok]).T, k, torch.float32)
    # scale 2^-127 with activations as they are: the products are subnormal floats or small normal ones
    assert np.all(np.abs(got[:, 3] - small @ w[3]) <= k * 2.0 ** -149 + 2.0 ** -16 * (np.abs(small) @ np.abs(w[3])))


@pytest.mark.parametrize("m", [1, 6, 24, 80, 200])
def test_a_token_that_is_not_finite_stays_its_own(m):
    """Infinities and NaN in a token's activations concern that token's outputs, in the weights that feature's; what lies
    between the rows and behind the last one is not read."""
    from fastllm_py_b200.native import mxfp4

    n, k = 140, 200
    x, data, w = operands(m, n, k, m)
    bad = m // 2
    x[bad, 7] = np.inf
    buf = torch.full((m + 3, 208), float("nan"), dtype=torch.bfloat16, device=DEV)
    buf[:m, :k] = torch.from_numpy(x).to(DEV).to(torch.bfloat16)
    out = torch.full((m + 3, n), -5.0, dtype=torch.bfloat16, device=DEV)
    mxfp4.linear(buf[:m, :k], matrix(data, n, k), out[:m])
    assert bool((out[m:] == -5.0).all())
    with np.errstate(invalid="ignore"):
        want = x @ w.T
    got = out[:m].double().cpu().numpy()
    assert np.array_equal(np.isnan(got[bad]), np.isnan(want[bad])) and not np.isfinite(got[bad]).any()
    keep = [t for t in range(m) if t != bad]
    check_sum(out[keep], want[keep], np.abs(x[keep]) @ np.abs(w).T, k, torch.bfloat16)


def test_no_tokens():
    from fastllm_py_b200.native import mxfp4

    w = mxfp4.Matrix.of(torch.randn(64, 96, device=DEV))
    mxfp4.linear(torch.empty(0, 96, dtype=torch.bfloat16, device=DEV), w, torch.empty(0, 64, dtype=torch.bfloat16, device=DEV))
    mxfp4.linear_gated(torch.empty(0, 96, dtype=torch.bfloat16, device=DEV), w, torch.empty(0, 32, dtype=torch.bfloat16, device=DEV))
    torch.cuda.synchronize()


def layer(m, hidden, inter, seed):
    rng = np.random.default_rng(seed)
    x = bf16(rng.standard_normal((m, hidden)))
    gate_up = rng.standard_normal((2 * inter, hidden)) / np.sqrt(hidden)
    down = rng.standard_normal((hidden, inter)) / np.sqrt(inter)
    return x, gate_up.astype(np.float32), down.astype(np.float32)


def run_layer(x, q_gate_up, q_down, act, out):
    from fastllm_py_b200.native import mxfp4

    mxfp4.linear_gated(x, q_gate_up, act)
    mxfp4.linear(act, q_down, out)


@pytest.mark.parametrize("m", [1, 12, 90, 400])
def test_a_feed_forward_in_four_bits(m):
    """quantize, linear_gated and linear one after another, as a layer runs them, eagerly, on another stream and captured and
    replayed twice with other activations: the same bits each time, and the plain layer's values."""
    from fastllm_py_b200.native import mxfp4

    hidden, inter = 264, 712
    x, gate_up, down = layer(m, hidden, inter, m)
    q1, q2 = mxfp4.Matrix.of(torch.from_numpy(gate_up).to(DEV)), mxfp4.Matrix.of(torch.from_numpy(down).to(DEV))
    xs = rows_in(x, torch.bfloat16)
    act, out = torch.empty(m, inter, dtype=torch.bfloat16, device=DEV), torch.empty(m, hidden, dtype=torch.bfloat16, device=DEV)
    run_layer(xs, q1, q2, act, out)
    torch.cuda.synchronize()
    w1, w2 = plain.values(plain.pack(gate_up), 2 * inter, hidden), plain.values(plain.pack(down), hidden, inter)
    check_gated(act, x, w1, "silu", (0, 0), hidden, torch.bfloat16)
    a = act.double().cpu().numpy()
    check_sum(out, a @ w2.T, np.abs(a) @ np.abs(w2).T, inter, torch.bfloat16)
    first = out.clone()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out.fill_(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        run_layer(xs, q1, q2, act, out)
    torch.cuda.synchronize()
    assert torch.equal(out, first)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_layer(xs, q1, q2, act, out)
    other = rows_in(x[::-1].copy(), torch.bfloat16)
    keep = xs.clone()
    for source, want in ((keep, first), (other, None), (keep, first)):
        xs.copy_(source)
        out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        if want is not None:
            assert torch.equal(out, want)
        else:
            assert torch.equal(out, first.flip(0)) or m > 1


def test_two_streams_at_once():
    """Products of two streams that run at the same time do not touch one another's results."""
    from fastllm_py_b200.native import mxfp4

    jobs = []
    for i, (m, n, k) in enumerate([(9, 2000, 3000), (200, 1500, 2000)]):
        x, data, _ = operands(m, n, k, i)
        jobs.append((rows_in(x, torch.bfloat16), matrix(data, n, k), torch.cuda.Stream(), [torch.empty(m, n, dtype=torch.bfloat16, device=DEV) for _ in range(9)]))
    for x, w, _, outs in jobs:
        mxfp4.linear(x, w, outs[0])
    torch.cuda.synchronize()
    for i in range(1, 9):
        for x, w, stream, outs in jobs:
            with torch.cuda.stream(stream):
                mxfp4.linear(x, w, outs[i])
    torch.cuda.synchronize()
    for _, _, _, outs in jobs:
        assert all(torch.equal(o, outs[0]) for o in outs)


def test_long_rows_and_many_tokens():
    """Offsets past 2^31 elements of the output, and many tokens: the last rows are as good as the first."""
    from fastllm_py_b200.native import mxfp4

    m, n, k = 70000, 33000, 64
    x, data, w = operands(300, n, k, 1)
    xs = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
    xs[:150], xs[-150:] = rows_in(x, torch.bfloat16)[:150], rows_in(x, torch.bfloat16)[150:]
    out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    mxfp4.linear(xs, matrix(data, n, k), out)
    got = torch.cat([out[:150], out[-150:]])
    check_sum(got, x @ w.T, np.abs(x) @ np.abs(w).T, k, torch.bfloat16)
    assert bool((out[150:-150] == 0).all())


@pytest.mark.parametrize("m, n, k", [(1, 65536 * 256 + 5, 24), (9, 65536 * 256 + 5, 24), (65536 * 128 + 5, 8, 8)])
def test_more_tiles_than_a_grid_has_places(m, n, k):
    """65536 tiles and a few rows more, of W or of tokens: zeros but for the last rows, whose sums come out where they belong."""
    from fastllm_py_b200.native import mxfp4

    rng = np.random.default_rng(m)
    rows = n % 128 or 128
    last = plain.pack((rng.standard_normal((rows, k)) / np.sqrt(k)).astype(np.float32))
    q = mxfp4.Matrix.empty(n, k, DEV)
    q.data.zero_()
    q.data[-1].copy_(torch.from_numpy(np.ascontiguousarray(last)).to(DEV)[0])
    w = plain.values(last, rows, k)
    some = bf16(rng.standard_normal((130, k)))
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
    take = min(m, 130)
    x[-take:] = torch.from_numpy(some[:take]).to(DEV).to(torch.bfloat16)
    out = torch.full((m, n), -5.0, dtype=torch.bfloat16, device=DEV)
    mxfp4.linear(x, q, out)
    check_sum(out[-take:, n - rows:], some[:take] @ w.T, np.abs(some[:take]) @ np.abs(w).T, k, torch.bfloat16)
    assert not bool(out[:, :n - rows].any()) and not bool(out[:m - take].any())
    a = mxfp4.Matrix.of(x)
    av = torch.empty(m, k, device=DEV)
    mxfp4.dequantize(a, av)
    av = av[-take:].double().cpu().numpy()
    out.fill_(-5.0)
    mxfp4.product(a, q, out)
    check_sum(out[-take:, n - rows:], av @ w.T, np.abs(av) @ np.abs(w).T, k, torch.bfloat16)
    assert not bool(out[:, :n - rows].any()) and not bool(out[:m - take].any())


def test_a_layer_multiplies_as_soon_as_it_is_made():
    """Two layers made one after the other and used at once: their matrices are there before a product reads them as constant."""
    from fastllm_py_b200.parts.linear import Linear

    rng = np.random.default_rng(5)
    x = bf16(rng.standard_normal((3, 4096)))
    xs = rows_in(x, torch.bfloat16)
    ws = [bf16(rng.standard_normal((2048, 4096)) / 64) for _ in range(2)]
    layers = [Linear([torch.from_numpy(w).to(DEV).to(torch.bfloat16)], "mxfp4") for w in ws]
    outs = [torch.empty(3, 2048, dtype=torch.bfloat16, device=DEV) for _ in ws]
    for layer, out in zip(layers, outs):
        layer.forward(xs, out)
    for w, out in zip(ws, outs):
        v = plain.values(plain.pack(w.astype(np.float32)), 2048, 4096)
        check_sum(out, x @ v.T, np.abs(x) @ np.abs(v).T, 4096, torch.bfloat16)


def test_two_captured_products_replayed_at_the_same_time():
    """Graphs of the same calls on different outputs, replayed on two streams: nothing but the operands is shared."""
    from fastllm_py_b200.native import mxfp4

    m, n, k = 40, 520, 2048
    x, data, w = operands(m, 2 * n, k, 3)
    xs, q = rows_in(x, torch.bfloat16), matrix(data, 2 * n, k)
    a = mxfp4.Matrix.of(xs)
    mxfp4.reserve(DEV)
    graphs, outs = [], []
    for _ in range(2):
        out = [torch.empty(m, 2 * n, dtype=torch.float32, device=DEV) for _ in range(2)] + [torch.empty(m, n, dtype=torch.float32, device=DEV)]
        mxfp4.linear(xs, q, out[0]), mxfp4.product(a, q, out[1]), mxfp4.linear_gated(xs, q, out[2])
        outs.append((out, [o.clone() for o in out]))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            mxfp4.linear(xs, q, out[0]), mxfp4.product(a, q, out[1]), mxfp4.linear_gated(xs, q, out[2])
        graphs.append(g)
    for out, _ in outs:
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, want in outs:
        assert all(torch.equal(o, v) for o, v in zip(out, want))
    check_sum(outs[0][0][0], x @ w.T, np.abs(x) @ np.abs(w).T, k, torch.float32)


@pytest.mark.parametrize("m, n, k", [(1, 4096, 20000), (8, 4096, 20000), (2, 40000, 2048), (7, 40000, 2048)])
def test_few_rows_with_a_large_matrix(m, n, k):
    """Matrices of more than 2^26 values, for which one or the other kernel takes less: a plain product and a gated one of each, at
    chosen features against 64 bits and as a whole against the other kernel."""
    from fastllm_py_b200.native import mxfp4

    g = torch.Generator(device=DEV).manual_seed(m + n)
    x = torch.randn(m, k, generator=g, device=DEV).to(torch.bfloat16)
    q = mxfp4.Matrix.of(torch.randn(n, k, generator=g, device=DEV) / k ** 0.5)
    some = torch.arange(0, n, 997, device=DEV)
    w = torch.empty(n, k, dtype=torch.bfloat16, device=DEV)
    mxfp4.dequantize(q, w)
    xs, ws = x.double().cpu().numpy(), w[some].double().cpu().numpy()
    outs = [torch.empty(m, n, dtype=torch.float32, device=DEV) for _ in range(2)]
    units = [torch.empty(m, n // 2, dtype=torch.float32, device=DEV) for _ in range(2)]
    for kernel in (0, 1):
        mxfp4.linear(x, q, outs[kernel], kernel=kernel)
        mxfp4.linear_gated(x, q, units[kernel], kernel=kernel)
    check_sum(outs[0][:, some], xs @ ws.T, np.abs(xs) @ np.abs(ws).T, k, torch.float32)
    # the other kernel's sums differ by twice what either may be off
    off = 2 * (k / 16 + 64) * 2.0 ** -23 * (x.abs().double() @ w.abs().double().T)
    assert bool(((outs[0].double() - outs[1].double()).abs() <= off).all())
    gate, up = outs[0].double().split(n // 2, dim=1)
    eg, eu = off.split(n // 2, dim=1)
    # silu's slope is at most 1.1, its value at most |g|; its own evaluation in float is within 2^-18, twice
    unit = up * gate * torch.sigmoid(gate)
    assert bool(((units[0].double() - units[1].double()).abs() <= 1.1 * eg * up.abs() + gate.abs() * eu + eg * eu + 2.0 ** -17 * unit.abs()).all())


@pytest.mark.parametrize("name, kernel, m, n, k", [("linear", 1, 64, 4096, 11008), ("linear", 1, 128, 4096, 5504), ("linear", 1, 96, 2304, 8192), ("linear", 2, 600, 4096, 5504),
                                                   ("linear_gated", 1, 40, 2048, 8192), ("linear_gated", 2, 900, 2048, 5504), ("product", 1, 100, 4096, 11008),
                                                   ("product", 2, 1024, 8192, 5504), ("product", 2, 4096, 8192, 11008)])
def test_the_same_sums_every_time(name, kernel, m, n, k):
    """Many launches of a large product, with the operands in and out of the L2: bits are the same, and no warp has given up.  (Copies
    land in any order, and warps that share a ring's stages must not take one phase of a barrier for another.)"""
    from fastllm_py_b200.native import gemm_tc, mxfp4

    g = torch.Generator(device=DEV).manual_seed(k)
    x = torch.randn(m, k, generator=g, device=DEV).to(torch.bfloat16)
    gated = name == "linear_gated"
    q = mxfp4.Matrix.of(torch.randn(2 * n if gated else n, k, generator=g, device=DEV) / k ** 0.5)
    first = mxfp4.Matrix.of(x) if name == "product" else x
    outs = [torch.full((m, n), -5.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    flush = torch.empty(160 << 20, dtype=torch.uint8, device=DEV)
    call = getattr(mxfp4, name)
    call(first, q, outs[0], kernel=kernel)
    differ = torch.zeros((), dtype=torch.int64, device=DEV)
    for i in range(150):
        if i % 3 == 0:
            flush.fill_(i)
        call(first, q, outs[1], kernel=kernel)
        differ += (outs[0] != outs[1]).sum()
    assert int(gemm_tc.status_word(torch.device(DEV)).item()) == 0 and int(differ) == 0
    assert not bool((outs[0] == -5.0).all())
