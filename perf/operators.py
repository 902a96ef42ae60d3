"""Cases of the operators on microscaled 4-bit floating point (MXFP4): rounding to it, the product of bfloat16 rows with a matrix
held in it, the gated unit on such a matrix, and the product of two matrices held in it.

The format: along K a matrix is cut into blocks of 32; a block has one scale, a power of two 2^(s - 127) with a byte s (255: the
block is NaN), and 32 elements of 4 bits (a sign and the magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6).  The packed form is a byte
tensor [row tiles of 128][K chunks of 128][8704]: four pieces (one for each block of the chunk) of 128 rows x 16 bytes of codes,
then 512 bytes of scales, row r's four at (r % 32) * 16 + (r // 32) * 4.  A little-endian 4-byte word of codes holds 8 elements:
nibble j is element 2 j for j < 4 and 2 (j - 4) + 1 after that.

`own` False computes everything with elementary torch operations; True calls fastllm_py_b200.native.mxfp4.
"""
import math

import torch

own = False

DEV = "cuda"
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
ORDER = (0, 2, 4, 6, 1, 3, 5, 7)                 # the element that nibble j of a word of codes holds
CHUNK = 8704


def listed():
    return [
        # one token's activations of a model of 7B size on their way to a 4-bit product: latency
        {"name": "round-1x4096", "op": "round", "m": 1, "k": 4096, "dtype": "bfloat16"},
        # the feed-forward activations of a prompt of 2048 tokens
        {"name": "round-2048x11008", "op": "round", "m": 2048, "k": 11008, "dtype": "bfloat16"},
        # a 32-bit checkpoint's matrix when a model is loaded, of odd sizes
        {"name": "round-32bit-5503x4097", "op": "round", "m": 5503, "k": 4097, "dtype": "float32"},
        # one token through the stacked q|k|v matrix of 7B size
        {"name": "linear-1-4096-12288", "op": "linear", "m": 1, "n": 12288, "k": 4096},
        # a batch of 8 through its down projection
        {"name": "linear-8-11008-4096", "op": "linear", "m": 8, "n": 4096, "k": 11008},
        # a batch of 64 through the down projection of 67B size
        {"name": "linear-64-22016-8192", "op": "linear", "m": 64, "n": 8192, "k": 22016},
        # a prompt portion of odd length, odd sizes
        {"name": "linear-517-2047-5503", "op": "linear", "m": 517, "n": 5503, "k": 2047},
        # one token through the gated unit of 7B size
        {"name": "gated-1-4096-11008", "op": "gated", "m": 1, "n": 11008, "k": 4096},
        # a prompt of 2048 tokens through it
        {"name": "gated-2048-4096-11008", "op": "gated", "m": 2048, "n": 11008, "k": 4096},
        # a batch of 40 through the q|k|v matrix with 4-bit activations
        {"name": "product-40-4096-12288", "op": "product", "m": 40, "n": 12288, "k": 4096},
        # odd sizes, a few tiles
        {"name": "product-261-1000-1537", "op": "product", "m": 261, "n": 1537, "k": 1000},
        # prompts of 4096 tokens with 4-bit activations through the up projections of 67B size
        {"name": "product-4096-8192-22016", "op": "product", "m": 4096, "n": 22016, "k": 8192},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("round", "linear", "gated", "product"))
    if op == "round":
        return {"op": op, "m": _log(rng, 1, 5600), "k": _log(rng, 1, 11008), "dtype": rng.choice(("bfloat16", "float32"))}
    most = 2 * 2048 * 4096 * 11008
    while True:
        m, n, k = _log(rng, 1, 4096), _log(rng, 16, 22016), _log(rng, 24, 22016)
        if rng.random() < 0.5:                   # as models have them
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        if m * n * k * (2 if op == "gated" else 1) <= most:
            return {"op": op, "m": m, "n": n, "k": k}


def work(case):
    m, k = case["m"], case["k"]
    packed = lambda rows: rows * -(-k // 32) * 17  # noqa: E731
    if case["op"] == "round":                    # read, written as 4-bit codes, and the values that those stand for
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": 2 * m * k * size + packed(m), "flops": 2 * m * k}
    n = case["n"]
    if case["op"] == "gated":
        return {"bytes": packed(2 * n) + 2 * m * k + 2 * m * n, "flops": 4 * m * n * k}
    if case["op"] == "product":
        return {"bytes": packed(n) + packed(m) + 2 * m * n, "flops": 2 * m * n * k}
    return {"bytes": packed(n) + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------------------- plain forms

def _blocks(x):
    """[rows, k] -> float32 [rows, blocks, 32], zeros behind k."""
    rows, k = x.shape
    full = torch.zeros((rows, -(-k // 32) * 32), dtype=torch.float32, device=x.device)
    full[:, :k] = x
    return full.view(rows, -1, 32)


def _encode(x):
    """Scale bytes [rows, blocks] (int32), signed magnitudes [rows, blocks, 32] on the grid, and the scales."""
    b = _blocks(x)
    amax = b.abs().amax(2)
    s = ((amax.contiguous().view(torch.int32) >> 23) - 2).clamp(min=0)
    s = torch.where(torch.isfinite(amax), s, torch.full_like(s, 255))
    scale = torch.ldexp(torch.ones_like(amax), (s - 127).clamp(max=127))
    v = b / scale[:, :, None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)
    return s, v, torch.where(s == 255, torch.full_like(scale, math.nan), scale)


def _pack(x):
    """The packed form of x [rows, k], in torch."""
    rows, k = x.shape
    s, v, _ = _encode(x)
    tiles, chunks = -(-rows // 128), -(-k // 128)
    codes = torch.bucketize(v.abs(), torch.tensor(GRID, device=x.device)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    codes = codes * (s != 255)[:, :, None].to(torch.uint8)
    full = torch.zeros((tiles * 128, chunks * 4, 32), dtype=torch.uint8, device=x.device)
    full[:rows, :codes.shape[1]] = codes
    full = full.view(tiles, 128, chunks, 4, 4, 8)[..., list(ORDER)]
    full = full[..., 0::2] | (full[..., 1::2] << 4)
    scales = torch.zeros((tiles * 128, chunks * 4), dtype=torch.uint8, device=x.device)
    scales[:rows, :s.shape[1]] = s.to(torch.uint8)
    data = torch.empty((tiles, chunks, CHUNK), dtype=torch.uint8, device=x.device)
    data[:, :, :8192] = full.permute(0, 2, 3, 1, 4, 5).reshape(tiles, chunks, 8192)
    data[:, :, 8192:] = scales.view(tiles, 4, 32, chunks, 4).permute(0, 3, 2, 1, 4).reshape(tiles, chunks, 512)
    return data


def _unpack(data, rows, k):
    """The values that a packed form stands for, float32 [rows, k]."""
    tiles, chunks, _ = data.shape
    codes = data[:, :, :8192].reshape(tiles, chunks, 4, 128, 4, 4).permute(0, 3, 1, 2, 4, 5)      # tile, row, chunk, block, word, byte
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int32)                  # ..., nibble
    place = [ORDER.index(e) for e in range(8)]
    codes = codes[..., place]
    mag, e = codes & 1, (codes >> 1) & 3
    v = torch.where(e == 0, 0.5 * mag, torch.ldexp(1 + 0.5 * mag, e - 1)) * (1 - 2 * (codes >> 3))
    s = data[:, :, 8192:].reshape(tiles, chunks, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles, 128, chunks, 4).to(torch.int32)
    scale = torch.where(s == 255, math.nan, torch.ldexp(torch.ones_like(s, dtype=torch.float32), (s - 127).clamp(max=127)))
    return (v.flatten(-2) * scale[..., None]).reshape(tiles * 128, chunks * 128)[:rows, :k].contiguous()


# ------------------------------------------------------------------------------------------------------------------ inputs

def _rows(m, k, g, dtype):
    """Activations: channels of different sizes, a few of them far out, in a buffer whose rows begin on 16 bytes."""
    size = torch.exp(0.5 * torch.randn(k, generator=g, device=DEV))
    size = torch.where(torch.rand(k, generator=g, device=DEV) < 0.002, 20 * size, size)
    buf = torch.full((m, -(-k // 8) * 8), 7.0, dtype=dtype, device=DEV)
    buf[:, :k] = (torch.randn((m, k), generator=g, device=DEV) * size).to(dtype)
    return buf[:, :k]


def _matrix(n, k, g):
    return _pack(torch.randn((n, k), generator=g, device=DEV) / math.sqrt(k))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    m, k, op = case["m"], case["k"], case["op"]
    if op == "round":
        x = _rows(m, k, g, getattr(torch, case["dtype"]))
        return {"case": case, "x": x, "data": torch.empty((-(-m // 128), -(-k // 128), CHUNK), dtype=torch.uint8, device=DEV),
                "out": torch.empty((m, k), dtype=x.dtype, device=DEV)}
    n = case["n"]
    state = {"case": case, "w": _matrix(2 * n if op == "gated" else n, k, g), "out": torch.empty((m, n), dtype=torch.bfloat16, device=DEV)}
    x = _rows(m, k, g, torch.bfloat16)
    state["x"] = _pack(x.float()) if op == "product" else x
    return state


def run(state):
    case, x, out = state["case"], state["x"], state["out"]
    op, m, k, n = case["op"], case["m"], case["k"], case.get("n")
    if own:
        from fastllm_py_b200.native import mxfp4

        if op == "round":
            q = mxfp4.Matrix(state["data"], m, k)
            mxfp4.quantize(x, q)
            mxfp4.dequantize(q, out)
        elif op == "linear":
            mxfp4.linear(x, mxfp4.Matrix(state["w"], n, k), out)
        elif op == "gated":
            mxfp4.linear_gated(x, mxfp4.Matrix(state["w"], 2 * n, k), out)
        else:
            mxfp4.product(mxfp4.Matrix(x, m, k), mxfp4.Matrix(state["w"], n, k), out)
        return out
    if op == "round":
        _, v, scale = _encode(x)
        return (v * scale[:, :, None]).reshape(m, -1)[:, :k].to(x.dtype)
    if op == "linear":
        return (x.float() @ _unpack(state["w"], n, k).t()).to(torch.bfloat16)
    if op == "gated":
        y = x.float() @ _unpack(state["w"], 2 * n, k).t()
        gate, up = y[:, :n], y[:, n:]
        return (gate / (1 + torch.exp(-gate)) * up).to(torch.bfloat16)
    return (_unpack(x, m, k) @ _unpack(state["w"], n, k).t()).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------- the same from the definition

def _values64(data, rows, k):
    """A packed form's values in 64 bits, gathered element by element through its addresses."""
    table = torch.tensor(list(GRID) + [-v for v in GRID], dtype=torch.float64, device=data.device)
    flat = data.reshape(-1)
    chunks = data.shape[1]
    c = torch.arange(k, device=data.device)
    within = c % 8
    nibble = torch.where(within % 2 == 0, within // 2, 4 + within // 2)
    code_at = (c // 128) * CHUNK + (c % 128) // 32 * 2048 + (c % 32) // 8 * 4 + nibble // 2
    scale_at = (c // 128) * CHUNK + 8192 + (c % 128) // 32
    out = torch.empty((rows, k), dtype=torch.float64, device=data.device)
    for r0 in range(0, rows, 1024):
        r = torch.arange(r0, min(rows, r0 + 1024), device=data.device)[:, None]
        base = (r // 128) * chunks * CHUNK
        byte = flat[base + (r % 128) * 16 + code_at].to(torch.int64)
        s = flat[base + (r % 32) * 16 + (r % 128) // 32 * 4 + scale_at].to(torch.float64)
        out[r0:r0 + 1024] = table[(byte >> (4 * (nibble % 2))) & 15] * torch.where(s == 255, math.nan, torch.exp2(s - 127))
    return out


def _rounded64(x):
    """x on the grid of its blocks: the nearest of the eight magnitudes, of two equally near ones that with the even code."""
    rows, k = x.shape
    out = torch.empty((rows, k), dtype=torch.float64, device=x.device)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    for c0 in range(0, k, 32 * 64):
        part = x[:, c0:c0 + 32 * 64].double()
        wide = torch.nn.functional.pad(part, (0, -part.shape[1] % 32)).reshape(rows, -1, 32)
        top = wide.abs().amax(2, keepdim=True)
        unit = torch.where(top > 0, torch.exp2((torch.frexp(top).exponent - 3).clamp(min=-127).double()), torch.ones_like(top))
        a = wide.abs() / unit
        best, value = torch.full_like(a, math.inf), torch.zeros_like(a)
        for code in (0, 2, 4, 6, 1, 3, 5, 7):
            off = (a - grid[code]).abs()
            value, best = torch.where(off < best, grid[code], value), torch.minimum(off, best)
        out[:, c0:c0 + 32 * 64] = (torch.sign(wide) * value * unit).reshape(rows, -1)[:, :part.shape[1]]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    m, k, n = case["m"], case["k"], case.get("n")
    if case["op"] == "round":
        return _rounded64(state["x"])
    if case["op"] == "product":
        return _values64(state["x"], m, k) @ _values64(state["w"], n, k).t()
    x = state["x"].double()
    if case["op"] == "linear":
        return x @ _values64(state["w"], n, k).t()
    w = _values64(state["w"], 2 * n, k)
    gate = x @ w[:n].t()
    return gate * torch.sigmoid(gate) * (x @ w[n:].t())
