"""Calls of the 4-bit operators that are refused on the host, and rules of their kernels that are checked on the sources."""
import re
from pathlib import Path

import pytest
import torch

from fastllm_py_b200.native import mxfp4
from fastllm_py_b200.native.ops import KernelError

CSRC = Path(__file__).resolve().parent.parent / "fastllm-py_b200" / "csrc"


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("kernel", [0, 1, 2])
def test_a_gated_product_has_a_unit(kernel):
    """Without one the up half would have no place in the result; a plain product goes without."""
    w = mxfp4.Matrix.empty(64, 96, "cpu")
    with pytest.raises(KernelError, match="activation"):
        mxfp4.linear_gated(bf(5, 96), w, bf(5, 32), activation=None, kernel=kernel)
    with pytest.raises(KernelError, match="activation"):
        mxfp4.linear_gated(bf(0, 96), w, bf(0, 32), None)
    with pytest.raises(KernelError, match="CUDA device only"):
        mxfp4.linear(bf(5, 96), w, bf(5, 64), activation=None, kernel=kernel)


def test_a_recorded_fault_is_raised_once(monkeypatch):
    """The status word's code is raised and cleared; no word, no error; the host has none."""
    from fastllm_py_b200.native import gemm_tc

    word, waited = torch.zeros(1, dtype=torch.int32), []
    monkeypatch.setattr(gemm_tc, "status_word", lambda device: word)
    monkeypatch.setattr(torch.cuda, "synchronize", waited.append)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    mxfp4.check("cuda:0")
    word.fill_(121)
    with pytest.raises(KernelError, match="121"):
        mxfp4.check("cuda:0")
    mxfp4.check(torch.device("cuda:0"))
    assert waited == [torch.device("cuda:0")] * 3 and int(word) == 0
    with pytest.raises(KernelError, match="CUDA device only"):
        mxfp4.check("cpu")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(KernelError, match="captured"):
        mxfp4.check("cuda:0")


def test_every_launch_is_counted(monkeypatch):
    """One kernel a call, whichever launcher takes it; a refused or an empty call counts none."""
    from fastllm_py_b200.native import ops

    rc = {"fl_mxt_product": 0}
    monkeypatch.setattr(mxfp4, "_stream_of", lambda *tensors: 0)
    monkeypatch.setattr(mxfp4, "_known", lambda t: (0, 148))
    monkeypatch.setattr(mxfp4, "_fns", {name: (lambda *args, name=name: rc.get(name, 0)) for name in
                                        ("fl_mx_quantize", "fl_mx_dequantize", "fl_mx_few", "fl_mxt_product", "fl_mxq_product")})
    w, a = mxfp4.Matrix.empty(64, 96, "cpu"), mxfp4.Matrix.empty(20, 96, "cpu")
    calls = [lambda: mxfp4.quantize(bf(20, 96), a), lambda: mxfp4.dequantize(a, bf(20, 96)), lambda: mxfp4.linear(bf(3, 96), w, bf(3, 64)),
             lambda: mxfp4.linear(bf(20, 96), w, bf(20, 64)), lambda: mxfp4.linear_gated(bf(20, 96), w, bf(20, 32)),
             lambda: mxfp4.linear_gated(bf(2, 96), w, bf(2, 32)), lambda: mxfp4.product(a, w, bf(20, 64)), lambda: mxfp4.Matrix.of(bf(20, 96))]
    for call in calls:
        before = ops.counter.launches
        call()
        assert ops.counter.launches == before + 1
    before = ops.counter.launches
    mxfp4.linear(bf(0, 96), w, bf(0, 64))
    rc["fl_mxt_product"] = 1
    with pytest.raises(KernelError, match="CUDA error 1"):
        mxfp4.linear(bf(20, 96), w, bf(20, 64))
    assert ops.counter.launches == before
    # a launcher that has left the call to the one for few rows has launched nothing
    rc["fl_mxt_product"] = mxfp4.LESS
    monkeypatch.setattr(mxfp4, "FEW_VALUES", 0)
    mxfp4.linear(bf(3, 96), w, bf(3, 64))
    assert ops.counter.launches == before + 1


def test_a_model_counts_its_matrices_in_four_bits():
    """What `weights="mxfp4"` has come to: the stacked matrices of a Linear are one, those held as stored are none."""
    from types import SimpleNamespace as Thing

    from fastllm_py_b200 import Model
    from fastllm_py_b200.parts.linear import Linear

    def linear(q4):
        lin = Linear([bf(8, 16)])
        lin._q4 = q4
        return lin

    q = mxfp4.Matrix.empty(8, 16, "cpu")
    parts = [Thing(qkv=linear(q), o=linear(q)), Thing(router=linear(None), size=3), Thing(gate_up=linear(q), down=linear(None))]
    model = Model(None, None, Thing(all_parts=lambda: iter(parts)), None)
    assert model.matrices_in_four_bits == 3
    parts[:] = [Thing(head=linear(None))]
    assert model.matrices_in_four_bits == 0


def body_of(file, name):
    """From a function's name to the brace that closes it."""
    text = (CSRC / file).read_text()
    body = text[re.search(rf"\n(?:\S[^\n]*[ *])?{name}\(", text).start():]
    return body[:body.index("\n}\n")]


@pytest.mark.parametrize("file, function, roles", [
    ("mxfp4_tc.cu", "mxt_produce", []), ("mxfp4_tc.cu", "mxt_kernel", ["// ---- codes to bfloat16", "// ---- MMA issuer."]),
    ("mxfp4_tc.cu", "mxq_kernel", []), ("gemm_tcgen05.cu", "gemm_tc_kernel", ["// ---- producer", "// ---- MMA issuer", "// ---- epilogue"])])
def test_time_limits_begin_when_the_preceding_kernel_is_over(file, function, roles):
    """A kernel launched programmatically may wait for its predecessor as long as that takes.  A role whose barrier comes after that wait of
    another role waits for the predecessor first itself: the limit after which it gives up is for what its own kernel does."""
    body = body_of(file, function)
    cuts = [0] + [body.rindex("{", 0, body.index(mark)) for mark in roles] + [len(body)]
    parts = [body[a:b] for a, b in zip(cuts, cuts[1:])]
    waits = 0
    for part in parts:
        wait = re.search(r"mxt_wait\(|mbar_wait\(", part)
        if wait:
            waits += 1
            assert "pdl_wait();" in part[:wait.start()], part[:200]
    assert waits == max(1, len(roles))


WAITS = {
    "mxt_produce": ["empty_bar[s], ph ^ 1u"],
    "mxt_kernel": ["full_bar[s], ph", "a_empty[place], pa ^ 1u", "a_full[place], pa"],
    "mxq_kernel": ["empty_bar[s], ph ^ 1u", "full_bar[s], ph"],
    "mxp_kernel": ["w_full[s], ph", "x_full[x], xph", "a_empty[turn], pa ^ 1u", "acc_full[b], (uint32_t)(i >> 1) & 1u", "x_empty[s], ph ^ 1u",
                   "w_empty[s], ph ^ 1u", "acc_empty[b], ((uint32_t)(i >> 1) & 1u) ^ 1u", "a_full[turn], pa"],
    "mxqp_kernel": ["empty_bar[s], ph ^ 1u", "full_bar[s], ph", "acc_full, (uint32_t)i & 1u", "empty_bar[s], ph ^ 1u",
                    "acc_empty, ((uint32_t)i & 1u) ^ 1u", "scales_bar[s], ph"],
}


@pytest.mark.parametrize("function", list(WAITS))
def test_the_kernels_wait_as_their_model_does(function):
    """The hand-overs that tests/test_mxfp4_barriers.py runs on the host, in the sources: every wait of each kernel, in its order.  One
    that changes is changed in the model too, which then says whether a phase can be taken for another."""
    body = body_of("mxfp4_pair.cuh" if function in ("mxp_kernel", "mxqp_kernel") else "mxfp4_tc.cu", function)
    assert re.findall(r"mxt_wait\(&?(.*?), abort_flag\)", body) == WAITS[function]
