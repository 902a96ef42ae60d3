"""`weights="mxfp4"` in models whose dense feed-forwards stand beside other mixers and experts: gated and plain units, units shared beside
experts, widths that are no multiples of 8.  The engine is held to the plain model with the same matrices rounded by the plain
implementation of the format, within the bounds that the bfloat16 engine is held to with the stored ones (0.08 of the logits' spread in
the median of the positions, 0.3 at the ninth decile: tests/test_saberax_gpu.py and its neighbours)."""
import re

import numpy as np
import pytest
import torch

import kerirax_tiny
import lufozen_tiny
import plain_kerirax
import plain_lufozen
import plain_mxfp4
import plain_saberax
import replay
import saberax_tiny
import test_kerirax_gpu
import test_lufozen_gpu
import test_saberax_gpu

pytestmark = pytest.mark.gpu

ROUNDED = re.compile(r"l\d+\.mlp\.(shared\.)?(gate|up|down)$")


def make(family, name):
    if family == "kerirax":
        m = test_kerirax_gpu.MODELS[name]
        raw = kerirax_tiny.config(m["layers"], **m["kw"])
        return raw, kerirax_tiny.weights(raw, seed=5), kerirax_tiny, plain_kerirax, m["page"], test_kerirax_gpu.LENGTHS[name]
    if family == "lufozen":
        m = test_lufozen_gpu.MODELS[name]
        raw = lufozen_tiny.config(m["layers"], **m["kw"])
        return raw, lufozen_tiny.weights(raw, seed=5, rank=m["rank"]), lufozen_tiny, plain_lufozen, m["page"], test_lufozen_gpu.LENGTHS[name]
    m = test_saberax_gpu.MODELS[name]
    raw = saberax_tiny.config(m["layers"], m["vocab"], m["width"], m["eps"], m["mult"])
    return raw, saberax_tiny.weights(raw, seed=5, rank=m["rank"]), saberax_tiny, plain_saberax, m["page"], test_saberax_gpu.LENGTHS[name]


def held(model):
    """The Linears in 4 bits, of a gated unit one for both its matrices."""
    return [lin for part in model.decoder.all_parts() for lin in vars(part).values() if type(lin).__name__ == "Linear" and lin._q4 is not None]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("family, name", [(f, n) for f in ("kerirax", "lufozen", "saberax") for n in ("mix", "odd", "even")])
def test_models_of_other_families_in_four_bits(family, name, graph, tmp_path):
    from fastllm_py_b200 import Model

    raw, weights, tiny, plain, page, lengths = make(family, name)
    names = [k for k in weights if ROUNDED.match(k)]
    rounded = dict(weights)
    for k in names:
        x = weights[k].float().numpy()
        rounded[k] = torch.from_numpy(plain_mxfp4.values(plain_mxfp4.pack(x), *x.shape).astype(np.float32))
    rng = np.random.default_rng(40)
    requests = {f"q{i}": rng.integers(0, raw["vocab"], size=n).tolist() for i, n in enumerate(lengths)}
    want = {rid: plain.forward(raw, rounded, toks).float() for rid, toks in requests.items()}
    stored = {rid: plain.forward(raw, weights, toks).float() for rid, toks in requests.items()}
    spread = float(torch.cat([v.flatten() for v in want.values()]).std())
    model = Model.load(tiny.write(raw, weights, tmp_path / "model"), weights="mxfp4", page_size=page, max_tokens=512, max_requests=3,
                       max_batched_tokens=256, max_model_len=256, cuda_graph=graph, check_cache=True)
    gates = sum(k.endswith("gate") for k in names)
    assert len(held(model)) == len(names) - gates > 0
    steps = replay.mixed(requests, live=3, seed=3, prefill_sizes=(9, 2, 17, 5, 70), decode_tail=6)
    got = replay.run_in_process(model.engine, steps)
    off = lambda target: np.array([float((got[k] - target[k[0]][k[1]]).pow(2).mean().sqrt()) for k in got]) / spread  # noqa: E731
    errs = off(want)
    assert np.median(errs) <= 0.08 and np.quantile(errs, 0.9) <= 0.3, (np.median(errs), np.quantile(errs, 0.9))
    assert np.median(off(stored)) > np.median(errs), "the test's model does not tell rounded matrices from stored ones"
    model.engine.check_status()


@pytest.mark.parametrize("family, mlp, count", [("kerirax", "dense", 2), ("kerirax", None, 0)])
def test_the_load_line_says_how_many_matrices_are_in_four_bits(family, mlp, count, tmp_path, capsys):
    from fastllm_py_b200.cli import main

    raw = kerirax_tiny.config([(kerirax_tiny.latent(2, 8, 4, 12, 10, 14), kerirax_tiny.dense(32) if mlp else None)], width=24, vocab=50)
    folder = kerirax_tiny.write(raw, kerirax_tiny.weights(raw, seed=1), tmp_path / "model")
    assert main([str(folder), "", "3", "--weights", "mxfp4", "--prompt-ids", "3,14,15", "--page-size", "16", "--max-model-len", "64"]) == 0
    assert f"weights=mxfp4 ({count} matrices in 4 bits)" in capsys.readouterr().out
