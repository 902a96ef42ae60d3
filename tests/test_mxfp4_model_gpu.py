"""Models whose dense layers' matrices are held in microscaled 4-bit floating point: the engine against the plain model with the
same matrices rounded by the plain implementation of the format."""
import numpy as np
import pytest
import torch

import plain_llama as plain
import plain_mxfp4
import tiny

pytestmark = pytest.mark.gpu


def rounded(weights):
    """The model's matrices in the layers replaced by what their 4-bit form stands for."""
    out = {}
    for name, w in weights.items():
        if "layers." in name and w.dim() == 2:
            x = w.float().numpy()
            w = torch.from_numpy(plain_mxfp4.values(plain_mxfp4.pack(x), *x.shape).astype(np.float32))
        out[name] = w
    return out


def check_greedy(weights, config, prompt, got):
    """Every token is the plain model's best one, or nearly tied with it: within twice what storing the plain model's activations
    in bfloat16 does to that row."""
    ids = list(prompt)
    for tok in got:
        row = plain.forward(weights, config, ids, store=plain.store_bf16)[-1]
        best = int(row.argmax())
        if tok != best:
            noise = float((row - plain.forward(weights, config, ids)[-1]).abs().max())
            assert float(row[best] - row[tok]) <= 2 * noise + 1e-3, (len(ids), tok, best)
        ids.append(tok)


@pytest.mark.parametrize("name", list(tiny.CONFIGS))
@pytest.mark.parametrize("use_graph", [False, True])
def test_model_in_four_bits(name, use_graph, model_folders):
    """Single prompts and a batch of prompts of different lengths, so that steps have from one to some two hundred tokens."""
    from fastllm_py_b200 import Model

    weights, config = plain.load_folder(model_folders[name])
    weights = rounded(weights)
    model = Model.load(model_folders[name], dtype="bfloat16", weights="mxfp4", page_size=tiny.CONFIGS[name]["page_size"], max_tokens=1024,
                       max_requests=8, max_batched_tokens=256, max_model_len=128, cuda_graph=use_graph)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 256, length).tolist() for length in (3, 17, 40, 1, 90, 8, 5, 33)]
    one = model.generate(prompts[1], max_new_tokens=6, use_graph=use_graph)
    check_greedy(weights, config, prompts[1], one)
    for prompt, got in zip(prompts, model.generate(prompts, max_new_tokens=5, use_graph=use_graph)):
        assert len(got) == 5
        check_greedy(weights, config, prompt, got)
    model.engine.check_status()
    held = [lin._q4 is not None for part in model.decoder.all_parts() for lin in vars(part).values() if type(lin).__name__ == "Linear"]
    assert sum(held) == 4 * config["num_hidden_layers"]


def test_rounded_matrices_matter(model_folders):
    """The engine's 4-bit logits follow the plain model with rounded matrices, and not the one with the stored ones."""
    from fastllm_py_b200 import Model, StepEntry

    name = "tiny_c"
    weights, config = plain.load_folder(model_folders[name])
    ids = list(range(5, 65))
    model = Model.load(model_folders[name], dtype="bfloat16", weights="mxfp4", page_size=32, max_tokens=256, max_requests=2,
                       max_batched_tokens=128, max_model_len=128, cuda_graph=False)
    model.engine.begin("a")
    got = model.engine.step([StepEntry("a", ids, [len(ids) - 1])])[0].float().cpu()
    model.engine.end("a")
    near = plain.forward(rounded(weights), config, ids, store=plain.store_bf16)[-1]
    exact = plain.forward(rounded(weights), config, ids)[-1]
    stored = plain.forward(weights, config, ids)[-1]
    noise = float((near - exact).abs().max())
    assert float((got - near).abs().max()) <= 2 * noise + 1e-3
    assert float((stored - exact).abs().max()) > 4 * noise, "the test's model does not tell the two apart"


def test_command_line(model_folders, capsys):
    from fastllm_py_b200.cli import main

    assert main([str(model_folders["tiny_a"]), "", "4", "--weights", "mxfp4", "--prompt-ids", "3,141,59,26", "--page-size", "16"]) == 0
    said = capsys.readouterr().out
    assert "weights=mxfp4" in said and "[4 tokens in" in said
