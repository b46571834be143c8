"""Whole models with their matrices in 4 bits on the device, against the plain implementation with the values that packing leaves."""
import pytest
import torch

import fokurax_models
import gitipel_models
import helpers
import lefavik_models
import plain_qwen3
import tiny_configs
from packed_models import packed_values, packed_weights

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16"]


def runner_of(folder, dtype, group, page_size=16, pool=512, max_requests=8):
    from chibillm_b200.engine.runner import ModelRunner
    runner = ModelRunner.from_folder(folder, dtype=dtype, page_size=page_size, pool_tokens=pool, max_requests=max_requests,
                                     weight_group=group)
    runner.storage.poison()
    return runner


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name,group", [("A", 64), ("B", 32), ("C", 128)])
def test_tiny_models(tmp_path, name, group, dtype):
    folder = helpers.make_model_dir(tmp_path, name, seed=3)
    config, weights = plain_qwen3.read_model_folder(folder)
    weights = packed_weights(weights, group)
    vocab = tiny_configs.get(name)["vocab_size"]
    requests = helpers.random_requests(vocab, [5, 40, 70, 90], seed=1)
    want = {rid: plain_qwen3.forward(config, weights, ids).float() for rid, ids in requests.items()}
    runner = runner_of(folder, dtype, group)
    for trace, what in ((helpers.trace_whole(requests), "whole"), (helpers.trace_last_decoded(requests, 20), "decoded"),
                        (helpers.trace_portions(requests, seed=2), "portions"), (helpers.trace_mixed(requests, 512, seed=4), "mixed")):
        helpers.assert_logits_close(helpers.run_trace(runner, trace), want, helpers.TOL[dtype], f"4 bits {name} {dtype} {what}")
    runner.runtime.kernels.check_error_word()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_of_real_sizes(tmp_path, dtype):
    """Two layers of width 1,024 with prompts long enough for the product of many rows, and single tokens of several requests."""
    folder = helpers.make_model_dir(tmp_path, "A", seed=5, hidden_size=1024, num_attention_heads=16, num_key_value_heads=8, head_dim=128,
                                    intermediate_size=2048, vocab_size=4099, max_position_embeddings=1024)
    config, weights = plain_qwen3.read_model_folder(folder)
    weights = packed_weights(weights, 64)
    requests = helpers.random_requests(4099, [300, 230, 17], seed=7)
    want = {rid: plain_qwen3.forward(config, weights, ids).float() for rid, ids in requests.items()}
    runner = runner_of(folder, dtype, 64, pool=1024)
    for trace, what in ((helpers.trace_whole(requests), "whole"), (helpers.trace_last_decoded(requests, 12), "decoded"),
                        (helpers.trace_mixed(requests, 1024, seed=4), "mixed")):
        helpers.assert_logits_close(helpers.run_trace(runner, trace), want, helpers.TOL[dtype], f"4 bits width 1024 {dtype} {what}")
    assert runner.graph_replays > 0


def test_generation_is_the_plain_implementations(tmp_path):
    import chibillm_b200
    folder = helpers.make_model_dir(tmp_path, "B", seed=6)
    config, weights = plain_qwen3.read_model_folder(folder)
    weights = packed_weights(weights, 64)
    prompts = list(helpers.random_requests(384, [9, 33, 4, 60], seed=8).values())
    want = [plain_qwen3.generate_greedy(config, weights, p, 10) for p in prompts]
    llm = chibillm_b200.LLM(folder, dtype="float32", context_length=128, max_sequences=4, weight_group=64)
    assert llm.generate(prompts, max_tokens=10, ignore_eos=True) == want
    assert llm.generate(prompts[:1], max_tokens=10, ignore_eos=True) == want[:1]
    one = chibillm_b200.LLM(folder, dtype="bfloat16", context_length=128, max_sequences=4, weight_group=64)
    assert one.generate(prompts, max_tokens=10, ignore_eos=True) == one.generate(prompts, max_tokens=10, ignore_eos=True)


@pytest.mark.parametrize("config", [lefavik_models.get("L1"), lefavik_models.get("L3"), lefavik_models.get("L4"),
                                    fokurax_models.get("F1"), fokurax_models.get("F3")], ids=["L1", "L3", "L4", "F1", "F3"])
def test_other_architectures(config):
    """The same model with matrices in 4 bits, and with the values that those stand for as 32-bit matrices."""
    from chibillm_b200.config.registry import find_architecture
    from chibillm_b200.engine.model import DecoderModel
    from chibillm_b200.engine.runner import ModelRunner, make_runtime
    from chibillm_b200.parts.attention import PagedAttention
    from chibillm_b200.parts.mlp import DenseMLP, GatedMLP
    from chibillm_b200.weights.random_init import random_tensors
    arch = find_architecture(config)
    spec = arch.model_spec(arch.read_config(config))
    logits = []
    for group in (32, None):
        runtime = make_runtime("float32", "cuda:0", spec=spec, weight_group=group)
        model = DecoderModel(spec, runtime)
        tensors = {n: (t if t.dtype == torch.int32 else t.float()).to("cuda:0") for n, t in
                   random_tensors(model, 3, torch.bfloat16, torch.device("cuda:0"))}
        if group is None:
            packed = set()
            for part in parts_of(model):
                if isinstance(part, (PagedAttention, GatedMLP, DenseMLP)):
                    packed |= {t.name for t in part.expected_tensors() if len(t.shape) == 2}
            assert packed
            for n in packed:
                tensors[n] = packed_values(tensors[n], 32)
            output = packed_values(tensors.get(spec.output_name, tensors[spec.embedding_name]), 32)
        model.bind(tensors)
        if group is None:
            model.output = output
        runner = ModelRunner(model, runtime, 16, 512, 4)
        requests = helpers.random_requests(spec.vocab_size, [33, 7, 50], seed=9)
        logits.append(helpers.run_trace(runner, helpers.trace_last_decoded(requests, 6)))
    helpers.assert_logits_close(logits[0], logits[1], helpers.TOL["float32"], "4 bits, another architecture")


@pytest.mark.parametrize("name", ["G1", "G3"])
def test_a_recurrent_architecture_cut_in_different_ways(tmp_path, name):
    """Gitipel: attention and feed-forwards in 4 bits beside a recurrence as it is; whole prompts against single tokens."""
    config = gitipel_models.get(name)
    folder = gitipel_models.write_model(config, str(tmp_path / "model"), 4)
    vocab = int(config["vocab"]) if "vocab" in config else int(config["vocab_size"])
    requests = helpers.random_requests(vocab, [33, 7, 50], seed=9)
    logits = []
    for group in (32, None):
        runner = runner_of(folder, "float32", group)
        whole = helpers.run_trace(runner, helpers.trace_whole(requests))
        helpers.assert_logits_close(helpers.run_trace(runner, helpers.trace_last_decoded(requests, 6)), whole, helpers.TOL["float32"],
                                    f"4 bits {name} decoded")
        logits.append(whole)
    # the matrices did change, and not by much
    for rid in requests:
        off = float((logits[0][rid] - logits[1][rid]).norm() / logits[1][rid].norm())
        assert 1e-3 < off < 0.7, off


def parts_of(model):
    seen, todo = [], list(model.blocks)
    while todo:
        part = todo.pop()
        if part in seen or isinstance(part, (torch.Tensor, str)):
            continue
        seen.append(part)
        for value in vars(part).values() if hasattr(part, "__dict__") else ():
            for v in value if isinstance(value, (list, tuple)) else (value,):
                if type(v).__module__.startswith("chibillm_b200.parts") and hasattr(v, "expected_tensors"):
                    todo.append(v)
    return seen

