"""Matrices in 4 bits without a GPU: how work is shared out, options and refusals, and models with such matrices on stand-in
kernels."""
import io

import pytest
import torch

import helpers
import plain_qwen3
import tiny_configs
from chibillm_b200 import cli
from chibillm_b200.kernels.packed import GROUPS, FewRowsPlan, PackedWeights, few_rows_plan, many_rows_cut
from packed_models import PackedReferenceKernels, packed_weights
from reference_ops import ReferenceKernels

SMS = 148
CLUSTERS = {1: 148, 2: 74, 3: 45, 4: 33, 5: 26, 6: 22, 7: 15, 8: 15}      # as a B200 says


def smem_kb(wide, group, columns):
    def kb(tokens, warps, splits, batch, depth, run):
        plane = -(-(-(-columns // 128)) // splits) * 4 * tokens * 64
        stage = -(-run * (2048 + 128 // group * 64) // 128) * 128
        return -(-(warps * depth * stage + (2 if wide else 1) * plane + batch * warps * (1024 if tokens <= 8 else 2048) + 64
                   + warps * depth * 8) // 1024)
    return kb


def plan_of(rows, columns, paired, m, wide=False, group=64):
    return few_rows_plan(rows, columns, paired, m, wide, smem_kb(wide, group, columns),
                         lambda tokens, warps, splits, kb: CLUSTERS[splits] * (2 if warps == 8 and kb <= 113 else 1), SMS)


SIZES = [(1, 1), (16, 128), (2048, 1024), (2051, 1021), (4096, 4096), (4096, 12288), (12288, 4096), (151936, 4096), (64, 65536),
         (100, 20000), (1023, 2000)]


@pytest.mark.parametrize("rows,columns", SIZES)
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 12, 16, 17, 40, 300])
@pytest.mark.parametrize("paired,wide,group", [(False, False, 64), (True, False, 128), (False, True, 32), (True, True, 64)])
def test_a_plan_for_few_rows_fits_and_takes_every_record(rows, columns, m, paired, wide, group):
    p = plan_of(rows, columns, paired, m, wide, group)
    assert isinstance(p, FewRowsPlan)
    chunks, blocks = -(-columns // 128), -(-rows // (16 if paired else 32))
    assert p.warps in (8, 16) and p.tokens <= min(16, p.warps) and p.along_k in (1, 2, 4, 8, 16) and p.along_k <= p.warps
    assert p.splits in (1, 2, 4, 8) and p.splits <= chunks and p.depth >= 1 and 1 <= p.run <= 4 and p.batch >= 1
    assert smem_kb(wide, group, columns)(p.tokens, p.warps, p.splits, p.batch, p.depth, p.run) <= 226
    # the kernel's loops: every (block of rows, block of columns) once
    per_unit = p.warps // p.along_k
    units = -(-blocks // per_unit)
    assert 1 <= p.clusters <= units
    if blocks * chunks > 20000:
        return
    seen = set()
    for cluster in range(p.clusters):
        for unit in range(cluster, units, p.clusters):
            for rank in range(p.splits):
                c0, c1 = chunks * rank // p.splits, chunks * (rank + 1) // p.splits
                for warp in range(p.warps):
                    wk, wr = warp % p.along_k, warp // p.along_k
                    if unit * per_unit + wr >= blocks:
                        continue
                    for c in range(c0 + (c1 - c0) * wk // p.along_k, c0 + (c1 - c0) * (wk + 1) // p.along_k):
                        assert (unit * per_unit + wr, c) not in seen
                        seen.add((unit * per_unit + wr, c))
    assert len(seen) == blocks * chunks


@pytest.mark.parametrize("rows,columns", SIZES)
@pytest.mark.parametrize("m", [13, 17, 48, 49, 96, 97, 192, 193, 300, 1999, 2048, 5000])
@pytest.mark.parametrize("paired", [False, True])
def test_a_cut_for_many_rows_takes_every_tile_once(rows, columns, m, paired):
    cut = many_rows_cut(rows, columns, paired, m, lambda splits: CLUSTERS[splits])
    assert cut.tokens in (48, 96, 192) and 1 <= cut.splits <= min(8, -(-columns // 128))
    tiles = -(-rows // (64 if paired else 128)) * -(-m // cut.tokens)
    grid = cut.clusters * cut.splits
    assert grid <= CLUSTERS[cut.splits] * cut.splits
    whole = cut.rounds * grid
    if cut.splits == 1:
        assert whole >= tiles > whole - grid
    else:
        assert 0 < tiles - whole <= cut.clusters


def test_a_machine_that_takes_no_clusters_still_has_a_cut():
    assert many_rows_cut(4096, 4096, False, 200, lambda splits: 148 if splits == 1 else 0).splits == 1
    assert few_rows_plan(4096, 4096, False, 1, False, smem_kb(False, 64, 4096),
                         lambda tokens, warps, splits, kb: 148 if splits == 1 else 0, SMS).splits == 1


@pytest.mark.parametrize("group", GROUPS)
def test_bytes_and_first_rows(group):
    record = 2048 + 128 // group * 64
    assert PackedWeights.bytes_for(32, 128, group) == record == PackedWeights.bytes_for(16, 1, group, paired=True)
    assert PackedWeights.bytes_for(33, 129, group) == 4 * record
    w = PackedWeights(torch.empty(PackedWeights.bytes_for(100, 300, group), dtype=torch.uint8), 100, 300, group, False)
    first = w[:40]
    assert tuple(w.shape) == (100, 300) and tuple(first.shape) == (40, 300) and first.data is w.data and w[:40] is first
    for bad in (slice(0, 40), slice(None, 101), slice(None, 0), slice(None, 10, 2), 5):
        with pytest.raises(IndexError):
            w[bad]
    pair = PackedWeights(w.data, 50, 300, group, True)
    assert tuple(pair.shape) == (100, 300)
    with pytest.raises(IndexError):
        pair[:10]


def test_no_kernels_without_a_device():
    from chibillm_b200.kernels.ops import CudaKernels, KernelError
    k = CudaKernels.__new__(CudaKernels)
    k._device_index = 0
    w = torch.zeros(32, 64)
    for call in (lambda: k.pack_weights(w), lambda: k.pack_gate_up(w, w), lambda: k.pack_weights(w, 48),
                 lambda: k.pack_weights(w[0], 32), lambda: k.pack_gate_up(w, w[:3]),
                 lambda: k.pack_codes(w.to(torch.int8), w, 64),
                 lambda: k.linear(w, PackedWeights(w, 32, 64, 64, False), w),
                 lambda: k.linear(w, PackedWeights(w, 32, 64, 64, True), w),
                 lambda: k.linear_swiglu(w, PackedWeights(w, 32, 64, 64, False), w),
                 lambda: k.linear_swiglu(w, PackedWeights(w, 32, 64, 64, True), w, kind="tanh"),
                 lambda: k.unpack_weights(PackedWeights(w, 32, 64, 64, False), w)):
        with pytest.raises(KernelError):
            call()


def test_options():
    assert cli.parse_cli_options([]).weight_group is None
    assert cli.parse_cli_options(["--weight-group", "128"]).weight_group == 128
    for argv, message in ((["--weight-group"], "missing value"), (["--weight-group", "16"], "invalid weight group: 16")):
        with pytest.raises(cli.CliError) as e:
            cli.parse_cli_options(argv)
        assert message in str(e.value)
    assert "--weight-group" in cli.USAGE


def test_refusals_when_a_model_is_made(tmp_path):
    from chibillm_b200.engine.runner import ModelRunner
    folder = helpers.make_model_dir(tmp_path, "A", seed=1)
    with pytest.raises(ValueError, match="weight_group 48"):
        ModelRunner.from_folder(folder, device="cpu", kernels=PackedReferenceKernels(), weight_group=48)
    with pytest.raises(ValueError, match="no matrices in 4 bits"):
        ModelRunner.from_folder(folder, device="cpu", kernels=ReferenceKernels(), weight_group=64)


@pytest.mark.parametrize("name,group", [("A", 32), ("B", 64), ("C", 128)])
def test_models_with_matrices_in_4_bits_on_cpu(tmp_path, name, group):
    from chibillm_b200.engine.runner import ModelRunner
    folder = helpers.make_model_dir(tmp_path, name, seed=3)
    kernels = PackedReferenceKernels()
    runner = ModelRunner.from_folder(folder, dtype="float32", device="cpu", page_size=8, pool_tokens=192, kernels=kernels,
                                     weight_group=group)
    config, weights = plain_qwen3.read_model_folder(folder)
    weights = packed_weights(weights, group)
    requests = helpers.random_requests(tiny_configs.get(name)["vocab_size"], [5, 40, 70], seed=1)
    want = {rid: plain_qwen3.forward(config, weights, ids).float() for rid, ids in requests.items()}
    for trace in (helpers.trace_whole(requests), helpers.trace_portions(requests, seed=2)):
        helpers.assert_logits_close(helpers.run_trace(runner, trace), want, helpers.TOL["float32"], f"{name} in 4 bits")
    layers = config["num_hidden_layers"]
    assert kernels.calls["pack_weights"] == 3 * layers + 1 and kernels.calls["pack_gate_up"] == layers


def test_the_command_line_passes_it_on(tmp_path):
    folder = helpers.make_model_dir(tmp_path, "A", seed=2)
    config, weights = plain_qwen3.read_model_folder(folder)
    want = plain_qwen3.generate_greedy(config, packed_weights(weights, 32), [5, 6, 7], 4)
    kernels = PackedReferenceKernels()
    options = cli.parse_cli_options([folder, "--context-length", "64", "--max-tokens", "4", "--dtype", "float32", "--ignore-eos",
                                     "--no-stream", "--prompt-ids", "5,6,7", "--weight-group", "32"])
    out, err = io.StringIO(), io.StringIO()
    assert cli.run(options, io.StringIO(), out, err, kernels=kernels, device="cpu") == 0, err.getvalue()
    assert kernels.calls["packed gate and up"] > 0
    assert " ".join(map(str, want)) in out.getvalue()
