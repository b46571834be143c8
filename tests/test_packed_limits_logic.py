"""Matrices in 4 bits without a GPU: what must be refused or looked at before a kernel runs."""
import math
import os
import re
import weakref

import pytest
import torch

import chibillm_b200.csrc
import helpers
import tiny_configs
from chibillm_b200.config import GatedMLPSpec
from chibillm_b200.engine.runner import ModelRunner, make_runtime
from chibillm_b200.kernels.ops import CudaKernels, KernelError
from chibillm_b200.kernels import ops
from chibillm_b200.kernels.packed import PackedWeights, few_rows_plan, many_rows_cut
from chibillm_b200.parts import make_feed_forward
from chibillm_b200.weights import loader, random_init
from packed_models import PackedReferenceKernels
from reference_ops import ReferenceKernels


def smem_kb(wide, group, columns):
    """Shared memory of a CTA of the kernel for few rows, by its layout: rings, x, sums, the rows' notes and barriers."""
    def kb(tokens, warps, splits, batch, depth, run):
        plane = -(-(-(-columns // 128)) // splits) * 4 * tokens * 64
        stage = -(-run * (2048 + 128 // group * 64) // 128) * 128
        return -(-(warps * depth * stage + (2 if wide else 1) * plane + batch * warps * (1024 if tokens <= 8 else 2048) + 128
                   + warps * depth * 8) // 1024)
    return kb


def plan_of(rows, columns, paired, m, wide=False, group=64, clusters=lambda tokens, warps, splits, kb: 148 // splits):
    return few_rows_plan(rows, columns, paired, m, wide, smem_kb(wide, group, columns), clusters, 148)


def bare_kernels():
    """Kernels without a device: what stands before a launch."""
    k = CudaKernels.__new__(CudaKernels)
    k._device_index = 0
    return k


def test_both_matrices_of_a_pair_are_looked_at(monkeypatch):
    """Each tensor whose address a kernel gets has to be on the kernels' device."""
    k, seen = bare_kernels(), []
    monkeypatch.setattr(k, "_on_this_device", lambda what, *tensors: seen.extend(tensors))
    monkeypatch.setattr(k, "_packed_room", lambda *sizes: (_ for _ in ()).throw(KernelError("no room")))
    gate, up = torch.zeros(32, 64), torch.zeros(32, 64)
    with pytest.raises(KernelError, match="no room"):
        k.pack_gate_up(gate, up, 32)
    assert any(t is gate for t in seen) and any(t is up for t in seen)


def kernel_bodies(name):
    with open(os.path.join(os.path.dirname(chibillm_b200.csrc.__file__), name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^)]*\)\s*)?(\w+)\([^{;]*\)\n\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


def test_kernels_that_write_a_matrix_let_no_product_start_early():
    """bfloat16 products fetch their matrix before the kernel ahead of them has ended, so a kernel that makes one (its values read
    back are one, too) neither triggers the next launch nor ends with stores that a tile copy might miss."""
    bodies = dict(kernel_bodies("packed_weights.cu"))
    writers = ["pack_kernel", "pack_codes_kernel", "unpack_kernel"]
    assert set(writers) < set(bodies)
    for name in writers:
        assert "pdl_enter()" not in bodies[name] and "pdl_trigger" not in bodies[name], name
        assert bodies[name].lstrip().startswith("pdl_wait_now();") and "packed_done();" in bodies[name], name


@pytest.mark.parametrize("paired", [False, True])
def test_records_that_are_not_all_there_are_refused(monkeypatch, paired):
    """A kernel reads as many bytes as the matrix's sizes say."""
    k = bare_kernels()
    monkeypatch.setattr(k, "_on_this_device", lambda what, *tensors: None)
    k._current_device = lambda: (_ for _ in ()).throw(AssertionError("a launch"))
    k.error, k.lib, k.packed_few_rows_max = torch.zeros(1, dtype=torch.int32), None, 16
    rows, columns, group = 40, 200, 64
    need = PackedWeights.bytes_for(rows, columns, group, paired)
    whole = torch.zeros(need + 16, dtype=torch.uint8)
    whole = whole[-whole.data_ptr() % 16:][:need]
    x, out = torch.zeros(3, columns), torch.zeros(2 * rows if paired else rows, columns)
    for data in (whole[:-1], whole[:0], whole[1:], torch.zeros(need, dtype=torch.int8), torch.zeros(2 * need, dtype=torch.uint8)[::2],
                 torch.cat([whole, whole])[1:]):
        w = PackedWeights(data, rows, columns, group, paired)
        with pytest.raises(KernelError, match="bytes"):
            k.unpack_weights(w, out)
        with pytest.raises(KernelError, match="bytes"):
            k._packed_call(x, w, torch.zeros(3, rows), "silu" if paired else None, False, "linear")


@pytest.mark.parametrize("group", [64.0, True, "64", None, 0, 48, 256])
def test_groups_are_whole_numbers_of_the_list(monkeypatch, group):
    k = bare_kernels()
    monkeypatch.setattr(k, "_on_this_device", lambda what, *tensors: None)
    w = torch.zeros(32, 64)
    for call in (lambda: k.pack_weights(w, group), lambda: k.pack_gate_up(w, w, group),
                 lambda: k.pack_codes(w.to(torch.int8), torch.zeros(32, 1, dtype=torch.bfloat16), group)):
        with pytest.raises(KernelError, match="groups of"):
            call()
    if group is not None:
        with pytest.raises(ValueError, match="weight_group"):
            make_runtime("bfloat16", "cpu", kernels=PackedReferenceKernels(), weight_group=group)


CLUSTER_SIZES = [(1, 1), (64, 4096), (100, 20000), (64, 65536), (2051, 1021), (4096, 4096), (4096, 12288), (151936, 4096)]


@pytest.mark.parametrize("rows,columns", CLUSTER_SIZES)
@pytest.mark.parametrize("m", [1, 2, 8, 16, 17, 300])
@pytest.mark.parametrize("paired,wide", [(False, False), (True, False), (False, True)])
def test_clusters_that_do_not_run_are_no_plan(rows, columns, m, paired, wide):
    """A device that takes no clusters (or none of 8): a plan keeps to what runs, or there is none."""
    for largest in (1, 4):
        p = plan_of(rows, columns, paired, m, wide, clusters=lambda tokens, warps, splits, kb: 148 // splits if splits <= largest else 0)
        whole = plan_of(rows, columns, paired, m, wide)
        assert p is None or p.splits <= largest
        # nothing fits only where x of one row is beyond what CTAs of such clusters hold
        if p is None:
            assert whole.splits > largest and smem_kb(wide, 64, columns)(1, 8, largest, 1, 1, 1) > 226
    assert plan_of(rows, columns, paired, m, wide, clusters=lambda *cut: 0) is None


def test_a_device_that_runs_nothing_has_no_cut_for_many_rows():
    assert many_rows_cut(4096, 4096, False, 200, lambda splits: 0) is None
    assert many_rows_cut(4096, 4096, False, 20, lambda splits: 74 if splits == 2 else 0).splits == 2


def test_a_query_that_failed_is_asked_again(monkeypatch):
    """What the device says about clusters is kept, but not an error, and no plan that came of one."""
    class Library:
        answers = {"few": 0, "many": 0}

        def chibi_packed_few_rows_kb(self, x32, group, columns, *cut):
            return smem_kb(bool(x32), group, columns)(*cut)

        def chibi_packed_few_rows_clusters(self, x32, group, tokens, warps, splits, kb):
            return self.answers["few"] // splits

        def chibi_packed_many_rows_clusters(self, splits):
            return self.answers["many"] // splits

    monkeypatch.setattr(ops, "_PACKED_CLUSTERS", {})
    k = bare_kernels()
    k.lib, k.sm_count, k._packed_plans, k._packed_cuts = Library(), 148, {}, {}
    w = PackedWeights(torch.zeros(1, dtype=torch.uint8), 64, 4096, 64, False)
    for ask, which in ((lambda: k.packed_plan(w, 1, False), "few"), (lambda: k.packed_cut(w, 200), "many")):
        with pytest.raises(KernelError):
            ask()
        Library.answers[which] = 148
        assert ask().clusters >= 1


@pytest.mark.parametrize("activation,biases", [("silu", False), ("gelu_tanh", False), ("gelu_tanh", True)])
def test_feed_forwards_take_matrices_in_another_order(activation, biases):
    """Tensors whose rows are not contiguous are put in order before they are packed, as the other layouts do."""
    class Strict(PackedReferenceKernels):
        def pack_weights(self, w, group=64):
            assert w.is_contiguous()
            return super().pack_weights(w, group)

        def pack_gate_up(self, gate, up, group=64):
            assert gate.is_contiguous() and up.is_contiguous()
            return super().pack_gate_up(gate, up, group)

    g = torch.Generator().manual_seed(3)
    names = {n: n for n in ("gate_proj", "up_proj", "down_proj", "gate_bias", "up_bias", "down_bias")}
    tensors = {"gate_proj": torch.randn(96, 64, generator=g), "up_proj": torch.randn(96, 64, generator=g),
               "down_proj": torch.randn(64, 96, generator=g), "gate_bias": torch.randn(96, generator=g),
               "up_bias": torch.randn(96, generator=g), "down_bias": torch.randn(64, generator=g)}
    spec = GatedMLPSpec("gated_mlp", hidden_size=64, intermediate_size=96, activation=activation, biases=biases)
    bound = []
    for order in (lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        runtime = make_runtime("float32", "cpu", kernels=Strict(), weight_group=32)
        part = make_feed_forward(spec, names, runtime)
        part.bind({n: order(t) for n, t in tensors.items()})
        bound.append(part)
    for name in ("gate_up", "gate_up_interleaved", "down"):
        one, other = (getattr(p, name) for p in bound)
        assert (one is None) == (other is None) and (one is None or torch.equal(one.values, other.values)), name


def live_bytes_while(monkeypatch, load):
    """The most bytes of source tensors on the device at any time while ``load`` runs (counted where a part asks for one)."""
    live, most = {}, [0]

    def watched(make):
        def made(*args, **kw):
            t = make(*args, **kw)
            key = id(t)
            live[key] = t.numel() * t.element_size()
            weakref.finalize(t, live.pop, key, None)
            most[0] = max(most[0], sum(live.values()))
            return t
        return made

    monkeypatch.setattr(loader, "put_on_device", watched(loader.put_on_device))
    monkeypatch.setattr(random_init, "stored_tensor", watched(random_init.stored_tensor))
    load()
    return most[0]


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("from_folder", [True, False])
def test_a_model_is_never_whole_on_the_device_beside_its_packed_matrices(tmp_path, monkeypatch, name, from_folder):
    """Packing while a model is loaded: a matrix goes when it has been packed, so what fits in 4 bits can be loaded."""
    config = dict(tiny_configs.get(name), num_hidden_layers=12)
    folder = helpers.make_model_dir(tmp_path, name, seed=3, num_hidden_layers=12)
    kernels = PackedReferenceKernels()
    common = dict(dtype="float32", device="cpu", page_size=8, pool_tokens=192, kernels=kernels, weight_group=32)
    runners = []
    most = live_bytes_while(monkeypatch, lambda: runners.append(
        ModelRunner.from_folder(folder, **common) if from_folder else ModelRunner.from_random(config, seed=3, **common)))
    spec = runners[0].model.spec
    sizes = {t.name: math.prod(t.shape) * 4 for t in runners[0].model.expected_tensors(None)}
    kept = sum(n for name, n in sizes.items() if "norm" in name) + sizes[spec.embedding_name] + sizes.get(spec.output_name, 0)
    layer = sum(n for name, n in sizes.items() if ".layers.0." in name)
    assert most <= kept + layer < sum(sizes.values()) / 3


def test_loaded_tensors_are_one_while_somebody_holds_them(tmp_path):
    folder = helpers.make_model_dir(tmp_path, "A", seed=3)
    runner = ModelRunner.from_folder(folder, dtype="float32", device="cpu", page_size=8, pool_tokens=192, kernels=ReferenceKernels())
    tensors = loader.load_weights(runner.model, folder, runner.runtime)
    names = list(tensors)
    held = tensors[names[0]]
    assert tensors[names[0]] is held and names[0] in tensors and "no such" not in tensors and None not in tensors
    assert tensors.get(None) is None and len(tensors) == len(names) == len(set(names))
    with pytest.raises(KeyError):
        tensors["no such"]
