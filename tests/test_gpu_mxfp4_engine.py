"""The engine with projections in 4 bits: logits against the plain implementation with the weights that the codes stand for, every
product of a run against 64-bit sums of its own inputs, recorded steps, generation, refusals."""
import pytest
import torch
from conftest import REAL_LAYERS, TINY

import bench
import plain_qwen3 as P
import trace_tools as T
from mini_rsglang_b200 import RuntimeConfig, SamplingParams, kernels
from mini_rsglang_b200.engine import EngineHandle, ModelRunner, SequenceStep
from mini_rsglang_b200.errors import InvalidRequest
from mini_rsglang_b200.models import config_from_dict
from mini_rsglang_b200.parts import FEED_FORWARDS, Runtime
from mini_rsglang_b200.weights import write_random_model
from test_gpu_mxfp4 import close_to_sums, plain_quantise, plain_values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# widths that are whole blocks of 32, odd numbers of them and of heads
CONFIG = dict(model_type="qwen3", architectures=["Qwen3ForCausalLM"], hidden_size=160, intermediate_size=224, num_hidden_layers=3,
              num_attention_heads=6, num_key_value_heads=2, head_dim=32, vocab_size=389, max_position_embeddings=1024, rms_norm_eps=1e-6,
              rope_theta=100000.0, tie_word_embeddings=False, hidden_act="silu", eos_token_id=5)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("four_bits"))
    write_random_model(path, config_from_dict(CONFIG), seed=77, dtype=torch.bfloat16)
    return path


def runner_for(folder, activations="held", **limits):
    return ModelRunner.load(folder, limits=RuntimeConfig(max_seq_len=512, page_size=8, max_running=4, weight_format="mxfp4",
                                                         activation_format=activations, **limits), num_pages=96)


def plain_weights(folder):
    """The checkpoint with every projection replaced by what its 4 bits stand for."""
    weights = P.load_plain_weights(folder)
    return {name: plain_quantise(w.bfloat16())[0].to(w.dtype) if name.endswith("_proj.weight") else w for name, w in weights.items()}


def feed(runner, request, tokens, cuts):
    out, pos = [], 0
    runner.cache.open(request)
    for n in cuts:
        runner.cache.extend(request, pos + n)
        out.append(runner.step([SequenceStep(request, tokens[pos:pos + n], pos, list(range(n)))]).double().cpu())
        pos += n
    return torch.cat(out)


def test_logits_are_those_of_the_values(folder):
    tokens = [(13 * i + 7) % CONFIG["vocab_size"] for i in range(230)]
    want = P.logits_of_sequence(P.PlainConfig.load(folder), plain_weights(folder), tokens)
    runner = runner_for(folder)
    assert runner.model.projections_in_4_bits() == 4 * CONFIG["num_hidden_layers"]
    T.check_rows(feed(runner, 1, tokens, [230]), want, "bfloat16", "whole")
    T.check_rows(feed(runner, 2, tokens[:40], [17, 1, 1, 9, 12]), want[:40], "bfloat16", "portions")
    T.check_rows(feed(runner, 3, tokens[:24], [1] * 24), want[:24], "bfloat16", "one by one")


def test_recorded_decode_steps(folder):
    """Three requests decode together through recorded steps, beside a prompt."""
    tokens = [[(31 * i + 11 * r) % CONFIG["vocab_size"] for i in range(60)] for r in range(3)]
    weights = plain_weights(folder)
    want = [P.logits_of_sequence(P.PlainConfig.load(folder), weights, t) for t in tokens]
    runner = runner_for(folder)
    heads = [30, 3, 17]
    for r in range(3):
        runner.cache.open(r + 1)
        runner.cache.extend(r + 1, heads[r])
        runner.step([SequenceStep(r + 1, tokens[r][:heads[r]], 0, [])])
    for k in range(20):
        batch = []
        for r in range(3):
            runner.cache.extend(r + 1, heads[r] + k + 1)
            batch.append(SequenceStep(r + 1, [tokens[r][heads[r] + k]], heads[r] + k, [0]))
        T.check_rows(runner.step(batch).double().cpu(), torch.stack([want[r][heads[r] + k] for r in range(3)]), "bfloat16", f"step {k}")
    assert runner.recorded_steps > 0


@pytest.mark.parametrize("activations", ["held", "mxfp4"])
def test_every_product_of_a_run(folder, activations, monkeypatch):
    """A prompt and single tokens: each product's output against 64-bit sums of the very rows it read."""
    seen = []
    product = kernels.mxfp4_gemm

    def watched(x, weight, out, quantise=False, plan=None):
        product(x, weight, out, quantise=quantise, plan=plan)
        assert quantise == (activations == "mxfp4")
        values = plain_quantise(x)[0] if quantise else x.double()
        w = plain_values(weight.codes, weight.block_scales())
        close_to_sums(out, values @ w.T, values.abs() @ w.abs().T, x.shape[1], f"{tuple(x.shape)} x {weight.shape}")
        seen.append((x.shape[0], weight.shape))

    monkeypatch.setattr(kernels, "mxfp4_gemm", watched)
    runner = runner_for(folder, activations, record_mixed_steps=False)
    runner.record_decode = False
    tokens = [(29 * i + 3) % CONFIG["vocab_size"] for i in range(150)]
    logits = feed(runner, 1, tokens, [131, 1, 1, 17])
    assert logits.isfinite().all() and len(seen) == 4 * 4 * CONFIG["num_hidden_layers"]


@pytest.mark.parametrize("activations", ["held", "mxfp4"])
def test_generation(folder, activations):
    """The same greedy tokens with recorded steps and without, and again from the same engine."""
    prompts = [[5 + i, 17, 3, 99] * 6 for i in range(3)] + [[7] * 41]
    results = []
    for record in (True, False):
        limits = RuntimeConfig(max_seq_len=128, page_size=8, prefill_budget=32, max_running=4, weight_format="mxfp4", activation_format=activations,
                               record_mixed_steps=record)
        engine = EngineHandle.load(folder, 0, config=limits, num_pages=96)
        engine.runner.record_decode = record
        sampling = SamplingParams(max_tokens=12, ignore_eos=True)
        first, again = ([r.token_ids for r in engine.generate_many(prompts, sampling)] for _ in range(2))
        assert first == again and all(len(t) == 12 for t in first)
        results.append(first)
        engine.shutdown()
    # padded steps may take other kernels for their rows: rounding only, so single requests differ at most where two logits are near
    assert sum(a == b for a, b in zip(*results)) >= 3


@pytest.mark.parametrize("kind", ["swiglu", "gated_mlp", "dense_mlp", "clamped_glu"])
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_feed_forwards_take_4_bits(kind, rows):
    """Every dense feed-forward: with weights that 4 bits hold exactly it computes what it computes with those weights in bfloat16."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    width, inner = 96, 160
    extra = {"clamped_glu": {"limit": 7.0}}.get(kind, {})
    parts = [FEED_FORWARDS.get(kind)(prefix="f", width=width, inner=inner, **extra) for _ in range(2)]
    tensors = {}
    for spec in parts[0].weight_specs():
        w = torch.randn(spec.shape, device=DEV, generator=g) * 0.2
        tensors[spec.name] = plain_quantise(w.bfloat16())[0].bfloat16()
        assert torch.equal(plain_quantise(tensors[spec.name])[0], tensors[spec.name].double())
    for part, form in zip(parts, ("held", "mxfp4")):
        part.bind(dict(tensors), Runtime(torch.device(DEV), torch.bfloat16, 16, form))
    h = torch.randn(rows, width, device=DEV, generator=g).bfloat16()
    held, four = (part.forward(h.clone(), None) for part in parts)
    assert held.dtype is four.dtype and four.isfinite().all()
    # both round the inner activations to bfloat16 once (two roundings a part of the gate: 2^-8 each) and sum in float32
    assert (held.double() - four.double()).norm() <= 3 * 2.0 ** -8 * held.double().norm()


def test_refusals(folder, model_folders, tmp_path):
    with pytest.raises(InvalidRequest, match="32-bit path"):
        ModelRunner.load(folder, dtype="float32", limits=RuntimeConfig(max_seq_len=64, weight_format="mxfp4"), num_pages=8)
    with pytest.raises(InvalidRequest, match="whole blocks of 32"):          # a width of 136
        ModelRunner.load(model_folders["D"], limits=RuntimeConfig(max_seq_len=64, page_size=TINY["D"][1], weight_format="mxfp4"), num_pages=8)
    with pytest.raises(InvalidRequest, match="weight_format"):
        ModelRunner.load(folder, limits=RuntimeConfig(max_seq_len=64, activation_format="mxfp4"), num_pages=8)


def test_real_layer_sizes(real_size_folder):
    """Two layers with the sizes of a real checkpoint: a prompt, then single tokens, in the kernels that serve them."""
    tokens = [(101 * i + 13) % REAL_LAYERS["vocab_size"] for i in range(70)]
    want = P.logits_of_sequence(P.PlainConfig.load(real_size_folder), plain_weights(real_size_folder), tokens)
    runner = ModelRunner.load(real_size_folder, limits=RuntimeConfig(max_seq_len=512, max_running=2, weight_format="mxfp4"), num_pages=32)
    T.check_rows(feed(runner, 1, tokens, [60, 1, 1, 8]), want, "bfloat16", "real sizes")


def model_with_4_bits(name, folder, activations):
    """The engine's dense model, or a small one of each other design with a mixer of every kind that the design has."""
    if name == "qwen3":
        return runner_for(folder, activations)
    raw = bench.DESIGNS[name][3](dict(width=512, ff=512, heads=4, kv_heads=2, layers=8), CONFIG["vocab_size"])[0]
    limits = RuntimeConfig(max_seq_len=512, page_size=16, max_running=4, weight_format="mxfp4", activation_format=activations)
    return ModelRunner.from_random(config_from_dict(raw), 5, limits=limits, num_pages=96)


@pytest.mark.parametrize("name,activations", [("qwen3", "held"), ("qwen3", "mxfp4")] + [(name, "held") for name in bench.DESIGNS])
def test_padding_rows_are_ordinary_numbers(folder, name, activations, monkeypatch):
    """Recorded steps have rows that belong to no sequence, which attention, scans and gates leave out.  What the memory held before reaches no
    product: one row far from the others, or not finite, would choose the operands of all."""
    poisoned = [False]
    for entry in ("empty", "empty_like"):
        def make(*args, _plain=getattr(torch, entry), **kwargs):
            made = _plain(*args, **kwargs)
            return made.fill_(float("nan")) if poisoned[0] and made.is_cuda and made.is_floating_point() else made

        monkeypatch.setattr(torch, entry, make)
    seen = {}
    product = kernels.mxfp4_gemm

    def watched(x, weight, out, quantise=False, plan=None):
        product(x, weight, out, quantise=quantise, plan=plan)
        if torch.cuda.is_current_stream_capturing():
            seen.setdefault(x.shape[0], []).append(x.clone())

    monkeypatch.setattr(kernels, "mxfp4_gemm", watched)
    runner = model_with_4_bits(name, folder, activations)
    poisoned[0] = True
    tokens = [(29 * i + 3) % CONFIG["vocab_size"] for i in range(90)]

    def step(batch, rows):
        assert runner.step(batch).isfinite().all()
        assert seen[rows] and all(x.isfinite().all() for x in seen[rows])

    for request, n, rows in ((1, 30, 32), (2, 3, 16), (3, 17, 32)):
        runner.cache.open(request)
        runner.cache.extend(request, n)
        step([SequenceStep(request, tokens[:n], 0, [n - 1])], rows)
    for k in range(3):                                             # three decoded tokens in a step of four
        for request, n in ((1, 30), (2, 3), (3, 17)):
            runner.cache.extend(request, n + k + 1)
        step([SequenceStep(request, [tokens[n + k]], n + k, [0]) for request, n in ((1, 30), (2, 3), (3, 17))], 4)
    assert runner.recorded_steps == 6
