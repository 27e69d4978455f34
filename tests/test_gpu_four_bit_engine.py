"""The engine on a cache of 4 bits an element against the plain implementation with keys and values kept that way."""
import numpy as np
import pytest
import torch

from tests import schedules
from tests.four_bit_util import quantised
from tests.plain import qwen3_plain
from tests.test_gpu_engine import SCHEDULES, compare, run_steps
from tests.util import TINY, make_model_dir, random_tokens, read_config, read_weights, tolerance

pytestmark = pytest.mark.gpu
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
LENGTHS = {"B": [5, 23, 40], "M": [90, 45, 130, 17]}


@pytest.fixture(scope="module")
def cases(tmp_path_factory):
    cache = {}

    def get(name, dtype_name):
        key = (name, dtype_name)
        if key not in cache:
            folder = str(tmp_path_factory.mktemp(f"four_bit_{name}_{dtype_name}"))
            make_model_dir(folder, TINY[name], seed=3 + len(cache), dtype=DTYPES[dtype_name])
            config, weights = read_config(folder), read_weights(folder)
            requests = {f"r{i}": random_tokens(10 * i + 3, n, config["vocab_size"]) for i, n in enumerate(LENGTHS[name])}
            cache[key] = (folder, config, weights, requests)
        return cache[key]

    return get


def _engine(folder, dtype_name, **options):
    from leone_amd.engine.engine import Engine
    from leone_amd.runtime import load_model
    model = load_model(folder, DTYPES[dtype_name], "cuda:0")
    return Engine(model, max_requests=4, cache_bits=4, **options)


def _plain(config, weights, tokens, kept, windows=None):
    """The plain implementation whose attention reads ``kept(layer, keys, values)``; logits, and the layers' own keys and values.
    ``windows``: of layers that have one."""
    exact, seen = qwen3_plain.causal_attention, []

    def attention(q, k, v, window=None):
        seen.append((k, v))
        return exact(q, *kept(len(seen) - 1, k, v), (windows or {}).get(len(seen) - 1, window))

    try:
        qwen3_plain.causal_attention = attention
        return qwen3_plain.forward(weights, config, tokens).numpy(), seen
    finally:
        qwen3_plain.causal_attention = exact


def _cached(engine, request):
    """What the cache holds of a request, layer by layer: (keys, values) float64 ``[tokens, heads, dim]``."""
    from leone_amd import ops
    table = torch.tensor([engine.cache.table(request, 0)], dtype=torch.int32, device="cuda:0")
    positions = torch.arange(engine.length(request), dtype=torch.int32, device="cuda:0")
    found = []
    for slot in sorted(engine.pools.paged):
        pools = engine.pools.paged[slot]
        k, v = ops.cache_rows_4bit(pools, positions, torch.zeros_like(positions), table)
        found.append(tuple(x.double().cpu().reshape(len(positions), pools[0].shape[1], -1) for x in (k, v)))
    return found


@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("schedule", list(SCHEDULES))
def test_float32_schedules(cases, schedule, page_tokens):
    """Held to what the model is held to without such a cache.  (A hidden state off by some 1e-6 puts one element in 10^5 on the other
    side of the border between two codes; the three requests have 13,000.)"""
    folder, config, weights, requests = cases("B", "float32")
    expected = {rid: _plain(config, weights, toks, lambda layer, k, v: (quantised(k), quantised(v)))[0] for rid, toks in requests.items()}
    engine = _engine(folder, "float32", max_tokens=512, page_tokens=page_tokens, poison_freed=True)
    steps = list(SCHEDULES[schedule](requests))
    compare(steps, run_steps(engine, steps), expected, tolerance("float32"), schedule)


@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("schedule", list(SCHEDULES))
def test_bfloat16_schedules(cases, schedule, page_tokens):
    """Given what the cache holds, the logits are held to what the model is held to without such a cache.  What it holds are the plain
    implementation's keys and values but for elements whose neighbouring code is as near: the hidden states are rounded to 2^-8 at
    every step, some 0.5 % of an element, 0.01 of its block's unit, and borders lie 0.5 to 2 units apart, so that some 2 % of the
    elements are on the other side of one (and a block in a hundred has another unit): one in ten at most."""
    from leone_amd.engine.engine import StepEntry
    folder, config, weights, requests = cases("M", "bfloat16")
    engine = _engine(folder, "bfloat16", max_tokens=512, page_tokens=page_tokens, poison_freed=True)
    steps, outputs, held = list(SCHEDULES[schedule](requests)), {}, {}
    for s in steps:
        out = engine.step([StepEntry(e["id"], e["tokens"], e["want"]) for e in s["entries"]])
        if out.logits is not None:
            outputs[s["step"]] = out.logits.float().cpu().numpy()
        for rid in s["end"]:
            held[rid] = _cached(engine, rid)
            engine.release(rid)
        engine.cache.check()
    got = schedules.collect(steps, outputs)
    for rid, toks in requests.items():
        want, seen = _plain(config, weights, toks, lambda layer, k, v: held[rid][layer])
        off = np.abs(np.stack(got[rid]) - want).max()
        assert off <= tolerance("bfloat16"), (rid, off)
        for layer, kept in enumerate(held[rid]):
            for x, y in zip(kept, seen[layer]):
                other = (x != quantised(y)).double().mean().item()
                assert other <= 0.1, (rid, layer, other)


@pytest.mark.parametrize("graphs", [False, True])
def test_recorded_and_eager_steps(cases, graphs):
    """Decode steps from a recording, replayed with other work and synchronizations between, and kernel by kernel."""
    from leone_amd.engine.engine import StepEntry
    folder, config, weights, requests = cases("M", "bfloat16")
    engine = _engine(folder, "bfloat16", max_tokens=1024, page_tokens=64, graphs=graphs)
    for rid, toks in requests.items():
        engine.step([StepEntry(rid, toks[:-8], [])])
    got = []
    for i in range(8, 0, -1):
        out = engine.step([StepEntry(rid, [toks[-i]], [0]) for rid, toks in requests.items()])
        got.append(out.logits.float().cpu().numpy())
        torch.zeros(1 << 16, device="cuda:0").add_(1.0)
        torch.cuda.synchronize()
    for at, (rid, toks) in enumerate(requests.items()):
        held = _cached(engine, rid)
        want = _plain(config, weights, toks, lambda layer, k, v: held[layer])[0][-8:]
        assert np.abs(np.stack([rows[at] for rows in got]) - want).max() <= tolerance("bfloat16"), rid


def test_generation_and_what_a_token_takes(cases):
    from leone_amd.api import Runtime, cache_bytes_per_token, sampling_params
    folder, _, _, requests = cases("M", "bfloat16")
    prompts = list(requests.values())
    runtime = Runtime.load(folder, "bfloat16", "cuda:0", max_requests=4, max_context=512, cache_bits=4)
    greedy = runtime.generate_tokens(prompts, 12, eos_token_id=None)
    again = runtime.generate_tokens(prompts, 12, eos_token_id=None)
    assert [r.tokens for r in greedy] == [r.tokens for r in again] and all(len(r.tokens) == 12 for r in greedy)
    drawn = runtime.generate_tokens(prompts, 6, sampling_params(temperature=0.8, seed=3, top_k=20), eos_token_id=None)
    assert all(len(r.tokens) == 6 for r in drawn)
    model = runtime.model
    assert runtime.engine.pools.bytes_per_token() == cache_bytes_per_token(model, 4) == cache_bytes_per_token(model) * 17 // 64


def test_forks_share_pages_and_requests_are_cut_back(cases):
    from leone_amd.engine.engine import StepEntry
    folder, _, _, requests = cases("B", "float32")
    toks = requests["r2"]
    engine = _engine(folder, "float32", max_tokens=1024, page_tokens=16)
    whole = engine.step([StepEntry("a", toks, [len(toks) - 1])]).logits.clone()
    held = engine.fork("a", "b", 35)
    out = engine.step([StepEntry("b", toks[held:], [len(toks) - held - 1])]).logits
    assert held == 32 and (out - whole).abs().max() <= tolerance("float32")
    engine.truncate("a", 32)                                   # (within a page that is shared it cannot be cut)
    out = engine.step([StepEntry("a", toks[32:], [len(toks) - 33])]).logits
    assert (out - whole).abs().max() <= tolerance("float32")


@pytest.mark.parametrize("schedule", list(SCHEDULES))
def test_windows_and_attention_as_a_branch(cases, schedule):
    """A layer that sees the last 20 tokens (its pages behind them are given back) and one whose attention is a branch of a mixer of
    several, which keeps its cache under a name."""
    import dataclasses
    from leone_amd.architectures import config_from_dict, model_spec_for
    from leone_amd.engine.engine import Engine
    from leone_amd.parts.base import PartSpec
    from leone_amd.parts.model import DecoderModel
    from leone_amd.weights import loader
    folder, config, weights, requests = cases("B", "float32")
    spec = model_spec_for(config_from_dict(config))
    first, second = (dict(layer.params) for layer in spec.layers[:2])
    first["mixer"] = PartSpec("gqa_attention", {**first["mixer"].params, "window": 20})
    second["mixer"] = PartSpec("parallel", {"hidden": config["hidden_size"], "eps": 1e-6, "weights": {"only": 1.0},
                                            "branches": {"only": PartSpec("gqa_attention", {**second["mixer"].params, "float_output": True})}})
    spec = dataclasses.replace(spec, layers=[PartSpec("prenorm", first), PartSpec("prenorm", second), *spec.layers[2:]])
    model = DecoderModel(spec, torch.float32, "cuda:0")
    model.bind(loader.load_from_dir(folder, model.tensor_specs(), torch.float32, torch.device("cuda:0"), ignore=spec.ignore_tensors))
    expected = {rid: _plain(config, weights, toks, lambda layer, k, v: (quantised(k), quantised(v)), {0: 20})[0] for rid, toks in requests.items()}
    engine = Engine(model, max_requests=4, cache_bits=4, max_tokens=512, page_tokens=16, poison_freed=True)
    steps = list(SCHEDULES[schedule](requests))
    compare(steps, run_steps(engine, steps), expected, tolerance("float32"), schedule)


def test_models_and_sizes_that_do_not_fit_are_refused(cases, tmp_path):
    from leone_amd.engine.engine import Engine
    from leone_amd.runtime import load_model
    folder = str(tmp_path / "a")
    make_model_dir(folder, TINY["A"], seed=1, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="4 bits"):
        Engine(load_model(folder, "bfloat16", "cuda:0"), max_tokens=64, cache_bits=4)
    model = load_model(cases("M", "bfloat16")[0], "bfloat16", "cuda:0")
    with pytest.raises(ValueError, match="bits"):
        Engine(model, max_tokens=64, cache_bits=8)
    with pytest.raises(ValueError):
        Engine(model, max_tokens=64, page_tokens=12, cache_bits=4)
