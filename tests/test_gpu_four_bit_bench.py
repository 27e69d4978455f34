"""The measurement program on a cache of 4 bits an element: what it reads is random numbers, not the zeros a cache begins with."""
import json

import pytest
import torch

from tests.util import TINY

pytestmark = pytest.mark.gpu


def test_a_measured_cache_holds_random_numbers():
    """Every page of every layer: keys and values of about the size the other caches are filled with (normal, 0.5), and none that is
    no number."""
    from leone_amd import benchmark, ops
    from leone_amd.architectures import config_from_dict
    from leone_amd.engine.engine import Engine
    from leone_amd.runtime import random_model
    model = random_model(config_from_dict(TINY["M"]), seed=0, dtype="bfloat16")
    engine = Engine(model, num_pages=12, page_tokens=16, max_requests=2, max_context=128, cache_bits=4)
    benchmark.fill_cache(engine, 2, 80)
    where = torch.arange(12 * 16, dtype=torch.int32, device="cuda:0")
    pages = torch.arange(12, dtype=torch.int32, device="cuda:0")[None]
    seen = []
    for pools in engine.pools.paged.values():
        for held in ops.cache_rows_4bit(pools, where, torch.zeros_like(where), pages):
            held = held.double()
            # 12 pages of 16 tokens and at least 32 elements: mean squares of 6,144 numbers of one eighth or one quarter times 8.56 on average
            assert torch.isfinite(held).all() and abs(held.square().mean().item() - 8.5625 * (1 / 64 + 1 / 16) / 2) < 0.05
            assert (held.square().mean(dim=1) > 0.05).all() and abs(held.mean().item()) < 0.1
            seen.append(held)
    assert all(not torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])
    for request in (("bench", 0), ("bench", 1)):
        engine.release(request)
    assert benchmark.time_decode(engine, 1, 20, 4, 2)[0] > 0


def test_the_record_says_what_it_measured(capsys):
    from leone_amd import benchmark
    records = []
    for more in ([], ["--cache-bits", "4"]):
        assert benchmark.main(["--layers", "1", "--steps", "2", "--warmup", "1", "--batch", "2", "--context", "256", "--no-peaks", "--no-points",
                               "--no-prefill", *more]) == 0
        records.append(json.loads(capsys.readouterr().out.splitlines()[-1]))
    plain, small = records
    assert "cache_bits" not in plain["bytes"] and small["bytes"]["cache_bits"] == 4
    assert plain["bytes"]["cache_a_token"] == 2 * 8 * 128 * 2 and small["bytes"]["cache_a_token"] == 8 * (128 + 8)
    assert plain["config"] == small["config"] and small["bytes"]["a_step"] < plain["bytes"]["a_step"]
    assert "attention" in small["kernels"]
