"""The operators of a cache of 4 bits an element where a value is no number, however little it weighs."""
import math

import pytest
import torch

from leone_amd import ops
from tests.four_bit_util import attended, pools_of

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def _low_then_high(dim, heads, page, keys, low):
    """A request's cache in which the first ``low`` keys are all -8 and the others 8, values 1 to 3; its pools, block table, keys and values."""
    k = torch.full((keys, heads, dim), 8.0, dtype=torch.float64)
    k[:low] = -8.0
    gen = torch.Generator().manual_seed(dim + keys)
    v = torch.tensor([1.0, 1.5, 2.0, 3.0], dtype=torch.float64)[torch.randint(0, 4, (keys, heads, dim), generator=gen)]
    paged = [x.reshape(keys // page, page, heads, dim).transpose(1, 2).contiguous() for x in (k, v)]
    pools = ops.FourBitPools(*(p.to(DEVICE) for p in pools_of(*paged)))
    return pools, torch.arange(keys // page, dtype=torch.int32, device=DEVICE)[None], k.to(DEVICE), v.to(DEVICE)


@pytest.mark.parametrize("splits", [None, 1, 2, 4, 8])
@pytest.mark.parametrize("operator", ["rows", "rows float32", "single tokens", "portions"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_value_that_is_no_number_counts_however_little_it_weighs(operator, dim, splits):
    """Queries of ones see 64 keys of -8 and 448 of 8: the former weigh exp(-16 sqrt(dim)), 2^-184 or less, nothing in float.  One of them has a
    value block of NaN; in 64 bits no weight is zero, so that the block's elements are NaN and no other is touched, wherever the keys
    are cut and in whichever wave the block is."""
    heads, q_heads, page, keys, at = 2, 4, 64, 512, 10
    pools, table, k, v = _low_then_high(dim, heads, page, keys, 64)
    rows = 40
    positions = torch.arange(keys - rows, keys, dtype=torch.int32, device=DEVICE)
    entries = torch.zeros_like(positions)
    q = torch.ones(rows, q_heads * dim, dtype=torch.float32 if operator == "rows float32" else torch.bfloat16, device=DEVICE)

    def run():
        where = (table, q_heads, dim ** -0.5)
        if operator == "portions":
            return ops.attention_prefill_4bit(q, torch.zeros_like(q), pools, positions, ops.prefill_tiles([(0, 0, rows)]).to(DEVICE), *where,
                                              mean_keys=keys, splits=splits)
        if operator == "single tokens":
            return ops.attention_decode_4bit(q, pools, positions, entries, *where, splits=splits)
        return ops.attention_rows_4bit(q, pools, positions, entries, *where, splits=splits)

    before = run()
    assert torch.isfinite(before).all()
    pools.v_powers[at // page, 1, at % page // 4, 1, at % 4] = 255
    v[at, 1, 32:64] = math.nan
    out = run().reshape(rows, q_heads, dim)
    want = attended(q[-1].reshape(q_heads, dim), k, v, keys - 1, dim ** -0.5)[0]
    spoiled = torch.isnan(want)
    assert spoiled.sum() == 2 * 32
    assert torch.equal(torch.isnan(out), spoiled.expand_as(out))
    assert torch.equal(out[:, ~spoiled], before.reshape(rows, q_heads, dim)[:, ~spoiled])


@pytest.mark.parametrize("splits", [1, 3])
def test_portions_recorded_and_replayed(splits):
    """A portion's attention in a recorded run, its ranges' merge with it: every replay, with other work, calls of its own and synchronizations
    between, gives the eager call's bits, and so does the eager call every time."""
    dim, heads, q_heads, page, keys, rows = 128, 2, 4, 64, 512, 200
    pools, table, _, _ = _low_then_high(dim, heads, page, keys, 300)
    gen = torch.Generator(device=DEVICE).manual_seed(3)
    positions = torch.arange(keys - rows, keys, dtype=torch.int32, device=DEVICE)
    tiles = ops.prefill_tiles([(0, 0, rows)]).to(DEVICE)
    inputs = [torch.randn(rows, q_heads * dim, generator=gen, device=DEVICE).to(torch.bfloat16) for _ in range(3)]
    given, out = inputs[0].clone(), torch.zeros_like(inputs[0])

    def call(into):
        return ops.attention_prefill_4bit(given, into, pools, positions, tiles, table, q_heads, dim ** -0.5, splits=splits)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call(out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(out)
    for turn in range(5):
        given.copy_(inputs[turn % 3])
        out.fill_(7.0)
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        want = call(torch.zeros_like(out))
        assert torch.equal(out, want) and torch.equal(want, call(torch.full_like(out, 3.0))), turn
        torch.randn(1 << 18, generator=gen, device=DEVICE).sum().item()
