"""Filling a cache of 4 bits an element next to the borders between two codes and two powers."""
import math

import pytest
import torch

from leone_amd import ops
from tests.four_bit_util import held, quantised

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
BORDERS = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]              # between neighbouring codes, in units of the block's power


def _blocks(exponent):
    """float64 rows of 32 elements: every border in its block's units, on it and 2^-40 of it to either side, with both signs; and blocks whose
    largest element is on a border of powers, or to either side of it.  Each is a float and a float 2^-40 of it."""
    unit, sides = 2.0 ** exponent, (-1.0, 0.0, 1.0)
    near = [s * b * (1 + side * 2.0 ** -40) for b in BORDERS for side in sides for s in (1.0, -1.0)]
    rows = [[6.0] + near[i:i + 31] for i in (0, 31)]
    rows += [[s * 7.0 * (1 + side * 2.0 ** -40)] + near[:31] for side in sides for s in (1.0, -1.0)]
    rows += [[7.0 * (1 + side * 2.0 ** -40)] + [b * (1 + other * 2.0 ** -40) for b in BORDERS for other in sides] for side in sides]
    return torch.tensor([(row + [0.0] * 32)[:32] for row in rows], dtype=torch.float64) * unit


@pytest.mark.parametrize("turn", ["none", "halves", "part", "neighbours"])
@pytest.mark.parametrize("dim", [32, 96, 128])
@pytest.mark.parametrize("exponent", [0, -3, 40, -60])
def test_next_to_a_border(exponent, dim, turn):
    """Keys and values of two planes whose sum lies on a border or 2^-40 of it to either side (far below half a step of float), and of
    one plane next to it in float: the very codes of the definition, whatever rotation by an angle of zero the key passes."""
    blocks = _blocks(exponent)
    n = -(-blocks.shape[0] // (dim // 32))
    x = torch.zeros(n * (dim // 32), 32, dtype=torch.float64)
    x[:blocks.shape[0]] = blocks
    x = x.reshape(n, dim).to(DEVICE)
    first = x.float()
    planes = torch.stack([first, (x - first.double()).float()])
    assert torch.equal(planes.double().sum(0), x) and not torch.equal(first.double(), x)
    beside = [torch.nextafter(first, first * way) for way in (0.0, 2.0)]
    rotary = {"none": 0, "halves": dim, "part": 20, "neighbours": dim}[turn]
    cos = torch.ones(8 * n, rotary // 2, device=DEVICE) if rotary else None
    sin = torch.zeros(8 * n, rotary // 2, device=DEVICE) if rotary else None
    page = 16
    positions = torch.arange(n, dtype=torch.int32, device=DEVICE)
    entries = torch.zeros_like(positions)
    table = torch.arange(-(-n // page), dtype=torch.int32, device=DEVICE)[None]
    for given, want in [(planes, x), (first, first.double()), *((b, b.double()) for b in beside)]:
        pools = ops.four_bit_pools(table.shape[1], 1, dim, page, DEVICE)
        qkv = given.repeat_interleave(3, dim=-2).reshape(*given.shape[:-2], n, 3 * dim)
        ops.qk_norm_rope_write_4bit(qkv.contiguous(), 1, 1, dim, None, None, 1e-6, cos, sin, positions, entries, table, pools, out_dtype=torch.float32,
                                    pairing="adjacent" if turn == "neighbours" else "half_split")
        want = quantised(want).cpu()
        kept = [p.cpu() for p in pools]                        # (powers of two are exact there)
        for row in range(n):
            key, value = held(kept, row // page, 0, row % page)
            assert torch.equal(key, want[row]) and torch.equal(value, want[row]), row


def test_the_largest_numbers():
    """Blocks at the end of float's range, and (sums of planes) behind it: up to 1.75 x 2^127 they read back as numbers; above, a block's units
    are coarser and what rounds to 2^128 or more is kept, but is an infinity as a bfloat16.  Infinities and NaN that are given
    make the whole block NaN."""
    dim, page = 32, 16
    largest = torch.finfo(torch.float32).max
    below, above = 1.75 * 2.0 ** 127, math.nextafter(1.75 * 2.0 ** 127, math.inf)
    rows = [(below, 0.0), (-below, 0.0), (torch.nextafter(torch.tensor(below), torch.tensor(math.inf)).item(), 0.0), (3.0e38, 0.0), (-3.0e38, 0.0),
            (largest, 0.0), (-largest, 0.0), (3.0e38, 3.0e38), (-largest, -largest), (largest, largest), (below, above - below), (math.inf, 0.0),
            (-math.inf, 0.0), (math.nan, 0.0), (math.inf, -math.inf)]
    first, second = (torch.tensor([r[i] for r in rows], dtype=torch.float64).float()[:, None].repeat(1, dim).to(DEVICE) for i in (0, 1))
    first[:, 1::2] *= 0.375
    second[:, 1::2] *= 0.375
    planes = torch.stack([first, second])
    n = len(rows)
    positions = torch.arange(n, dtype=torch.int32, device=DEVICE)
    entries, table = torch.zeros_like(positions), torch.zeros(1, 1, dtype=torch.int32, device=DEVICE)
    for given in (planes, first):
        pools = ops.four_bit_pools(1, 1, dim, page, DEVICE)
        x = given.double().sum(0) if given.dim() == 3 else given.double()
        ops.qk_norm_rope_write_4bit(given.repeat(*[1] * (given.dim() - 1), 3).contiguous(), 1, 1, dim, None, None, 1e-6, None, None, positions, entries,
                                    table, pools, out_dtype=torch.float32)
        want = quantised(x).cpu()
        read = [r.cpu() for r in ops.cache_rows_4bit(pools, positions, entries, table)]
        for row in range(n):
            spoiled = bool(torch.isnan(want[row]).any())
            for kept, back in zip(held([p.cpu() for p in pools], 0, 0, row), read):
                if spoiled:
                    assert torch.isnan(want[row]).all() and torch.isnan(kept).all() and torch.isnan(back[row]).all(), row
                    continue
                assert torch.equal(kept, want[row]), row
                # (what 2^128 is as a float and a bfloat16)
                assert torch.equal(back[row].double(), torch.where(want[row].abs() >= 2.0 ** 128, want[row] * math.inf, want[row])), row
        assert torch.isfinite(read[0][:2]).all() and torch.isinf(read[0][3:7, 0]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_smallest_numbers(dtype):
    """Blocks of the least power there is, 2^-126, whose elements are numbers below float's least normal one: kept and read back as they are,
    and attended as such (a value of which is all that is seen comes out as it is)."""
    dim, page = 64, 16
    steps = torch.arange(0, 64, dtype=torch.float64) / 8 * 2.0 ** -126              # 0 to 7 7/8 units in eighths
    x = torch.stack([steps[:dim], -steps[:dim], steps[:dim] / 4, (steps[:dim] * 2.0 ** -7)]).to(dtype).to(DEVICE)
    n = x.shape[0]
    positions = torch.arange(n, dtype=torch.int32, device=DEVICE)
    entries, table = torch.zeros_like(positions), torch.zeros(1, 1, dtype=torch.int32, device=DEVICE)
    pools = ops.four_bit_pools(1, 1, dim, page, DEVICE)
    ops.qk_norm_rope_write_4bit(x.repeat(1, 3).contiguous(), 1, 1, dim, None, None, 1e-6, None, None, positions, entries, table, pools)
    want = quantised(x).cpu()
    kept = [p.cpu() for p in pools]
    read = [r.cpu().double() for r in ops.cache_rows_4bit(pools, positions, entries, table)]
    for row in range(n):
        for got, back in zip(held(kept, 0, 0, row), read):
            assert torch.equal(got, want[row]) and torch.equal(back[row], want[row]), row
    one = torch.zeros_like(positions)
    q = torch.zeros(n, dim, dtype=dtype, device=DEVICE)
    for row in range(n):
        at = torch.full((1,), row, dtype=torch.int32, device=DEVICE)
        outs = [ops.attention_rows_4bit(q[:1], pools, at, one[:1], table, 1, 1.0, 1)]
        if dtype == torch.bfloat16:
            outs.append(ops.attention_decode_4bit(q[:1], pools, at, one[:1], table, 1, 1.0, 1))
            tiles = torch.tensor([(0, 0, 1)] + [(0, 0, 0)] * 3, dtype=torch.int32, device=DEVICE)
            outs.append(ops.attention_prefill_4bit(q[:1], torch.zeros_like(q[:1]), pools, at, tiles, table, 1, 1.0, 1))
        for out in outs:
            # (below the least normal number what a product or a sum gives may be nothing)
            got = out[0].double().cpu()
            assert torch.equal(torch.where(want[row].abs() >= 2.0 ** -126, got, 0.0), torch.where(want[row].abs() >= 2.0 ** -126, want[row], 0.0)), row
            assert (got - want[row]).abs().max() < 2.0 ** -126
