"""What the operators of a cache of 4 bits an element refuse: lengths, heads and operands that do not go together."""
import pytest
import torch

from leone_amd import ops
from leone_amd.ops.library import KernelError

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def test_more_refusals():
    """Lengths that do not go together, gains that start off a run of eight elements, pools of other heads, operands that are not there."""
    pools = ops.four_bit_pools(2, 2, 64, 64, DEVICE)
    positions = torch.zeros(3, dtype=torch.int32, device=DEVICE)
    entries, table = torch.zeros_like(positions), torch.zeros(1, 2, dtype=torch.int32, device=DEVICE)
    apart = torch.ones(64 + 1, device=DEVICE)[1:]
    ones = torch.ones(64, device=DEVICE)
    fill = dict(qkv=torch.zeros(3, 8 * 64, device=DEVICE), q_heads=4, kv_heads=2, head_dim=64, q_gain=ones, k_gain=ones, eps=1e-6, cos=None, sin=None,
                positions=positions, row_entry=entries, block_table=table, pools=pools)
    ops.qk_norm_rope_write_4bit(**fill)
    untouched = [p.clone() for p in pools]
    for change in (dict(positions=positions[:0]), dict(positions=positions[:2]), dict(positions=positions.repeat(2)), dict(row_entry=entries[:2]),
                   dict(row_entry=entries.repeat(2)), dict(row_entry=entries[None]), dict(positions=None), dict(row_entry=None), dict(block_table=None),
                   dict(block_table=table[0]), dict(block_table=table[:, :0]), dict(q_gain=apart), dict(k_gain=apart), dict(q_gain=apart, k_gain=apart),
                   dict(pools=ops.four_bit_pools(2, 1, 64, 64, DEVICE)), dict(pools=ops.four_bit_pools(2, 4, 64, 64, DEVICE)),
                   dict(pools=ops.four_bit_pools(2, 1, 128, 64, DEVICE)), dict(pools=ops.four_bit_pools(2, 4, 32, 64, DEVICE)), dict(pools=None),
                   dict(q_heads=2, kv_heads=3), dict(out=torch.zeros(2, 256, device=DEVICE)), dict(head_dim=32, q_heads=8, kv_heads=4)):
        with pytest.raises(KernelError):
            ops.qk_norm_rope_write_4bit(**{**fill, **change})
    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16, device=DEVICE)
    tiles = ops.prefill_tiles([(0, 0, 3)]).to(DEVICE)
    rows = dict(q=q, pools=pools, positions=positions, row_entry=entries, block_table=table, q_heads=4, scale=0.125)
    portions = dict(q=q, out=torch.zeros_like(q), pools=pools, positions=positions, tiles=tiles, block_table=table, q_heads=4, scale=0.125)
    ops.attention_prefill_4bit(**portions)
    for change in (dict(positions=positions[:0]), dict(positions=positions.repeat(2)), dict(positions=None), dict(block_table=None), dict(pools=None),
                   dict(block_table=table[:, :0]), dict(q_heads=8), dict(q_heads=0), dict(q_heads=-4)):
        for operator, good in ((ops.attention_rows_4bit, rows), (ops.attention_decode_4bit, rows), (ops.attention_prefill_4bit, portions)):
            with pytest.raises(KernelError):
                operator(**{**good, **change})
    for operator in (ops.attention_rows_4bit, ops.attention_decode_4bit):
        for change in (dict(row_entry=None), dict(row_entry=entries[:1]), dict(row_entry=entries.repeat(2))):
            with pytest.raises(KernelError):
                operator(**{**rows, **change})
    for change in (dict(tiles=None), dict(tiles=tiles[:3]), dict(tiles=tiles.reshape(-1)), dict(tiles=tiles.long()), dict(out=None), dict(splits=33)):
        with pytest.raises(KernelError):
            ops.attention_prefill_4bit(**{**portions, **change})
    for change in ((pools, None, entries, table), (pools, positions, None, table), (pools, positions, entries, None), (pools, positions, entries[:1], table),
                   (None, positions, entries, table)):
        with pytest.raises(KernelError):
            ops.cache_rows_4bit(*change)
    assert all(torch.equal(a, b) for a, b in zip(pools, untouched))
