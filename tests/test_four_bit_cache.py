"""What a cache of 4 bits an element needs and which layers take it (no GPU)."""
import pytest
import torch

from leone_amd import ops
from leone_amd.api import cache_bytes_per_token
from leone_amd.architectures import config_from_dict, model_spec_for
from leone_amd.ops.library import KernelError
from leone_amd.parts.base import FourBitKvNeed, KvNeed, StateNeed
from leone_amd.parts.model import DecoderModel
from tests import fosulix_util, sonulorn_util, zukinex_util
from tests.four_bit_util import codes_of, held, pools_of, quantised
from tests.util import TINY


def _model(raw, dtype=torch.bfloat16):
    return DecoderModel(model_spec_for(config_from_dict(raw)), dtype, "cpu")


@pytest.mark.parametrize("name,dim,heads", [("B", 32, 1), ("M", 128, 2)])
def test_plain_attention_takes_it(name, dim, heads):
    model = _model(TINY[name])
    plain, small = model.cache_needs(), model.cache_needs(4)
    assert set(plain) == set(small) and all(type(n) is FourBitKvNeed and (n.kv_heads, n.head_dim) == (heads, dim) for n in small.values())
    assert len({n.group_key() for n in small.values()}) == 1
    assert cache_bytes_per_token(model) == len(plain) * heads * dim * 4
    assert cache_bytes_per_token(model, 4) == len(plain) * heads * (dim + dim // 16)
    storage = next(iter(small.values())).allocate(3, 64, torch.bfloat16, "cpu")
    assert ops.four_bit_dims(storage) == (3, heads, 64, dim)
    assert sum(p.numel() for p in storage) == 3 * 64 * heads * (dim + dim // 16)
    need = next(iter(small.values()))
    need.poison(storage, torch.tensor([1]))
    assert (storage.k_powers[1] == 255).all() and (storage.v_powers[1] == 255).all() and (storage.k_powers[0] == 0).all()
    view = need.view(storage, None, 64)
    assert view.pools is storage and view.page_tokens == 64 and view.writes


@pytest.mark.parametrize("raw", [TINY["A"], TINY["C"]])
def test_heads_that_hold_no_whole_blocks_are_refused(raw):
    with pytest.raises(ValueError, match="4 bits"):
        _model(raw).cache_needs(4)


@pytest.mark.parametrize("raw", [zukinex_util.SMALL["A"], fosulix_util.SMALL["A"], sonulorn_util.SMALL["A"]])
def test_layers_of_other_kinds_are_refused(raw):
    model = _model(raw)
    assert model.cache_needs()
    with pytest.raises(ValueError, match="4 bits"):
        model.cache_needs(4)


def test_needs_are_equal_whatever_the_mixer_takes():
    assert KvNeed(2, 64, four_bits=True) == KvNeed(2, 64) and hash(KvNeed(2, 64, four_bits=True)) == hash(KvNeed(2, 64))
    assert KvNeed(2, 64, 128, four_bits=True).in_four_bits() == FourBitKvNeed(2, 64, 128)


@pytest.mark.parametrize("bits", [2, 8, 0, 16])
def test_other_sizes_are_refused(bits):
    with pytest.raises(ValueError, match="bits"):
        _model(TINY["M"]).cache_needs(bits)


def test_pools_of_other_shapes_are_refused():
    good = ops.four_bit_pools(2, 3, 64, 16, "cpu")
    assert ops.four_bit_dims(good) == (2, 3, 16, 64) == ops.four_bit_dims(tuple(good))
    for bad in (good[:3], (good[0], good[1], good[3], good[2]), (good[0][:1],) + tuple(good[1:]), (good[0], good[1][:, :, :8], good[2], good[3])):
        with pytest.raises(KernelError):
            ops.four_bit_dims(bad)
    with pytest.raises(KernelError):
        ops.attention_rows_4bit(torch.zeros(1, 128), good, torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                torch.zeros(1, 1, dtype=torch.int32), 2, 1.0)                     # no GPU tensors


def test_the_oracle_keeps_its_own_numbers():
    """Values of the format are kept as they are, packed and read back element by element; a planted change shows."""
    gen = torch.Generator().manual_seed(1)
    k, v = (quantised(torch.randn(2, 3, 8, 64, generator=gen) * 3) for _ in range(2))
    assert torch.equal(quantised(k), k)
    pools = pools_of(k, v)
    for page in range(2):
        for head in range(3):
            for token in range(8):
                assert torch.equal(held(pools, page, head, token)[0], k[page, head, token])
                assert torch.equal(held(pools, page, head, token)[1], v[page, head, token])
    pools[2][1, 2, 1, 5, 3, 1] ^= 0x10
    assert not torch.equal(held(pools, 1, 2, 7)[1], v[1, 2, 7])
    codes, powers = codes_of(torch.tensor([[float("nan")] + [1.0] * 31]))
    assert int(powers[0, 0]) == 255
