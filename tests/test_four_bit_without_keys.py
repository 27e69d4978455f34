"""A model that caches no keys has nothing to keep in 4 bits: asked to, it says so."""
import pytest
import torch

from leone_amd.api import cache_bytes_per_token
from leone_amd.architectures import config_from_dict, model_spec_for
from leone_amd.parts.model import DecoderModel
from tests import pamevik_util


def test_a_model_of_memories_alone_is_refused():
    model = DecoderModel(model_spec_for(config_from_dict(pamevik_util.config(48, 130, 4, [pamevik_util.mlstm(2, 16, 16, 12.0)] * 2))), torch.bfloat16, "cpu")
    needs = model.cache_needs()
    assert needs and not any(getattr(need, "paged", False) for need in needs.values())
    with pytest.raises(ValueError, match="no keys"):
        model.cache_needs(4)
    with pytest.raises(ValueError, match="no keys"):
        cache_bytes_per_token(model, 4)
