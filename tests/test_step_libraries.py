"""What a step launches for itself is among the libraries that a model builds before its first step."""
import pytest
import torch

from paged_batch_engine_b200.cache.storage import CacheStorage
from paged_batch_engine_b200.engine.runner import build_model
from tests import helpers

MODELS = dict(TINY_D=helpers.TINY_D, GEB_A=helpers.GEB_A, BAV_A=helpers.BAV_A, GUS_A=helpers.GUS_A, MOB_A=helpers.MOB_A,
              TUT_A=helpers.TUT_A, MAL_A=helpers.MAL_A, BAV_STATE_ONLY=helpers.BAV_STATE_ONLY)


@pytest.mark.parametrize("name", MODELS)
def test_the_maps_of_a_step_are_built_with_the_model(name):
    """Steps of many rows have their maps made on the device wherever a model has pages of one entry a token."""
    model = build_model(MODELS[name], torch.bfloat16, "cpu")
    storage = CacheStorage(model.cache_needs, 16, 4, 4, torch.bfloat16, "cpu")
    listed = ("page_maps", None) in model.kernel_libraries()
    assert listed == bool(storage.groups)


def test_with_a_4_bit_cache_too():
    model = build_model(helpers.TINY_D, torch.bfloat16, "cpu", cache_bits=4)
    assert ("page_maps", None) in model.kernel_libraries()
