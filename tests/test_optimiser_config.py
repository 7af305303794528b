"""The runners' ``optimiser`` block: its name chooses the optimiser (no GPU)."""
import pytest
import torch

from gncde import run


def cfg(**block):
    return {"optimiser": {"schedule": {"name": "constant_schedule", "value": "1e-2"}, **block}}


@pytest.mark.parametrize("block,error,words", [
    (dict(name="lamb"), NotImplementedError, "lamb"),
    (dict(name="sgd", weight_decay=1e-4), ValueError, "weight_decay"),
    (dict(name="adam", weight_decay="1e-4"), ValueError, "weight_decay"),
    (dict(name="sgd"), ValueError, "ClippedOptimiser.*GPU"),  # built, and refused for a model that is not on a GPU
    (dict(name="adam", gradient_clipping=False), ValueError, "ClippedOptimiser.*GPU"),
    (dict(name="adamw", weight_decay=1e-4), ValueError, "ClipAdamW.*GPU"),
    (dict(), ValueError, "ClipAdamW.*GPU"),
])
def test_the_name_chooses(block, error, words):
    with pytest.raises(error, match=words):
        run._build_optimiser(cfg(**block), torch.nn.Linear(2, 2))
