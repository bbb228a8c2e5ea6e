"""A config whose precision was changed behind its checks."""
import pytest
import torch

import alto_amd.mxfp4 as mx


def test_swap_params_names_a_precision_that_it_does_not_have():
    config = mx.TrainingOpConfig()
    config.precision = "nvfp4"
    with pytest.raises(ValueError, match="Unsupported training op config.*nvfp4"):
        mx.swap_params(torch.nn.Linear(32, 32), config=config)
