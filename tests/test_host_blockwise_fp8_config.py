"""Training options of the 8-bit layers: MXFP4's have no effect on them, so one that was set is refused."""
import pickle

import pytest

from alto_amd.mxfp4 import TrainingOpConfig

SET = [dict(use_2dblock_x=True), dict(use_2dblock_w=False), dict(use_hadamard=False), dict(use_sr_grad=False), dict(use_dge=True), dict(clip_mode="dynamic"), dict(clip_mode="static"),
       dict(two_level_scaling="blockwise"), dict(two_level_scaling="tensorwise"), dict(use_uos=True)]


@pytest.mark.parametrize("options", SET)
def test_an_option_of_the_other_precision_is_refused(options):
    TrainingOpConfig(**options)
    with pytest.raises(ValueError, match=next(iter(options))):
        TrainingOpConfig(precision="blockwise_fp8", **options)


def test_without_options():
    config = TrainingOpConfig(precision="blockwise_fp8")
    assert config == TrainingOpConfig(precision="blockwise_fp8", use_2dblock_w=True, clip_mode="none") != TrainingOpConfig()
    assert pickle.loads(pickle.dumps(config)) == config
    with pytest.raises(ValueError, match="use_dge, clip_mode"):
        TrainingOpConfig(precision="blockwise_fp8", use_dge=True, clip_mode="static")
