"""Sizes beyond one launch are refused on the host by name: a launch counts its threads, 256 a workgroup, in 32 bits."""
import pytest

from tests.test_host_training import attention, refused, rotary


@pytest.mark.parametrize("changes", [dict(B=32768, Hq=32, Hk=32, Sq=256, Sk=256, Sk_used=256, D=64),    # 2^24 tiles of queries and as many of keys
                                     dict(B=1024, Hq=1, Hk=1, Sq=32, Sk=16384 * 32, Sk_used=32, D=64),  # of keys alone
                                     dict(B=65535, Hq=256, Hk=1, Sq=32, Sk=32, Sk_used=32, D=64)])
def test_attention_backward_of_too_many_tiles(changes):
    refused("alto_mxfp4_attention_bwd", attention(**changes), "2^24 tiles", None)
    refused("alto_mxfp4_attention_bwd_workspace_bytes", attention(**changes), "2^24 tiles")


@pytest.mark.parametrize("changes", [dict(B=64, S=1 << 21, Hq=1, Hk=0, D=2, R=2), dict(B=1, S=1 << 30, Hq=1, Hk=1), dict(B=16, S=1 << 20, Hq=64, Hk=64, D=2048, R=2048)])
def test_rotary_of_too_many_tokens(changes):
    refused("alto_mxfp4_rotary", rotary(**changes), "too many tokens for one launch", None)
