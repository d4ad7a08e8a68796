"""Where the gated-scan memory is asked for and cannot be had."""
import pytest


def test_r2d2_says_that_its_memory_is_an_lstm():
    from ray_memory_management_amd.rllib.algorithms.r2d2 import R2D2Config

    with pytest.raises(ValueError, match="use_gated_scan"):
        R2D2Config().environment("CartPole-v1").training(model={"use_gated_scan": True}).build()
