"""Scales that leave the range of 32 bits on their way to powers of two, before any GPU is asked."""
import pytest

import test_serve_ops_cpu as S


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_scales_beyond_32_bits_are_refused(L, scale):
    """(A score of 0 would be 0 times infinity.)"""
    S.refused(L, S.attention(L, scale=scale), "scale")
