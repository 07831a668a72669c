"""Rotary configurations whose numbers leave what they are held in: refused
(hale-token_amd/csrc/rope_freq.cpp on the CPU)."""
import numpy as np
import pytest

from test_kv_pages import rope  # noqa: F401


@pytest.mark.parametrize("att", [1e39, 3.5e38, 1e-46, 1e300])
def test_attention_factors_that_no_f32_holds(rope, att):  # noqa: F811
    # cosines and sines are f32 numbers times it
    assert rope(att=att) == "refused: attention_factor must be positive, and a finite f32 number"


@pytest.mark.parametrize("att", [3.4e38, 1e-45, 1e-30, 0.5, 2.0])
def test_attention_factors_that_an_f32_holds(rope, att):  # noqa: F811
    assert rope(att=att).size == 64
