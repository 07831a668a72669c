"""Rotary configurations whose numbers leave what they are held in: refused
(hale-token_amd/csrc/rope_freq.cpp on the CPU)."""
import pytest

from test_kv_pages import rope  # noqa: F401


@pytest.mark.parametrize("att", [1e39, 3.5e38, 1e-46, 1e300])
def test_attention_factors_that_no_f32_holds(rope, att):  # noqa: F811
    # cosines and sines are f32 numbers times it
    assert rope(att=att) == "refused: attention_factor must be positive, and a finite f32 number"


@pytest.mark.parametrize("att", [3.4e38, 1e-45, 1e-30, 0.5, 2.0])
def test_attention_factors_that_an_f32_holds(rope, att):  # noqa: F811
    assert rope(att=att).size == 64


def test_a_scaled_base_that_is_not_finite(rope):  # noqa: F811
    # base factor^(r / (r - 2)): infinite, all frequencies but the first would be 0
    assert rope(base=1e6, scaling=2, factor=1e305) == "refused: base times its scaling is not finite"
    assert rope(base=1e6, scaling=2, factor=8.0, r=4).size == 2
    assert (rope(base=1e6, scaling=2, factor=1e200) > 0).all()
