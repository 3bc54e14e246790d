"""Frequency tables of rotary positions where the ramp between kept and stretched pairs is empty."""
import math

import numpy as np
import pytest

import eahmmf_b200 as eb


@pytest.mark.parametrize("n_rot,base,factor,ctx", [(64, 1e4, 8.0, 6), (128, 1e6, 4.0, 1), (2, 1e4, 2.0, 5)])
def test_a_context_of_less_than_a_turn_stretches_every_pair(n_rot, base, factor, ctx):
    """Even pair 0, of angle 1 a position, turns ctx / 2 pi < 1 times."""
    got, m = eb.rope_inv_freq(n_rot, base, "yarn", factor, ctx)
    np.testing.assert_allclose(got, base ** (-2.0 * np.arange(n_rot // 2) / n_rot) / factor, rtol=1.01 * 2.0 ** -24)
    assert m == pytest.approx(0.1 * math.log(factor) + 1, rel=2.0 ** -23)


@pytest.mark.parametrize("n_rot,base,ctx", [(64, 1.01, 1 << 30), (2, 1e4, 4096)])
def test_a_context_of_many_turns_keeps_every_pair(n_rot, base, ctx):
    """The slowest pair, too, turns more than 32 times."""
    got, _ = eb.rope_inv_freq(n_rot, base, "yarn", 8.0, ctx)
    np.testing.assert_allclose(got, base ** (-2.0 * np.arange(n_rot // 2) / n_rot), rtol=1.01 * 2.0 ** -24)
