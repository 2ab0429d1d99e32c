"""Where an 8-bit moment's code changes, to the last bits of float64."""
import numpy as np
import pytest
import torch

import adamw_reference as R
from util import npy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('units,reached', [(0, True), (1, True), (255, True), (256, True), (257, False), (1000, False), (1 << 20, False)])
def test_borders_are_reached_from_256_units_below(device, units, reached):
    """From moments of 1 and a gradient of 2: with 1 - b = 1/16 - units 2^-52, exactly, m is 1 + 1/16 - units 2^-52 and v 1 + 3/16 - 3 units 2^-52,
    half-way between two codes but for the units. The noise of a half is the one that tells."""
    from fast_sp_gs_amd.adamw import adamw8_pack, adamw8_step
    n = 1 << 20
    one = torch.ones(n, device=device)
    state, = adamw8_pack([one], [one])
    b = 15 / 16 + units * 2.0 ** -52
    assert 1 - b == 1 / 16 - units * 2.0 ** -52
    step = torch.tensor(6.0)
    adamw8_step([torch.zeros(n, device=device)], [2 * one], [state], [step], lr=0.0, betas=(b, 0.0), seed=4)
    u, _ = R.noise(n, 7, 4)
    assert (u == 0.5).any()
    expected = np.where(u >= 0.5 if reached else u > 0.5, 9 / 8, 1.0)
    assert np.array_equal(R.unpack(npy(state), n)[0], expected)
    state, = adamw8_pack([one], [one])
    adamw8_step([torch.zeros(n, device=device)], [2 * one], [state], [torch.tensor(6.0)], lr=0.0, betas=(0.0, b), seed=4)
    _, u = R.noise(n, 7, 4)
    assert (u == 0.5).any()
    expected = np.where(u >= 0.5 if 3 * units <= 256 else u > 0.5, 10 / 8, 9 / 8)
    assert np.array_equal(R.unpack(npy(state), n)[1], expected)
