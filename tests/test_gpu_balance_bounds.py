"""Sizes that are refused are refused before anything is allocated for them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _peak(call, text):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match=text):
        call()
    return torch.cuda.max_memory_allocated() - before


def test_nothing_is_allocated_for_what_is_refused(device):
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    w, index = torch.full((4, 2), 0.5, device=device), torch.zeros(4, 2, dtype=torch.long, device=device)
    for M in ((1 << 26) - 15, 1 << 28, 1 << 40):
        assert _peak(lambda: neighbour_balance(w, index, M), 'superpoints') == 0
    wide = torch.zeros(1, device=device).expand(1, 1 << 26)  # one number's memory
    assert _peak(lambda: balance_loss(wide, 1), 'superpoints') == 0
    long = torch.zeros(1, dtype=torch.float16, device=device).expand((1 << 31) - 1, 1)
    assert _peak(lambda: balance_loss(long, 1), 'points') == 0


def test_weights_a_rounding_above_one(device):
    """Up to float32's 1.0001 a weight is one, and counts as what it is; the next number is none, nor is the first below 0."""
    import numpy as np
    from fast_sp_gs_amd.balance import neighbour_balance
    most = np.float32(1.0001)
    index = torch.arange(300, device=device).remainder(7)[:, None].expand(300, 2).contiguous()
    for value, fits in ((1.0, True), (float(np.nextafter(np.float32(1), np.float32(2))), True), (float(most), True),
                        (float(np.nextafter(most, np.float32(2))), False), (-0.0, True), (-1e-45, False), (0.0, True)):
        w = torch.zeros(300, 2, device=device)
        w[123, 0] = value
        loss, counts, importance = neighbour_balance(w, index, 7)
        assert bool(torch.isfinite(loss)) == fits and bool(torch.isfinite(importance).all()) == fits and int(counts.sum()) == 300
        if fits:
            # units of 2^-31, the mean's rounding
            assert abs(float(importance[123 % 7]) - value / 300) <= 2.0 ** -32 / 300 + 2.0 ** -24 * value / 300
