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
