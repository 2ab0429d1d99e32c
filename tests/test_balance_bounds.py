"""Where the balance losses' bounds lie (no GPU is needed to be refused)."""
import pytest


@pytest.mark.parametrize('M,fits', [((1 << 26) - 17, True), ((1 << 26) - 16, True), ((1 << 26) - 15, False), ((1 << 26) - 1, False), (1 << 26, False), ((1 << 31) - 1, False)])
def test_superpoints_of_a_launch(M, fits):
    """Sixteen superpoints take 1024 threads of the totals' launch; a launch has fewer than 2^32. What fits gets as far as its workspace's size."""
    from fast_sp_gs_amd import lib
    L = lib.load()
    A = 4096  # an address that is not followed
    assert (-(-M // 16) * 1024 < 1 << 32) == fits
    for rc in (L.fsgs_balance_loss_forward(4, M, M, 1, 0, A, None, A, A, A, A, A, A, 16, None),
               L.fsgs_neighbour_balance_forward(4, M, 3, A, A, None, A, A, A, A, A, 16, None)):
        assert rc == 3 if fits else rc not in (0, 3)
        assert (b'workspace' if fits else b'superpoints') in L.fsgs_last_error()
