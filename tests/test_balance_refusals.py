"""What the balance losses refuse, before anything is launched (no GPU is needed to be refused)."""
import pytest
import torch


def test_wrong_places_and_shapes():
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    x = torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match='CUDA'):
        balance_loss(x, 1)
    with pytest.raises(RuntimeError, match='CUDA'):
        neighbour_balance(x, torch.zeros(4, 5, dtype=torch.long), 5)


def test_c_entries_refuse_without_touching_the_gpu():
    from fast_sp_gs_amd import lib
    L = lib.load()
    most = L.fsgs_balance_max_choices()
    A = 4096  # an address that is not followed
    big = 1 << 40
    forward = lambda N=4, M=70, ld=70, K=1, dtype=0, logits=A, stats=A, ws=A, n=big: L.fsgs_balance_loss_forward(
        N, M, ld, K, dtype, logits, None, A, A, A, A, stats, ws, n, None)
    for wrong in (dict(N=-1), dict(N=1 << 31), dict(M=0), dict(ld=69), dict(K=0), dict(K=71), dict(K=most + 1, M=500, ld=500), dict(dtype=1),
                  dict(dtype=7), dict(logits=None), dict(logits=A + 2), dict(stats=A + 4), dict(ws=None), dict(ws=A + 4), dict(n=100)):
        assert forward(**wrong) != 0 and b'balance_loss' in L.fsgs_last_error(), wrong
    need = L.fsgs_balance_loss_workspace_bytes(4, 70, 0)
    assert need > 0 and forward(n=need - 1) == 3
    assert L.fsgs_balance_loss_workspace_bytes(-1, 70, 0) == 0 and L.fsgs_balance_loss_workspace_bytes(4, 0, 0) == 0
    backward = lambda N=4, M=70, ld=70, dtype=0, logits=A, stats=A, g=A, grad=A: L.fsgs_balance_loss_backward(
        N, M, ld, dtype, logits, stats, A, A, g, None, grad, None)
    for wrong in (dict(N=-1), dict(M=0), dict(ld=3), dict(dtype=1), dict(logits=None), dict(stats=None), dict(g=None), dict(grad=None),
                  dict(grad=A + 1), dict(stats=A + 4)):
        assert backward(**wrong) != 0, wrong
    assert backward(N=0) == 0
    near = lambda N=4, M=70, K=3, w=A, i=A, ws=A, n=big: L.fsgs_neighbour_balance_forward(N, M, K, w, i, None, A, A, A, A, ws, n, None)
    for wrong in (dict(N=-1), dict(N=1 << 31), dict(M=0), dict(K=0), dict(w=None), dict(i=None), dict(w=A + 1), dict(i=A + 4), dict(ws=A + 1), dict(n=10)):
        assert near(**wrong) != 0 and b'neighbour_balance' in L.fsgs_last_error(), wrong
    near_back = lambda N=4, i=A, g=A, grad=A: L.fsgs_neighbour_balance_backward(N, 70, 3, i, None, A, A, g, None, grad, None)
    for wrong in (dict(N=-1), dict(i=None), dict(g=None), dict(grad=None), dict(grad=A + 2), dict(i=A + 4)):
        assert near_back(**wrong) != 0, wrong
    assert near_back(N=0) == 0


def test_what_sums_and_launches_cannot_hold():
    from fast_sp_gs_amd import lib
    L = lib.load()
    A, big = 4096, 1 << 60
    assert L.fsgs_balance_loss_forward(4, 1 << 26, 1 << 26, 1, 0, A, None, A, A, A, A, A, A, big, None) != 0
    assert b'superpoints' in L.fsgs_last_error()
    assert L.fsgs_neighbour_balance_forward(4, 1 << 26, 3, A, A, None, A, A, A, A, A, big, None) != 0
    assert b'superpoints' in L.fsgs_last_error()
    # 2^33 weights of 1 at one superpoint, in units of 2^-31, are 2^64
    assert L.fsgs_neighbour_balance_forward(1 << 30, 70, 8, A, A, None, A, A, A, A, A, big, None) != 0
    assert b'pairs' in L.fsgs_last_error()
