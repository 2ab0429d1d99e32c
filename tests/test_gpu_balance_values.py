"""Balance losses of logits far from 0 and of zeros of both signs, in every width of row, against their definition in 64 bits."""
import numpy as np
import pytest
import torch

from test_gpu_balance import _check, _reference

pytestmark = pytest.mark.gpu

# every number of lanes and of values a lane, whole rows and rows that end inside them
WIDTHS = [7, 16, 31, 64, 100, 128, 200, 256, 500, 512, 1000, 1500, 2048, 2500, 4096, 4097]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M', WIDTHS)
def test_logits_of_any_magnitude(device, M, dtype):
    """Rows about a large value of either sign: all equal, one ahead of the others, some steps of the type apart; and as a mask, over a part
    of a row or the whole of it. Tolerances are those of ordinary rows: differences from the row's largest logit are what counts."""
    g = torch.Generator().manual_seed(M)
    x = []
    for size in (1e5, 1e6, 1.1e6, 1e8, 3e9, 1e10, 1e20, 1e30, 9e37, 1.1e38, 3e38):
        for v in (size, -size):
            at = torch.tensor(v).to(dtype).float()
            equal = at.expand(M).clone()
            ahead = equal * (0.9375 if v > 0 else 1.0625)
            ahead[M // 3] = at
            apart = at * (1 + torch.randint(-3, 4, (M,), generator=g) * float(torch.finfo(dtype).eps))
            masked = torch.randn(M, generator=g)
            masked[torch.rand(M, generator=g) < 0.5] = -abs(at)
            x += [equal, ahead, apart, masked]
    x = torch.stack(x).to(dtype)
    assert torch.isfinite(x).all()
    N = len(x)
    rows = torch.rand(N, generator=g) < 0.8
    for K, on in ((1, None), (3, rows)):
        r = _reference(x.double().numpy(), K, np.ones(N, bool) if on is None else on.numpy())
        _check(x.to(device), K, None if on is None else on.to(device), r, dtype, (0.7, torch.randn(M, generator=g).to(device)))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M', WIDTHS)
def test_zeros_of_both_signs_are_equal(device, M, dtype):
    """Negative logits, many of them multiplied by 0: -0 and +0 tie, the lowest index first, whichever sign the lanes' largest have."""
    g = torch.Generator().manual_seed(M + 1)
    N = 48
    x = -torch.rand(N, M, generator=g) - 0.01
    kept = torch.rand(N, M, generator=g) < torch.linspace(0, 1, N)[:, None]
    zero = torch.where(torch.rand(N, M, generator=g) < torch.tensor([0.0, 0.02, 0.5, 1.0]).repeat(N // 4)[:, None], 0.0, -0.0)
    x = torch.where(kept, x, zero).to(dtype)
    for K in (1, 2, 3, 4, 5, 7):
        r = _reference(x.double().numpy(), K, np.ones(N, bool))
        _check(x.to(device), K, None, r, dtype)


@pytest.mark.parametrize('M', WIDTHS)
def test_rows_that_do_not_count_have_no_gradient(device, M):
    """Whatever comes from above: a NaN or an infinity in the importance's gradient reaches the rows that count and no other."""
    from fast_sp_gs_amd.balance import balance_loss
    g = torch.Generator().manual_seed(M + 2)
    N = 40
    x = torch.randn(N, M, generator=g).to(device)
    x[5] = float('-inf')
    rows = torch.rand(N, generator=g) < 0.6
    rows[:6] = True
    on = rows.clone()
    on[5] = False
    x.requires_grad_(True)
    for bad in (float('nan'), float('inf')):
        up = torch.zeros(M, device=device)
        up[M // 2] = bad
        grad, = torch.autograd.grad(balance_loss(x, 2, rows.to(device))[2], x, up)
        assert not bool(grad[(~on).to(device)].any())
        assert not bool(torch.isfinite(grad[on.to(device)]).any())
