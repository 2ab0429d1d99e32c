"""Structural changes of 16-bit points that `AdamW` steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_opacity_reset_of_points_in_any_type(device, dtype, bits):
    """Moments stay in the optimiser's type, float32 or 8 bits, through pruning and a reset, and the next step takes them."""
    from fast_sp_gs_amd.adamw import AdamW
    from fast_sp_gs_amd.adaptive_control import GaussianPoints
    g = torch.Generator().manual_seed(5)
    P = 301
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)
    pts = GaussianPoints(make(P, 3), make(P, 1, 3), make(P, 15, 3), make(P, 2), make(P, 4), make(P, 1))
    opt = AdamW(pts.param_groups(1e-3), lr=1e-3, weight_decay=0.0, state_bits=bits)
    def step():
        for group in opt.param_groups:
            p = group['params'][0]
            p.grad = torch.randn(p.shape, generator=g).to(dtype).to(device)
        opt.step()
    step()
    pts.prune_points(opt, torch.rand(P, generator=g).to(device) < 0.4)
    step()
    pts.reset_opacity(opt)
    state = opt.state[pts._opacity]
    moments = [state[k] for k in (('exp_avg', 'exp_avg_sq') if bits == 32 else ('moments8',))]
    assert all(m.dtype == (torch.float32 if bits == 32 else torch.uint8) and not bool(m.any()) for m in moments)
    step()
    # (an update of 1e-3 is less than half a spacing of 16-bit numbers at -4.6, logit(0.01): 2^-6 and 2^-9, so the parameters need not move)
    moments = [state[k] for k in (('exp_avg', 'exp_avg_sq') if bits == 32 else ('moments8',))]
    assert pts._opacity.dtype == dtype and all(bool(m.any()) for m in moments) and float(state['step']) == 3.0
    assert all(bool(torch.isfinite(p.detach()).all()) for p in pts.parameters())


def test_opacity_reset_with_the_other_optimisers(device):
    """Their moments have the parameter's type."""
    from fast_sp_gs_amd.adaptive_control import GaussianPoints
    pts = GaussianPoints(*(torch.randn(50, *s, device=device) for s in ((3,), (1, 3), (15, 3), (2,), (4,), (1,))))
    opt = torch.optim.Adam(pts.param_groups(1e-3), lr=1e-3)
    for group in opt.param_groups:
        group['params'][0].grad = torch.ones_like(group['params'][0])
    opt.step()
    pts.reset_opacity(opt)
    assert opt.state[pts._opacity]['exp_avg'].dtype == torch.float32 and not bool(opt.state[pts._opacity]['exp_avg_sq'].any())
