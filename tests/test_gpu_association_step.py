"""The training step of a dynamic scene with a learned association (neighbour logits, balance loss, AdamW), and density control over
8-bit moments."""
import numpy as np
import pytest
import torch

import adamw_reference as R
from util import npy

pytestmark = pytest.mark.gpu


def _step(device, P=4000, M=48, **kw):
    from fast_sp_gs_amd import scenes
    from fast_sp_gs_amd.dynamic_step import DynamicStep
    scene, cam = scenes.config2(P=P, size=128, seed=3)
    g = torch.Generator().manual_seed(3)
    ctrl = (torch.rand(M, 3, generator=g) * 2 - 1).to(device)
    target = torch.rand(3, cam.H, cam.W, generator=g).to(device)
    torch.manual_seed(3)
    if kw.get('LBS_method') == 'W':
        kw['sp_W'] = (torch.randn(P, M, generator=g) * 0.1).to(device)
    return DynamicStep(scene.to(device), cam.to(device), ctrl, target, **kw)


@pytest.mark.parametrize('bits', [32, 8])
def test_learned_association(device, bits):
    from fast_sp_gs_amd.adamw import AdamW
    from fast_sp_gs_amd.balance import balance_loss
    state = _step(device, LBS_method='W', balance=0.5, weight_decay=0.01, state_bits=bits, max_norm=1.0, net_lr=1e-4)
    assert isinstance(state.net_opt, AdamW)
    t = torch.full((1,), 0.3, device=device)
    # the logits' gradient is that of the picture plus that of the balance
    loss, _ = state.forward_loss(t)
    whole, = torch.autograd.grad(loss, state.sp_W)
    state.balance, weight = 0.0, state.balance
    picture = torch.autograd.grad(state.forward_loss(t)[0], state.sp_W)[0]
    state.balance = weight
    alone, = torch.autograd.grad(weight * balance_loss(state.sp_W, 1)[0], state.sp_W)
    scale = float(picture.abs().max() + alone.abs().max())
    # both pictures' gradients pass through the same ordered sums; one addition more on one side
    assert float((whole - picture - alone).abs().max()) <= 4 * R.U * scale and float(alone.abs().max()) > 0
    before = [p.detach().clone() for p in [state.sp_W, state.ctrl, *state.net.parameters()]]
    packed = state.net._packed_versions
    for k in range(2):
        loss, _ = state.step(t)
        assert np.isfinite(float(loss))
    after = [state.sp_W, state.ctrl, *state.net.parameters()]
    assert all(torch.isfinite(p).all() for p in after) and sum(not torch.equal(p.detach(), b) for p, b in zip(after, before)) > len(after) // 2
    assert state.net._packed_versions != packed  # the network saw its weights change
    assert float(state.net_opt.last_norm) > 0 and state.sp_W.grad is None


def test_plain_steps_are_what_they_were(device):
    from fast_sp_gs_amd.sparse_gaussian_adam import DenseAdam
    assert isinstance(_step(device).net_opt, DenseAdam)
    for wrong in (dict(LBS_method='dist', sp_W=torch.zeros(4000, 48, device=device)), dict(balance=0.1)):
        with pytest.raises(ValueError, match='sp_W'):
            _step(device, **wrong)
    from fast_sp_gs_amd import scenes
    from fast_sp_gs_amd.dynamic_step import DynamicStep
    scene, cam = scenes.config2(P=100, size=64, seed=3)
    with pytest.raises(ValueError, match='sp_W'):
        DynamicStep(scene.to(device), cam.to(device), torch.zeros(8, 3, device=device), torch.zeros(3, 64, 64, device=device), LBS_method='W')


def test_density_control_carries_8_bit_moments(device):
    """Pruned, cloned and split points: the moments of the points that stay are their old values to the nearest code of their new
    block, those of new points are 0, and the next step works on."""
    from fast_sp_gs_amd.adamw import AdamW, adamw8_moments
    from fast_sp_gs_amd.adaptive_control import GaussianPoints
    g = torch.Generator().manual_seed(4)
    P = 3001
    make = lambda *s: torch.randn(*s, generator=g).to(device)
    pts = GaussianPoints(make(P, 3), make(P, 1, 3), make(P, 15, 3), make(P, 2) * 0.3 - 4, make(P, 4), make(P, 1))
    opt = AdamW(pts.param_groups(1e-3), lr=1e-3, weight_decay=0.0, eps=1e-15, state_bits=8)
    def step():
        for group in opt.param_groups:
            p = group['params'][0]
            p.grad = torch.randn(p.shape, generator=g).to(device) * 1e-3
        opt.step()
    def moments():
        out = {}
        for group in opt.param_groups:
            p = group['params'][0]
            (m, v), = adamw8_moments([opt.state[p]['moments8']], [p])
            out[group['name']] = (npy(m).reshape(p.shape[0], -1), npy(v).reshape(p.shape[0], -1))
        return out
    for _ in range(3):
        step()
    old = moments()
    mask = torch.rand(P, generator=g).to(device) < 0.4
    pts.prune_points(opt, mask)
    new = moments()
    keep = npy(~mask)
    for name in old:
        for a, b, bits in zip(old[name], new[name], (4, 5)):
            a = a[keep].astype(np.float64)
            assert a.shape == b.shape
            flat = abs(a.reshape(-1))
            # to the nearest: half a spacing is added before rounding down
            kept, spacing = R.rounded(flat, np.full(flat.shape, 0.5), bits)
            if bits == 5:
                kept = np.where((kept == 0) & (flat > 0), spacing, kept)
            assert np.array_equal(abs(b.reshape(-1)), kept) and (np.sign(b) * np.sign(a) >= 0).all()
    step()
    old = moments()
    count = pts._xyz.shape[0]
    pts.xyz_gradient_accum += torch.rand(count, 1, generator=g).to(device)
    pts.denom += 1
    pts.densify(opt, 0.7, 1.0)
    grown = pts._xyz.shape[0]
    assert grown > count
    new = moments()
    for name in old:
        rows = (new[name][1] != 0).any(1)
        # new points stand at the end and have no moments yet
        assert not rows[-(grown - int(rows.sum())):].any() and rows[:int(rows.sum())].all()
    step()
    pts.reset_opacity(opt)
    assert not opt.state[pts._opacity]['moments8'].any()
    step()
    assert all(torch.isfinite(p).all() for p in pts.parameters())
    assert all(float(opt.state[group['params'][0]]['step']) == 6.0 for group in opt.param_groups)
