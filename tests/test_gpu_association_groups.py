"""What the training step of a dynamic scene decays, and which association it balances."""
import pytest
import torch

from test_gpu_association_step import _step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('kw', [dict(), dict(LBS_method='W', balance=0.5), dict(LBS_method='W', state_bits=8, max_norm=1.0)])
def test_positions_and_logits_do_not_decay(device, kw):
    """Without a gradient a control point stays where it is and a logit what it is; the network's weights shrink by 1 - lr decay."""
    state = _step(device, weight_decay=0.1, net_lr=1e-2, **kw)
    network = list(state.net.parameters())
    kept = [p for p in (state.ctrl, state.sp_W) if p is not None]
    before = [p.detach().clone() for p in kept + network]
    for p in kept + network:
        p.grad = torch.zeros_like(p)
    for _ in range(3):
        state.net_opt.step()
    for p, b in zip(kept, before):
        assert torch.equal(p.detach(), b)
    for p, b in zip(network, before[len(kept):]):
        # three products, each by 0.999 rounded to float32, and their roundings
        assert float((p.detach() - b * 0.999 ** 3).abs().max()) <= 6 * 2.0 ** -24 * float(b.abs().max())
    assert sum(len(g['params']) for g in state.net_opt.param_groups) == len(kept) + len(network)


@pytest.mark.parametrize('bits', [32, 8])
def test_balance_of_the_weights_that_the_warp_uses(device, bits):
    """Its gradient is that of `neighbour_balance` of the neighbours' softmax, beside the picture's, and 0 for control points that a point does not
    see; the weights and indices are those of `calc_LBS_weight`. Of all logits it is another quantity."""
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    from fast_sp_gs_amd.deform import calc_LBS_weight
    state = _step(device, LBS_method='W', balance=0.5, balance_of='neighbours', state_bits=bits, max_norm=1.0, net_lr=1e-4, weight_decay=0.01)
    t = torch.full((1,), 0.3, device=device)
    loss, _ = state.forward_loss(t)
    whole, = torch.autograd.grad(loss, state.sp_W)
    state.balance, weight = 0.0, state.balance
    without, _ = state.forward_loss(t)
    picture, = torch.autograd.grad(without, state.sp_W)
    state.balance = weight
    M = state.sp_W.shape[1]
    weights, indices = calc_LBS_weight(state.params[0], state.ctrl, K=state.K, LBS_method='W', sp_W=state.sp_W)
    value = neighbour_balance(weights, indices, M)[0]
    alone, = torch.autograd.grad(weight * value, state.sp_W)
    U = 2.0 ** -24
    assert abs(float(loss) - float(without) - weight * float(value)) <= 4 * U * (abs(float(loss)) + weight * abs(float(value)))
    # both pictures' gradients pass through the same ordered sums; one addition more on one side
    scale = float(picture.abs().max() + alone.abs().max())
    assert float((whole - picture - alone).abs().max()) <= 4 * U * scale and float(alone.abs().max()) > 0
    seen = torch.zeros(state.sp_W.shape, dtype=torch.bool, device=device).scatter_(1, indices, True)
    assert not bool(whole[~seen].any())
    assert abs(float(value) - float(balance_loss(state.sp_W, 1)[0])) > 1e-3
    for _ in range(2):
        assert bool(torch.isfinite(state.step(t)[0]))
    assert bool(torch.isfinite(state.sp_W.detach()).all()) and state.sp_W.grad is None


def test_fresh_logits_choose_what_is_near(device):
    """Equal logits: the neighbours' choice follows the neighbours, that of all logits is the first control point for every point."""
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    from fast_sp_gs_amd.deform import calc_LBS_weight
    state = _step(device, LBS_method='W', balance=0.5, balance_of='neighbours')
    with torch.no_grad():
        state.sp_W.zero_()
        weights, indices = calc_LBS_weight(state.params[0], state.ctrl, K=state.K, LBS_method='W', sp_W=state.sp_W)
        counts = neighbour_balance(weights, indices, state.sp_W.shape[1])[1]
        assert torch.equal(counts, torch.bincount(indices[:, 0], minlength=len(counts)).int())
        assert int(balance_loss(state.sp_W, 1)[1][0]) == len(indices)


def test_what_is_balanced_has_a_name(device):
    with pytest.raises(ValueError, match='balance_of'):
        _step(device, LBS_method='W', balance=0.5, balance_of='weights')
