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
