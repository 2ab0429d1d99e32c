"""Checkpoints that lack what later ones have (on the CPU: nothing is stepped)."""
import copy

import pytest
import torch


def test_groups_without_capturable():
    """Loaded as not capturable; values, counts and moments are taken over, the saved ones left alone."""
    from fast_sp_gs_amd.adamw import AdamW
    theirs = torch.nn.Parameter(torch.ones(5))
    opt = torch.optim.AdamW([theirs], lr=0.1, foreach=False)
    theirs.grad = torch.linspace(0, 1, 5)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    for key in ('capturable', 'foreach', 'fused', 'differentiable', 'maximize', 'decoupled_weight_decay'):
        saved['param_groups'][0].pop(key, None)
    saved['state'][0]['step'] = 1  # a plain number
    ours = torch.nn.Parameter(torch.ones(5))
    loaded = AdamW([ours], capturable=False)
    loaded.load_state_dict(saved)
    assert loaded.param_groups[0]['capturable'] is False and loaded.param_groups[0]['lr'] == 0.1
    state = loaded.state[ours]
    assert torch.equal(state['exp_avg'], opt.state[theirs]['exp_avg']) and state['exp_avg'].data_ptr() != saved['state'][0]['exp_avg'].data_ptr()
    assert float(state['step']) == 1.0 and state['step'].dtype == torch.float32 and saved['state'][0]['step'] == 1
    assert copy.deepcopy(loaded).param_groups[0]['capturable'] is False


def test_moments_of_another_shape_are_refused():
    """Also where they could be spread over the parameter's elements."""
    from fast_sp_gs_amd.adamw import AdamW
    for shape in ((1, 4), (4,), (3, 1), (12,), (4, 3)):
        theirs = torch.nn.Parameter(torch.ones(shape))
        opt = torch.optim.AdamW([theirs], foreach=False)
        theirs.grad = torch.ones(shape)
        opt.step()
        ours = AdamW([torch.nn.Parameter(torch.ones(3, 4))], lr=0.25)
        with pytest.raises(ValueError, match='shape'):
            ours.load_state_dict(opt.state_dict())
        assert not ours.state and ours.param_groups[0]['lr'] == 0.25  # as it was
    saved = AdamW([torch.nn.Parameter(torch.ones(256))], state_bits=8).state_dict()
    for bits in (8, 32):
        saved['state'][0] = {'step': torch.tensor(1.0), 'moments8': torch.zeros(514, dtype=torch.uint8)}
        with pytest.raises(ValueError, match='shape'):
            AdamW([torch.nn.Parameter(torch.ones(257))], state_bits=bits).load_state_dict(saved)
