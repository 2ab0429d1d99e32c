"""Checkpoints that lack what later ones have (on the CPU: nothing is stepped)."""
import copy

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
