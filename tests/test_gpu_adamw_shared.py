"""Tensors of an AdamW step that share memory. None of these calls may reach the GPU: what is refused is refused before anything is counted or
launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _call(device, bits, **given):
    """A step of two tensors of 600 elements, with some of its arguments given; (call, step counts)."""
    from fast_sp_gs_amd.adamw import adamw8_state, adamw8_step, adamw_step
    make = lambda: [torch.zeros(600, device=device) for _ in range(2)]
    args = dict(params=make(), grads=make(), m=make(), v=make(), steps=[torch.tensor(3.0) for _ in range(2)])
    args['states'] = [adamw8_state(p) for p in args['params']]
    args.update(given)
    a = args
    if bits == 8:
        return lambda: adamw8_step(a['params'], a['grads'], a['states'], a['steps']), a['steps']
    return lambda: adamw_step(a['params'], a['grads'], a['m'], a['v'], a['steps']), a['steps']


def _wrong(device, bits):
    part = lambda at, n=600: torch.zeros(4 * 600, device=device)[at:at + n]
    whole = torch.zeros(4 * 600, device=device)
    two = [whole[:600], whole[599:1199]]
    cases = [('share memory', dict(params=two)), ('share memory', dict(params=[whole[600:1200], whole[1199:1799]][::-1])),
             ('share memory', dict(params=[whole[:600], part(0)], grads=[part(0), whole[1:601]])),
             ('share memory', dict(params=[whole[:600], whole[600:1200]], grads=[whole[600:1200], whole[:600]])),
             ('there twice', dict(params=[whole[:600]] * 2)), ('there twice', dict(steps=[torch.tensor(3.0)] * 2))]
    if bits == 32:
        cases += [('share memory', dict(m=[whole[:600], part(0)], v=[whole[:600], part(0)])), ('share memory', dict(m=two)),
                  ('share memory', dict(m=[whole[:600], part(0)], v=[part(0), whole[300:900]])), ('there twice', dict(v=[whole[:600]] * 2)),
                  ('share memory', dict(params=[whole[:600], part(0)], m=[part(0), whole[599:1199]])),
                  ('share memory', dict(grads=[whole[:600], part(0)], v=[part(0), whole[599:1199]]))]
    else:
        bytes_ = torch.zeros(8 * 514, dtype=torch.uint8, device=device)
        floats = torch.zeros(4096, device=device)
        cases += [('share memory', dict(states=[bytes_[:1542], bytes_[1536:1536 + 1542]])), ('there twice', dict(states=[bytes_[:1542]] * 2)),
                  ('share memory', dict(params=[floats[:600], part(0)], states=[bytes_[:1542], floats.view(torch.uint8)[2384:2384 + 1542]]))]
    return cases


@pytest.mark.parametrize('bits', [32, 8])
def test_tensors_that_share_memory_are_refused(device, bits):
    for text, given in _wrong(device, bits):
        call, steps = _call(device, bits, **given)
        with pytest.raises(RuntimeError, match=text):
            call()
        assert all(float(s) == 3.0 for s in steps)


def test_step_counts_on_the_device(device):
    counts = torch.full((3,), 3.0, device=device)
    for steps in ([counts[0], counts[0]],):
        call, _ = _call(device, 32, steps=steps)
        with pytest.raises(RuntimeError, match='there twice'):
            call()
    call, _ = _call(device, 32, params=[counts[1:2], counts[2:3]], grads=[counts[:1], counts[:1]], m=[torch.zeros(1, device=device) for _ in range(2)],
                    v=[torch.zeros(1, device=device) for _ in range(2)], steps=[counts[0], counts[1]])
    with pytest.raises(RuntimeError, match='share memory'):
        call()
    assert bool((counts == 3.0).all())


@pytest.mark.parametrize('bits', [32, 8])
def test_neighbours_in_memory_are_stepped(device, bits):
    """Parts of one allocation side by side, in falling order; gradients that are one and the same; a parameter that is its own gradient: as copies
    of their own."""
    from fast_sp_gs_amd.adamw import adamw8_state
    n, state_bytes = 600, adamw8_state(torch.zeros(600, device=device)).numel()
    results = []
    for shared in (True, False):
        g = torch.Generator().manual_seed(1)
        flat = torch.randn(8 * n, generator=g).to(device)
        parts = [flat[k * n:(k + 1) * n] for k in range(8)][::-1]
        parts[6].square_(), parts[7].square_()
        grad = torch.randn(n, generator=g).to(device)
        room = torch.zeros(2 * 1552, dtype=torch.uint8, device=device)
        given = dict(params=parts[:2], grads=[grad, parts[1]], m=parts[4:6], v=parts[6:8], states=[room[1552:1552 + state_bytes], room[:state_bytes]])
        if not shared:
            given = {k: [t.clone() for t in ts] for k, ts in given.items()}
        call, steps = _call(device, bits, **given)
        call()
        assert all(float(s) == 4.0 for s in steps)
        results.append(given['params'] + (given['states'] if bits == 8 else given['m'] + given['v']))
    assert all(torch.equal(a, b) for a, b in zip(*results))
