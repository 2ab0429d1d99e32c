"""AdamW steps over many tensors (fast_sp_gs_amd/adamw.py) against the step in 64 bits, at sizes around a lane's, a wavefront's and a
block's share, element types, layouts and addresses; the 8-bit moments against their restatement on integers; norms, streams, graphs,
checkpoints and structural changes."""
import numpy as np
import pytest
import torch

import adamw_reference as R
from util import npy

pytestmark = pytest.mark.gpu

SIZES = [1, 3, 4, 63, 64, 255, 256, 257, 1023, 1024, 1025, 5000]
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # relative, of the parameters' last rounding


def _flat(t):
    return np.asarray(t.detach().float().cpu().reshape(-1), np.float64)


def _problem(device, sizes, dtype, seed, offset=0, fresh=False):
    """Parameters, gradients, moments and host step counts; `offset`: elements between an allocation's start and a tensor's."""
    g = torch.Generator().manual_seed(seed)
    def at(values, type):
        room = torch.zeros(values.numel() + offset, dtype=type, device=device)
        room[offset:].copy_(values)
        return room[offset:]
    params, grads, ms, vs = [], [], [], []
    for n in sizes:
        params.append(at(torch.randn(n, generator=g) * 0.3, dtype))
        grad = torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g) - 4)
        grad[torch.rand(n, generator=g) < 0.2] = 0
        grads.append(at(grad, dtype))
        r = torch.exp(torch.randn(n, generator=g) - 4)
        ms.append(at(torch.zeros(n) if fresh else r * torch.tanh(torch.randn(n, generator=g)), torch.float32))
        vs.append(at(torch.zeros(n) if fresh else r * r, torch.float32))
    steps = [torch.tensor(0.0 if fresh else float(10 + 7 * k)) for k in range(len(sizes))]
    return params, grads, ms, vs, steps


def _check_params(p, want, off, dtype):
    got = _flat(p)
    bound = off + HALF[dtype] * (abs(want) + off) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert (abs(got - want) <= bound).all(), (abs(got - want) / bound).max()


@pytest.mark.parametrize('clip', [False, True])
@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_step_against_64_bits(device, dtype, offset, clip):
    from fast_sp_gs_amd.adamw import adamw_step
    params, grads, ms, vs, steps = _problem(device, SIZES, dtype, 1, offset)
    lr, wd, eps = [1e-3 * (k + 1) for k in range(len(SIZES))], [0.1 * (k % 3) for k in range(len(SIZES))], [1e-8] * len(SIZES)
    before = [[_flat(t) for t in ts] for ts in (params, grads, ms, vs)]
    total = np.sqrt(sum((g ** 2).sum() for g in before[1]))
    max_norm = 0.25 * total if clip else None
    norm = adamw_step(params, grads, ms, vs, steps, lr, (0.9, 0.999), eps, wd, max_norm)
    if clip:
        assert abs(float(norm) - total) <= 8 * R.U * total
    else:
        assert norm is None
    factor = min(1.0, max_norm / (total + 1e-6)) if clip else 1.0
    for k in range(len(SIZES)):
        assert float(steps[k]) == 11 + 7 * k
        p, m, v, (off_p, off_m, off_v) = R.step64(*(b[k] for b in before), 11 + 7 * k, lr[k], eps=eps[k], wd=wd[k], factor=factor)
        _check_params(params[k], p, off_p, dtype)
        assert (abs(_flat(ms[k]) - m) <= off_m).all() and (abs(_flat(vs[k]) - v) <= off_v).all()
        assert np.array_equal(_flat(grads[k]), before[1][k])


@pytest.mark.parametrize('clip', [False, True])
@pytest.mark.parametrize('fresh', [False, True])
@pytest.mark.parametrize('dtype,offset', [(torch.float32, 0), (torch.float32, 1), (torch.bfloat16, 0), (torch.bfloat16, 3), (torch.float16, 1)])
def test_8_bit_step_against_64_bits(device, dtype, offset, fresh, clip):
    from fast_sp_gs_amd.adamw import adamw8_moments, adamw8_pack, adamw8_state, adamw8_step
    params, grads, ms, vs, steps = _problem(device, SIZES, dtype, 2, offset, fresh)
    states = [adamw8_state(p) for p in params] if fresh else adamw8_pack(ms, vs)
    before = [[_flat(t) for t in ts] for ts in (params, grads)]
    old = [R.unpack(npy(s), n) for s, n in zip(states, SIZES)]
    for (m, v), kept in zip(old, adamw8_moments(states, params)):
        assert np.array_equal(_flat(kept[0]), m) and np.array_equal(_flat(kept[1]), v)
    total = np.sqrt(sum((g ** 2).sum() for g in before[1]))
    max_norm = 0.25 * total if clip else None
    factor = min(1.0, max_norm / (total + 1e-6)) if clip else 1.0
    adamw8_step(params, grads, states, steps, 1e-3, max_norm=max_norm, seed=5)
    clashes = 0
    for k, n in enumerate(SIZES):
        t = int(steps[k])
        p, m, v, (off_p, off_m, off_v) = R.step64(before[0][k], before[1][k], *old[k], t, 1e-3, factor=factor)
        # p follows from the moments before they are rounded
        _check_params(params[k], p, off_p, dtype)
        got_m, got_v = R.unpack(npy(states[k]), n)
        u_m, u_v = R.noise(n, t, 5)
        for x, off, got, u, bits in ((abs(m), off_m, abs(got_m), u_m, 4), (v, off_v, got_v, u_v, 5)):
            kept, spacing = R.rounded(x, u, bits)
            if bits == 5:
                kept = np.where((kept == 0) & (x > 0), spacing, kept)
            differ = got != kept
            # a value so near to a border that float32 may see it on the other side, one code further
            at = x / spacing + u
            near = abs(at - np.round(at)) <= 2 * off / spacing + 2.0 ** -19
            assert (near | ~differ).all() and (abs(got - kept)[differ] <= spacing[differ]).all()
            clashes += int(differ.sum())
        assert (np.sign(got_m) == np.where(got_m == 0, 0, np.sign(m))).all()
        assert ((got_v > 0) == (v > 0)).all()
    assert clashes <= 3  # of 2 x 10 000 values; a part in 10^5 is near a border


def test_rounding_is_right_on_average(device):
    """One value, a million noises: the mean of what is kept is the value (what is kept has a standard deviation of at most half a
    spacing; five sigma). The same along the steps of many elements."""
    from fast_sp_gs_amd.adamw import adamw8_moments, adamw8_pack, adamw8_state, adamw8_step
    n = 1 << 20
    for value in (0.3, 1.9, 2.0 ** -10 * 1.3, 2.0 ** -16 * 1.4):
        p = torch.zeros(n, device=device)
        g = torch.full((n,), value, device=device)
        g[::256] = 1.96  # above 1.875: the highest binade of m begins at 2, that of v at 4 (1.96^2 > 3.75)
        state = adamw8_state(p)
        adamw8_step([p], [g], [state], [torch.zeros(())], betas=(0.0, 0.0), seed=1)
        for kept, x, lowest in zip(adamw8_moments([state], [p])[0], (value, value * value), (1 - 14, 2 - 30)):
            kept = kept.double().view(-1, 256)[:, 1:]
            spacing = 2.0 ** (max(np.floor(np.log2(x)), lowest) - 3)
            if lowest == 2 - 30 and x < spacing:  # by definition v > 0 below the lowest code is that code's value, not 0
                assert bool((kept == spacing).all())
                continue
            # noise comes in steps of 2^-16 spacings, float32 squares within U
            assert abs(float(kept.mean()) - x) < 5 * 0.5 * spacing / np.sqrt(kept.numel()) + spacing * 2.0 ** -16 + 4 * R.U * x
            assert float((kept - x).abs().max()) < spacing * (1 + 2.0 ** -16)
    # v decays from 2.25 towards the constant squared gradient 1, by a thousandth of the way at a time, though spacings are an eighth
    n, steps = 1 << 16, 400
    p, g, step = torch.zeros(n, device=device), torch.ones(n, device=device), torch.tensor(0.0)
    state, = adamw8_pack([g], [g * 2.25])
    expected = 2.25
    for _ in range(steps):
        adamw8_step([p], [g], [state], [step], lr=0.0)
        expected = 0.999 * expected + 0.001
    (m, v), = adamw8_moments([state], [p])
    # a step's rounding has a variance of at most a quarter of spacing^2 (an eighth of 2 squared): sums over the steps and elements
    sigma = np.sqrt(steps * 0.25) * 0.25 / np.sqrt(n)
    assert abs(float(v.double().mean()) - expected) < 5 * sigma + steps * 4 * R.U * 2.25
    assert bool((m == 1.0).all())


def test_norms(device):
    from fast_sp_gs_amd.adamw import grad_norm
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for sizes in ([1], [3, 5, 8191, 8192, 8193], [100_003, 7], [0, 5], [0], [11] * 150):
            ts = [torch.randn(n, generator=g).to(dtype).to(device) for n in sizes]
            want = np.sqrt(sum((_flat(t) ** 2).sum() for t in ts))
            got = grad_norm(ts, 0.5)
            # squares of 8 elements at a time are added in float32, the rest in float64
            assert abs(float(got[0]) - want) <= 8 * R.U * want
            assert abs(float(got[1]) - min(1.0, 0.5 / (want + 1e-6))) <= 16 * R.U
    mixed = [torch.ones(3, device=device), torch.ones(4, device=device, dtype=torch.bfloat16), torch.ones(2, 3, device=device).t()]
    assert float(grad_norm(mixed)[0]) == pytest.approx(np.sqrt(13), rel=8 * R.U) and float(grad_norm(mixed)[1]) == 1.0
    strided = torch.arange(20, device=device, dtype=torch.float32)[::3]
    assert float(grad_norm([strided])[0]) == pytest.approx(float(strided.double().norm()), rel=8 * R.U)
    bad = torch.ones(1000, device=device)
    bad[500] = float('nan')
    assert bool(torch.isnan(grad_norm([bad], 1.0)).all())
    bad[500] = float('inf')
    out = grad_norm([bad], 1.0)
    assert float(out[0]) == float('inf') and float(out[1]) == 0.0


def test_equal_calls_give_equal_results(device):
    from fast_sp_gs_amd.adamw import adamw8_pack, adamw8_step
    runs = []
    for _ in range(2):
        params, grads, ms, vs, steps = _problem(device, [300_000, 7, 4099], torch.float32, 4)
        states = adamw8_pack(ms, vs)
        norm = adamw8_step(params, grads, states, steps, max_norm=0.1, seed=9)
        runs.append(params + states + [norm])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize('bits', [32, 8])
def test_many_tensors_of_mixed_types(device, bits):
    """More tensors than a launch takes, three element types in turn, empty ones among them, against one tensor at a time."""
    from fast_sp_gs_amd.adamw import adamw8_pack, adamw8_step, adamw_step
    types = [torch.float32, torch.bfloat16, torch.float16]
    made = []
    for k in range(160):
        made.append(_problem(device, [0 if k % 31 == 5 else 1 + (37 * k) % 700], types[k % 3], 100 + k))
    def run(together):
        params, grads, ms, vs, steps = ([m[i][0].clone() for m in made] for i in range(5))
        lr = [1e-3 + 1e-4 * k for k in range(160)]
        if bits == 8:
            more = [adamw8_pack(ms, vs)]
            step = lambda i, j: adamw8_step(params[i:j], grads[i:j], more[0][i:j], steps[i:j], lr[i:j], seed=3)
        else:
            more = [ms, vs]
            step = lambda i, j: adamw_step(params[i:j], grads[i:j], more[0][i:j], more[1][i:j], steps[i:j], lr[i:j])
        if together:
            step(0, 160)
        else:
            for k in range(160):
                step(k, k + 1)
        return params + sum(more, []) + steps
    assert all(torch.equal(a, b) for a, b in zip(run(True), run(False)))


def test_layouts(device):
    """Parameters in any order of memory, gradients in another, strided and expanded ones."""
    from fast_sp_gs_amd.adamw import AdamW
    g = torch.Generator().manual_seed(6)
    base = torch.randn(40, 24, generator=g)
    grad = torch.randn(40, 24, generator=g)
    wide = torch.zeros(40, 48, device=device)
    wide[:, ::2] = grad.to(device)
    forms = {'rows': (base.to(device).clone(), grad.to(device)),
             'columns': (base.t().contiguous().to(device).t(), grad.to(device)),
             'columns, gradient too': (base.t().contiguous().to(device).t(), grad.t().contiguous().to(device).t()),
             'strided gradient': (base.to(device).clone(), wide[:, ::2])}
    for bits in (32, 8):
        results = {}
        for name, (value, given) in forms.items():
            p = torch.nn.Parameter(value.clone(memory_format=torch.preserve_format))
            opt = AdamW([p], lr=1e-2, state_bits=bits)
            for _ in range(3):
                p.grad = given
                opt.step()
            results[name] = p.detach().contiguous()
        for name, value in results.items():
            # 8 bits: the moments' blocks follow the memory, and with them what is rounded
            if bits == 32 or name in ('rows', 'strided gradient'):
                assert torch.equal(value, results['rows']), name
        assert torch.equal(results['columns'], results['columns, gradient too'])
    p = torch.nn.Parameter(torch.zeros(30, 5, device=device))
    opt = AdamW([p], lr=0.5, weight_decay=0.0)
    p.grad = torch.ones(1, 5, device=device).expand(30, 5)
    opt.step()
    assert float((p.detach() + 0.5).abs().max()) < 1e-6


def test_against_torch(device):
    """Ten steps beside torch's AdamW, groups of their own rates: the sums of ten roundings of the step."""
    from fast_sp_gs_amd.adamw import AdamW
    g = torch.Generator().manual_seed(7)
    values = [torch.randn(s, generator=g).to(device) for s in ((17,), (33, 65), (4, 5, 6))]
    ours, theirs = ([torch.nn.Parameter(v.clone()) for v in values] for _ in range(2))
    groups = lambda ps: [{'params': ps[:2], 'lr': 1e-2}, {'params': ps[2:], 'weight_decay': 0.3, 'betas': (0.8, 0.99), 'eps': 1e-6}]
    a, b = AdamW(groups(ours), lr=1e-3, max_norm=2.0), torch.optim.AdamW(groups(theirs), lr=1e-3, foreach=False)
    for k in range(10):
        for p, q in zip(ours, theirs):
            p.grad = torch.randn(p.shape, generator=g).to(device)
            q.grad = p.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(theirs, 2.0)
        a.step(), b.step()
        assert float(a.last_norm) == pytest.approx(float(norm), rel=1e-6)
    for p, q, v in zip(ours, theirs, values):
        # an update is at most 7.3 lr; each side rounds it to 20 U, and the parameter itself to 3 U a step
        bound = 2 * 10 * (20 * R.U * 7.3 * 1e-2 + 3 * R.U * v.abs().max().item())
        assert float((p - q).detach().abs().max()) < bound


@pytest.mark.parametrize('bits', [32, 8])
def test_values_at_the_edges(device, bits):
    """Zero gradients move nothing but the decay; zero and tiny moments stay apart from each other; infinities and NaN stay where they
    are (with 8 bits: in their block of 256)."""
    from fast_sp_gs_amd.adamw import AdamW
    p = torch.nn.Parameter(torch.ones(1000, device=device))
    opt = AdamW([p], lr=1e-2, weight_decay=0.5, eps=0.0 if bits == 32 else 1e-15, state_bits=bits)
    p.grad = torch.zeros(1000, device=device)
    opt.param_groups[0]['eps'] = 1e-15
    for _ in range(2):
        opt.step()
    assert float((p.detach() - 0.995 ** 2).abs().max()) < 4 * R.U
    # magnitudes far below the block's largest, then no gradient at all: the update dies out instead of blowing up
    p = torch.nn.Parameter(torch.zeros(512, device=device))
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, eps=1e-15, state_bits=bits)
    g = 10.0 ** -torch.linspace(0, 18, 512, device=device)
    for k in range(40):
        before = p.detach().clone()
        p.grad = g if k == 0 else torch.zeros_like(g)
        opt.step()
        # |m| / sqrt(v) is at most sqrt(c1 terms): 0.1 / sqrt(0.001) = 3.2 at the first step and less after, over 1 - b1^t >= 0.1
        assert bool(torch.isfinite(p.detach()).all()) and float((p.detach() - before).abs().max()) <= 1e-3 * 7.3
    p = torch.nn.Parameter(torch.zeros(1024, device=device))
    opt = AdamW([p], lr=1e-3, state_bits=bits)
    for bad in (float('nan'), float('inf')):
        with torch.no_grad():
            p.zero_()
        opt.state.clear()
        g = torch.ones(1024, device=device)
        g[300] = bad
        for _ in range(2):
            p.grad = g
            opt.step()
        finite = torch.isfinite(p.detach())
        assert not bool(finite[300])
        if bits == 32:
            assert int((~finite).sum()) == 1
        else:
            assert bool(finite[:256].all()) and bool(finite[512:].all())


@pytest.mark.parametrize('bits', [32, 8])
def test_captured_steps(device, bits):
    """A captured step with its counts on the device equals eager steps, replay by replay, another stream's work in between."""
    from fast_sp_gs_amd.adamw import AdamW
    g = torch.Generator().manual_seed(8)
    shapes = [(300, 7), (5,), (1031,)]
    values = [torch.randn(s, generator=g).to(device) for s in shapes]
    feeds = [[torch.randn(s, generator=g).to(device) for s in shapes] for _ in range(6)]
    made = []
    for captured in (False, True):
        params = [torch.nn.Parameter(v.clone()) for v in values]
        opt = AdamW(params, lr=1e-2, state_bits=bits, max_norm=3.0, capturable=captured)
        for p in params:
            p.grad = torch.zeros_like(p)
        made.append((params, opt))
    (eager, eager_opt), (params, opt) = made
    def feed(ps, k):
        for p, f in zip(ps, feeds[k]):
            p.grad.copy_(f)
    feed(eager, 0), eager_opt.step()
    feed(params, 0), opt.step()  # makes the states
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 6):
        feed(eager, k), eager_opt.step()
        feed(params, k)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(params, eager):
            # pow on the device and on the host may differ in the last bit of a correction; 8-bit codes then in a code at a border
            off = (p.detach() - q.detach()).abs()
            assert float(off.max()) <= (k * 1e-2 * 7.3 * (8 * R.U if bits == 32 else 0.13)) and float((off > 1e-6).float().mean()) < 1e-2
        assert all(float(opt.state[p]['step']) == k + 1 for p in params)
        assert float(opt.last_norm) == pytest.approx(float(eager_opt.last_norm), rel=1e-6)
    opt = AdamW(params, lr=1e-2, state_bits=bits)
    opt.step()
    refused = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='captured'):
        with torch.cuda.graph(refused):
            opt.step()


@pytest.mark.parametrize('bits', [32, 8])
def test_another_stream(device, bits):
    from fast_sp_gs_amd.adamw import AdamW
    results = []
    for other in (False, True):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 100_001, device=device))
        opt = AdamW([p], state_bits=bits, max_norm=0.5)
        stream = torch.cuda.Stream() if other else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for k in range(3):
                p.grad = torch.cos(p.detach() * (k + 1))
                opt.step()
        torch.cuda.current_stream().wait_stream(stream)
        results.append(p.detach().clone())
    assert torch.equal(*results)


def test_autograd_sees_the_step(device):
    from fast_sp_gs_amd.adamw import AdamW
    w, x = torch.nn.Parameter(torch.randn(4, 4, device=device)), torch.randn(4, 4, device=device, requires_grad=True)
    opt = AdamW([w])
    y = (x @ w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_checkpoints(device, dtype):
    """A state saved and loaded goes on bit for bit; 32-bit states load into 8 bits and back; torch's own load too."""
    import copy
    from fast_sp_gs_amd.adamw import AdamW
    g = torch.Generator().manual_seed(9)
    start = [torch.randn(s, generator=g).to(dtype).to(device) for s in ((700,), (3, 5))]
    feeds = [[torch.randn(t.shape, generator=g).to(dtype).to(device) for t in start] for _ in range(4)]
    def run(params, opt, which):
        for k in which:
            for p, f in zip(params, feeds[k]):
                p.grad = f
            opt.step()
    for bits in (32, 8):
        params = [torch.nn.Parameter(t.clone()) for t in start]
        opt = AdamW(params, state_bits=bits)
        run(params, opt, (0, 1))
        saved, values = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in params]
        again = [torch.nn.Parameter(v) for v in values]
        other = AdamW(again, state_bits=bits)
        other.load_state_dict(saved)
        run(params, opt, (2, 3)), run(again, other, (2, 3))
        assert all(torch.equal(p, q) for p, q in zip(params, again))
        for p in again:
            kinds = {k: t.dtype for k, t in other.state[p].items()}
            assert kinds == ({'step': torch.float32, 'moments8': torch.uint8} if bits == 8 else
                             {'step': torch.float32, 'exp_avg': torch.float32, 'exp_avg_sq': torch.float32})
        width = AdamW([torch.nn.Parameter(v.clone()) for v in values], state_bits=40 - bits, capturable=True)
        width.load_state_dict(saved)
        for p, q in zip(width.param_groups[0]['params'], start):
            p.grad = torch.ones_like(p)
        width.param_groups[0]['capturable'] = False
        assert ('moments8' in width.state[width.param_groups[0]['params'][0]]) == (bits == 32)
    theirs = [torch.nn.Parameter(t.float().clone()) for t in start]
    from_torch = torch.optim.AdamW(theirs, foreach=False)
    for p, f in zip(theirs, feeds[0]):
        p.grad = f.float()
    from_torch.step()
    ours = [torch.nn.Parameter(t.detach().clone()) for t in theirs]
    opt = AdamW(ours)
    opt.load_state_dict(from_torch.state_dict())
    for p, q in zip(ours, theirs):
        assert torch.equal(opt.state[p]['exp_avg'], from_torch.state[q]['exp_avg']) and float(opt.state[p]['step']) == 1.0
        p.grad = torch.ones_like(p)
    opt.step()
    assert float(from_torch.state[theirs[0]]['step']) == 1.0


def test_offsets_beyond_32_bits(device):
    """More than 2^31 elements in one tensor: the far end steps like a tensor of its own."""
    from fast_sp_gs_amd.adamw import adamw8_moments, adamw8_state, adamw8_step, adamw_step
    n, far = (1 << 31) + 1027, 5003
    p = torch.zeros(n, dtype=torch.bfloat16, device=device)
    g = torch.zeros(n, dtype=torch.bfloat16, device=device)
    values = torch.randn(far, generator=torch.Generator().manual_seed(10)).to(torch.bfloat16).to(device)
    p[-far:], g[-far:] = values, values.flip(0)
    state = adamw8_state(p)
    adamw8_step([p], [g], [state], [torch.tensor(4.0)], 1e-2, seed=2)
    want, m, v, (off, off_m, _) = R.step64(_flat(values), _flat(values.flip(0)), np.zeros(far), np.zeros(far), 5, 1e-2)
    _check_params(p[-far:], want, off, torch.bfloat16)
    assert not bool(p[:-far].any())
    b = (n + 255) // 256
    first = (n - far) // 256 * 256  # the block that the far end begins in
    codes = [npy(state[k * 256 * b + first:(k + 1) * 256 * b]) for k in (0, 1)]
    got_m, _ = R.unpack(np.concatenate(codes + [npy(state[512 * b + 2 * (first // 256):])]), n - first)
    x = np.concatenate([np.zeros(n - far - first), abs(m)])
    u, _ = R.noise(n - first, 5, 2, first)
    kept, spacing = R.rounded(x, u, 4)
    assert (abs(got_m) != kept).sum() <= 2 and (abs(abs(got_m) - kept) <= spacing).all()
    del state
    ms, vs = torch.zeros(n, device=device), torch.zeros(n, device=device)
    p[-far:] = values
    adamw_step([p], [g], [ms], [vs], [torch.tensor(4.0)], 1e-2)
    _check_params(p[-far:], want, off, torch.bfloat16)
    assert not bool(ms[:-far].any())


def test_first_step_is_not_captured(device):
    """The states that a first step makes would be zeroed again by every replay."""
    from fast_sp_gs_amd.adamw import AdamW
    p = torch.nn.Parameter(torch.ones(10, device=device))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], capturable=True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='before'):
        with torch.cuda.graph(graph):
            opt.step()


def test_copies_and_pickles_of_the_optimiser(device):
    import copy
    import pickle
    from fast_sp_gs_amd.adamw import AdamW
    for make in (copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))):
        p = torch.nn.Parameter(torch.linspace(0, 1, 600, device=device))
        opt = AdamW([p], lr=1e-2, state_bits=8, max_norm=0.5, seed=3)
        p.grad = torch.cos(p.detach())
        opt.step()
        other = make(opt)
        q = other.param_groups[0]['params'][0]
        for o, t in ((opt, p), (other, q)):
            t.grad = torch.sin(t.detach())
            o.step()
        assert torch.equal(p.detach(), q.detach()) and float(other.last_norm) == float(opt.last_norm)


def test_wrong_tensors_are_refused(device):
    """Before anything is counted or written."""
    from fast_sp_gs_amd.adamw import AdamW, adamw8_moments, adamw8_pack, adamw8_state, adamw8_step, adamw_step
    p, step = torch.ones(8, device=device), torch.tensor(3.0)
    ok = lambda: torch.zeros(8, device=device)
    cases = [('there twice', dict(params=[p, p])), ('shape', dict(grads=[torch.ones(2, 4, device=device)])), ('dtype', dict(grads=[p.half()])),
             ('differ', dict(m=[torch.zeros(4, 2, device=device)])), ('torch.float32', dict(m=[ok().half()])), ('one number', dict(steps=[torch.zeros(2)])),
             ('CUDA', dict(grads=[torch.ones(8)])), ('gaps', dict(params=[torch.ones(16, device=device)[::2]])),
             ('dtype', dict(params=[p.double()], grads=[p.double()])), ('there twice', dict(params=[ok(), ok()], m=[p, p])),
             ('there twice', dict(params=[ok(), ok()], steps=[step, step]))]
    for text, wrong in cases:
        n = max(len(v) for v in wrong.values())
        args = dict(params=[ok() for _ in range(n)], grads=[ok() for _ in range(n)], m=[ok() for _ in range(n)], v=[ok() for _ in range(n)],
                    steps=[step.clone() for _ in range(n)])
        args.update(wrong)
        with pytest.raises(RuntimeError, match=text):
            adamw_step(args['params'], args['grads'], args['m'], args['v'], args['steps'])
        assert all(float(s.max()) in (0.0, 3.0) for s in args['steps'])
    with pytest.raises(RuntimeError, match='all be on the host or all on the device'):
        adamw_step([ok(), ok()], [ok(), ok()], [ok(), ok()], [ok(), ok()], [step, step.to(device)])
    with pytest.raises(RuntimeError, match='another number of elements'):
        adamw8_step([p], [p], [adamw8_state(torch.ones(300, device=device))], [step])
    with pytest.raises(RuntimeError, match='another number of elements'):
        adamw8_moments([adamw8_state(p)], [torch.ones(300, device=device)])
    with pytest.raises(RuntimeError, match='uint8'):
        adamw8_step([p], [p], [torch.zeros(514, device=device)], [step])
    with pytest.raises(RuntimeError, match='boundary of 16 bytes'):
        adamw8_step([p], [p], [torch.zeros(515, dtype=torch.uint8, device=device)[1:]], [step])
    with pytest.raises(RuntimeError, match='differ'):
        adamw8_pack([p], [p.view(2, 4)])
    assert float(step) == 3.0 and torch.equal(p, torch.ones_like(p))
    theirs = torch.optim.AdamW([torch.nn.Parameter(ok())], amsgrad=True)
    with pytest.raises(ValueError, match='amsgrad'):
        AdamW([torch.nn.Parameter(ok())]).load_state_dict(theirs.state_dict())


def test_more_elements_than_a_launch_takes_are_refused(device):
    from fast_sp_gs_amd.adamw import adamw8_step
    n = 1 << 34  # nothing of it is touched
    p = torch.empty(n, dtype=torch.bfloat16, device=device)
    step, state = torch.zeros(()), torch.empty(n // 256 * 514, dtype=torch.uint8, device=device)
    with pytest.raises(RuntimeError, match='elements'):
        adamw8_step([p], [p], [state], [step])
    assert float(step) == 0.0


@pytest.mark.parametrize('clip', [False, True])
def test_codes_are_those_of_the_exact_moments(device, clip):
    """Values that lie within a float32's rounding of a border fall on the side that the definition puts them on: not one of a million
    codes differs (in float64 both sides are off by parts in 10^16, a border is that near for none of them)."""
    from fast_sp_gs_amd.adamw import adamw8_pack, adamw8_step
    n = 1 << 18
    params, grads, ms, vs, steps = _problem(device, [n, n], torch.float32, 31)
    states = adamw8_pack(ms, vs)
    old = [R.unpack(npy(s), n) for s in states]
    total = np.sqrt(sum((_flat(g) ** 2).sum() for g in grads))
    factor = min(1.0, 0.3 * total / (total + 1e-6)) if clip else 1.0
    adamw8_step(params, grads, states, steps, max_norm=0.3 * total if clip else None, seed=8)
    for k in range(2):
        t = int(steps[k])
        _, m, v, _ = R.step64(0.0, _flat(grads[k]), *old[k], t, 1e-3, factor=factor)
        got_m, got_v = R.unpack(npy(states[k]), n)
        u_m, u_v = R.noise(n, t, 8)
        kept_m, _ = R.rounded(abs(m), u_m, 4)
        kept_v, spacing = R.rounded(v, u_v, 5)
        assert np.array_equal(got_m, np.sign(m) * kept_m)
        assert np.array_equal(got_v, np.where((kept_v == 0) & (v > 0), spacing, kept_v))


def test_a_moment_that_equals_its_gradient_stays(device):
    """Codes' own values as gradients, with every noise there is (0 among them): m and v are on their codes' borders and keep them."""
    from fast_sp_gs_amd.adamw import adamw8_pack, adamw8_step
    n = 1 << 20
    values = torch.tensor([1.0, 1.125, 0.625, 0.01171875], device=device).repeat(n // 4)
    p, step = torch.zeros(n, device=device), torch.tensor(3.0)
    m, = adamw8_pack([values], [torch.ones_like(values)])
    before = m.clone()
    adamw8_step([p], [values.clone()], [m], [step], lr=0.0, betas=(0.9, 0.0))
    assert torch.equal(m[:n], before[:n])
    ones = torch.tensor([1.0, 0.5, 2.0, 0.25], device=device).repeat(n // 4)
    state, = adamw8_pack([ones], [ones * ones])
    before = state.clone()
    for seed in range(4):
        adamw8_step([p], [ones], [state], [step], lr=0.0, seed=seed)
        assert torch.equal(state, before)


def test_moments_on_a_border_by_decimal_betas(device):
    """0.9 * 9 / 8 + 0.1 * 8 is 14.5 / 8: with a noise of a half it reaches 15 / 8, though 1 - 0.9 in binary falls short of 0.1 by 2e-17."""
    from fast_sp_gs_amd.adamw import adamw8_pack, adamw8_step
    n = 1 << 20
    p, m = torch.zeros(n, device=device), torch.full((n,), 9 / 8, device=device)
    state, = adamw8_pack([m], [torch.ones(n, device=device)])
    adamw8_step([p], [torch.full((n,), 8.0, device=device)], [state], [torch.tensor(5.0)], lr=0.0, seed=2)
    u, _ = R.noise(n, 6, 2)
    assert (u == 0.5).any()
    assert np.array_equal(R.unpack(npy(state), n)[0], np.where(u >= 0.5, 15 / 8, 14 / 8))
