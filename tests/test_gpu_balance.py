"""Balance losses of an association (fast_sp_gs_amd/balance.py) against their definition in 64 bits: widths around a lane's, a row of
lanes', a wavefront's and beyond; ties, -inf, masks, NaN; strides and addresses; gradients against the formula and differences; bad
weights and indices; graphs and streams; and the association's training with the optimiser that goes with it."""
import numpy as np
import pytest
import torch

from util import npy

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _reference(x, K, on):
    """x [N,M] float64, on [N] -> dict with p, counts, importance, loss and D, the largest distance of a weight above 2^-126 from the largest."""
    N, M = x.shape
    on = on & (x > -np.inf).any(1) if N else on
    p, counts, D = np.zeros((N, M)), np.zeros(M, np.int64), np.zeros(N)
    for n in np.flatnonzero(on):
        d = x[n] - x[n].max()
        e = np.exp(d)
        p[n] = e / e.sum()
        D[n] = min(90.0, -d[d > -np.inf].min())
        order = np.argsort(-x[n], kind='stable')[:K]
        counts[order[x[n][order] > -np.inf]] += 1
    T, C = max(1, on.sum()), max(1, counts.sum())
    importance = p.sum(0) / T
    return dict(p=p, counts=counts, importance=importance, loss=M * (counts / C * importance).sum(), D=D, T=T, C=C, on=on)


def _off_p(r):
    """A weight's relative error: a difference, its product with log2 e (itself rounded) and exp2 in the weight and in the sum, up to 64
    additions a lane and six between them, a quotient and a product."""
    return (6 * r['D'] + 80) * U


def _grad(r, M, g_loss, g_importance):
    a = (g_loss * M * r['counts'] / r['C'] + g_importance) / r['T']
    mean = (r['p'] * a).sum(1, keepdims=True)
    size = abs(a) + (r['p'] * abs(a)).sum(1, keepdims=True)
    # the weights' errors in both places, a's own five roundings, the mean's up to 70 additions, two operations after
    return r['p'] * (a - mean), r['p'] * size * (2 * _off_p(r)[:, None] + 90 * U)


def _check(logits, K, rows, r, dtype, upstream=(0.7, None)):
    from fast_sp_gs_amd.balance import balance_loss
    M = logits.shape[1]
    leaf = logits.detach().requires_grad_(True) if logits.is_contiguous() else logits.detach().as_strided(
        logits.size(), logits.stride(), logits.storage_offset()).requires_grad_(True)
    loss, counts, importance = balance_loss(leaf, K, rows)
    assert counts.dtype == torch.int32 and importance.dtype == torch.float32 and loss.shape == ()
    assert np.array_equal(npy(counts), r['counts'])
    # rows in turn in float32 within a lane (their errors of one sign at worst), blocks in float64
    off = (r['p'] * _off_p(r)[:, None]).sum(0) / r['T'] + (r['p'].shape[0] + 8) * U * r['importance'] + 2.0 ** -126
    assert (abs(npy(importance) - r['importance']) <= off).all()
    assert abs(float(loss) - r['loss']) <= M * (r['counts'] / r['C'] * off).sum() + 2 * U * r['loss']
    with torch.no_grad():
        again = balance_loss(leaf, K, rows)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts) and torch.equal(again[2], importance)
    g_importance = torch.zeros(M, device=logits.device) if upstream[1] is None else upstream[1]
    outs, ups = ([loss], [torch.tensor(upstream[0], device=logits.device)])
    if upstream[1] is not None:
        outs, ups = [loss, importance], ups + [upstream[1]]
    grad, = torch.autograd.grad(outs, leaf, ups)
    assert grad.dtype == dtype and grad.shape == logits.shape
    want, off = _grad(r, M, float(ups[0]), npy(g_importance).astype(np.float64))
    bound = off + HALF[dtype] * (abs(want) + off) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
    got = npy(grad.float()).astype(np.float64)
    assert (abs(got - want) <= bound).all()
    assert not got[~r['on']].any()
    return grad


WIDTHS = [(1, 1), (5, 3), (7, 8), (33, 16), (40, 17), (64, 31), (100, 32), (50, 33), (90, 64), (257, 65), (129, 128), (60, 130),
          (50, 256), (70, 512), (31, 513), (20, 1000), (13, 1024), (9, 1500), (6, 2048), (6, 2049), (5, 4096), (4, 4097), (3, 6001)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('N,M', WIDTHS)
def test_loss_counts_and_gradient(device, N, M, dtype):
    g = torch.Generator().manual_seed(N * 10007 + M)
    for K in sorted({1, min(2, M), min(5, M), min(16, M)}):
        x = torch.randn(N, M, generator=g) * 2
        x[torch.rand(N, M, generator=g) < 0.2] = float('-inf')
        x[0, 1:] = float('-inf')  # a point that may use one superpoint
        if N > 2:
            x[2] = float('-inf')  # and one that may use none
        x = x.to(dtype)
        rows = torch.rand(N, generator=g) < 0.8 if K != 1 else None
        on = np.ones(N, bool) if rows is None else npy(rows)
        r = _reference(x.double().numpy(), K, on)
        up = torch.randn(M, generator=g).to(device) if K == 2 else None
        _check(x.to(device), K, None if rows is None else rows.to(device), r, dtype, (0.7, up))


@pytest.mark.parametrize('N,M,dtype', [(1000, 4500, torch.float32), (900, 8192, torch.bfloat16), (7, 8193, torch.float32), (5, 16384, torch.float16),
                                       (4, 16385, torch.float32), (3, 20001, torch.bfloat16)])
def test_rows_that_take_a_block(device, N, M, dtype):
    """More superpoints than a wavefront's lanes hold, blocks with a second row, with ties and with points left out."""
    g = torch.Generator().manual_seed(M)
    x = (torch.randn(N, M, generator=g) * 2).round(decimals=1).to(dtype)
    rows = torch.rand(N, generator=g) < 0.8
    rows[0] = True
    for K in (1, 5):
        r = _reference(x.double().numpy(), K, npy(rows))
        _check(x.to(device), K, rows.to(device), r, dtype, (0.7, torch.randn(M, generator=g).to(device)))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M', [7, 16, 64, 100, 512, 1030, 4097])
def test_ties_go_to_the_lowest_index(device, M, dtype):
    """All equal, few distinct values, zeros of both signs, and the type's lowest value, which is no mask."""
    g = torch.Generator().manual_seed(M)
    N = 40
    x = torch.randint(-2, 3, (N, M), generator=g).float() / 2
    x[0] = 0.0
    x[1] = torch.where(torch.arange(M) % 2 == 0, -0.0, 0.0)
    x[2, : M // 2] = float('-inf')
    x[2, M // 2:] = 1.0
    x = x.to(dtype)
    x[3] = torch.finfo(dtype).min
    x[4, 1:] = torch.finfo(dtype).min
    for K in sorted({1, 2, min(6, M), min(33, M)}):
        _check(x.to(device), K, None, _reference(x.double().numpy(), K, np.ones(N, bool)), dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M', [5, 64, 500, 512, 2000])
def test_strides_and_addresses(device, M, dtype):
    g = torch.Generator().manual_seed(M + 1)
    N, K = 37, 3
    x = torch.randn(N, M, generator=g).to(dtype)
    r = _reference(x.double().numpy(), K, np.ones(N, bool))
    first = _check(x.to(device), K, None, r, dtype)
    for at, width in ((0, M + 8), (1, M + 9), (8, M + 16), (3, M + 3)):
        wide = torch.full((N, width), float('nan'), dtype=dtype, device=device)
        wide[:, at:at + M] = x.to(device)
        assert torch.equal(_check(wide[:, at:at + M], K, None, r, dtype), first)
    flat = torch.full((N * M + 1,), float('nan'), dtype=dtype, device=device)
    flat[1:] = x.to(device).view(-1)
    assert torch.equal(_check(flat[1:].view(N, M), K, None, r, dtype), first)
    assert torch.equal(_check(x.to(device).t().contiguous().t(), K, None, r, dtype), first)
    one = x[:1].to(device).expand(N, M)  # rows that share their memory
    _check(one, K, None, _reference(x[:1].double().numpy().repeat(N, 0), K, np.ones(N, bool)), dtype)
    mask = torch.zeros(2 * N, dtype=torch.bool, device=device)
    mask[::4] = True
    on = npy(mask[::2])
    _check(x.to(device), K, mask[::2], _reference(x.double().numpy(), K, on), dtype)


@pytest.mark.parametrize('M', [8, 48, 512, 1500, 4100])
def test_values_that_are_no_numbers(device, M):
    """NaN and infinities in rows that do not count are not seen; in rows that do they reach every result but the counts."""
    from fast_sp_gs_amd.balance import balance_loss
    g = torch.Generator().manual_seed(M + 2)
    N, K = 25, 2
    x = torch.randn(N, M, generator=g)
    rows = torch.rand(N, generator=g) < 0.6
    x[~rows] = torch.tensor([float('nan'), float('inf'), float('-inf'), 3e38])[torch.randint(0, 4, (int((~rows).sum()), M), generator=g)]
    clean = torch.where(rows[:, None], x, 0.0)
    _check(x.to(device), K, rows.to(device), _reference(clean.double().numpy(), K, npy(rows)), torch.float32)
    for bad in (float('nan'), float('inf')):
        for whole in (False, True):
            y = torch.randn(N, M, generator=g).to(device)
            if whole:
                y[7] = bad
            else:
                y[7, M // 2] = bad
            y.requires_grad_(True)
            loss, counts, importance = balance_loss(y, K)
            grad, = torch.autograd.grad(loss, y)
            assert bool(torch.isnan(loss)) and bool(torch.isnan(importance).any()) and bool(torch.isnan(grad[7]).any())
            assert int(counts.sum()) <= N * K
    # far apart logits: all of the weight on one, and magnitudes whose squares overflow
    y = torch.zeros(N, M)
    y[:, 1] = torch.linspace(0, 1e4, N)
    y[3] = -3e38
    y[4] = 3e38
    y[4, 0] = -3e38
    _check(y.to(device), 1, None, _reference(y.double().numpy(), 1, np.ones(N, bool)), torch.float32)


def test_nothing_to_count(device):
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    for N, rows in ((0, None), (5, torch.zeros(5, dtype=torch.bool, device=device)), (5, None)):
        x = torch.full((N, 6), float('-inf') if rows is None else 1.0, device=device, requires_grad=True)
        loss, counts, importance = balance_loss(x, 2, rows)
        assert float(loss) == 0 and not bool(counts.any()) and not bool(importance.any())
        assert not bool(torch.autograd.grad(loss, x)[0].any())
    for N, rows in ((0, None), (5, torch.zeros(5, dtype=torch.bool, device=device))):
        w = torch.full((N, 3), 0.5, device=device, requires_grad=True)
        loss, counts, importance = neighbour_balance(w, torch.zeros(N, 3, dtype=torch.long, device=device), 4, rows)
        assert float(loss) == 0 and not bool(counts.any()) and not bool(importance.any())
        assert not bool(torch.autograd.grad(loss, w)[0].any())


def test_many_rows(device):
    """More rows than the blocks take in one turn, and than 2^31 elements."""
    from fast_sp_gs_amd.balance import balance_loss
    g = torch.Generator(device=device).manual_seed(5)
    N, M = 70_001, 40
    x = torch.randn(N, M, generator=g, device=device)
    _check(x, 3, None, _reference(npy(x).astype(np.float64), 3, np.ones(N, bool)), torch.float32)
    N, M = 1_100_000, 2000
    rows = torch.zeros(N, dtype=torch.bool, device=device)
    rows[-50:] = True
    rows[5] = True
    x = torch.empty(N, M, dtype=torch.bfloat16, device=device)
    x[rows] = torch.randn(51, M, generator=g, device=device).bfloat16()
    part = x[rows]
    r = _reference(part.double().cpu().numpy(), 4, np.ones(51, bool))
    x.requires_grad_(True)
    loss, counts, importance = balance_loss(x, 4, rows)
    grad, = torch.autograd.grad(loss, x)
    alone = part.requires_grad_(True)
    want = balance_loss(alone, 4)
    assert np.array_equal(npy(counts), r['counts']) and torch.equal(counts, want[1])
    assert abs(float(loss) - r['loss']) <= 700 * U * r['loss']
    assert float((importance - want[2]).abs().max()) <= 60 * U * float(want[2].max())
    got, same = grad[rows].double(), torch.autograd.grad(want[0], alone)[0].double()
    assert float((got - same).abs().max()) <= 2.0 ** -7 * float(same.abs().max())
    assert not bool(grad[:5].any()) and not bool(grad[6:-50:1000].any()) and not bool(grad[-150:-50].any())


def test_gradient_against_differences(device):
    """The choices held, as they are in the derivative: central differences of the 64-bit loss."""
    from fast_sp_gs_amd.balance import balance_loss
    g = torch.Generator().manual_seed(6)
    N, M, K = 9, 11, 2
    x = torch.randn(N, M, generator=g)
    r = _reference(x.double().numpy(), K, np.ones(N, bool))
    share = r['counts'] / r['C']
    leaf = x.to(device).requires_grad_(True)
    grad, = torch.autograd.grad(balance_loss(leaf, K)[0], leaf)
    h, y = 1e-5, x.double().numpy()
    def loss(y):
        e = np.exp(y - y.max(1, keepdims=True))
        return M * (share * (e / e.sum(1, keepdims=True)).mean(0)).sum()
    for n in range(N):
        for m in range(M):
            up, down = y.copy(), y.copy()
            up[n, m] += h
            down[n, m] -= h
            # differences: h^2 / 6 of third derivatives (below 1) and 1e-16 / h of rounding; the kernel: 400 U of values below 1
            assert abs(float(grad[n, m]) - (loss(up) - loss(down)) / (2 * h)) < 1e-10 + 1e-10 + 400 * U


# ---- neighbour weights --------------------------------------------------------------------------------------------------------------
def _neighbour_reference(w, index, M, on):
    w, index = w[on], index[on]
    counts = np.bincount(index[np.arange(len(w)), w.argmax(1)], minlength=M) if len(w) else np.zeros(M, np.int64)
    T = max(1, len(w))
    importance = np.bincount(index.reshape(-1), weights=w.reshape(-1), minlength=M) / T
    return counts, importance, M * (counts / max(1, counts.sum()) * importance).sum(), T


@pytest.mark.parametrize('N,M,K', [(1, 1, 1), (1, 5, 3), (3, 2, 7), (1000, 512, 3), (1025, 64, 4), (4097, 2048, 8), (300, 5400, 2),
                                   (300, 5401, 2), (500, 20_000, 5), (300_000, 37, 1), (262_145, 512, 2), (50, 10, 20)])
def test_neighbour_balance(device, N, M, K):
    from fast_sp_gs_amd.balance import neighbour_balance
    g = torch.Generator().manual_seed(N + M + K)
    w = torch.softmax(torch.randn(N, K, generator=g) * 2, dim=-1)
    w[0] = 1.0 / K  # equal weights: the first is chosen
    index = torch.randint(0, M, (N, K), generator=g)
    if K > 2:
        index[:, 2] = index[:, 0]  # an index that is there twice
    for masked in (False, True):
        rows = torch.rand(N, generator=g) < 0.7 if masked else torch.ones(N, dtype=torch.bool)
        given, where = w.clone(), index.clone()
        given[~rows], where[~rows] = float('nan'), -77  # not looked at
        counts, importance, loss, T = _neighbour_reference(w.double().numpy(), npy(index), M, npy(rows))
        leaf = given.to(device).requires_grad_(True)
        got = neighbour_balance(leaf, where.to(device), M, rows.to(device) if masked else None)
        assert np.array_equal(npy(got[1]), counts)
        # every weight in units of 2^-31: half a unit each; the sum's and the mean's rounding
        off = np.bincount(npy(index[rows]).reshape(-1), minlength=M) * 2.0 ** -32 / T + 2 * U * importance
        assert (abs(npy(got[2]) - importance) <= off).all()
        assert abs(float(got[0]) - loss) <= M * (counts / max(1, counts.sum()) * off).sum() + 2 * U * loss
        again = neighbour_balance(leaf.detach(), where.to(device), M, rows.to(device) if masked else None)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
        up = torch.randn(M, generator=g)
        grad, = torch.autograd.grad([got[0], got[2]], leaf, [torch.tensor(1.3, device=device), up.to(device)])
        a, b = 1.3 * M * counts / max(1, counts.sum()) / T, up.double().numpy() / T
        want = np.where(npy(rows)[:, None], (a + b)[npy(index)], 0.0)
        bound = np.where(npy(rows)[:, None], (abs(a) + abs(b))[npy(index)], 0.0) * 8 * U
        assert (abs(npy(grad).astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize('N,M,K', [(300, 10_800, 3), (300, 10_801, 4), (700, 86_400, 3), (700, 86_401, 4), (20_000, 30_000, 2)])
def test_neighbour_balance_of_many_superpoints(device, N, M, K):
    """Several ranges of superpoints, and more than there are ranges for."""
    test_neighbour_balance(device, N, M, K)


def test_bad_weights_and_indices_show(device):
    from fast_sp_gs_amd.balance import neighbour_balance
    for M in (50, 6000, 90_000):
        for bad_w, bad_i in ((float('nan'), 3), (-0.1, 3), (1.5, 3), (float('inf'), 3), (0.5, -1), (0.5, M), (0.5, 1 << 40)):
            w = torch.full((2000, 3), 1 / 3, device=device)
            index = torch.randint(0, M, (2000, 3), device=device)
            w[1234, 1], index[1234, 1] = bad_w, bad_i
            w.requires_grad_(True)
            loss, counts, importance = neighbour_balance(w, index, M)
            assert bool(torch.isnan(loss)) and bool(torch.isnan(importance).all()) and int(counts.sum()) == 2000
            grad, = torch.autograd.grad(loss, w)
            assert bool(torch.isnan(grad[1234, 1])) == (bad_i != 3) and int(torch.isnan(grad).sum()) == int(bad_i != 3)
            rows = torch.ones(2000, dtype=torch.bool, device=device)
            rows[1234] = False
            assert bool(torch.isfinite(neighbour_balance(w.detach(), index, M, rows)[0]))


# ---- calls as a program makes them ---------------------------------------------------------------------------------------------------
def _both(x, w, index, M, rows):
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    a, b = balance_loss(x, 2, rows), neighbour_balance(w, index, M, rows)
    return [*a, *b, *torch.autograd.grad(a[0] + 2 * b[0], (x, w))]


def test_captured_and_on_another_stream(device):
    g = torch.Generator(device=device).manual_seed(11)
    N, M, K = 5000, 96, 4
    def inputs():
        return (torch.randn(N, M, generator=g, device=device), torch.softmax(torch.randn(N, K, generator=g, device=device), -1),
                torch.randint(0, M, (N, K), generator=g, device=device), torch.rand(N, generator=g, device=device) < 0.8)
    sets = [inputs() for _ in range(4)]
    def eager(k):
        x, w, index, rows = sets[k]
        return [t.clone() for t in _both(x.clone().requires_grad_(True), w.clone().requires_grad_(True), index, M, rows)]
    want = [eager(k) for k in range(4)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = eager(1)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    x, w, index, rows = (t.clone() for t in sets[0])
    x.requires_grad_(True), w.requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _both(x, w, index, M, rows)
    for k in (0, 1, 2, 3, 1):
        with torch.no_grad():
            for t, s in zip((x, w, index, rows), sets[k]):
                t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
        assert all(torch.equal(a, b) for a, b in zip(eager(k), want[k]))


def test_captured_beside_an_eager_graph_of_the_same_leaves(device):
    """The default stream, on which the eager graph accumulates, cannot join a capture: refused before anything is recorded."""
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    x = torch.randn(300, 20, device=device, requires_grad=True)
    w = torch.full((300, 2), 0.5, device=device, requires_grad=True)
    index = torch.randint(0, 20, (300, 2), device=device)
    calls = [lambda: balance_loss(x)[0], lambda: neighbour_balance(w, index, 20)[0]]
    for leaf, call in zip((x, w), calls):
        alive = call()
        want, = torch.autograd.grad(alive, leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match='eager graph'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(call(), leaf)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_differentiated_once(device):
    from fast_sp_gs_amd.balance import balance_loss
    x = torch.randn(6, 5, device=device, requires_grad=True)
    loss, counts, importance = balance_loss(x, 1)
    assert not counts.requires_grad and importance.requires_grad
    up = torch.ones((), device=device, requires_grad=True)  # as after any further operation of a graph
    g, = torch.autograd.grad(loss, x, up, create_graph=True)
    with pytest.raises(RuntimeError, match='once'):
        g.sum().backward()
    loss, counts, importance = balance_loss(x, 1)
    counts += 1  # what the backward reads
    with pytest.raises(RuntimeError, match='inplace'):
        loss.backward()


def test_training_of_an_association(device):
    """Learned logits over the superpoints as a model trains them: neighbours by distance, weights by `sp_W`, the warp, a loss on the
    warped points plus both balances, one clipped AdamW step with 8-bit moments; the logits' gradient is the sum of its parts."""
    from fast_sp_gs_amd.adamw import AdamW
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    from fast_sp_gs_amd.deform import calc_LBS_weight, superpoint_deform
    g = torch.Generator().manual_seed(12)
    N, M, K = 3000, 40, 4
    points, ctrl = torch.randn(N, 3, generator=g).to(device), torch.randn(M, 3, generator=g).to(device)
    sp_t, sp_r = torch.randn(M, 3, generator=g).to(device), torch.randn(M, 4, generator=g).to(device)
    target = torch.randn(N, 3, generator=g).to(device)
    sp_W = torch.nn.Parameter((torch.randn(N, M, generator=g) * 0.1).to(device))
    opt = AdamW([{'params': [sp_W], 'name': 'sp_W'}], lr=1e-2, weight_decay=0.0, state_bits=8, max_norm=1.0)
    def parts():
        d_xyz, _, _, _, index = superpoint_deform(points, ctrl, sp_t, sp_r, None, K=K, LBS_method='W', sp_W=sp_W)
        weights, same = calc_LBS_weight(points, ctrl, K=K, LBS_method='W', sp_W=sp_W)
        assert torch.equal(index, same)
        return [((points + d_xyz - target) ** 2).mean(), balance_loss(sp_W, 1)[0], 0.5 * neighbour_balance(weights, index, M)[0]]
    for k in range(3):
        grads = [torch.autograd.grad(p, sp_W)[0] for p in parts()]
        opt.zero_grad()
        sum(parts()).backward()
        # one accumulation order against another, of three terms
        assert float((sp_W.grad - sum(grads)).abs().max()) <= 4 * U * float(sum(t.abs() for t in grads).max())
        before, norm = sp_W.detach().clone(), float(sp_W.grad.double().norm())
        opt.step()
        assert float(opt.last_norm) == pytest.approx(norm, rel=8 * U)
        moved = (sp_W.detach() - before).abs()
        assert bool(torch.isfinite(sp_W.detach()).all()) and 0 < float(moved.max()) <= 1e-2 * 7.3
    assert float(opt.state[sp_W]['step']) == 3.0


def test_wrong_calls_are_refused(device):
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    x, w, i = torch.zeros(4, 5, device=device), torch.zeros(4, 2, device=device), torch.zeros(4, 2, dtype=torch.long, device=device)
    for text, call in (('K must be', lambda: balance_loss(x, 0)), ('K must be', lambda: balance_loss(x, 6)),
                       ('K must be', lambda: balance_loss(torch.zeros(4, 100, device=device), 65)), ('N, M', lambda: balance_loss(x[0], 1)),
                       ('N, M', lambda: balance_loss(x[:, :0], 1)), ('dtype', lambda: balance_loss(x.double(), 1)),
                       ('shape', lambda: balance_loss(x, 1, torch.ones(5, dtype=torch.bool, device=device))),
                       ('torch.bool', lambda: balance_loss(x, 1, torch.ones(4, device=device))), ('CUDA', lambda: balance_loss(x, 1, torch.ones(4, dtype=torch.bool))),
                       ('float32', lambda: neighbour_balance(w.half(), i, 3)), ('int64', lambda: neighbour_balance(w, i.int(), 3)),
                       ('shape', lambda: neighbour_balance(w, i[:, :1], 3)), ('M must', lambda: neighbour_balance(w, i, 0)),
                       ('N, K', lambda: neighbour_balance(w[0], i[0], 3)), ('shape', lambda: neighbour_balance(w, i, 3, torch.ones(3, dtype=torch.bool, device=device)))):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_two_threads_at_once(device):
    """Calls of two host threads on streams of their own."""
    import threading
    g = torch.Generator(device=device).manual_seed(13)
    sets = [(torch.randn(3000, 70 + 30 * k, generator=g, device=device), torch.softmax(torch.randn(3000, 3, generator=g, device=device), -1),
             torch.randint(0, 70, (3000, 3), generator=g, device=device)) for k in range(2)]
    run = lambda s: _both(s[0].clone().requires_grad_(True), s[1].clone().requires_grad_(True), s[2], 70, None)
    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    wrong = []
    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = run(sets[k])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    wrong.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
