"""What the AdamW steps refuse, before anything is launched or counted (no GPU is needed to be refused)."""
import numpy as np
import pytest
import torch

import adamw_reference as R


def test_wrong_places_and_numbers():
    from fast_sp_gs_amd.adamw import AdamW, adamw8_moments, adamw8_pack, adamw8_step, adamw_step, grad_norm
    t, step = torch.zeros(4), torch.zeros(())
    with pytest.raises(RuntimeError, match='CUDA'):
        adamw_step([t], [t], [t], [t], [step])
    with pytest.raises(RuntimeError, match='CUDA'):
        adamw8_step([t], [t], [t.byte()], [step])
    with pytest.raises(RuntimeError, match='CUDA'):
        grad_norm([t])
    with pytest.raises(RuntimeError, match='no gradients'):
        grad_norm([])
    with pytest.raises(RuntimeError, match='CUDA'):
        adamw8_moments([torch.zeros(514, dtype=torch.uint8)], [t])
    with pytest.raises(RuntimeError, match='CUDA'):
        adamw8_pack([t], [t])
    with pytest.raises(RuntimeError, match='not supported'):
        adamw8_moments([], [], torch.float64)
    for wrong in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=float('nan')), dict(betas=(1.0, 0.9))):
        with pytest.raises(RuntimeError):
            adamw_step([t], [t], [t], [t], [step], **wrong)
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(t)], **wrong)
    with pytest.raises(RuntimeError, match='for each parameter'):
        adamw_step([t, t], [t], [t, t], [t, t], [step, step])
    with pytest.raises(RuntimeError, match='for each parameter'):
        adamw_step([t], [t], [t], [t], [step], lr=[1e-3, 1e-3])
    with pytest.raises(ValueError, match='state_bits'):
        AdamW([torch.nn.Parameter(t)], state_bits=16)
    with pytest.raises(ValueError, match='max_norm'):
        AdamW([torch.nn.Parameter(t)], max_norm=-1.0)
    assert float(step) == 0.0  # nothing was counted
    assert adamw_step([], [], [], [], []) is None and adamw8_moments([], []) == [] and adamw8_pack([], []) == []


def test_c_entries_refuse_without_touching_the_gpu():
    import ctypes
    from fast_sp_gs_amd import lib
    L = lib.load()
    most = L.fsgs_adamw_max_tensors()
    assert L.fsgs_adamw8_state_bytes(1) == 514 and L.fsgs_adamw8_state_bytes(256) == 514 and L.fsgs_adamw8_state_bytes(257) == 1028
    assert L.fsgs_adamw8_state_bytes(0) == 0 and L.fsgs_adamw8_state_bytes(-1) == 0
    one = (ctypes.c_double * 1)(1.0)
    count = (ctypes.c_int64 * 1)(4)
    odd = (ctypes.c_void_p * 1)(4097)  # an address that is no float's
    null = (ctypes.c_void_p * 1)(None)
    A = ctypes.addressof
    step = lambda n, dtype, counts, p: L.fsgs_adamw_update_multi(n, dtype, A(counts), A(one), A(one), 0.9, 0.999, A(one), A(one), None,
                                                                None, A(p), A(p), A(p), A(p), None)
    assert step(most + 1, 0, count, odd) != 0 and b'adamw' in L.fsgs_last_error()
    assert step(1, 1, count, odd) != 0  # float64
    assert step(1, 0, count, odd) != 0 and step(1, 0, count, null) != 0
    assert step(1, 0, (ctypes.c_int64 * 1)(-4), odd) != 0
    assert step(0, 0, count, odd) == 0 and step(1, 0, (ctypes.c_int64 * 1)(0), null) == 0
    assert L.fsgs_adamw_update_multi(1, 0, None, None, None, 0.9, 0.999, None, None, None, None, None, None, None, None, None) != 0
    assert L.fsgs_adamw8_update_multi(1, 0, A(count), A(one), A(one), 0.9, 0.999, A(one), A(one), 0, None, None, A(odd), A(odd), A(odd),
                                      None) != 0
    assert L.fsgs_grad_square_sums(1, 0, A(count), A(null), 4, 4096, None) != 0
    assert L.fsgs_grad_square_sums(1, 0, A(count), A(odd), L.fsgs_grad_square_sums_max() + 1, 4096, None) != 0
    assert L.fsgs_grad_norm_factor(4, None, 1.0, 4096, None) != 0
    assert L.fsgs_adamw_rates(1, A(null), A(one), 0.9, 0.999, 0, 4096, None) != 0
    assert L.fsgs_adamw8_unpack_multi(1, 0, A(count), A(odd), A(odd), A(odd), None) != 0
    assert L.fsgs_adamw8_pack_multi(1, A(count), A(odd), A(odd), A(odd), None) != 0


def test_more_than_a_launch_holds_is_refused():
    import ctypes
    from fast_sp_gs_amd import lib
    L = lib.load()
    A = ctypes.addressof
    one, at = (ctypes.c_double * 1)(1.0), (ctypes.c_void_p * 1)(4097)  # an address that is no float's
    many = (ctypes.c_int64 * 1)(1 << 34)  # 2^24 blocks of 1024 elements, 256 threads each
    assert L.fsgs_adamw_update_multi(1, 0, A(many), A(one), A(one), 0.9, 0.999, A(one), A(one), None, None, A(at), A(at), A(at), A(at), None) != 0
    assert b'elements' in L.fsgs_last_error()
    assert L.fsgs_adamw8_update_multi(1, 0, A(many), A(one), A(one), 0.9, 0.999, A(one), A(one), 0, None, None, A(at), A(at), A(at), None) != 0
    assert b'elements' in L.fsgs_last_error()
    assert L.fsgs_adamw8_unpack_multi(1, 0, A(many), A(at), A(at), A(at), None) != 0 and b'elements' in L.fsgs_last_error()
    assert L.fsgs_adamw8_pack_multi(1, A(many), A(at), A(at), A(at), None) != 0 and b'elements' in L.fsgs_last_error()


def test_the_roundings_noise_is_even():
    """The hash's two halves over elements, steps and seeds: means, variances and correlations of uniform numbers (five sigma)."""
    n = 1 << 18
    series = [R.noise(n, t, s) for t, s in ((1, 0), (2, 0), (1, 1), (40, 7))]
    for a, b in series:
        for x in (a, b):
            assert abs(x.mean() - 0.5) < 5 * (1 / 12 / n) ** 0.5 + 2 ** -17 and abs(x.var() - 1 / 12) < 5 * (1 / 180 / n) ** 0.5
            for lag in (1, 2, 64, 256):
                assert abs(np.corrcoef(x[:-lag], x[lag:])[0, 1]) < 5 / n ** 0.5
        assert abs(np.corrcoef(a, b)[0, 1]) < 5 / n ** 0.5
        counts = np.bincount((a * 256).astype(int), minlength=256)
        assert ((counts - n / 256) ** 2 / (n / 256)).sum() < 255 + 5 * (2 * 255) ** 0.5
    for i in range(4):
        for j in range(i):
            assert abs(np.corrcoef(series[i][0], series[j][0])[0, 1]) < 5 / n ** 0.5
    # along the steps of one element
    x = np.array([R.noise(4, t, 0)[1][3] for t in range(1, 4097)])
    assert abs(x.mean() - 0.5) < 5 * (1 / 12 / 4096) ** 0.5 and abs(np.corrcoef(x[:-1], x[1:])[0, 1]) < 5 / 64
