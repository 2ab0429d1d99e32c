"""The norm of all gradients to the last bit that float32 can have."""
import numpy as np
import pytest
import torch

from test_gpu_adamw import _flat

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sizes', [[1], [3, 5, 8191, 8192, 8193], [100_003, 7], [0, 5], [11] * 150, [1 << 21]])
def test_norms_are_rounded_once(device, sizes, dtype):
    """Squares and sums are float64 from the first element on: n additions of 2^-53 each, far below what is left, the norm's and the factor's
    rounding to float32."""
    from fast_sp_gs_amd.adamw import grad_norm
    g = torch.Generator().manual_seed(len(sizes) + sizes[0])
    ts = [torch.randn(n, generator=g).to(dtype).to(device) for n in sizes]
    want = np.sqrt(sum((_flat(t) ** 2).sum() for t in ts))
    inside = sum(sizes) * 2.0 ** -53 + 2.0 ** -50
    for max_norm in (0.5 * want, 2.0 * want):
        norm, factor = (float(x) for x in grad_norm(ts, max_norm))
        assert abs(norm - want) <= (U + inside) * want
        assert abs(factor - min(1.0, max_norm / (want + 1e-6))) <= U + inside
