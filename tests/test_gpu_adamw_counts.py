"""Step counts that cannot count, or have not begun."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(device, bits, count):
    from fast_sp_gs_amd.adamw import adamw8_state, adamw8_step, adamw_step
    p, g = (torch.ones(8, device=device) for _ in range(2))
    if bits == 8:
        adamw8_step([p], [g], [adamw8_state(p)], [count])
    else:
        adamw_step([p], [g], [torch.zeros_like(p)], [torch.zeros_like(p)], [count])
    return p


@pytest.mark.parametrize('bits', [32, 8])
def test_counts(device, bits):
    """In types whose numbers end their steps at 256 or 2048 the bias corrections and the rounding's random numbers would stand still."""
    for value, dtype, text in ((2048, torch.float16, 'dtype'), (256, torch.bfloat16, 'dtype'), (127, torch.int8, 'dtype'), (255, torch.uint8, 'dtype'),
                               (True, torch.bool, 'dtype'), (32767, torch.int16, 'dtype'), (-1.0, torch.float32, 'negative'), (-7, torch.int64, 'negative'),
                               (float('nan'), torch.float64, 'negative')):
        count = torch.tensor(value, dtype=dtype)
        with pytest.raises(RuntimeError, match=text):
            _step(device, bits, count)
        assert torch.equal(count, torch.tensor(value, dtype=dtype)) or value != value
    want = _step(device, bits, torch.tensor(300.0))
    for dtype in (torch.float64, torch.int32, torch.int64):
        count = torch.tensor([300], dtype=dtype)
        assert torch.equal(_step(device, bits, count), want) and int(count) == 301
