"""The gradient norm, clipping and the clipped Adam step on the host: rows, references, refusals (no GPU needed)."""
import math
import struct

from nvdiffrecmc_amd import _lib, optim


def _row(**kw):
    f = dict(dict(grad_scale=1.0, lo=-math.inf, hi=math.inf, lr_scale=1.0), **kw)
    return _lib.NvdrAdamTensor.from_buffer_copy(optim._ADAM_ROW(16, 32, 48, 64, 5, f['grad_scale'], f['lo'], f['hi'], 0, 0, 0, 0, f['lr_scale'], 0, 0, 0, 0))


def test_a_row_with_numbers_beyond_fp32():
    """Bounds and scales outside fp32 are infinite, as they are in the structure itself; everything else is rounded once."""
    for name in ('grad_scale', 'lo', 'hi', 'lr_scale'):
        for value in (1e39, -1e39, 1e308, 10 ** 39, 3.4028235e38, 0.1, -0.0, 1e-50, math.inf, math.nan):
            plain = _lib.NvdrAdamTensor()
            setattr(plain, name, value)
            got = getattr(_row(**{name: value}), name)
            assert struct.pack('f', got) == struct.pack('f', getattr(plain, name)), (name, value)
    r = _row(hi=1e39)
    assert (r.param, r.grad, r.exp_avg, r.exp_avg_sq, r.n, r.lo, r.hi) == (16, 32, 48, 64, 5, -math.inf, math.inf)
