"""The gradient norm, clipping and the clipped Adam step on the host: rows, references, refusals (no GPU needed)."""
import itertools
import math
import random
import struct
import time
from types import SimpleNamespace

import pytest
import torch

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


# ---- which strided tensors share memory ----------------------------------------------------------------------------------------------------

def _bytes(t, base):
    """Every byte of every element, one by one."""
    size, out = t.element_size(), []
    for idx in itertools.product(*(range(n) for n in t.shape)):
        at = t.data_ptr() - base + size * sum(i * s for i, s in zip(idx, t.stride()))
        out += range(at, at + size)
    return out


def _check(tensors, base):
    got = _lib.gradops().shared(tensors)
    sets = [_bytes(t, base) for t in tensors]
    own = [len(set(s)) != len(s) for s in sets]
    pairs = {(i, j) for i in range(len(sets)) for j in range(i + 1, len(sets)) if set(sets[i]) & set(sets[j])}
    what = [(t.dtype, t.storage_offset(), t.shape, t.stride()) for t in tensors]
    if got is None:
        assert not any(own) and not pairs, what
    else:
        assert own[got[0]] if got[0] == got[1] else got in pairs, (what, got)
    return got


def test_shared_memory_of_strided_views_against_every_byte():
    rng = random.Random(7)
    buf = torch.zeros(4096, dtype=torch.uint8)
    base, found = buf.data_ptr(), [0, 0]
    for _ in range(6000):
        tensors = []
        for _ in range(rng.choice([1, 2, 2, 2, 3])):
            dtype = rng.choice([torch.float32, torch.bfloat16])
            shape = [rng.choice([1, 2, 3, 4, 5, 0] if rng.random() < 0.1 else [1, 2, 3, 4]) for _ in range(rng.randrange(4))]
            strides, reach = [], 1
            for n in shape:                                                 # mostly one inside the other, sometimes anything
                s = rng.randrange(0, 12) if rng.random() < 0.25 else reach + rng.choice([0, 0, 1, 2, 5])
                strides.append(s)
                reach = max(reach, s * n)
            order = list(range(len(shape)))
            rng.shuffle(order)
            tensors.append(buf.view(dtype).as_strided([shape[k] for k in order], [strides[k] for k in order], rng.randrange(24)))
        found[_check(tensors, base) is None] += 1
    assert min(found) > 1000, found                                         # both answers were met often


def test_shared_memory_of_views_that_a_model_has():
    w = torch.zeros(60, 70)
    none = [[w[:, :11], w[:, 11:40], w[:, 40:]], [w[::2], w[1::2]], [w[:30, :35], w[30:, 35:], w[:30, 35:], w[30:, :35]], [w.t()[5:9], w[:, :5], w[3, 9:]],
            [torch.zeros(8).as_strided((2, 3), (3, 2))], [w[:0], w], [w[:, 3:3], w[:, :]], []]
    for views in none:
        assert _check(views, w.data_ptr()) is None
    a = w[:, :11]
    assert _check([a, a], w.data_ptr()) == (0, 1)
    assert _check([w, torch.zeros(3), w[:, :11]], w.data_ptr()) == (0, 2)
    assert _check([w[:, :12], w[:, 11:]], w.data_ptr()) == (0, 1)
    assert _check([w[::2], w[1::2], w[7, 3:5]], w.data_ptr()) == (1, 2)
    assert _check([torch.zeros(1).expand(9)], w.data_ptr()) == (0, 0)
    assert _check([w, w.view(-1).as_strided((10, 8), (5, 1))], w.data_ptr()) == (1, 1)
    # large: nothing is enumerated
    v = torch.empty((1 << 16, 64))
    views = [v[:, k:k + 2] for k in range(0, 64, 2)]
    start = time.perf_counter()
    assert _lib.gradops().shared(views) is None and _lib.gradops().shared(views + [v[5, 63:]]) == (31, 32)
    assert _lib.gradops().shared([v.t()[k::3] for k in range(3)]) is None and _lib.gradops().shared([v[k::5] for k in range(5)] + [v[4::10]]) == (4, 5)
    assert time.perf_counter() - start < 2.0
    c = torch.empty(1 << 24, dtype=torch.bfloat16)
    assert _lib.gradops().shared([c.as_strided((1 << 20, 2), (3, 1), 0), c.as_strided((1 << 20,), (3,), 2)]) is None
    with pytest.raises(TypeError, match='list'):
        _lib.gradops().shared((w,))
    with pytest.raises(TypeError, match='tensors'):
        _lib.gradops().shared([1])


# ---- tensors of a step that share memory -----------------------------------------------------------------------------------------------------

def _step(*rows, m=(1, 1), v=(2, 2)):
    """nvdr_adam_step_factor on rows of (parameter, gradient, elements, zero_grad): addresses that nobody reads, since the last row is refused for its
    rate if for nothing else."""
    A, lib = 1 << 30, _lib.load()
    tab = b''.join(optim._ADAM_ROW(p, g, m[k] * A + k * 4096, v[k] * A + k * 4096, n, 1.0, -math.inf, math.inf, 0, 0, 0, 0, -1.0 if k == len(rows) - 1 else 1.0, 0, 3 * A if z else 0, z, 0)
                   for k, (p, g, n, z) in enumerate(rows))
    assert lib.nvdr_adam_step_factor(tab, len(rows), 1e-3, 0.9, 0.999, 1e-8, A, 1, None, None) == -1
    return lib.nvdr_last_error().decode()


def test_a_step_refuses_tensors_that_overlap():
    B, G = 1 << 20, 1 << 22
    apart = [(B, G, 12, 0), (B + 48, G + 48, 12, 0)]
    assert 'lr_scale' in _step(*apart) and 'lr_scale' in _step(*apart[::-1])
    assert 'lr_scale' in _step((B, G, 12, 0), (B, G, 0, 0))                 # nothing of nothing
    for other in (B, B + 44, B + 16, B - 44):
        for n in (12, 15):
            assert 'tensors 0 and 1 are the same or overlap' in _step((B, G, 12, 0), (other, G + 4096, n, 0))
    assert 'tensors 0 and 2 are the same' in _step((B, G, 12, 0), (B + 4096, G + 4096, 12, 0), (B + 8, G + 8192, 12, 0), m=(1, 1, 1), v=(2, 2, 2))
    A = 1 << 30
    assert 'are the same or overlap' in _step((B, G, 3000, 0), (B + (1 << 19), G + (1 << 19), 3000, 0))          # (the moments, 4096 bytes apart)
    assert 'are the same or overlap' in _step((B, G, 12, 0), (A, G + 4096, 12, 0))                               # a parameter in another one's moments


def test_a_step_refuses_a_shared_gradient_that_it_would_clear():
    B, G = 1 << 20, 1 << 22
    far = B + 4096
    assert 'lr_scale' in _step((B, G, 12, 0), (far, G, 12, 0))              # only read
    assert 'lr_scale' in _step((B, G, 12, 1), (far, G + 48, 12, 1))
    for z in ((1, 0), (0, 1), (1, 1)):
        for at in (G, G + 44, G - 44):
            assert 'share a gradient that zero_grad clears' in _step((B, G, 12, z[0]), (far, at, 12, z[1]))


def test_per_channel_bounds_are_checked():
    dev = torch.device('cpu')
    good = torch.tensor([0.0, 0.1, 0.2])
    optim._check_bounds([None, (0.0, 1.0), (None, None, good), [None, 1.0, None, good], (0.0, 1.0, None, None), (0.0, 1.0, good, good[1:])], dev)
    for bad in (good.double(), good.half(), good.long(), torch.zeros(6)[::2], torch.zeros(1).expand(3), good[:0], torch.empty(3, device='meta')):
        for c in ((0.0, 1.0, bad), (0.0, 1.0, None, bad), [0.0, 1.0, good, bad]):
            with pytest.raises(ValueError, match='bounds of parameter 1'):
                optim._check_bounds([None, c], dev)


def test_parameters_lie_on_one_gpu():
    def fake(index, **kw):
        return SimpleNamespace(**dict(dict(dtype=torch.float32, is_contiguous=lambda: True, is_cuda=True, device=torch.device('cuda', index)), **kw))
    for params in ([fake(0), fake(1)], [fake(1), fake(0)], [fake(0), fake(0, is_cuda=False, device=torch.device('cpu'))], [fake(0, dtype=torch.float16)],
                   [fake(0, is_contiguous=lambda: False)]):
        with pytest.raises(ValueError, match='on the GPU'):
            optim.FusedAdam(params)
