"""Gradient norm, clipping and the clipped Adam step where values, memory and callers reach their limits (beside test_gpu_gradnorm.py)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = torch.float32


def _values(shape, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen) * scale


def _adam(start, dev, **kw):
    from nvdiffrecmc_amd.optim import FusedAdam
    return FusedAdam([torch.nn.Parameter(s.to(dev)) for s in start], lr=0.01, **kw)


def _same(a, b):
    """Equal, NaN in the same places."""
    a, b = a.detach().cpu(), b.detach().cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.nan_to_num(a, nan=7.0), torch.nan_to_num(b, nan=7.0))


# ---- tiles and a norm that is not finite -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('when', [0, 2], ids=['first step', 'third step'])
@pytest.mark.parametrize('subsets', [False, True], ids=['whole', 'subsets'])
def test_tiles_follow_the_dense_step_where_the_norm_is_not_finite(subsets, when, bad, dev):
    """A norm of NaN makes every parameter a NaN in a dense tensor, and so in one of tiles, whether they have gradient or history or neither;
    an infinite norm makes the factor zero, and 0 * inf a NaN where the infinity stands.  The steps behind it agree too.  A texel of a normal
    map that is skipped is not normalised again: each time a quotient by a length of 1 +- 2^-23, 2^-22 at most with its own rounding."""
    shapes = [(40, 40, 3), (33, 21, 3), (5, 3)]                             # 25 tiles; 11, the last of 53 texels; and a plain tensor
    start = [_values(s, 3 + i).clamp(-0.9, 0.9) for i, s in enumerate(shapes)]
    kw = dict(max_norm=1.0, clamps=[(0.0, 1.0), (-1.0, 1.0), None], normalize3=[False, True, False])
    a = _adam(start, dev, sparse=[False] * 3, **kw)
    b = _adam(start, dev, sparse=[True, True, False], **kw)
    for t in range(5):
        h = [_values(s, 10 * t + i) for i, s in enumerate(shapes)]
        for g in h[:2]:
            flat = g.view(-1, 3)
            flat[64:] *= (torch.arange(flat.shape[0] - 64) // 64 % 5 == t)[:, None]       # tiles with a gradient: the first, and others every step
        if t == when:
            h[2].view(-1)[4] = bad
        for x, y, g in zip(a.params, b.params, h):
            x.grad, y.grad = g.to(dev), g.to(dev)
        for opt in (a, b):
            if subsets:
                opt.measure_norm()
                opt.step(subset=[2, 1], advance=False)
                opt.step(subset=[0], advance=True)
            else:
                opt.step()
        for i in range(3):
            assert _same(a.exp_avg[i], b.exp_avg[i]) and _same(a.exp_avg_sq[i], b.exp_avg_sq[i]), (t, i)
            x, y = a.params[i].detach(), b.params[i].detach()
            assert torch.equal(x.isnan(), y.isnan()) and float((x - y).nan_to_num().abs().max()) <= (6 * 2.0 ** -22 if i == 1 else 0.0), (t, i)
            if t >= when and math.isnan(bad):
                assert bool(b.params[i].isnan().all()) and (b.active[i] is None or bool((b.active[i] != 0).all())), (t, i)
            elif i < 2:
                assert not bool(b.params[i].isnan().any()), (t, i)
