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


# ---- an outlier that only clipping keeps in range ----------------------------------------------------------------------------------------

@pytest.mark.parametrize('kind', ['plain', 'normal map', 'tiles'])
@pytest.mark.parametrize('subsets', [False, True], ids=['whole', 'subsets'])
def test_an_outlier_beyond_fp32_behind_its_scale_is_clipped(subsets, kind, dev):
    """1e37 * 64 is over fp32's range, its clipped value is max_norm.  The factor, 10 / 6.4e38 = 1.6e-38, is a normal number: rounded once, the
    product with 64 exact, the product with the gradient rounded once: 2^-23 relative; the first moment (0.1 rounded, one product) 2^-23
    more, the second (0.001 rounded, two products, the gradient's error twice) 6 * 2^-24 more, each 2^-21 at most."""
    shape = (20, 16, 3)
    g = _values(shape, 1).view(-1)
    g[7], g[300] = 1e37, -3e36
    g = g.view(shape)
    opt = _adam([torch.full(shape, 0.5), torch.full((9,), 0.5)], dev, max_norm=10.0, grad_scales=[64.0, 1.0], sparse=[kind == 'tiles', False], normalize3=[kind == 'normal map', False])
    h = [g, torch.full((9,), 2.0)]
    for q, x in zip(opt.params, h):
        q.grad = x.to(dev)
    if subsets:
        opt.measure_norm()
        opt.step(subset=[0], advance=False)
        opt.step(subset=[1])
    else:
        opt.step()
    eff = [h[0].double() * 64.0, h[1].double()]
    norm = math.sqrt(sum(float((x * x).sum()) for x in eff))
    assert math.isinf(opt.grad_norm.item()) and 2.0 ** -126 < 10.0 / norm
    for i in range(2):
        want = eff[i] * (10.0 / (norm + 1e-6))
        for got, ref in ((opt.exp_avg[i], 0.1 * want), (opt.exp_avg_sq[i], 0.001 * want * want)):
            off = (got.cpu().double() - ref).abs()
            assert bool((off <= 2.0 ** -21 * ref.abs() + 2.0 ** -149).all()), (i, float(off.max()))
        assert bool(torch.isfinite(opt.params[i]).all())
    assert float(opt.exp_avg[0].view(-1)[7]) > 0.9                          # the outlier is what is left


def test_the_factor_enters_a_step_as_a_power_of_two_would(dev):
    """grad_scale * factor as one product: the same bits as gradients scaled beforehand where both are powers of two, whatever the gradient."""
    start = [_values((700, 3), 2)]
    a, b = _adam(start, dev, max_norm=1.0, grad_scales=[64.0]), _adam(start, dev, grad_scales=[64.0])
    for t in range(3):
        g = _values((700, 3), 5 + t, 10.0 ** (t - 1))
        norm = math.sqrt(float(((64.0 * g.double()) ** 2).sum()))
        a.max_norm = 2.0 ** -6 * (norm + 1e-6)                              # rounded to fp32 the factor is 2^-6
        a.params[0].grad, b.params[0].grad = g.to(dev), (g * 2.0 ** -6).to(dev)
        a.step()
        b.step()
        assert torch.equal(a.params[0], b.params[0]) and torch.equal(a.exp_avg[0], b.exp_avg[0]) and torch.equal(a.exp_avg_sq[0], b.exp_avg_sq[0]), t


# ---- numbers beyond fp32 from the host ---------------------------------------------------------------------------------------------------

def test_bounds_beyond_fp32_do_not_bind(dev):
    start = [_values((70, 3), 4)]
    a = _adam(start, dev, clamps=[(-1e39, 1e39)])
    b = _adam(start, dev)
    for t in range(2):
        g = _values((70, 3), t)
        a.params[0].grad, b.params[0].grad = g.to(dev), g.to(dev)
        a.step()
        b.step()
        assert torch.equal(a.params[0], b.params[0])


def test_a_rate_below_fp32_is_no_plain_rate(dev):
    start = [_values((70, 3), 4), _values((9,), 5)]
    for tiny in (1e-46, 5e-324, 2.0 ** -149):
        opt = _adam(start, dev, lr_scales=[tiny, 1.0])
        for q in opt.params:
            q.grad = torch.ones_like(q)
        opt.step()
        assert torch.equal(opt.params[0].cpu(), start[0]) and bool((opt.exp_avg[0] > 0).all())      # (no step that fp32 can hold; the moments go on)
        assert not torch.equal(opt.params[1].cpu(), start[1])


# ---- another thread drops a gradient during the call ---------------------------------------------------------------------------------------

def _entry_that_drops(params, seen):
    """What another thread may do while a call has released the interpreter's lock; nothing is launched."""
    def entry(*_):
        before = torch.cuda.memory_allocated()
        for p in params:
            p.grad = None
        seen.append(before - torch.cuda.memory_allocated())
        return 0
    return entry


def test_clip_holds_the_gradients_it_scales(dev):
    import ctypes
    from nvdiffrecmc_amd import _lib
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    ops, lib = _lib.gradops(), _lib.load()
    names = ('nvdr_grad_norm', 'nvdr_grad_clip', 'nvdr_grad_norm_workspace', 'nvdr_last_error')
    own = {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names}
    params = [torch.nn.Parameter(torch.zeros(1 << 20, device=dev)) for _ in range(3)]
    for p in params:
        p.grad = torch.ones_like(p)
    before, seen = torch.cuda.memory_allocated(), []
    entry = ctypes.CFUNCTYPE(ctypes.c_int, *([ctypes.c_void_p] * 3), ctypes.c_int64, ctypes.c_int, ctypes.c_double, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p)(
        _entry_that_drops(params, seen))
    try:
        ops.bind(*(ctypes.cast(entry, ctypes.c_void_p).value if n == 'nvdr_grad_clip' else own[n] for n in names), torch._C._cuda_getCurrentRawStream)
        clip_grad_norm_(params, 1.0)
    finally:
        ops.bind(*own.values(), torch._C._cuda_getCurrentRawStream)
    assert seen == [0]
    assert torch.cuda.memory_allocated() <= before - (3 << 22) + 512        # ... and no longer (the norm is there)


@pytest.mark.parametrize('how', ['plain', 'clipped', 'subset'])
def test_a_step_holds_the_gradients_it_reads(how, dev, monkeypatch):
    from types import SimpleNamespace
    from nvdiffrecmc_amd import _lib
    opt = _adam([torch.zeros(1 << 20)] * 2, dev, max_norm=None if how == 'plain' else 1.0)
    for p in opt.params:
        p.grad = torch.ones_like(p)
    if how == 'subset':
        opt.measure_norm()
    before, seen = torch.cuda.memory_allocated(), []
    entry = _entry_that_drops(opt.params, seen)
    monkeypatch.setattr(_lib, 'load', lambda: SimpleNamespace(nvdr_adam_step_clipped=entry, nvdr_adam_step_factor=entry))
    opt.step(subset=[0, 1] if how == 'subset' else None)
    assert seen == [0]
    assert torch.cuda.memory_allocated() <= before - (2 << 22)


# ---- versions ------------------------------------------------------------------------------------------------------------------------------

def _with_grads(grads):
    ps = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


def test_a_refused_clip_leaves_the_versions(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    a, b, c = torch.ones(5, device=dev), torch.ones(7, device=dev), torch.ones(9, 4, device=dev)
    cpu, wide, expanded = torch.ones(5), torch.ones(5, device=dev, dtype=torch.float64), torch.ones(1, device=dev).expand(6)
    lists = {'CPU': [a, b, cpu], 'type': [a, wide], 'twice': [a, b, a], 'overlap': [a, b, b[2:]], 'expanded': [a, expanded, c[:, :2]]}
    for name, grads in lists.items():
        versions = [g._version for g in grads]
        with pytest.raises((RuntimeError, ValueError)):
            clip_grad_norm_(_with_grads(grads), 0.5)
        assert [g._version for g in grads] == versions, name
    bad = torch.tensor([1.0, math.nan], device=dev)
    versions = a._version, bad._version
    with pytest.raises(RuntimeError, match='nan'):
        clip_grad_norm_(_with_grads([a, bad]), 0.5, error_if_nonfinite=True)
    assert (a._version, bad._version) == versions


def test_a_clip_raises_each_version_once(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    for strided in (False, True):
        grads = [torch.ones(5, device=dev), torch.ones(9, 4, device=dev)[:, :2] if strided else torch.ones(9, 2, device=dev), torch.ones(300000, device=dev, dtype=torch.bfloat16)]
        versions = [g._version for g in grads]
        clip_grad_norm_(_with_grads(grads), 0.5)
        assert [g._version for g in grads] == [v + 1 for v in versions]
    # what autograd has saved of a gradient is known to have changed
    w = torch.ones(4, device=dev, requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    later = (g * g).sum()
    clip_grad_norm_(_with_grads([g.detach()]), 0.5)
    with pytest.raises(RuntimeError, match='inplace'):
        later.backward()
    with torch.inference_mode():
        i = torch.ones(5, device=dev)
    p = torch.nn.Parameter(torch.ones(5, device=dev))
    with torch.inference_mode():
        p.grad = i
        clip_grad_norm_(p, 0.5)
        assert float(i[0]) < 0.23


# ---- strided gradients that share memory, and that only seem to ----------------------------------------------------------------------------

def test_strided_gradients_that_share_memory_are_refused(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    h = _values((60, 70), 3)
    d = h.to(dev)
    a = d[:, :11]
    for name, grads in {'the same view twice': [a, a], 'equal views': [d[:, :11], d[:, :11]], 'a buffer and its columns': [d, a], 'columns that overlap': [d[:, :12], d[:, 11:]],
                        'a row and columns': [d[7], d[:, 69:]]}.items():
        ps = _with_grads(grads)
        with pytest.raises(RuntimeError, match='share memory'):
            clip_grad_norm_(ps, 1e-3)
        with pytest.raises(RuntimeError, match='share memory'):
            clip_grad_norm_(ps[::-1], 1e-3)
        assert torch.equal(d.cpu(), h), name
    p = torch.nn.Parameter(torch.empty(60, 11, device=dev))
    p.grad = a
    with pytest.raises(RuntimeError, match='share memory'):
        clip_grad_norm_([p, p], 1e-3)


def test_strided_gradients_that_interleave_are_scaled(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    h = _values((6000,), 5)
    makers = {'rows that pass one another': lambda b: [b.as_strided((2, 3), (3, 2))],                         # offsets 0 2 4 3 5 7
              'every third': lambda b: [b[0::3], b[1::3], b[2::3]],
              'a row between columns': lambda b: [b.view(60, 100)[:, :50], b.view(60, 100)[31, 50:], b.view(60, 100)[32:, 50:]]}
    for name, f in makers.items():
        d = h.to(dev)
        grads, want = f(d), f(h.double())
        norm = math.sqrt(sum(float((x * x).sum()) for x in want))
        got = clip_grad_norm_(_with_grads(grads), 0.5 * norm)
        assert abs(got.item() - norm) <= (2.0 ** -24 + 1e-10) * norm
        factor = 0.5 * norm / (norm + 1e-6)
        for g, x in zip(grads, want):
            assert bool(((g.cpu().double() - x * factor).abs() <= 2.0 ** -23 * (x * factor).abs()).all()), name
        rest = torch.ones(6000, dtype=torch.bool)
        for x in f(rest):
            x.fill_(False)
        assert torch.equal(d.cpu()[rest], h[rest]), name


def test_bounds_on_the_host_are_refused(dev):
    bound = torch.tensor([0.0, 0.1, 0.2])
    for c in ((None, None, bound), (None, None, None, bound.double().to(dev))):
        with pytest.raises(ValueError, match='bounds of parameter 0'):
            _adam([torch.zeros(5, 3)], dev, clamps=[c])
    _adam([torch.zeros(5, 3)], dev, clamps=[(None, None, bound.to(dev))])


def test_parameters_of_a_subclass(dev):
    """Asking whether a subclass is a tensor may run Python code."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm

    class Mine(torch.Tensor):
        pass
    p = torch.nn.Parameter(torch.zeros(5, device=dev))
    q = torch.zeros(3, device=dev).as_subclass(Mine).requires_grad_(True)
    p.grad, q.grad = torch.full((5,), 2.0, device=dev), torch.full((3,), 2.0, device=dev)
    assert float(grad_norm([p.grad, q.grad])) == float(clip_grad_norm_([p, q], 1.0)) == torch.tensor(32.0).sqrt().item()
    assert abs(float(q.grad[0]) - 2.0 / math.sqrt(32.0)) < 1e-6
    with pytest.raises(TypeError, match='int'):
        clip_grad_norm_([p, q, 1], 1.0)


@pytest.mark.parametrize('order', ['as they lie', 'backwards', 'shuffled'])
def test_the_order_of_a_list_does_not_matter(order, dev):
    """Neighbours, gaps and tensors of their own, in any order: scaled once, versions raised once, and refused with one of them twice."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    buf = torch.zeros(40000, device=dev)
    sizes = [1, 700, 0, 3000, 5, 64, 9000]
    at, grads = 3, []
    for k, n in enumerate(sizes):
        grads.append(buf[at:at + n])
        at += n + (k % 2) * 7
    grads += [torch.zeros(n, device=dev) for n in (11, 30000, 2)]
    if order != 'as they lie':
        grads.sort(key=lambda g: -g.data_ptr())
    if order == 'shuffled':
        grads = grads[1::2] + grads[::2]
    host = [_values(g.shape, 3 + k) for k, g in enumerate(grads)]
    for g, h in zip(grads, host):
        g.copy_(h)
    norm = math.sqrt(sum(float((h.double() ** 2).sum()) for h in host))
    with pytest.raises(RuntimeError, match='share memory'):
        clip_grad_norm_(_with_grads(grads + [grads[-1] if grads[-1].numel() else grads[0]]), 0.5 * norm)
    ps, versions = _with_grads(grads), {id(g): g._version for g in grads if g.untyped_storage().data_ptr() != buf.untyped_storage().data_ptr()}
    got = clip_grad_norm_(ps, 0.5 * norm)
    assert abs(got.item() - norm) <= (2.0 ** -24 + 1e-10) * norm
    factor = 0.5 * norm / (norm + 1e-6)
    for g, h in zip(grads, host):
        x = h.double() * factor
        assert bool(((g.cpu().double() - x).abs() <= 2.0 ** -23 * x.abs() + 2.0 ** -150).all())
        assert g._version == versions.get(id(g), g._version - 1) + 1
