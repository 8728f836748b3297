"""The global gradient norm, clipping by it and the clipped Adam step (csrc/gradnorm.hip, optim.py) against their formulas in 64 bits.

Tolerances.  The norm is a sum in fp64 (its own error is below 1e-12 here) rounded once to fp32: 2^-24 relative.  The factor is rounded once
to fp32 and the product once to fp32: 2^-23 for an fp32 gradient, plus half a step of the type for the others (bf16 2^-8, fp16 2^-11); values
below the smallest normal number are off by half of the smallest subnormal instead."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SUBNORMAL = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}
NORM_TOL = 2.0 ** -24 + 1e-10


def norm64(tensors, p, scales=None):
    parts = []
    for k, t in enumerate(tensors):
        x = t.detach().cpu().double().reshape(-1).abs() * (abs(scales[k]) if scales is not None else 1.0)
        if x.numel():
            parts.append(x)
    if not parts:
        return 0.0
    x = torch.cat(parts)
    return float(x.max() if p == math.inf else x.sum() if p == 1.0 else (x * x).sum().sqrt())


def factor64(norm, max_norm):
    return 1.0 if math.isinf(max_norm) else min(1.0, max_norm / (norm + 1e-6))


def close(got, want, tol, what=''):
    assert abs(got - want) <= tol * abs(want), (what, got, want)


def assert_scaled(got, before, factor, what=''):
    """got = before * factor, each element to the roundings of its type."""
    g, b = got.detach().cpu().double(), before.detach().cpu().double() * factor
    tol = (2.0 ** -23 + HALF_STEP[got.dtype]) * b.abs() + SUBNORMAL[got.dtype] / 2 + 2.0 ** -150
    bad = (g - b).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float((g - b).abs().max()))


def values(n, seed, dtype, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, generator=gen).pow(3) * scale).to(dtype)


def params_of(grads):
    ps = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


LISTS = {
    'one': [1],
    'many empties': [0] * 12,
    'empties behind a full table': [3] * 160 + [0] * 300,
    'one behind a full table and empties': [3] * 160 + [0] * 300 + [5],
    'empty': [0],
    'empties between': [0, 5, 0, 0, 70000, 0],
    'around a vector': [2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33],
    'around a chunk': [4095, 4096, 4097, 8191, 8192, 8193, 16383, 16385],
    'around an unrolled round': [2047, 2048, 2049, 6144, 6145, 8190],
    'full table': [37] * 160,
    'over the table': [37] * 161,
    'three tables': [(k * 37) % 101 for k in range(400)],
    'more chunks than workgroups': [5000001, 3, 4200000, 1],
    'long and short': [1] * 90 + [2500000] + [2] * 90,
}


@pytest.mark.parametrize('p', [2.0, 1.0, math.inf], ids=['two', 'one', 'max'])
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('name', sorted(LISTS))
def test_norm_and_clip_of_lists(name, dtype, p, dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    host = [values(n, 17 * k + n, dtype) for k, n in enumerate(LISTS[name])]
    grads = [h.to(dev) for h in host]
    want = norm64(host, p)
    got = grad_norm(grads, norm_type=p)
    assert got.shape == () and got.dtype == F32 and got.device == grads[0].device
    close(float(got), want, NORM_TOL, 'norm')
    for h, g in zip(host, grads):
        assert torch.equal(h, g.cpu())
    max_norm = 0.3 * want if want else 1.0
    norm = clip_grad_norm_(params_of(grads), max_norm, norm_type=p)
    assert norm.item() == got.item()                                # the same sums in the same order
    for h, g in zip(host, grads):
        assert_scaled(g, h, factor64(want, max_norm), name)


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('lead', [0, 1, 3, 5])
def test_views_of_a_buffer_at_odd_places(lead, dtype, dev):
    """Adjacent views (one entry of the table), then views with gaps; what lies around and between them stays as it was."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    sizes = [7, 1, 0, 12345, 4096, 3, 100001]
    for gap in (0, 1, 6):
        buf = torch.full((lead + sum(sizes) + gap * len(sizes) + 9,), 0.125, dtype=dtype)
        at, where = lead, []
        for k, n in enumerate(sizes):
            buf[at:at + n] = values(n, 5 * k + gap, dtype)
            where.append((at, n))
            at += n + gap
        d = buf.to(dev)
        grads = [d[a:a + n] for a, n in where]
        want = norm64([buf[a:a + n] for a, n in where], 2.0)
        close(float(grad_norm(grads)), want, NORM_TOL)
        clip_grad_norm_(params_of(grads), 0.5 * want)
        inside = torch.zeros(buf.numel(), dtype=torch.bool)
        for a, n in where:
            inside[a:a + n] = True
        assert torch.equal(d.cpu()[~inside], buf[~inside])
        assert_scaled(d.cpu()[inside], buf[inside], factor64(want, 0.5 * want), (lead, gap))


def test_mixed_types_and_scales(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    host = [values(1001, 1, F32), values(70001, 2, BF16), values(333, 3, F16), values(5, 4, F32), values(40000, 5, BF16)]
    scales = [64.0, -0.5, 0.0, 1.0, 0.09999999403953552]            # (the last: an fp32 number)
    grads = [h.to(dev) for h in host]
    for p in (2.0, 1.0, math.inf):
        close(float(grad_norm(grads, norm_type=p, scales=scales)), norm64(host, p, scales), NORM_TOL, p)
    want = norm64(host, 2.0)
    clip_grad_norm_(params_of(grads), 1.5)
    for g, h in zip(grads, host):
        assert_scaled(g, h, factor64(want, 1.5))
    with pytest.raises(ValueError, match='scales'):
        grad_norm(grads, scales=[1.0])


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['fp32', 'bf16', 'fp16'])
def test_strided_gradients(dtype, dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    base = values(6 * 70 * 90, 3, dtype).view(6, 70, 90)
    makers = {'permuted': lambda t: t.permute(2, 0, 1), 'columns': lambda t: t[:, :, 5:50], 'every other': lambda t: t[::2, 1::3], 'transposed slice': lambda t: t[:, 3:40].transpose(0, 2)}
    for name, f in makers.items():
        d = base.to(dev)
        g, h = f(d), f(base)
        want = norm64([h], 2.0)
        close(float(grad_norm([g])), want, NORM_TOL, name)
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=dtype, device=dev))
        p.grad = g
        clip_grad_norm_(p, 0.25 * want)
        assert_scaled(g, h, factor64(want, 0.25 * want), name)
        rest = torch.ones_like(base, dtype=torch.bool)
        f(rest).fill_(False)
        assert torch.equal(d.cpu()[rest], base[rest]), name
    e = values(1, 9, dtype).to(dev).expand(1000)
    close(float(grad_norm([e])), float(e[0]) .__abs__() * math.sqrt(1000.0), NORM_TOL + 1e-15)
    p = torch.nn.Parameter(torch.empty(1000, dtype=dtype, device=dev))
    p.grad = e
    with pytest.raises(RuntimeError, match='expanded'):
        clip_grad_norm_(p, 0.1)


def test_values_whose_squares_leave_fp32(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    for v in (3e30, 1e-30, 2.0 ** -149):
        h = torch.full((1000,), v)
        for p in (2.0, 1.0, math.inf):
            close(float(grad_norm([h.to(dev)], norm_type=p)), norm64([h], p), NORM_TOL + 2.0 ** -150 / norm64([h], p), (v, p))      # (a subnormal norm: half of the smallest)
    h = torch.tensor([2.0 ** -14, 2.0 ** -24, 65504.0], dtype=F16)
    close(float(grad_norm([h.to(dev)])), norm64([h], 2.0), NORM_TOL)
    g = torch.full((512,), 3e38, device=dev)                           # the norm is over fp32's range: infinite in fp32, finite where the factor is made
    want = norm64([g], 2.0)
    norm = clip_grad_norm_(params_of([g]), 1e6)                        # (a factor of 1.5e-34: still a normal number)
    assert math.isinf(float(norm))
    assert_scaled(g, torch.full((512,), 3e38), factor64(want, 1e6))


def test_values_that_are_not_finite(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    for dtype in (F32, BF16, F16):
        for bad, at in ((math.nan, 0), (math.nan, 9999), (math.inf, 5000), (-math.inf, 3)):
            h = values(10000, 1, dtype)
            h[at] = bad
            for p in (2.0, 1.0, math.inf):
                n = float(grad_norm([values(77, 2, dtype).to(dev), h.to(dev), values(8, 3, dtype).to(dev)], norm_type=p))
                assert math.isnan(n) if math.isnan(bad) else n == math.inf, (dtype, bad, p, n)
                g = h.to(dev)
                with pytest.raises(RuntimeError, match='norm of the gradients'):
                    clip_grad_norm_(params_of([g]), 1.0, norm_type=p, error_if_nonfinite=True)
                assert torch.equal(torch.nan_to_num(g.cpu(), nan=7.0), torch.nan_to_num(h, nan=7.0))       # untouched
                clip_grad_norm_(params_of([g]), 1.0, norm_type=p)
                if math.isnan(bad):
                    assert bool(g.isnan().all())                        # as torch.nn.utils does
                else:
                    keep = torch.arange(10000) != at
                    assert bool(g[at].isnan()) and bool((g.cpu()[keep] == 0).all())
    # a NaN next to an infinity is a NaN whichever comes first
    for pair in ((math.nan, math.inf), (math.inf, math.nan)):
        assert math.isnan(float(grad_norm([torch.tensor([v], device=dev) for v in pair], norm_type=math.inf)))


def test_below_the_threshold_nothing_changes(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    for dtype in (F32, BF16, F16):
        h = [values(50001, 4, dtype), values(3, 5, dtype)]
        for max_norm in (2.0 * norm64(h, 2.0), math.inf):
            g = [x.to(dev) for x in h]
            clip_grad_norm_(params_of(g), max_norm)
            assert all(torch.equal(a.cpu(), b) for a, b in zip(g, h))
    g = values(1000, 6, F32).to(dev)
    clip_grad_norm_(params_of([g]), 0.0)                                # a threshold of zero
    assert bool((g == 0).all())
    z = torch.zeros(1000, device=dev)
    assert clip_grad_norm_(params_of([z]), 0.0).item() == 0.0 and bool((z == 0).all())
    inf = torch.tensor([math.inf, 1.0], device=dev)
    assert math.isinf(clip_grad_norm_(params_of([inf]), math.inf).item()) and inf.tolist() == [math.inf, 1.0]      # only measured


def test_parameters_without_gradients_duplicates_and_versions(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    a, b, c = (torch.nn.Parameter(torch.ones(5, device=dev)) for _ in range(3))
    a.grad, c.grad = torch.full((5,), 3.0, device=dev), torch.full((5,), 4.0, device=dev)
    version = a.grad._version
    n = clip_grad_norm_((p for p in (a, b, c)), 1.0)
    close(n.item(), math.sqrt(125.0), NORM_TOL)
    assert b.grad is None and a.grad._version > version
    with pytest.raises(RuntimeError, match='share memory'):
        clip_grad_norm_([a, a], 1.0)
    b.grad = c.grad[:5]
    with pytest.raises(RuntimeError, match='share memory'):
        clip_grad_norm_([a, b, c], 1.0)
    if torch.cuda.device_count() == 1:
        b.grad = None
        d = torch.nn.Parameter(torch.ones(5))
        d.grad = torch.ones(5)
        with pytest.raises(RuntimeError, match='GPU'):
            clip_grad_norm_([a, d], 1.0)


def test_the_same_call_twice_gives_the_same_bits(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    h = [values(3000001, 1, F32), values(70003, 2, BF16), values(12, 3, F16)]
    runs = []
    for _ in range(3):
        g = [x.to(dev) for x in h]
        runs.append([clip_grad_norm_(params_of(g), 1.0)] + g)
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_on_another_stream(dev):
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    h = values(2000003, 8, F32)
    want = norm64([h], 2.0)
    s = torch.cuda.Stream()
    g = h.to(dev)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g.mul_(2.0)
        norm = clip_grad_norm_(params_of([g]), 1.0)
        g.mul_(0.5)
    torch.cuda.current_stream().wait_stream(s)
    close(norm.item(), 2.0 * want, NORM_TOL)
    assert_scaled(g, h, factor64(2.0 * want, 1.0))


def test_many_norms_at_once_on_several_streams(dev):
    """Norms that overlap on the device: each waits for its own workgroups only and has a workspace of its own."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    sizes = [(5000001, F32), (70001, BF16), (1200007, F16), (333, F32)]
    host = [[values(n, 50 * k + i, t) for i, (n, t) in enumerate(sizes)] for k in range(4)]
    want = [norm64(h, 2.0) for h in host]
    grads = [[x.to(dev) for x in h] for h in host]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = [[] for _ in range(4)]
    for _ in range(30):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(grad_norm(grads[k]))
                got[k].append(clip_grad_norm_(params_of(grads[k]), 2.0 * want[k]))        # (nothing to scale)
    torch.cuda.synchronize()
    for k in range(4):
        first = got[k][0].item()
        close(first, want[k], NORM_TOL, k)
        assert all(x.item() == first for x in got[k]), k


def test_two_captured_graphs_replayed_in_turn(dev):
    """Each graph owns its workspace; every replay sees the gradients of its moment, with eager calls in between."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    sets = [[torch.zeros(n, dtype=t, device=dev) for n, t in spec] for spec in ([(1000001, F32), (5, F32)], [(70001, BF16), (0, F16), (333, F16)] + [(3, F32)] * 170)]
    ps = [params_of(s) for s in sets]
    graphs, norms = [], []
    for p in ps:
        clip_grad_norm_(p, 1.0)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clip_grad_norm_(p, 1.0))
        graphs.append(g)
    with pytest.raises(RuntimeError, match='capture'):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            clip_grad_norm_(ps[0], 1.0, error_if_nonfinite=True)
    torch.cuda.synchronize()
    for it in range(4):
        hosts = []
        for k, s in enumerate(sets):
            h = [values(t.numel(), 100 * it + 10 * k + i, t.dtype, scale=10.0 ** (it - 2)) for i, t in enumerate(s)]
            hosts.append(h)
            for t, x in zip(s, h):
                t.copy_(x)
        eager = grad_norm(sets[it % 2])
        for g in (graphs if it % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        close(eager.item(), norm64(hosts[it % 2], 2.0), NORM_TOL)
        for h, s, n in zip(hosts, sets, norms):
            want = norm64(h, 2.0)
            close(n.item(), want, NORM_TOL, it)
            for x, t in zip(h, s):
                assert_scaled(t, x, factor64(want, 1.0), it)


def test_more_elements_than_32_bits_count(dev):
    """2^31 + 77 bf16 elements: every power of two of the sum is exact, the last elements are counted and scaled."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    n = (1 << 31) + 77
    g = torch.full((n,), 2.0 ** -10, dtype=BF16, device=dev)
    g[-1] = 1024.0
    want = math.sqrt((n - 1) * 2.0 ** -20 + 2.0 ** 20)
    norm = clip_grad_norm_(params_of([g]), 0.5 * want)
    close(norm.item(), want, NORM_TOL)
    f = factor64(want, 0.5 * want)
    close(float(g[-1]), 1024.0 * f, 2.0 ** -8 + 2.0 ** -23)
    lo, hi = float(g[:-1].min()), float(g[:-1].max())
    assert lo == hi
    close(lo, 2.0 ** -10 * f, 2.0 ** -8 + 2.0 ** -23)


@pytest.mark.parametrize('p', [2.0, 1.0, math.inf], ids=['two', 'one', 'max'])
def test_lists_longer_than_the_cache(p, dev):
    """Over 160 MB: streamed in several rounds of runs, the end kept in the cache, scaled from the end by larger workgroups.  Three tables,
    odd lengths, odd places, all types; the reference sums in fp64 on the GPU."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_, grad_norm
    gen = torch.Generator(device=dev).manual_seed(3)
    spec = [(30000001, F32), (7, F16), (50000003, BF16)] + [(1 + 13 * k, (F32, BF16, F16)[k % 3]) for k in range(400)] + [(20000005, F16), (3000001, F32)]
    grads, kept = [], []
    for k, (n, t) in enumerate(spec):
        b = torch.empty(n + 5, dtype=t, device=dev)
        b.normal_(generator=gen)
        grads.append(b[k % 4:k % 4 + n])
        kept.append((b, b.clone()))
    before = [g.clone() for g in grads]
    big = lambda g: g.double().abs()
    if p == math.inf:
        want = max(float(big(g).max()) for g in grads)
    else:
        want = sum(float((big(g) ** p).sum()) for g in grads) ** (1.0 / p)
    n = grad_norm(grads, norm_type=p)
    close(float(n), want, NORM_TOL)
    m = clip_grad_norm_(params_of(grads), 0.37 * want, norm_type=p)
    assert m.item() == n.item()
    f = factor64(want, 0.37 * want)
    for k, (g, b, (buf, old)) in enumerate(zip(grads, before, kept)):
        tol = (2.0 ** -23 + HALF_STEP[g.dtype]) * big(b) * f + SUBNORMAL[g.dtype] / 2 + 2.0 ** -150
        assert not bool(((g.double() - b.double() * f).abs() > tol).any()), k
        assert torch.equal(buf[:k % 4], old[:k % 4]) and torch.equal(buf[k % 4 + g.numel():], old[k % 4 + g.numel():]), k


def test_more_launches_than_the_reverse_order_remembers(dev):
    """65 tables and more: the ones behind the 64th are scaled in their own order, each tensor once."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    count = 160 * 66 + 7
    buf = values(count * 4, 11, F32)                                       # every fourth element: no two are neighbours
    d = buf.to(dev)
    grads = list(d.view(count, 4)[:, :1].unbind(0))
    h = buf.view(count, 4)[:, 0]
    want = norm64([h], 2.0)
    n = clip_grad_norm_(params_of(grads), 0.5 * want)
    close(n.item(), want, NORM_TOL)
    assert_scaled(d.view(count, 4)[:, 0], h, factor64(want, 0.5 * want))
    assert torch.equal(d.view(count, 4)[:, 1:].cpu(), buf.view(count, 4)[:, 1:])


def test_columns_of_one_buffer(dev):
    """Gradients that interleave in memory: each is scaled through its own copy, once."""
    from nvdiffrecmc_amd.optim import clip_grad_norm_
    h = values(60 * 70, 12, F32).view(60, 70)
    d = h.to(dev)
    want = norm64([h], 2.0)
    n = clip_grad_norm_(params_of([d[:, :11], d[:, 11:40], d[:, 40:]]), 0.5 * want)
    close(n.item(), want, NORM_TOL)
    assert_scaled(d, h, factor64(want, 0.5 * want))
    p = torch.nn.Parameter(torch.empty(10, 8, device=dev))
    p.grad = d.view(-1).as_strided((10, 8), (5, 1))                        # rows that overlap
    with pytest.raises(RuntimeError, match='share memory'):
        clip_grad_norm_(p, 1e-3)


# ---- the clipped step ------------------------------------------------------------------------------------------------------------------

def _adam(shapes, dev, seed, **kw):
    from nvdiffrecmc_amd.optim import FusedAdam
    gen = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.rand(s, generator=gen).to(dev)) for s in shapes]
    return FusedAdam(ps, lr=0.01, **kw)


def _grads(shapes, seed, scale=1.0):
    return [values(math.prod(s), 7 * seed + i, F32, scale).view(s) for i, s in enumerate(shapes)]


SHAPES = [(33, 33, 3), (17, 17, 3), (16, 16, 3), (1001, 3)]
SETUP = dict(grad_scales=[1.0, 1.0, 64.0, 1.0], lr_scales=[1.0, 1.0, 3.0, 0.5], clamps=[(0.0, 1.0), (-1.0, 1.0), (0.01, None), None], normalize3=[False, True, False, False])


@pytest.mark.parametrize('norm_type', [2.0, 1.0, math.inf], ids=['two', 'one', 'max'])
@pytest.mark.parametrize('sparse', [False, True], ids=['dense', 'tiles'])
def test_clipped_step_is_the_formula(sparse, norm_type, dev):
    """Five steps in fp64: the effective gradient g * grad_scale * grad_mult, its norm, Adam, clamps, renormalised normals.  A moment is off by
    a few fp32 roundings a step (5 * 4 * 2^-24); a parameter moves by lr * m / (sqrt(v) + eps), whose quotient's error is that of its
    parts (another 8 roundings) on a step of at most lr * lr_scale * 3.2 (|m| / sqrt(v) after 5 steps is at most (1 - b1^5) / (1 - b1) * ... < 3.2
    times its bias corrections), and is rounded itself."""
    opt = _adam(SHAPES, dev, 1, max_norm=2.0, norm_type=norm_type, sparse=[sparse, sparse, False, False], **SETUP)
    p = [q.detach().cpu().double() for q in opt.params]
    m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
    mult = 0.125
    for t in range(1, 6):
        h = _grads(SHAPES, t, scale=1.0 if t != 3 else 1e-6)                # the third lies below the threshold
        for q, g in zip(opt.params, h):
            q.grad = g.to(dev)
        opt.step(grad_mult=mult)
        eff = [g.double() * k * mult for g, k in zip(h, SETUP['grad_scales'])]
        want = norm64(eff, norm_type)
        close(opt.grad_norm.item(), want, NORM_TOL, t)
        f = factor64(want, 2.0)
        assert (f == 1.0) == (t == 3)
        for i in range(len(p)):
            g = eff[i] * f
            m[i] = 0.9 * m[i] + 0.1 * g
            v[i] = 0.999 * v[i] + 0.001 * g * g
            step = 0.01 * SETUP['lr_scales'][i] / (1 - 0.9 ** t)
            x = p[i] - step * m[i] / (v[i].sqrt() / math.sqrt(1 - 0.999 ** t) + 1e-8)
            c = SETUP['clamps'][i]
            if c is not None:
                x = x.clamp(c[0], c[1])
            if SETUP['normalize3'][i]:
                x = x / x.square().sum(-1, keepdim=True).clamp(min=1e-20).sqrt()
            p[i] = x
            assert torch.equal(opt.params[i].grad.cpu(), h[i])              # the gradients stay
    for i in range(len(p)):
        top = m[i].abs().max()
        assert float((opt.exp_avg[i].cpu().double() - m[i]).abs().max()) <= 20 * 2.0 ** -24 * float(top)
        assert float(((opt.exp_avg_sq[i].cpu().double() - v[i]).abs() / v[i].max()).max()) <= 40 * 2.0 ** -24
        # the quotient's relative error grows where the moment cancels: compared to the largest step an element can take
        assert float((opt.params[i].detach().cpu().double() - p[i]).abs().max()) <= 5 * (28 * 2.0 ** -24 * 3.2 * 0.03 * 4 + 2.0 ** -23), i
    assert opt.step_count == 5


def test_clipped_step_equals_scaled_gradients(dev):
    """max_norm is the plain step on gradients scaled by the factor: bit for bit with a factor that is a power of two."""
    a, b = _adam(SHAPES, dev, 2, max_norm=1.0, **SETUP), _adam(SHAPES, dev, 2, **SETUP)
    h = _grads(SHAPES, 3)
    norm = norm64([g.double() * k for g, k in zip(h, SETUP['grad_scales'])], 2.0)
    a.max_norm = 0.25 * (norm + 1e-6)                                       # a factor of 0.25 but for the last bit of the norm
    for t in range(3):
        for x, y, g in zip(a.params, b.params, h):
            x.grad, y.grad = g.to(dev), (g * 0.25).to(dev)
        a.step()
        assert a._norm_work.view(F32)[0].item() == 0.25                     # (what the step begins with: factor, step size, ...)
        b.step()
    for i in range(len(SHAPES)):
        assert torch.equal(a.params[i], b.params[i]) and torch.equal(a.exp_avg[i], b.exp_avg[i]) and torch.equal(a.exp_avg_sq[i], b.exp_avg_sq[i]), i
    # an infinite threshold measures and changes nothing
    c, d = _adam(SHAPES, dev, 2, max_norm=math.inf, **SETUP), _adam(SHAPES, dev, 2, **SETUP)
    assert c.grad_norm.item() == 0.0 and d.grad_norm is None
    for x, y, g in zip(c.params, d.params, h):
        x.grad, y.grad = g.to(dev), g.to(dev)
    c.step(); d.step()
    close(c.grad_norm.item(), norm, NORM_TOL)
    assert all(torch.equal(x, y) for x, y in zip(c.params, d.params))


def test_clipped_step_in_subsets_and_frozen_tensors(dev):
    a, b = _adam(SHAPES, dev, 4, max_norm=1.0, **SETUP), _adam(SHAPES, dev, 4, max_norm=1.0, **SETUP)
    for opt in (a, b):
        opt.lr_scales[1] = 0.0                                              # frozen: no update, and not in the norm
    for t in range(3):
        h = _grads(SHAPES, t)
        for x, y, g in zip(a.params, b.params, h):
            x.grad, y.grad = g.to(dev), g.to(dev)
        a.step()
        with pytest.raises(RuntimeError, match='measure_norm'):
            b.step(subset=[2, 3], advance=False)
        b.measure_norm()
        b.step(subset=[2, 3], advance=False)
        b.step(subset=[0, 1], advance=True)
        want = norm64([h[0], h[2] * 64.0, h[3]], 2.0)
        close(a.grad_norm.item(), want, NORM_TOL)
        assert a.grad_norm.item() == b.grad_norm.item()
    for x, y in zip(a.params, b.params):
        assert torch.equal(x, y)
    assert a.step_count == b.step_count == 3
    with pytest.raises(RuntimeError, match='no max_norm'):
        _adam(SHAPES, dev, 1).measure_norm()
    a.params[0].grad = None
    with pytest.raises(RuntimeError, match='parameter 0 has no gradient'):
        a.step()
    with pytest.raises(ValueError, match='max_norm'):
        _adam(SHAPES, dev, 1, max_norm=-1.0)
    with pytest.raises(ValueError, match='norm_type'):
        _adam(SHAPES, dev, 1, max_norm=1.0, norm_type=0.5)


def test_clipped_step_zeroes_consumed_gradients(dev):
    """zero_grad with the tile-sparse path: the norm has read them before."""
    opt = _adam([(64, 64, 3), (8, 3)], dev, 5, max_norm=1.0, sparse=[True, False], zero_grad=[True, False])
    for t in range(3):
        h = _grads([(64, 64, 3), (8, 3)], t)
        h[0].view(-1, 192)[::3] = 0.0                                       # tiles without a gradient
        buf = h[0].to(dev)
        opt.params[0].grad, opt.params[1].grad = buf, h[1].to(dev)
        opt.step()
        close(opt.grad_norm.item(), norm64(h, 2.0), NORM_TOL)
        assert bool((buf == 0).all()) and torch.equal(opt.params[1].grad.cpu(), h[1])


def test_clipped_step_captured(dev):
    a, b = _adam(SHAPES, dev, 6, max_norm=1.0, **SETUP), _adam(SHAPES, dev, 6, max_norm=1.0, **SETUP)
    for opt in (a, b):
        for q in opt.params:
            q.grad = torch.zeros_like(q)
    b.step(); a.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for t in range(4):
        for x, y, g in zip(a.params, b.params, _grads(SHAPES, t, scale=10.0 ** -t)):
            x.grad.copy_(g); y.grad.copy_(g)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert a.grad_norm.item() == b.grad_norm.item()
        for x, y in zip(a.params, b.params):
            assert torch.equal(x, y), t
    assert a.step_count == b.step_count == 5


def test_gradients_at_odd_places_update_alike(dev):
    """Gradients inside a bucket begin anywhere: the same parameters and moments as from gradients of their own, bit for bit, by every path
    (plain, normal map, sparse with and without zeroing), at lengths that are no multiple of four."""
    shapes = [(1001, 3), (13, 7, 3), (37, 3), (1,), (2053,), (65, 3)]
    kw = dict(max_norm=1.0, normalize3=[False, True, True, False, False, False], sparse=[True, False, True, False, False, True], zero_grad=[True, False, False, False, False, True],
              clamps=[(0.0, 1.0, torch.tensor([0.1, 0.0, 0.2], device=dev)), (-1.0, 1.0), None, (None, 0.7), (0.01, None), (None, None, None, torch.tensor([0.5, 0.6], device=dev))])
    a, b = _adam(shapes, dev, 7, **kw), _adam(shapes, dev, 7, **kw)
    buf = torch.full((20000,), 9.0, device=dev)
    for t in range(3):
        h = _grads(shapes, t)
        h[0][64:128] = 0.0                                                  # a tile without a gradient
        at = 3
        for x, y, g in zip(a.params, b.params, h):
            x.grad = g.to(dev)
            y.grad = buf[at:at + g.numel()].view(g.shape)
            y.grad.copy_(g)
            at += g.numel() + 1
        a.step()
        b.step()
        assert a.grad_norm.item() == b.grad_norm.item()
        for i in range(len(shapes)):
            assert torch.equal(a.params[i], b.params[i]) and torch.equal(a.exp_avg[i], b.exp_avg[i]) and torch.equal(a.exp_avg_sq[i], b.exp_avg_sq[i]), (t, i)
            assert torch.equal(a.params[i].grad, b.params[i].grad), (t, i)
            assert bool((b.params[i].grad == 0).all()) == kw['zero_grad'][i], (t, i)
            if a.active[i] is not None:
                assert torch.equal(a.active[i], b.active[i])
    gaps = torch.ones(20000, dtype=torch.bool)
    at = 3
    for s in shapes:
        gaps[at:at + math.prod(s)] = False
        at += math.prod(s) + 1
    assert bool((buf.cpu()[gaps] == 9.0).all())


def test_a_frozen_sparse_texture_only_loses_its_gradient(dev):
    opt = _adam([(40, 40, 3), (8, 3)], dev, 8, max_norm=1.0, sparse=[True, False], zero_grad=[True, False], lr_scales=[0.0, 1.0])
    h = _grads([(40, 40, 3), (8, 3)], 1)
    before = opt.params[0].detach().clone()
    for q, g in zip(opt.params, h):
        q.grad = g.to(dev)
    opt.step()
    close(opt.grad_norm.item(), norm64(h[1:], 2.0), NORM_TOL)
    assert torch.equal(opt.params[0], before) and bool((opt.params[0].grad == 0).all())
    assert bool((opt.exp_avg[0] == 0).all()) and bool((opt.active[0] == 0).all())


def test_a_step_longer_than_the_cache_is_the_same_step(dev):
    """7 M parameters at once (moments past the caches) and tensor by tensor (not): the same bits."""
    shapes = [(1201, 1203, 3), (1000, 1001, 3), (257, 3), (31, 33, 3)]
    kw = dict(max_norm=0.5, normalize3=[False, True, False, True], clamps=[(0.0, 1.0), (-1.0, 1.0), None, None])
    a, b = _adam(shapes, dev, 9, **kw), _adam(shapes, dev, 9, **kw)
    assert 28 * sum(p.numel() for p in a.params) > 160 << 20 > 28 * max(p.numel() for p in a.params)
    for t in range(2):
        for x, y, g in zip(a.params, b.params, _grads(shapes, t)):
            x.grad, y.grad = g.to(dev), g.to(dev)
        a.step()
        b.measure_norm()
        for i in range(4):
            b.step(subset=[i], advance=(i == 3))
        for i in range(4):
            assert torch.equal(a.params[i], b.params[i]) and torch.equal(a.exp_avg[i], b.exp_avg[i]) and torch.equal(a.exp_avg_sq[i], b.exp_avg_sq[i]), (t, i)


def test_the_same_tensor_twice_is_refused(dev):
    from nvdiffrecmc_amd.optim import FusedAdam
    opt = _adam(SHAPES, dev, 11, max_norm=1.0, **SETUP)
    for q, g in zip(opt.params, _grads(SHAPES, 1)):
        q.grad = g.to(dev)
    opt.measure_norm()
    with pytest.raises(RuntimeError, match='the same'):
        opt.step(subset=[1, 0, 1])
    opt.step(subset=[0, 1], advance=False)                                  # (a refused launch leaves the measured norm)
    if hasattr(opt.params[2], 'grad_dtype'):
        opt.params[2].grad = None
        opt.params[2].grad_dtype = BF16
        opt.params[2].grad = torch.ones(SHAPES[2], dtype=BF16, device=dev)
        with pytest.raises(RuntimeError, match='float32'):
            opt.step(subset=[2, 3])
    p = torch.nn.Parameter(torch.ones(5, device=dev))
    p.grad = torch.ones(5, device=dev)
    for kw in ({}, {'max_norm': 1.0}):
        with pytest.raises(RuntimeError, match='the same'):
            FusedAdam([p, p], **kw).step()
    assert bool((p == 1).all())


def test_a_threshold_given_later(dev):
    a, b = _adam(SHAPES, dev, 10, **SETUP), _adam(SHAPES, dev, 10, max_norm=0.5, **SETUP)
    a.max_norm = 0.5
    for x, y, g in zip(a.params, b.params, _grads(SHAPES, 1)):
        x.grad, y.grad = g.to(dev), g.to(dev)
    a.step(); b.step()
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params)) and a.grad_norm.item() == b.grad_norm.item() > 0.5


# ---- together, as the iteration uses them -------------------------------------------------------------------------------------------------

def test_iteration_with_clipping_fused_and_composed_agree(dev):
    """DirectLightingStep(max_grad_norm): the clipped fused update against clip_grad_norm_ in front of torch.optim.Adam, same samples."""
    from nvdiffrecmc_amd.trainer import DirectLightingStep
    a = DirectLightingStep('bob', 96, 4, view=[1], device=dev, tex_res=128, fused=True, max_grad_norm=0.004)
    b = DirectLightingStep('bob', 96, 4, view=[1], device=dev, tex_res=128, fused=False, max_grad_norm=0.004)
    for k in range(6):
        la, lb = float(a.step().detach()), float(b.step().detach())
        assert abs(la - lb) <= 2e-5 * max(abs(lb), 1e-3), (k, la, lb)
        assert a.opt.grad_norm.item() > 0.004                               # it did clip
    # the first moments after the steps: those of clipped gradients on both sides.  What differs beyond fp32 rounding comes from the order of the atomic
    # sums of the light's and the textures' gradients, as in the test of the unclipped iteration, and is compared to the largest moment.
    for p, m, name in zip(b.params, a.opt.exp_avg, a.param_names):
        want = b.opt.state[p]['exp_avg']
        top = float(want.abs().max())
        off = ((m - want).abs() > 2e-3 * top).float().mean()
        assert top > 0 and float(off) <= 1e-2, (name, float(off))


@pytest.mark.parametrize('graph', [False, True], ids=['eager', 'hip_graphs'])
@pytest.mark.parametrize('geometry', [False, True], ids=['locked', 'geometry_trained'])
def test_several_rank_schedule_with_clipping_follows_the_plain_one(geometry, graph, dev):
    """The schedule of several ranks (chunked exchange, pipelined geometry stage) with ONE rank: the norm over all chunks, then all updates --
    the losses of the plain iteration with clipping."""
    from nvdiffrecmc_amd.trainer import DirectLightingStep
    kw = dict(view=[0, 2], device=dev, tex_res=128, max_grad_norm=0.004, use_graph=graph, optimize_geometry=geometry, perturb_pos=0.002 if geometry else 0.0, lr_pos=1e-5)
    a = DirectLightingStep('bob', 96, 4, **kw)
    b = DirectLightingStep('bob', 96, 4, force_exchange=True, **kw)
    for k in range(8):
        la, lb = float(a.step().detach()), float(b.step().detach())
        assert abs(la - lb) <= 2e-3 * abs(lb), (k, la, lb)                  # (the order of atomic sums, steps of Adam where a gradient is rounding noise)
        na, nb = a.opt.grad_norm.item(), b.opt.grad_norm.item()
        assert na > 0.004 and abs(na - nb) <= 2e-2 * na, (k, na, nb)
    b.finish()
    assert (a._graphs is not None) == graph and (b._graphs is not None) == graph
    assert a.opt.step_count == b.opt.step_count == 8


_TWO_RANKS = r'''
import json, os, sys, torch, torch.distributed as dist
sys.path.insert(0, %r)
from nvdiffrecmc_amd.trainer import DirectLightingStep
rank, world = int(os.environ['RANK']), int(os.environ['WORLD_SIZE'])
torch.cuda.set_device(0)
if world > 1:
    dist.init_process_group('gloo', rank=rank, world_size=world)
per = 4 // world
mine = list(range(rank * per, (rank + 1) * per))
st = DirectLightingStep('bob', 96, 4, view=mine, n_views=4, device='cuda:0', lr=0.03, tex_res=512, pixel_index_offset=mine[0] * 96 * 96,
                        use_graph=os.environ['USE_GRAPH'] == '1', exchange_mode=os.environ['EXCHANGE'], max_grad_norm=0.002)
losses, norms = [], []
for it in range(8):
    losses.append(float(st.step(world).detach()))
    norms.append(st.opt.grad_norm.item())
st.finish()
out = {'rank': rank, 'losses': losses, 'norms': norms, 'steps': st.opt.step_count, 'sums': [float(p.detach().double().sum()) for p in st.params]}
print('RESULT ' + json.dumps(out), flush=True)
if world > 1:
    dist.barrier()
    dist.destroy_process_group()
'''


@pytest.mark.parametrize('graph,exchange', [('0', 'dense'), ('1', 'dense'), ('1', 'sparse')], ids=['eager', 'hip_graphs', 'hip_graphs_sparse'])
def test_two_ranks_clip_by_the_norm_of_the_batch(graph, exchange, dev):
    """Four views on two ranks: the norm is that of the averaged gradients, the same on both, and the run follows the one-rank run (to the
    tolerances of the test of the unclipped schedule; the norm, a sum of squares of such gradients, to 1e-2)."""
    import json
    import os
    import socket
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

    def run(world, rank, port):
        env = dict(os.environ, MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), USE_GRAPH=graph, EXCHANGE=exchange)
        return subprocess.Popen([sys.executable, '-c', _TWO_RANKS % root], env=env, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, cwd=root)

    def result(p):
        out, err = p.communicate(timeout=100)
        assert p.returncode == 0, out[-2000:] + err[-3000:]
        return json.loads([line for line in out.splitlines() if line.startswith('RESULT ')][-1][7:])

    def port():
        with socket.socket() as s:
            s.bind(('127.0.0.1', 0))
            return s.getsockname()[1]
    one = result(run(1, 0, port()))
    at = port()
    two = sorted((result(p) for p in [run(2, r, at) for r in range(2)]), key=lambda d: d['rank'])
    assert one['steps'] == two[0]['steps'] == two[1]['steps'] == 8
    assert two[0]['norms'] == two[1]['norms']
    for it in range(8):
        pair = 0.5 * (two[0]['losses'][it] + two[1]['losses'][it])
        assert abs(pair - one['losses'][it]) <= 2e-4 * abs(one['losses'][it]), (it, pair, one['losses'][it])
        assert one['norms'][it] > 0.002 and abs(two[0]['norms'][it] - one['norms'][it]) <= 1e-2 * one['norms'][it], (it, two[0]['norms'][it], one['norms'][it])
    for a, b, c in zip(two[0]['sums'], two[1]['sums'], one['sums']):
        assert abs(a - b) <= 1e-9 * abs(a) and abs(a - c) <= 1e-4 * abs(c)
