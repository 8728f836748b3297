"""What the gradient norm, the clipping and the clipped Adam step refuse, and what they do without a launch (no GPU needed)."""
import array
import ctypes
import math

import pytest
import torch

from nvdiffrecmc_amd import _lib, optim


def _param(grad):
    p = torch.nn.Parameter(torch.zeros(grad.shape, dtype=grad.dtype))
    p.grad = grad
    return p


def test_python_refusals():
    x = torch.zeros(3)
    for call in (lambda t, **k: optim.grad_norm([t], **k), lambda t, **k: optim.clip_grad_norm_([_param(t)], 1.0, **k)):
        with pytest.raises(RuntimeError, match='GPU'):
            call(x)
        with pytest.raises(ValueError, match='float64'):
            call(x.double())
        for p in (0.0, 3.0, -math.inf, math.nan):
            with pytest.raises(ValueError, match='norm_type'):
                call(x, norm_type=p)
    with pytest.raises(TypeError, match='grad_norm.*float'):
        optim.grad_norm([1.0])
    with pytest.raises(TypeError, match='clip_grad_norm_.*str'):
        optim.clip_grad_norm_(['w'], 1.0)
    with pytest.raises(RuntimeError):
        optim.grad_norm([torch.eye(3).to_sparse()])
    for m in (-1.0, math.nan, -math.inf):
        with pytest.raises(ValueError, match='max_norm'):
            optim.clip_grad_norm_([_param(x)], m)


def test_nothing_to_do():
    assert optim.grad_norm([]).item() == 0.0
    assert optim.clip_grad_norm_([], 1.0).item() == 0.0
    assert optim.clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0).item() == 0.0          # no gradient
    assert optim.clip_grad_norm_(torch.nn.Parameter(torch.ones(3)), 1.0).item() == 0.0
    assert optim.clip_grad_norm_((p for p in ()), 1.0).item() == 0.0


# ---- the C entries refuse before anything is launched -----------------------------------------------------------------------------------

def _call(entry, data, n, types, max_norm=1.0, norm_type=2, workspace=None, out=True, scale=None):
    """The entry on host lists (addresses are never dereferenced: every call here is refused)."""
    lib = _lib.load()
    d, c = array.array('Q', data).tobytes(), array.array('q', n).tobytes()
    need = lib.nvdr_grad_norm_workspace(c, bytes(types), len(n), int(entry == 'nvdr_grad_clip'))
    ws = torch.empty(max(need, 1) if workspace is None else workspace, dtype=torch.float64)
    o = torch.empty(2)
    args = [d, c, bytes(types)] + ([scale] if entry == 'nvdr_grad_norm' else [])
    args += [len(n), norm_type, max_norm, ws.data_ptr(), ws.numel(), o.data_ptr() if out else None] + ([None] if entry == 'nvdr_grad_norm' else []) + [None]
    rc = getattr(lib, entry)(*args)
    return rc, (lib.nvdr_last_error() or b'').decode()


@pytest.mark.parametrize('entry', ['nvdr_grad_norm', 'nvdr_grad_clip'])
def test_entries_refuse_bad_arguments(entry):
    A = 1 << 20
    cases = [
        (dict(data=[A], n=[4], types=[3]), 'type'),
        (dict(data=[A], n=[-1], types=[0]), 'elements'),
        (dict(data=[A], n=[1 << 40], types=[0]), 'elements'),
        (dict(data=[0], n=[4], types=[0]), 'no memory'),
        (dict(data=[A + 2], n=[4], types=[0]), 'aligned'),
        (dict(data=[A + 1], n=[4], types=[1]), 'aligned'),
        (dict(data=[A], n=[1 << 30], types=[0], workspace=8), 'workspace'),
        (dict(data=[A] * 9, n=[0] * 9, types=[0] * 9, workspace=8), 'workspace'),
        (dict(data=[A], n=[4], types=[0], out=False), 'norm'),
        (dict(data=[A], n=[4], types=[0], max_norm=-1.0), 'max_norm'),
        (dict(data=[A], n=[4], types=[0], max_norm=math.nan), 'max_norm'),
        (dict(data=[A], n=[4], types=[0], norm_type=3), 'norm type'),
        (dict(data=[A], n=[4], types=[0], norm_type=-1), 'norm type'),
    ]
    for kw, word in cases:
        rc, msg = _call(entry, **kw)
        assert rc == -1 and word in msg, (kw, rc, msg)
    lib = _lib.load()
    ws, o = torch.empty(8192, dtype=torch.float64), torch.empty(2)
    tail = [2, 1.0, ws.data_ptr(), ws.numel(), o.data_ptr()] + ([None] if entry == 'nvdr_grad_norm' else []) + [None]
    assert getattr(lib, entry)(*([None, None, None] + ([None] if entry == 'nvdr_grad_norm' else []) + [1] + tail)) == -1
    assert getattr(lib, entry)(*([None, None, None] + ([None] if entry == 'nvdr_grad_norm' else []) + [-1] + tail)) == -1


def test_clip_refuses_gradients_that_share_memory():
    A = 1 << 20
    for data, n, types in (([A, A], [4, 4], [0, 0]), ([A + 64, A], [4, 17], [0, 0]), ([A, A + 8], [4, 4], [0, 0]), ([A + 4096, A + 6, A], [8, 8, 4], [0, 1, 1])):
        rc, msg = _call('nvdr_grad_clip', data, n, types)
        assert rc == -1 and 'share memory' in msg, (data, n, rc, msg)


def test_workspace_of_a_list():
    lib = _lib.load()

    def need(sizes, clip=0, t=0):
        return lib.nvdr_grad_norm_workspace(array.array('q', sizes).tobytes(), bytes([t]) * len(sizes), len(sizes), clip)
    assert need([1], clip=1) == need([0, 7], clip=1) == need([], clip=1) == 0          # clipped by one workgroup
    assert need([1 << 30]) == need([1]) >= need([]) > 512 and need([1 << 30], clip=1) == need([1 << 30])
    assert need([1] * 9, clip=1) > 512                                                  # many tensors are no short list
    assert need([1] * 160) == need([1] * 9) < need([1] * 161) < need([1] * 1000)
    assert need([1 << 16], clip=1, t=1) <= need([1 << 16], clip=1)


def test_a_missing_extension_is_an_error(monkeypatch):
    from nvdiffrecmc_amd import _build
    monkeypatch.setattr(_lib, '_gradops', None)
    monkeypatch.setattr(_build, 'GRADOPS', '/nonexistent/_gradops.so')
    with pytest.raises(RuntimeError, match='not built'):
        optim.grad_norm([torch.zeros(3)])


def test_adam_entry_refuses_without_a_launch():
    lib = _lib.load()
    assert lib.nvdr_adam_step_factor(None, 0, 1e-3, 0.9, 0.999, 1e-8, None, 1, None, None) == -1 and b'NULL' in lib.nvdr_last_error()
    assert lib.nvdr_adam_step_clipped(None, 0, 1e-3, 0.9, 0.999, 1e-8, None, 2, 1.0, None, 0, None, None) == -1 and b'NULL' in lib.nvdr_last_error()
    A = 1 << 20
    row = optim._ADAM_ROW(A, A, A, A, 4, 1.0, -math.inf, math.inf, 0, 0, 0, 0, 1.0, 0, 0, 0, 0)
    ws, norm = torch.empty(8, dtype=torch.float64), torch.empty(1)
    at = ws.data_ptr() + (-ws.data_ptr()) % 16
    for kw, word in ((dict(workspace=None), b'workspace'), (dict(workspace=at + 8), b'workspace'), (dict(size=1), b'workspace'), (dict(norm=None), b'norm'),
                     (dict(norm_type=5), b'norm type'), (dict(max_norm=-1.0), b'max_norm'), (dict(lr=-1.0), b'hyper')):
        a = dict(dict(lr=1e-3, norm_type=2, max_norm=1.0, workspace=at, size=4, norm=norm.data_ptr()), **kw)
        rc = lib.nvdr_adam_step_clipped(row, 1, a['lr'], 0.9, 0.999, 1e-8, A, a['norm_type'], a['max_norm'], a['workspace'], a['size'], a['norm'], None)
        assert rc == -1 and word in lib.nvdr_last_error(), (kw, rc, lib.nvdr_last_error())


def test_the_packed_row_is_the_structure():
    row = optim._ADAM_ROW(1, 2, 3, 4, 5, 6.0, 7.0, 8.0, 9, 10, 11, 12, 13.0, 14, 15, 16, 17)
    t = _lib.NvdrAdamTensor.from_buffer_copy(row)
    assert len(row) == ctypes.sizeof(_lib.NvdrAdamTensor)
    assert [getattr(t, n) for n, _ in _lib.NvdrAdamTensor._fields_] == list(range(1, 18))
