"""What a build makes again, and what it leaves (compilers replaced by a stand-in)."""
import os
import types

import pytest

from nvdiffrecmc_amd import _build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A tree of two sources; calls: the outputs of each build, versions: what a compiler says of itself."""
    csrc = tmp_path / 'csrc'
    csrc.mkdir()
    (tmp_path / 'include').mkdir()
    for n in ('a.hip', 'b.hip', 'gradops.cpp', 'c.h'):
        (csrc / n).write_text('x')
        os.utime(csrc / n, (1e9, 1e9))
    t = types.SimpleNamespace(made=[], version='1.0', csrc=csrc, fail='')

    def run(cmd, **_):
        if cmd[-1] == '--version':
            return types.SimpleNamespace(returncode=0, stdout=t.version, stderr='')
        out = cmd[cmd.index('-o') + 1]
        if t.fail and t.fail in out:
            with open(out, 'w') as f:
                f.write('half')
            os.utime(out, (4e9, 4e9))
            return types.SimpleNamespace(returncode=1, stdout='', stderr='no')
        with open(out, 'w') as f:
            f.write('made')
        os.utime(out, ns=((len(t.made) + 2 * 10 ** 9) * 10 ** 9,) * 2)      # each younger than the one before
        t.made.append(os.path.basename(out))
        return types.SimpleNamespace(returncode=0, stdout='', stderr='')

    monkeypatch.setattr(_build, 'ROOT', str(tmp_path))
    monkeypatch.setattr(_build, 'CSRC', str(csrc))
    monkeypatch.setattr(_build, 'BUILD', str(csrc / 'build'))
    monkeypatch.setattr(_build, 'LIB', str(csrc / 'build' / 'lib.so'))
    monkeypatch.setattr(_build, 'GRADOPS', str(csrc / 'build' / '_gradops.so'))
    monkeypatch.setattr(_build, 'GRADOPS_SOURCE', str(csrc / 'gradops.cpp'))
    monkeypatch.setattr(_build, 'SOURCES', ['a.hip', 'b.hip'])
    monkeypatch.setattr(_build.subprocess, 'run', run)

    def build(**kw):
        start = len(t.made)
        assert _build.build(**kw) == _build.LIB
        return sorted(t.made[start:])
    t.build = build
    return t


EVERYTHING = ['_gradops.so', 'a.o', 'b.o', 'lib.so']


def test_a_build_makes_what_is_missing_or_old(tree):
    assert tree.build() == EVERYTHING and tree.build() == [] and tree.build(force=True) == EVERYTHING and tree.build() == []
    os.utime(tree.csrc / 'a.hip', (3e9, 3e9))
    assert tree.build() == ['a.o', 'lib.so']
    os.utime(tree.csrc / 'a.hip', (1e9, 1e9))
    os.remove(tree.csrc / 'build' / 'b.o')
    assert tree.build() == ['b.o', 'lib.so'] and tree.build() == []
    os.remove(tree.csrc / 'build' / 'lib.so')
    assert tree.build() == ['lib.so']
    os.utime(tree.csrc / 'gradops.cpp', (3e9, 3e9))
    assert tree.build() == ['_gradops.so']
    os.utime(tree.csrc / 'gradops.cpp', (1e9, 1e9))
    assert tree.build() in ([], ['_gradops.so']) and tree.build() == []
    os.utime(tree.csrc / 'c.h', (3e9, 3e9))
    assert tree.build() == EVERYTHING


def test_a_build_follows_flags_and_versions(tree, monkeypatch):
    import torch
    tree.build()
    monkeypatch.setattr(_build, 'FLAGS', _build.FLAGS + ['-DX=1'])
    assert tree.build() == ['a.o', 'b.o', 'lib.so'] and tree.build() == []
    monkeypatch.setattr(torch, '__version__', '0.0')
    assert tree.build() == ['_gradops.so'] and tree.build() == []
    tree.version = '2.0'
    assert tree.build() == EVERYTHING and tree.build() == []
    for f in os.listdir(_build.BUILD):
        if f.endswith('.recipe'):
            os.remove(os.path.join(_build.BUILD, f))                        # outputs of a build that kept none
    assert tree.build() == EVERYTHING and tree.build() == []


def test_a_failed_step_is_taken_again(tree):
    tree.build()
    os.utime(tree.csrc / 'a.hip', (3e9, 3e9))
    tree.fail = 'a.o'
    with pytest.raises(RuntimeError, match='a.hip'):
        tree.build()
    tree.fail = 'lib.so'
    with pytest.raises(RuntimeError, match='link'):
        tree.build()
    os.utime(tree.csrc / 'a.hip', (1e9, 1e9))
    tree.fail = ''
    assert tree.build() == ['lib.so'] and tree.build() == []


def test_packed_fp32_is_taken_away_from_every_source():
    at = _build.FLAGS.index('-packed-fp32-ops')
    assert _build.FLAGS[at - 3:at + 1] == ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops'] and '-ffp-contract=off' in _build.FLAGS
