"""What holds for the files of the tree as a whole."""
import ast
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIRS = ('nvdiffrecmc_amd', 'tools', 'tests', 'oracle', 'perf')


def _files(*suffixes):
    out = [f for d in DIRS for f in glob.glob(os.path.join(ROOT, d, '**', '*'), recursive=True) if f.endswith(suffixes)]
    return out + [f for f in glob.glob(os.path.join(ROOT, '*')) if f.endswith(suffixes)]


def test_every_stream_has_the_default_priority():
    """Work on streams of different priorities has hung on this runtime for good."""
    found = []
    for f in _files('.py'):
        for node in ast.walk(ast.parse(open(f).read())):
            if isinstance(node, ast.Call):
                found += [(f, node.lineno, k.arg) for k in node.keywords if k.arg in ('priority', 'is_high_priority_stream')]
    for f in _files('.hip', '.cpp', '.h', '.c'):
        if re.search(r'hip(StreamCreate|ExtStreamCreate)With(Priority|CUMask)', open(f).read()):
            found.append(f)
    assert not found


def test_tools_that_are_named_exist():
    """The documents and the sources point to no tool that is gone."""
    files = [os.path.join(ROOT, f) for f in ('README.md', 'DESIGN.md', 'INTEGRATION.md')] + _files('.py', '.hip', '.cpp', '.h')
    named = {(os.path.relpath(f, ROOT), m) for f in files for m in re.findall(r'\btools/[\w/]+\.(?:py|sh|hip|c|txt)\b', open(f).read())}
    assert len(named) > 20
    assert not sorted((f, m) for f, m in named if not os.path.exists(os.path.join(ROOT, m)))


def test_no_build_switch_leaves_work_out():
    """A build that skips work to time the rest has no place in the sources."""
    assert not [f for f in _files('.hip', '.h', '.cpp') if re.search(r'#define \w*(SKIP|EXPERIMENT)\w*', open(f).read())]


def test_no_memset_node_on_a_path_that_may_be_captured():
    """A memset inside a captured graph has given wrong results on replays: the library fills by kernels, but for the experiment switches and the
    arithmetic's self-test, which is not captured."""
    found = []
    for f in _files('.hip', '.h'):
        if 'ubench' in f:
            continue
        lines = open(f).read().splitlines()
        found += [(os.path.basename(f), line.strip()) for k, line in enumerate(lines) if 'hipMemsetAsync(' in line and 'c->debug &' not in line + lines[max(k - 1, 0)]]
    assert [(f, 'counters' in line) for f, line in found] == [('core.hip', True)], found
