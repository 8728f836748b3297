"""In-tree build of libnvdr_hip.so (explicit hipcc for gfx950; no JIT cache, no cmake).

The library is a plain C-ABI shared object (include/nvdr_hip.h) with no libtorch linkage.  It
links the HIP runtime by SONAME (libamdhip64.so.7); inside a Python process that has imported
torch first, the loader resolves that to the runtime torch already mapped, so device pointers
and stream handles coming from torch are valid in it.
"""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'nvdiffrecmc_amd', 'csrc')
BUILD = os.path.join(CSRC, 'build')
LIB = os.path.join(BUILD, 'libnvdr_hip.so')
ARCH = 'gfx950'

SOURCES = [
    'core.hip',
    'bvh.hip',
    'env_shade.hip',
    'denoise.hip',
    'renderutils.hip',
    'light.hip',
    'gbuffer.hip',
    'mesh.hip',
    'optim.hip',
    'gradnorm.hip',
    'exchange.hip',
]

# nvdr_grad_norm / nvdr_grad_clip for lists of Python tensors: a CPython extension against the installed torch (host code only)
GRADOPS_SOURCE = os.path.join(CSRC, 'gradops.cpp')
GRADOPS = os.path.join(BUILD, '_gradops.so')

# -ffp-contract=off: the sampling math must round exactly like the CPU oracle
# (see include/nvdr_detmath.h); fused operations are written as explicit fmaf.
# -packed-fp32-ops: the compiler makes v_pk_add / mul / fma_f32 from ordinary float code at -O3, and some of their forms have given wrong
# results now and then on MI355X; the target feature is taken away for every source (the host pass warns that it does not know it).
FLAGS = ['--offload-arch=' + ARCH, '-O3', '-std=c++17', '-fPIC', '-ffp-contract=off', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
         '-I' + os.path.join(ROOT, 'include'), '-I' + CSRC, '-Wno-unused-result', '-Wno-unused-value'] + os.environ.get('NVDR_EXTRA_FLAGS', '').split()


def _hipcc():
    exe = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    if not os.path.exists(exe):
        raise RuntimeError('hipcc not found: cannot build libnvdr_hip.so')
    return exe


def _deps_mtime():
    m = 0.0
    for d in (CSRC, os.path.join(ROOT, 'include')):
        for fn in os.listdir(d):
            if fn.endswith(('.h', '.hpp')):
                m = max(m, os.path.getmtime(os.path.join(d, fn)))
    return m


def _current(out, recipe, newest):
    """Is `out` younger than what it is made from, and was it made by this recipe (the command line and the versions behind it)?"""
    try:
        with open(out + '.recipe') as f:
            return os.path.getmtime(out) > newest and f.read() == recipe
    except OSError:
        return False


def _make(what, cmd, out, recipe, verbose):
    if verbose:
        print(' '.join(cmd), flush=True)
    if os.path.exists(out + '.recipe'):
        os.remove(out + '.recipe')              # (what a failed command leaves is not current)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError('%s failed:\n%s\n%s' % (what, r.stdout, r.stderr))
    if verbose and r.stderr.strip():
        print(r.stderr, file=sys.stderr)
    with open(out + '.recipe', 'w') as f:
        f.write(recipe)


def _version(exe):
    return subprocess.run([exe, '--version'], capture_output=True, text=True).stdout


def _compile(src, force, hdr_mtime, version, verbose):
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + '.o')
    sp = os.path.join(CSRC, src)
    cmd = [_hipcc()] + FLAGS + ['-c', sp, '-o', obj]
    recipe = '\n'.join(cmd + [version])
    if not force and _current(obj, recipe, max(os.path.getmtime(sp), hdr_mtime)):
        return obj, False
    _make('hipcc for ' + src, cmd, obj, recipe, verbose)
    return obj, True


def build(force=False, verbose=False):
    """Compile every HIP translation unit for gfx950 and link libnvdr_hip.so.  Returns its path.  What is there already stays when it was made from
    these sources by these commands, flags and versions."""
    os.makedirs(BUILD, exist_ok=True)
    hdr_mtime = _deps_mtime()
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    missing = [s for s in SOURCES if s not in srcs]
    if missing:
        raise RuntimeError('missing HIP sources: %s' % missing)
    version = _version(_hipcc())
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        res = list(ex.map(lambda s: _compile(s, force, hdr_mtime, version, verbose), srcs))
    objs = [o for o, _ in res]
    cmd = [_hipcc(), '--offload-arch=' + ARCH, '-shared', '-fPIC'] + objs + ['-ldl', '-o', LIB]
    recipe = '\n'.join(cmd + [version])
    if force or any(c for _, c in res) or not _current(LIB, recipe, max(os.path.getmtime(o) for o in objs)):
        _make('link', cmd, LIB, recipe, verbose)
    _build_gradops(force, hdr_mtime, verbose)
    return LIB


def _build_gradops(force, hdr_mtime, verbose):
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    cxx = os.environ.get('CXX', 'g++')
    cmd = [cxx, '-O2', '-std=c++17', '-fPIC', '-shared', '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch._C._GLIBCXX_USE_CXX11_ABI,
           '-I' + os.path.join(ROOT, 'include'), '-I' + sysconfig.get_paths()['include']] + ['-I' + d for d in cpp_extension.include_paths()]
    cmd += [GRADOPS_SOURCE, '-o', GRADOPS] + ['-L' + d for d in cpp_extension.library_paths()] + ['-ltorch_python', '-ltorch_cpu', '-lc10']
    recipe = '\n'.join(cmd + [torch.__version__, sys.version, _version(cxx)])
    if force or not _current(GRADOPS, recipe, max(os.path.getmtime(GRADOPS_SOURCE), hdr_mtime)):
        _make('g++ for gradops.cpp', cmd, GRADOPS, recipe, verbose)


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose=True))
