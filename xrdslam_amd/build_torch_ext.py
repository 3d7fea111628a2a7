"""Build the host C++ libraries that need the torch headers, in-tree under
_torch_ext/ (the .so are git-ignored):

* csrc_torch/svo_class.cpp -> xrd_svo_class.so: ``torch.classes.svo.Octree`` on
  top of the C-ABI octree;
* csrc_torch/token_ops.cpp -> xrd_token_ops.so: ``torch.ops.xrdslam.*``, the
  differentiable token and grouped-product operators over the C ABI.

    python -m xrdslam_amd.build_torch_ext
"""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OUT = os.path.join(HERE, '_torch_ext')
LIB = os.path.join(OUT, 'xrd_svo_class.so')
SRC = os.path.join(HERE, 'csrc_torch', 'svo_class.cpp')
TOKEN_LIB = os.path.join(OUT, 'xrd_token_ops.so')
TOKEN_SRC = os.path.join(HERE, 'csrc_torch', 'token_ops.cpp')


def _build(lib, src, force, verbose, cflags=(), ldflags=()):
    """compile ``src`` into ``lib`` unless that is newer than its sources.  One
    compiler call with torch's flags: torch.utils.cpp_extension.load counts
    versions per process and would skip a second forced build.  A build that
    fails leaves the library that is there."""
    import torch
    from torch.utils import cpp_extension
    header = os.path.join(ROOT, 'include', 'xrdslam_hip.h')
    if not force and os.path.exists(lib) and os.path.getmtime(lib) > max(
            os.path.getmtime(src), os.path.getmtime(header)):
        return
    os.makedirs(OUT, exist_ok=True)
    fresh = f'{lib}.{os.getpid()}.tmp'
    libs = os.path.join(os.path.dirname(torch.__file__), 'lib')
    cmd = [os.environ.get('CXX', 'c++'), '-O2', '-std=c++17', '-fPIC',
           '-shared', '-I' + os.path.join(ROOT, 'include')]
    for path in cpp_extension.include_paths():
        cmd += ['-isystem', path]
    cmd += [f'-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}',
            *cflags, src, '-o', fresh,
            # rpath = the package directory next to _torch_ext/
            f'-L{HERE}', '-lxrdslam_hip', '-Wl,-rpath,$ORIGIN/..',
            f'-L{libs}', *ldflags, '-lc10', '-ltorch_cpu', '-ltorch']
    if verbose:
        print('[xrdslam_amd.build_torch_ext]', *cmd)
    try:
        subprocess.run(cmd, check=True)
        os.replace(fresh, lib)
    finally:
        if os.path.exists(fresh):
            os.remove(fresh)


def build(verbose=False, force=False):
    from . import build as core
    core.build(verbose=verbose)  # libxrdslam_hip.so must exist to link
    _build(LIB, SRC, force, verbose)
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
    _build(TOKEN_LIB, TOKEN_SRC, force, verbose,
           cflags=['-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
                   f'-I{rocm}/include'],
           ldflags=['-lc10_hip'])
    return LIB


def load():
    """register torch.classes.svo (idempotent)"""
    import torch
    if not os.path.exists(LIB):
        build()
    torch.classes.load_library(LIB)
    return torch.classes.svo.Octree


if __name__ == '__main__':
    print(build(verbose=True))
