"""Build the host C++ libraries that need the torch headers, in-tree under
_torch_ext/ (the .so are git-ignored):

* csrc_torch/svo_class.cpp -> xrd_svo_class.so: ``torch.classes.svo.Octree`` on
  top of the C-ABI octree;
* csrc_torch/token_ops.cpp -> xrd_token_ops.so: ``torch.ops.xrdslam.*``, the
  differentiable token and grouped-product operators over the C ABI.

    python -m xrdslam_amd.build_torch_ext
"""
import os

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
OUT = os.path.join(HERE, '_torch_ext')
LIB = os.path.join(OUT, 'xrd_svo_class.so')
SRC = os.path.join(HERE, 'csrc_torch', 'svo_class.cpp')
TOKEN_LIB = os.path.join(OUT, 'xrd_token_ops.so')
TOKEN_SRC = os.path.join(HERE, 'csrc_torch', 'token_ops.cpp')


def _build(lib, src, force, verbose, cflags=(), ldflags=()):
    from torch.utils import cpp_extension
    header = os.path.join(ROOT, 'include', 'xrdslam_hip.h')
    if os.path.exists(lib):
        if not force and os.path.getmtime(lib) > max(
                os.path.getmtime(src), os.path.getmtime(header)):
            return
        os.remove(lib)
    os.makedirs(OUT, exist_ok=True)
    obj = os.path.join(OUT, os.path.basename(src)[:-4] + '.o')
    if force and os.path.exists(obj):     # compile anew whatever ninja thinks
        os.remove(obj)
    cpp_extension.load(
        name=os.path.basename(lib)[:-3], sources=[src],
        extra_include_paths=[os.path.join(ROOT, 'include')],
        extra_cflags=['-O2', *cflags],
        # rpath = the package directory next to _torch_ext/ ('$$' for ninja,
        # the backslash for the shell that runs the link line)
        extra_ldflags=[f'-L{HERE}', '-lxrdslam_hip',
                       '-Wl,-rpath,\\$$ORIGIN/..', *ldflags],
        build_directory=OUT, is_python_module=False, verbose=verbose)


def build(verbose=False, force=False):
    import torch

    from . import build as core
    core.build(verbose=verbose)  # libxrdslam_hip.so must exist to link
    _build(LIB, SRC, force, verbose)
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
    libs = os.path.join(os.path.dirname(torch.__file__), 'lib')
    _build(TOKEN_LIB, TOKEN_SRC, force, verbose,
           cflags=['-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
                   f'-I{rocm}/include'],
           ldflags=[f'-L{libs}', '-lc10_hip'])
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
