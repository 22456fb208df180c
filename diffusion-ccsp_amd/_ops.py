"""Loading and building of the operator libraries behind operators.py: libccsp_ops.so (the kernels and their C ABI, include/ccsp_ops.h) and
ccsp_ops_torch.so (the operators on torch tensors).  Like the sampling library they have no CPU fallback: if one cannot be loaded (or built)
every operator raises."""
import ctypes as C
import importlib.machinery
import importlib.util
import os
import shutil
import subprocess
import threading

from ._lib import CSRC, CcspError

OPS_SRC = os.path.join(CSRC, 'ops')
OPS_SO = os.path.join(CSRC, 'libccsp_ops.so')
TORCH_SO = os.path.join(CSRC, 'ccsp_ops_torch.so')
OPS_ABI_MAJOR = 1     # CCSP_OPS_VERSION_MAJOR of include/ccsp_ops.h this binding was written against
TYPES = {'float32': 0, 'bfloat16': 1, 'float16': 2}


def _compile(so, sources, cmd, force, verbose):
    if not force and os.path.isfile(so) and all(os.path.getmtime(so) >= os.path.getmtime(s) for s in sources):
        return
    tmp = '%s.%d.tmp' % (so, os.getpid())         # per process: the ranks of a first multi-rank run may all build at once
    cmd = cmd + ['-o', tmp]
    if verbose:
        print(' '.join(cmd))
    try:
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, universal_newlines=True)
        if r.returncode != 0:
            raise CcspError('%s failed:\n%s' % (os.path.basename(cmd[0]), r.stderr[-4000:]))
        os.replace(tmp, so)
    finally:
        if os.path.isfile(tmp):
            os.remove(tmp)


def build(force=False, verbose=False):
    """compile both libraries in-tree for gfx950 (cross-compiles without a GPU).  -packed-fp32-ops: no packed 32-bit float instructions, some forms of which have
    given wrong results on MI355X (hipcc's host pass warns that it does not know the feature: harmless)."""
    import sysconfig
    from torch.utils import cpp_extension
    header = os.path.join(CSRC, '..', '..', 'include', 'ccsp_ops.h')
    kernels = [os.path.join(OPS_SRC, f) for f in sorted(os.listdir(OPS_SRC)) if f.endswith(('.h', '.hip'))] + [header]
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    _compile(OPS_SO, kernels, [hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-shared', '-fPIC', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
                               os.path.join(OPS_SRC, 'ccsp_ops.hip')], force, verbose)
    source = os.path.join(OPS_SRC, 'ops_torch.cpp')
    cmd = [shutil.which('g++') or 'c++', '-O2', '-std=c++17', '-shared', '-fPIC', '-DTORCH_EXTENSION_NAME=ccsp_ops_torch', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1']
    cmd += ['-I' + p for p in cpp_extension.include_paths('cuda') + [sysconfig.get_paths()['include']]] + [source] + ['-L' + p for p in cpp_extension.library_paths('cuda')]
    _compile(TORCH_SO, [source, header], cmd + ['-L' + CSRC, '-l:' + os.path.basename(OPS_SO), '-Wl,-rpath,$ORIGIN', '-lc10', '-lc10_hip', '-ltorch_cpu', '-ltorch', '-ltorch_python'],
             force, verbose)
    return OPS_SO


def _check_version(so, ver):
    if ver // 1000 != OPS_ABI_MAJOR:
        raise CcspError('%s reports ABI version %d.%d, this binding is written against major version %d: rebuild it' % (so, ver // 1000, ver % 1000, OPS_ABI_MAJOR))


def _ensure():
    if not (os.path.isfile(OPS_SO) and os.path.isfile(TORCH_SO)):
        try:
            build()
        except Exception as e:  # noqa
            raise CcspError('the operator libraries are missing and could not be built (%s); the HIP extension is required -- there is no CPU fallback' % (e,))


_lib = _torch = None
_loading = threading.RLock()      # the first calls may come from several threads


def lib():
    """the C ABI (include/ccsp_ops.h) through ctypes"""
    global _lib
    if _lib is None:
        with _loading:
            if _lib is None:
                _lib = _load_lib()
    return _lib


def torch_ops():
    """the operators on torch tensors (csrc/ops/ops_torch.cpp)"""
    global _torch
    if _torch is None:
        with _loading:
            if _torch is None:
                _torch = _load_torch()
    return _torch


def _load_lib():
    _ensure()
    try:
        L = C.CDLL(OPS_SO)
    except OSError as e:
        raise CcspError('cannot load %s: %s (the HIP extension is required)' % (OPS_SO, e))
    vp, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.ccsp_ops_last_error.restype = C.c_char_p
    L.ccsp_ops_version.restype = i32
    _check_version(OPS_SO, int(L.ccsp_ops_version()))
    L.ccsp_ops_route_workspace.argtypes = [i64, i32, i64, i32]
    L.ccsp_ops_route_workspace.restype = i64
    L.ccsp_ops_route.argtypes = [vp, vp, i32, i64, i32, i32, i64] + [vp] * 8 + [i64, vp]
    L.ccsp_ops_rows_gather.argtypes = [i32, i64, i64, vp, i64] + [vp] * 6
    L.ccsp_ops_rows_combine.argtypes = [i32, i64, i64, i64, i32, vp, vp, vp, vp, i32, vp, i64, vp, vp]
    L.ccsp_ops_rows_back.argtypes = [i32, i64, i64] + [vp] * 5 + [i32, vp, i64, vp, i64, vp, vp, vp]
    L.ccsp_ops_linear_workspace.argtypes = [i32, i32, i32, i64, i64, i64, vp, i64, vp, i64]
    L.ccsp_ops_linear_workspace.restype = i64
    L.ccsp_ops_linear.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, vp, vp, i32, vp, vp, vp, i64, vp]
    L.ccsp_ops_linear_silu_back.argtypes = [i32, i32, i64, i64, vp, vp, i64, vp, vp, vp]
    L.ccsp_ops_linear_back_input.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, vp, vp, vp, i64, vp]
    L.ccsp_ops_linear_back_weight.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, vp, i64, vp, vp, vp, i64, vp]
    L.ccsp_ops_norm_workspace.argtypes = [i32, vp]
    L.ccsp_ops_norm_workspace.restype = i64
    L.ccsp_ops_clip_norm.argtypes = [i32, vp, vp, vp, vp, C.c_double, vp, vp, vp, i64, vp]
    return L


def _load_torch():
    _ensure()
    import torch  # noqa: F401  (its libraries come first)
    try:
        loader = importlib.machinery.ExtensionFileLoader('ccsp_ops_torch', TORCH_SO)
        m = importlib.util.module_from_spec(importlib.util.spec_from_file_location('ccsp_ops_torch', TORCH_SO, loader=loader))
        loader.exec_module(m)
    except ImportError as e:
        raise CcspError('cannot load %s: %s (the HIP extension is required)' % (TORCH_SO, e))
    _check_version(TORCH_SO, m.version())
    m.set_error(CcspError)
    return m
