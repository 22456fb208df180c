"""ctypes binding of libccsp_ops.so (include/ccsp_ops.h), the library behind operators.py.  Like the sampling library it has no CPU
fallback: if it cannot be loaded (or built) every operator raises."""
import ctypes as C
import os
import shutil
import subprocess

from ._lib import CSRC, CcspError

OPS_SRC = os.path.join(CSRC, 'ops')
OPS_SO = os.path.join(CSRC, 'libccsp_ops.so')
OPS_ABI_MAJOR = 1     # CCSP_OPS_VERSION_MAJOR of include/ccsp_ops.h this binding was written against
TYPES = {'float32': 0, 'bfloat16': 1, 'float16': 2}
MAX_EXPERTS = 1024    # CCSP_OPS_MAX_EXPERTS


def build(force=False, verbose=False):
    """hipcc --offload-arch=gfx950 the operator library in-tree (cross-compiles without a GPU).  -packed-fp32-ops: no packed 32-bit float instructions, some forms
    of which have given wrong results on these boards (hipcc's host pass warns that it does not know the feature: harmless)."""
    header = os.path.join(CSRC, '..', '..', 'include', 'ccsp_ops.h')
    sources = [os.path.join(OPS_SRC, f) for f in sorted(os.listdir(OPS_SRC)) if f.endswith(('.h', '.hip'))] + [header]
    if not force and os.path.isfile(OPS_SO) and all(os.path.getmtime(OPS_SO) >= os.path.getmtime(s) for s in sources):
        return OPS_SO
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    tmp = '%s.%d.tmp' % (OPS_SO, os.getpid())
    cmd = [hipcc, '--offload-arch=gfx950', '-O3', '-std=c++17', '-shared', '-fPIC', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops',
           '-o', tmp, os.path.join(OPS_SRC, 'ccsp_ops.hip')]
    if verbose:
        print(' '.join(cmd))
    try:
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, universal_newlines=True)
        if r.returncode != 0:
            raise CcspError('hipcc failed:\n' + r.stderr[-4000:])
        os.replace(tmp, OPS_SO)
    finally:
        if os.path.isfile(tmp):
            os.remove(tmp)
    return OPS_SO


_lib = None


def lib():
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.isfile(OPS_SO):
        try:
            build()
        except Exception as e:  # noqa
            raise CcspError('libccsp_ops.so is missing and could not be built (%s); the HIP extension is required -- there is no CPU fallback' % (e,))
    try:
        L = C.CDLL(OPS_SO)
    except OSError as e:
        raise CcspError('cannot load %s: %s (the HIP extension is required)' % (OPS_SO, e))
    vp, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.ccsp_ops_last_error.restype = C.c_char_p
    L.ccsp_ops_version.restype = i32
    ver = int(L.ccsp_ops_version())
    if ver // 1000 != OPS_ABI_MAJOR:
        raise CcspError('%s reports ABI version %d.%d, this binding is written against major version %d: rebuild it' % (OPS_SO, ver // 1000, ver % 1000, OPS_ABI_MAJOR))
    L.ccsp_ops_route_workspace.argtypes = [i64, i32, i64, i32]
    L.ccsp_ops_route_workspace.restype = i64
    L.ccsp_ops_route.argtypes = [vp, vp, i32, i64, i32, i32, i64] + [vp] * 7 + [i64, vp]
    L.ccsp_ops_rows_gather.argtypes = [i32, i64, i64, vp, i64, vp, vp, vp]
    L.ccsp_ops_rows_combine.argtypes = [i32, i64, i64, i32, vp, vp, vp, vp, i32, vp, i64, vp, vp]
    L.ccsp_ops_rows_back.argtypes = [i32, i64, i64, vp, vp, vp, i32, vp, i64, vp, i64, vp, vp, vp]
    L.ccsp_ops_linear_workspace.argtypes = [i32, i32, i32, i64, i64, i64, vp, i64, vp, i64]
    L.ccsp_ops_linear_workspace.restype = i64
    L.ccsp_ops_linear.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, vp, vp, i32, vp, vp, vp, i64, vp]
    L.ccsp_ops_linear_silu_back.argtypes = [i32, i32, i64, i64, vp, vp, i64, vp, vp, vp]
    L.ccsp_ops_linear_back_input.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, vp, vp, vp, i64, vp]
    L.ccsp_ops_linear_back_weight.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, vp, i64, vp, vp, vp, i64, vp]
    L.ccsp_ops_norm_workspace.argtypes = [i32, vp]
    L.ccsp_ops_norm_workspace.restype = i64
    L.ccsp_ops_clip_norm.argtypes = [i32, vp, vp, vp, vp, C.c_double, vp, vp, vp, i64, vp]
    _lib = L
    return L


def check(rc):
    if rc != 0:
        raise CcspError(lib().ccsp_ops_last_error().decode())
