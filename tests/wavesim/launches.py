"""The host side of kernel files alone: their entry points compiled for the host (tests/wavesim/build.py's rewrites and flags) with every
kernel launch RECORDED instead of executed, so that the launches of any accepted size can be looked at.  Pointers are never dereferenced.
TESTS ONLY (tests/test_layer_ops_launches.py)."""
import ctypes
import hashlib
import os
import subprocess

from . import build as _build

_HEAD = r"""
#include "pcm_attn.hpp"
#include <string>
#include <vector>
struct RecordedLaunch { std::string kernel; long grid, block; };
inline std::vector<RecordedLaunch> g_launches;
inline void record_launch(const char *kernel, dim3 g, dim3 b) { g_launches.push_back({kernel, (long)g.x * g.y * g.z, (long)b.x * b.y * b.z}); }
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) record_launch(#kernel, dim3(grid), dim3(block))
"""
_TAIL = r"""
extern "C" int recorded_launches() { return (int)g_launches.size(); }
extern "C" const char *recorded_launch(int i, long *grid, long *block)
{
    *grid = g_launches[i].grid, *block = g_launches[i].block;
    return g_launches[i].kernel.c_str();
}
extern "C" void forget_launches() { g_launches.clear(); }
"""


class Recorder:
    """Entry points as attributes; `launches(rc)` after a call: [(kernel, workgroups, threads of each)]."""

    def __init__(self, sources):
        from pointcloudmatters_amd import _lib

        _build.build()  # the wave model's core, which the kernels' bodies refer to
        text = _HEAD + "".join(_build.rewrite(n, open(_build.source_path(n)).read()) for n in sources) + _TAIL
        key = hashlib.sha1((text + open(_build.LIB, "rb").read().hex()[:4096]).encode()).hexdigest()[:16]
        so = os.path.join(_build.OUT, "launches.%s.so" % key)
        if not os.path.exists(so):
            tmp = "%s.%d" % (so, os.getpid())
            open(tmp + ".cpp", "w").write(text)
            subprocess.run([_build.CLANG] + _build.FLAGS + [tmp + ".cpp", "-x", "none", _build.LIB, "-Wl,-rpath," + _build.OUT, "-shared", "-o", tmp], check=True)
            os.replace(tmp, so)
        self._lib = ctypes.CDLL(so)
        self._lib.recorded_launch.restype = ctypes.c_char_p
        for name, args in _lib.SIGNATURES.items():
            fn = getattr(self._lib, name, None)
            if fn is not None:
                fn.argtypes, fn.restype = args, ctypes.c_long if name in _lib.LONG_RESULTS else ctypes.c_int
                setattr(self, name, fn)

    def launches(self):
        grid, block, out = ctypes.c_long(), ctypes.c_long(), []
        for i in range(self._lib.recorded_launches()):
            name = self._lib.recorded_launch(i, ctypes.byref(grid), ctypes.byref(block))
            out.append((name.decode(), grid.value, block.value))
        self._lib.forget_launches()
        return out
