"""The 8-bit products' schedule and choice of form (tests/f8_walk_host.cpp), built with the host's compiler once a process."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import numpy as np

from unpopped_b200 import build

FORMS = ["narrow", "wide 256", "pair 256", "wide 128"]
TOKENS, WEIGHTS, GROUP, CTAS = (32, 128, 256, 128), (128, 256, 256, 128), (4, 1, 1, 1), (1, 1, 2, 1)
_lib = None


def lib():
    global _lib
    if _lib is None:
        folder = tempfile.mkdtemp()
        try:
            out = os.path.join(folder, "f8_walk.so")
            here = os.path.join(os.path.dirname(os.path.abspath(__file__)), "f8_walk_host.cpp")
            subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", build.CSRC, here, "-o", out], check=True, capture_output=True)
            _lib = ctypes.CDLL(out)
        finally:
            shutil.rmtree(folder)
        _lib.f8_form.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_int]
        _lib.f8_panel_rows.argtypes = [ctypes.c_int64]
    return _lib


def form(m, n, k, experts=1, sms=148):
    return FORMS[lib().f8_form(m, experts, n, k, sms)]


def panel_rows(k):
    return lib().f8_panel_rows(k)


def runs(name, begin, n, k, owner, owners, panel=1 << 30):
    """[count, 9] of t, g0, g1, e, tb, m0, n, c0, c1: the runs of one owner; begin are the experts' first rows and the last's end."""
    begin = np.ascontiguousarray(begin, dtype=np.int32)
    kb = -(-k // 128)
    most = 4096
    while True:
        out = np.empty((most, 9), dtype=np.int32)
        count = lib().f8_runs(FORMS.index(name), len(begin) - 1, begin.ctypes.data_as(ctypes.c_void_p), n, kb, owner, owners, panel,
                              out.ctypes.data_as(ctypes.c_void_p), most)
        if count <= most:
            return out[:count]
        most = count


def shared(name, begin, n, k, sms=148, panel=1 << 30):
    """Whether some tile has parts."""
    owners = sms // CTAS[FORMS.index(name)]
    return any((runs(name, begin, n, k, o, owners, panel)[:, 7] >= 0).any() for o in range(owners))
