"""Child processes in which the library meets a stand-in for the HIP runtime (hip_standin.c)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEAD = """
import ctypes as C, sys
import numpy as np
gpu = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)   # its names come before those of the library's own dependencies
for name in ("taken", "largest", "frees", "launches"):
    getattr(gpu, "standin_" + name).restype = C.c_size_t
gpu.standin_memory.argtypes = [C.c_size_t]
gpu.standin_launch.argtypes = [C.c_size_t, C.POINTER(C.c_ulong)]
from nvllm_amd import capi
lib = capi.load_hip()
lib.init_ops()
def launches():   # (grid, block) of every one since the last standin_forget()
    out = []
    for i in range(gpu.standin_launches()):
        six = (C.c_ulong * 6)()
        gpu.standin_launch(i, six)
        out.append((tuple(six[:3]), tuple(six[3:])))
    return out
def ints(a):
    a = np.ascontiguousarray(a, np.int32)
    p = a.ctypes.data_as(C.POINTER(C.c_int))
    p.keep = a
    return p
def delta(ids, pos, slots, heads, dim, vdim, elem=2, qk_heads=None, q_ld=None, at=0x200000000000, eps=0.0):
    Q = qk_heads or heads
    T = len(ids)
    return lib.nvllm_gated_delta(at, at + (1 << 40), at + (2 << 40), at + (3 << 40), at + (4 << 40), at + (5 << 40), at + (6 << 40), ints(ids), ints(pos), slots, 1.0, eps, Q,
                                 heads, dim, vdim, q_ld or Q * dim, q_ld or Q * dim, heads * vdim, elem, T)
"""


def run(tmp_path, body):
    so = str(tmp_path / "standin.so")
    subprocess.check_call(["gcc", "-O1", "-shared", "-fPIC", "-w", "-I/opt/rocm/include", os.path.join(ROOT, "tests", "hip_standin.c"), "-o", so])
    r = subprocess.run([sys.executable, "-c", HEAD + body, so], capture_output=True, text=True, timeout=100,
                       env=dict(os.environ, PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", "")))
    assert r.returncode == 0, (r.returncode, r.stderr[-1500:])
    return r.stdout
