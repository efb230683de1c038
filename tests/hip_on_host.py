"""Host code of the library run without a GPU: a process of its own in which tests/cmirror/hip_on_host.cpp stands in for the HIP runtime."""
import functools
import os
import subprocess
import sys
import tempfile
import textwrap

import __graft_entry__ as ge

HEAD = """
import ctypes as C, sys
import numpy as np
fake = C.CDLL({so!r}, mode=C.RTLD_GLOBAL)          # in front of the library: its HIP calls land here
sys.modules["torch"] = None                        # (a runtime of its own)
sys.path.insert(0, {root!r})
import __graft_entry__ as ge
ge.load_package()
from importlib import import_module
hip = import_module(ge.PKG_NAME + ".hip")
L = hip.lib()
for f in ("fake_launches", "fake_most_threads", "fake_blocks"):
    getattr(fake, f).restype = C.c_uint64
"""


@functools.lru_cache(None)
def build():
    so = os.path.join(tempfile.mkdtemp(prefix="hip_on_host_"), "libhip_on_host.so")
    src = os.path.join(ge.ROOT, "tests", "cmirror", "hip_on_host.cpp")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", src, "-o", so])
    return so


def run(script):
    """`script` behind HEAD; what it prints."""
    out = subprocess.run([sys.executable, "-c", HEAD.format(so=build(), root=ge.ROOT) + textwrap.dedent(script)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-4000:]
    return out.stdout
