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


def tiny_plan(W=64, V=40, tied=False, flags=0, norm=None, **kw):          # one attention layer of the layer-list family, all but finalized
    rng = np.random.default_rng(1)
    layer, d, ctx = hip.LayerDesc(), hip.ModelDesc(), C.c_void_p()
    for k, v in dict(mixer=hip.MIX_ATTENTION, heads=2, kv_heads=2, dim=W // 2, vdim=W // 2, scale=0.2).items():
        setattr(layer, k, v)
    for k, v in dict(dict(struct_size=C.sizeof(d), arch=hip.ARCH_LAYERLIST, dim=W, vocab=V, ctx=16, n_layers=1, weight_type=hip.TYPE_F32, rms_eps=1e-5,
                          flags=flags | hip.FLAG_F32_COMPUTE, layer_descs=C.pointer(layer)), **kw).items():
        setattr(d, k, v)
    assert L.gl3_create(C.byref(d), C.byref(ctx)) == 0, L.gl3_last_error(None)
    tensors = {{"token_embd": rng.standard_normal((V, W)), "output_norm": np.ones(W) if norm is None else norm, "attn_norm": np.ones(W)}}
    tensors.update({{t: rng.standard_normal((W, W)) for t in ("attn_q", "attn_k", "attn_v", "attn_output")}})
    if not tied:
        tensors["output"] = rng.standard_normal((V, W))
    for name, a in tensors.items():
        a = np.ascontiguousarray(a, np.float32)
        assert L.gl3_upload_tensor(ctx, hip.T_IDS[name + ".weight"], 0, a.ctypes.data, a.nbytes, hip.TYPE_F32) == 0, L.gl3_last_error(ctx)
    return ctx
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
