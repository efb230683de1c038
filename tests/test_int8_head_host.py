"""A plan with an 8-bit head whose gl3_finalize fails and is called again: the logits' multiplier reaches the final norm once.  Without a GPU: HIP's calls land in
host memory (hip_on_host.py)."""
import pytest

import hip_on_host


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("fails", [0, 1, 2, 3])
def test_finalize_is_called_again(fails, tied):
    hip_on_host.run("""
    W, V, MUL = 64, 40, 3.0
    rng = np.random.default_rng(1)
    layer = hip.LayerDesc()
    for k, v in dict(mixer=hip.MIX_ATTENTION, heads=2, kv_heads=2, dim=32, vdim=32, scale=0.2).items():
        setattr(layer, k, v)
    d = hip.ModelDesc()
    for k, v in dict(struct_size=C.sizeof(d), arch=hip.ARCH_LAYERLIST, dim=W, vocab=V, ctx=16, n_layers=1, weight_type=hip.TYPE_F32, rms_eps=1e-5, logit_scale=MUL,
                     flags=hip.FLAG_INT8_HEAD | hip.FLAG_F32_COMPUTE, layer_descs=C.pointer(layer)).items():
        setattr(d, k, v)
    ctx = C.c_void_p()
    assert L.gl3_create(C.byref(d), C.byref(ctx)) == 0, L.gl3_last_error(None)

    def put(name, a):
        a = np.ascontiguousarray(a, np.float32)
        assert L.gl3_upload_tensor(ctx, hip.T_IDS[name + ".weight"], 0, a.ctypes.data, a.nbytes, hip.TYPE_F32) == 0, L.gl3_last_error(ctx)
    norm = rng.uniform(1, 2, W).astype(np.float32)
    put("token_embd", rng.standard_normal((V, W)))
    if not {tied}:
        put("output", rng.standard_normal((V, W)))
    put("output_norm", norm)
    put("attn_norm", np.ones(W))
    for t in ("attn_q", "attn_k", "attn_v", "attn_output"):
        put(t, rng.standard_normal((W, W)))
    fails = {fails}
    if fails:
        fake.fake_fail_malloc(fails)          # codes, scales, scratch
        assert L.gl3_finalize(ctx) != 0
        assert fake.fake_holds(norm.tobytes(), norm.nbytes) == 1 and fake.fake_pending() == 0
    assert L.gl3_finalize(ctx) == 0, L.gl3_last_error(ctx)
    once, twice = (norm * np.float32(MUL)).tobytes(), (norm * np.float32(MUL) * np.float32(MUL)).tobytes()
    assert fake.fake_holds(once, len(once)) == 1 and fake.fake_holds(twice, len(twice)) == 0
    assert L.gl3_finalize(ctx) == 0          # finalized: nothing happens
    assert fake.fake_holds(once, len(once)) == 1
    L.gl3_destroy(ctx)
    """.format(fails=fails, tied=tied))
