"""Operators on device memory: every refusal of the C entry points, before anything touches a GPU; workspace sizes; the Python twin's own checks."""
import ctypes as C
from importlib import import_module

import pytest
import torch

import __graft_entry__ as ge


@pytest.fixture(scope="module")
def hip(pkg):
    return import_module(ge.PKG_NAME + ".hip")


@pytest.fixture(scope="module")
def ops(pkg):
    return import_module(ge.PKG_NAME + ".ops")


A = 1 << 20            # an address that is 16-byte aligned and never followed
B = A + 1


def quantize(**kw):
    a = dict(device=0, stream=None, x=A, type=0, rows=2, cols=5, ldx=5, codes=A, ldq=128, scale=A)
    a.update(kw)
    return list(a.values())


def matmul(**kw):
    a = dict(device=0, stream=None, a=A, lda=128, a_scale=A, w=A, ldw=128, w_scale=A, bias=None, m=2, n=3, k=5, y=A, y_type=0, ldy=3, workspace=A, bytes=1 << 30)
    a.update(kw)
    return list(a.values())


def linear(**kw):
    a = dict(device=0, stream=None, x=A, x_type=0, ldx=5, w=A, ldw=128, w_scale=A, bias=None, m=2, n=3, k=5, y=A, y_type=0, ldy=3, workspace=A, bytes=1 << 30)
    a.update(kw)
    return list(a.values())


def logprobs(**kw):
    a = dict(device=0, stream=None, logits=A, type=0, rows=2, vocab=9, ld=9, targets=A, top=3, logprob=A, rank=A, entropy=A, top_ids=A, top_logprobs=A, workspace=A, bytes=1 << 30)
    a.update(kw)
    return list(a.values())


BAD = [("gl3_quantize_rows", quantize, kw) for kw in (
    dict(type=2), dict(type=8), dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(cols=-3), dict(cols=131072, ldx=131072, ldq=131072), dict(x=None), dict(codes=None), dict(scale=None),
    dict(x=B), dict(type=1, x=B), dict(scale=A + 2), dict(ldx=4), dict(ldx=-5), dict(ldx=1 << 62), dict(codes=A + 8), dict(ldq=120), dict(ldq=136), dict(ldq=0), dict(device=-1))]
BAD += [(name, make, kw) for name, make in (("gl3_int8_matmul", matmul), ("gl3_int8_linear", linear)) for kw in (
    dict(k=0), dict(k=131072), dict(m=-1), dict(n=-1), dict(m=1 << 31), dict(n=1 << 31), dict(y_type=8), dict(y_type=-1), dict(w=None), dict(w_scale=None), dict(y=None), dict(w=A + 4),
    dict(ldw=120), dict(ldw=0), dict(ldw=136), dict(w_scale=B), dict(bias=A + 2), dict(y=A + 2), dict(y_type=1, y=B), dict(ldy=2), dict(ldy=1 << 62), dict(device=-1))]
BAD += [("gl3_int8_matmul", matmul, kw) for kw in (dict(a=None), dict(a_scale=None), dict(a=A + 8), dict(lda=5), dict(lda=0), dict(a_scale=B),
                                                   dict(k=129, lda=256), dict(k=129, ldw=256))]
BAD += [("gl3_int8_linear", linear, kw) for kw in (dict(x=None), dict(x=B), dict(x_type=1, x=B), dict(x_type=8), dict(ldx=4), dict(ldx=0), dict(k=129, ldx=129), dict(m=200, workspace=None),
                                                   dict(m=200, workspace=A + 8), dict(m=200, bytes=0), dict(m=200, bytes=100))]
BAD += [("gl3_token_logprobs", logprobs, kw) for kw in (
    dict(type=8), dict(rows=-1), dict(rows=1 << 31), dict(vocab=0), dict(vocab=-1), dict(top=-1), dict(top=65), dict(targets=None), dict(logprob=None), dict(rank=None),
    dict(targets=None, rank=None), dict(logits=None), dict(logits=B), dict(type=1, logits=B), dict(ld=8), dict(ld=-9), dict(top_ids=None), dict(top_logprobs=None), dict(targets=B),
    dict(logprob=B), dict(rank=B), dict(entropy=B), dict(top_ids=B), dict(top_logprobs=B), dict(device=-1))]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_refused(hip, i):
    name, make, kw = BAD[i]
    assert getattr(hip.lib(), name)(*make(**kw)) == hip.E_ARG, (name, kw)
    assert hip.lib().gl3_last_error(None), (name, kw)


def test_nothing_to_do(hip):
    L = hip.lib()
    none = dict(x=None, codes=None, scale=None)
    assert L.gl3_quantize_rows(*quantize(rows=0, **none)) == 0
    for m, n in ((0, 3), (2, 0), (0, 0)):
        assert L.gl3_int8_matmul(*matmul(m=m, n=n, a=None, a_scale=None, w=None, w_scale=None, y=None, workspace=None, bytes=0)) == 0
        assert L.gl3_int8_linear(*linear(m=m, n=n, x=None, w=None, w_scale=None, y=None, workspace=None, bytes=0)) == 0
    assert L.gl3_token_logprobs(*logprobs(rows=0, logits=None, workspace=None, bytes=0)) == 0


def test_workspace_sizes(hip):
    L = hip.lib()
    a, b, c = C.c_uint64(7), C.c_uint64(7), C.c_uint64(7)
    assert L.gl3_int8_workspace(0, 5, 9, C.byref(a), C.byref(b)) == 0 and (a.value, b.value) == (0, 0)
    for m, n, k in ((1, 1, 1), (5, 300, 1000), (512, 128256, 4096), (2 ** 31 - 1, 2 ** 31 - 1, 131071)):
        assert L.gl3_int8_workspace(m, n, k, C.byref(a), C.byref(b)) == 0
        assert L.gl3_int8_workspace(m, n, k, None, None) == 0
        assert a.value <= b.value < 2 ** 63
    for bad in ((-1, 1, 1), (1, -1, 1), (1, 1, 0), (1, 1, 131072), (2 ** 31, 1, 1)):
        assert L.gl3_int8_workspace(*bad, C.byref(a), C.byref(b)) == hip.E_ARG
    assert L.gl3_logprobs_workspace(0, 9, 3, C.byref(c)) == 0 and c.value == 0
    for bad in ((-1, 9, 3), (1, 0, 3), (1, 9, -1), (1, 9, 65)):
        assert L.gl3_logprobs_workspace(*bad, C.byref(c)) == hip.E_ARG
    assert L.gl3_logprobs_workspace(1, 9, 3, None) == hip.E_ARG


def test_python_checks(hip, ops):
    x = torch.zeros(2, 5)
    with pytest.raises(hip.Gl3Error):
        ops.quantize_rows(x)
    with pytest.raises(hip.Gl3Error):
        ops.token_logprobs(x)
    w = ops.Int8Rows(torch.zeros(3, 128, dtype=torch.int8), torch.ones(3), 5)
    with pytest.raises(hip.Gl3Error):
        ops.int8_linear(x, w)
    with pytest.raises(hip.Gl3Error):
        ops.int8_matmul(w, w)
    assert torch.equal(w.dequantize(), torch.zeros(3, 5))
    assert (ops.CODE_BLOCK, ops.MAX_K, ops.MAX_TOP) == (128, 131071, 64)


def test_errors_belong_to_the_thread(hip):
    """Two threads' refused calls do not touch each other's message."""
    import threading
    L = hip.lib()
    seen = {}

    def work(i):
        for _ in range(300):
            bad = logprobs(top=65) if i % 2 else quantize(cols=0)
            assert (L.gl3_token_logprobs if i % 2 else L.gl3_quantize_rows)(*bad) == hip.E_ARG
            seen.setdefault(i, set()).add(L.gl3_last_error(None))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(v) == 1 for v in seen.values()) and len(seen) == 4
    assert all((b"top" in next(iter(v))) == bool(i % 2) for i, v in seen.items())


@pytest.mark.parametrize("i", range(12))
def test_strides_and_workspaces_that_do_not_do(hip, i):
    name, make, kw = [("gl3_int8_matmul", matmul, dict(ldw=(1 << 23) + 16)), ("gl3_int8_matmul", matmul, dict(lda=(1 << 23) + 16)), ("gl3_int8_matmul", matmul, dict(ldy=(1 << 26) + 1)),
                      ("gl3_int8_linear", linear, dict(ldw=(1 << 23) + 16)), ("gl3_int8_linear", linear, dict(ldy=(1 << 26) + 1)), ("gl3_int8_linear", linear, dict(ldx=1 << 62)),
                      ("gl3_token_logprobs", logprobs, dict(vocab=(1 << 30) + 1, ld=(1 << 30) + 1)), ("gl3_token_logprobs", logprobs, dict(ld=1 << 62)),
                      ("gl3_token_logprobs", logprobs, dict(vocab=128256, ld=128256, bytes=100)),
                      ("gl3_int8_matmul", matmul, dict(m=40, n=300, k=9000, lda=9088, ldw=9088, ldy=300, workspace=None, bytes=0)),
                      ("gl3_int8_matmul", matmul, dict(m=40, n=300, k=9000, lda=9088, ldw=9088, ldy=300, bytes=40 * 300 * 4)),
                      ("gl3_int8_linear", linear, dict(m=40, n=300, k=9000, ldx=9000, ldw=9088, ldy=300, bytes=40 * 9088 + 160))][i]
    assert getattr(hip.lib(), name)(*make(**kw)) == hip.E_ARG, (name, kw)


def test_a_thread_without_an_error_reads_the_newest(hip):
    """A plan that cannot be created in one thread, its message read in another that has none of its own."""
    import threading
    L = hip.lib()
    out = C.c_void_p()
    assert L.gl3_create(None, C.byref(out)) == hip.E_ARG
    seen = []
    t = threading.Thread(target=lambda: seen.append(L.gl3_last_error(None)))
    t.start()
    t.join()
    assert seen == [b"null argument"] == [L.gl3_last_error(None)]


@pytest.mark.parametrize("over", [dict(dim=131072), dict(vocab=(1 << 26) + 1)])
def test_an_int8_head_of_what_it_cannot_hold(hip, over):
    """Refused before anything is allocated."""
    d = hip.ModelDesc()
    layer = hip.LayerDesc()
    for k, v in dict(dict(struct_size=C.sizeof(d), arch=hip.ARCH_NODITAR, dim=64, vocab=100, ctx=16, n_layers=1, weight_type=30, flags=hip.FLAG_INT8_HEAD, layer_descs=C.pointer(layer)), **over).items():
        setattr(d, k, v)
    out = C.c_void_p()
    assert hip.lib().gl3_create(C.byref(d), C.byref(out)) == hip.E_ARG and b"INT8_HEAD" in hip.lib().gl3_last_error(None)


# ---- the host code behind the checks, without a GPU (hip_on_host.py): nothing is followed, launches are counted -------------------------------------
def test_an_error_of_somebody_else_is_not_an_operators():
    """A failed call that the program has dealt with leaves an error pending in its thread: operators return what their own launches return, and leave it be."""
    import hip_on_host
    hip_on_host.run("""
    A = 1 << 20
    calls = [lambda: L.gl3_quantize_rows(0, None, A, 0, 5, 300, 300, A, 384, A),
             lambda: L.gl3_int8_matmul(0, None, A, 384, A, A, 384, A, None, 5, 70, 300, A, 0, 70, A, 1 << 30),
             lambda: L.gl3_int8_linear(0, None, A, 0, 300, A, 384, A, None, 5, 70, 300, A, 0, 70, A, 1 << 30),
             lambda: L.gl3_int8_linear(0, None, A, 0, 300, A, 384, A, None, 500, 70, 300, A, 0, 70, A, 1 << 30),
             lambda: L.gl3_token_logprobs(0, None, A, 0, 3, 70000, 70000, A, 2, A, A, A, A, A, A, 1 << 30)]
    for call in calls:
        assert fake.hipSetDevice(1000) != 0          # pending until somebody asks
        fake.fake_reset()
        assert call() == 0, L.gl3_last_error(None)
        assert fake.fake_launches() >= 1 and fake.fake_pending() != 0
        fake.hipGetLastError()
    """)


def test_nothing_is_launched_behind_a_launch_that_failed():
    import hip_on_host
    hip_on_host.run("""
    A = 1 << 20
    calls = [lambda: L.gl3_quantize_rows(0, None, A, 0, 5, 300, 300, A, 384, A),
             lambda: L.gl3_int8_linear(0, None, A, 0, 300, A, 384, A, None, 500, 70, 300, A, 0, 70, A, 1 << 30),                     # codes, product
             lambda: L.gl3_int8_linear(0, None, A, 0, 30000, A, 30080, A, None, 40, 300, 30000, A, 0, 300, A, 1 << 30),              # codes, parts, their sums
             lambda: L.gl3_int8_matmul(0, None, A, 128, A, A, 128, A, None, 200000, 70, 100, A, 0, 70, A, 1 << 30),                  # pieces
             lambda: L.gl3_token_logprobs(0, None, A, 0, 3, 70000, 70000, A, 2, A, A, A, A, A, A, 1 << 30),                          # parts, join
             lambda: L.gl3_token_logprobs(0, None, A, 0, 200000, 7, 7, A, 2, A, A, A, A, A, A, 1 << 30)]
    seen = []
    for call in calls:
        fake.fake_reset()
        assert call() == 0, L.gl3_last_error(None)
        seen.append(fake.fake_launches())
        for n in range(1, seen[-1] + 1):
            fake.fake_reset()
            fake.fake_fail_launch(n)
            assert call() == hip.E_HIP and L.gl3_last_error(None)
            assert fake.fake_launches() == n and fake.fake_pending() == 0, (n, fake.fake_launches())
    assert seen == [1, 2, 3, 4, 2, 4], seen
    """)


def test_every_launch_has_fewer_threads_than_a_launch_may():
    """More rows than one launch takes, of every length that the quantiser tells apart: fewer than 2^32 threads a launch, and a workgroup's share for every row."""
    import hip_on_host
    hip_on_host.run("""
    A = 1 << 20
    for rows in (1, (1 << 21) - 1, 1 << 21, (1 << 21) + 1, 1 << 22, (1 << 23) + 5, 1 << 26):
        for cols, rows_a_group in ((300, 4), (1500, 4), (5000, 1), (8193, 1), (33000, 1), (131071, 1)):
            kp = -(-cols // 128) * 128
            fake.fake_reset()
            assert L.gl3_quantize_rows(0, None, A, 30, rows, cols, cols, A, kp, A) == 0, (rows, cols, L.gl3_last_error(None))
            assert fake.fake_most_threads() < 1 << 32 and fake.fake_blocks() * rows_a_group >= rows, (rows, cols)
    for rows, vocab in ((65536, 9), ((1 << 31) - 1, 9), (1, 1 << 30), (1300, 1 << 30)):
        fake.fake_reset()
        assert L.gl3_token_logprobs(0, None, A, 30, rows, vocab, vocab, A, 64, A, A, A, A, A, A, 1 << 62) == 0, (rows, vocab)
        assert fake.fake_most_threads() < 1 << 32 and fake.fake_blocks() >= rows
    for m, n, k in ((1 << 24, 5, 9), (5, 1 << 24, 9), (1 << 19, 1 << 19, 131071), (300, 1 << 30, 4096), (1, (1 << 31) - 1, 100), (8, 1 << 20, 2000)):
        ld = -(-k // 128) * 128
        fake.fake_reset()
        ldy = min(n, 1 << 26)
        r = L.gl3_int8_linear(0, None, A, 30, k, A, ld, A, None, m, n, k, A, 30, n if m == 1 else ldy, A, 1 << 62)
        assert r == (0 if m == 1 or n <= 1 << 26 else hip.E_ARG), (m, n, k, L.gl3_last_error(None))
        assert fake.fake_most_threads() < 1 << 32
    """)


def test_a_plan_that_could_not_be_made_is_told_to_every_thread(hip):
    """The newest such error, also in a thread that has had one of its own, or an operator's before its last call; an operator's own error stays until then."""
    import threading
    L = hip.lib()
    out = C.c_void_p()

    def elsewhere(call):
        t = threading.Thread(target=call)
        t.start()
        t.join()
    fails_here = lambda: L.gl3_create(C.byref(hip.ModelDesc()), C.byref(out))          # (no struct_size)
    fails_there = lambda: L.gl3_create(None, C.byref(out))
    assert fails_here() == hip.E_ARG and L.gl3_last_error(None) == b"gl3_model_desc.struct_size mismatch"
    elsewhere(fails_there)
    assert L.gl3_last_error(None) == b"null argument"
    assert L.gl3_token_logprobs(*logprobs(top=65)) == hip.E_ARG
    elsewhere(fails_there)
    elsewhere(lambda: L.gl3_quantize_rows(*quantize(cols=0)))
    assert b"top" in L.gl3_last_error(None)
    assert L.gl3_token_logprobs(*logprobs(rows=0)) == 0
    elsewhere(fails_there)
    assert L.gl3_last_error(None) == b"null argument"
    assert fails_here() == hip.E_ARG
    elsewhere(lambda: L.gl3_quantize_rows(*quantize(cols=0)))
    assert L.gl3_last_error(None) == b"gl3_model_desc.struct_size mismatch"


WORDS = {"gl3_quantize_rows": dict(type="GL3_TYPE_F32", rows="rows out of range", cols="cols out of range", x="null pointer", codes="null pointer", scale="null pointer", ldx="ldx is less", ldq="ldq",
                                   device="device"),
         "gl3_int8_matmul": dict(k="k out of range", m="m or n", n="m or n", y_type="results are", w="null pointer", w_scale="null pointer", y="null pointer", ldw="ldw", ldy="ldy", a="null pointer",
                                 a_scale="null pointer", lda="lda", device="device"),
         "gl3_int8_linear": dict(x_type="rows are GL3_TYPE_F32", x="x is null", ldx="ldx is less", workspace="workspace too small", bytes="workspace too small"),
         "gl3_token_logprobs": dict(type="logits are GL3_TYPE_F32", rows="rows or vocab", vocab="rows or vocab", top="top out of range", targets="all or none", logprob="all or none", rank="all or none",
                                    logits="logits are null", ld="ld is less", top_ids="top > 0 needs", top_logprobs="top > 0 needs", device="device")}
WORDS["gl3_int8_linear"] = dict(WORDS["gl3_int8_matmul"], **WORDS["gl3_int8_linear"])


def reason(name, kw):
    """A word of the message that names the first argument of kw (all have one that decides)."""
    if name == "gl3_int8_matmul" and "k" in kw and ("lda" in kw or "ldw" in kw):          # (the other one is too short then)
        return "ldw: " if "lda" in kw else "lda: "
    if name == "gl3_int8_linear" and kw == dict(k=129, ldx=129):
        return "ldw: "
    if kw.get("cols") == 131072:
        return "cols out of range"
    key, value = next(iter((k, v) for k, v in kw.items() if k not in ("type", "y_type", "x_type", "m") or len(kw) == 1))
    if key in ("codes", "ldq", "w", "ldw", "a", "lda") and value is not None and value % 16:
        return "start on 16 bytes"
    if isinstance(value, int) and value >= A and key in ("x", "scale", "w_scale", "bias", "y", "a_scale", "targets", "logprob", "rank", "entropy", "top_ids", "top_logprobs") and name + key != "gl3_int8_linearx":
        return "misaligned pointer"
    if key == "workspace" and value is not None:
        return "the workspace starts on 16 bytes"
    return WORDS[name][key]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_a_refusal_names_its_reason(hip, i):
    name, make, kw = BAD[i]
    L = hip.lib()
    assert L.gl3_int8_workspace(0, 0, 0, None, None) == hip.E_ARG and L.gl3_last_error(None) == b"sizes out of range"          # (the message before)
    assert getattr(L, name)(*make(**kw)) == hip.E_ARG
    assert reason(name, kw).encode() in L.gl3_last_error(None), (name, kw, L.gl3_last_error(None))


def test_scales_and_their_derivatives(hip, ops):
    """A scale that requires a gradient is refused where gradients are recorded, and only there; one with a tangent everywhere."""
    from torch.autograd import forward_ad
    codes, scale = torch.zeros(3, 128, dtype=torch.int8), torch.ones(3)
    learned = torch.ones(3, requires_grad=True)
    with pytest.raises(hip.Gl3Error):
        ops.Int8Rows(codes, learned, 5)
    with torch.no_grad():
        assert ops.Int8Rows(codes, learned, 5).rows == 3
    with forward_ad.dual_level():
        with pytest.raises(hip.Gl3Error):
            ops.Int8Rows(codes, forward_ad.make_dual(scale, torch.ones(3)), 5)
        with torch.no_grad(), pytest.raises(hip.Gl3Error):
            ops.Int8Rows(codes, forward_ad.make_dual(scale, torch.ones(3)), 5)
        assert ops.Int8Rows(codes, scale, 5).rows == 3


def test_matrices_that_meet(ops):
    """Against the bytes themselves, for small matrices; of one pitch, or a row and a matrix beside its columns, never too few, and too many only where a row
    would go on in one that the matrix does not have."""
    import itertools
    for rows, rows2, p, pitch, width, q, pitch2, width2 in itertools.product((1, 2, 3), (1, 2, 3), (0, 5), (6, 9), (1, 4, 6), range(0, 24), (6, 9), (2, 5)):
        if (rows > 1 and width > pitch) or (rows2 > 1 and width2 > pitch2):
            continue
        a = {p + r * pitch + c for r in range(rows) for c in range(width)}
        b = {q + r * pitch2 + c for r in range(rows2) for c in range(width2)}
        got = ops._meet(p, rows, pitch, width, q, rows2, pitch2, width2)
        assert got or not a & b, (rows, rows2, p, pitch, width, q, pitch2, width2)
        if rows == rows2 and (rows == 1 or pitch == pitch2):
            assert got == bool(a & b), (rows, p, pitch, width, q, pitch2, width2)
        one, many = ((q, width2), (p, pitch, width, rows)) if rows2 == 1 else ((p, width), (q, pitch2, width2, rows2))
        if min(rows, rows2) == 1 and many[0] <= one[0] and (one[0] - many[0]) % many[1] + one[1] <= many[1]:          # the row stands within one pitch of the matrix
            assert got == bool(a & b), (rows, rows2, p, pitch, width, q, pitch2, width2)
