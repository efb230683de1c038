"""Operators on device memory where their sizes change the kernel: every tile and strip with few and many stages, rows of every length, launches in
pieces, offsets that pass 32 bits, another stream's and the default stream's calls."""
from importlib import import_module

import numpy as np
import pytest
import torch

import __graft_entry__ as ge
from test_ops_gpu import DEV, NAMES, check_product, check_rows, codes_of, int8_rows, odd_rows, rng, targets_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return import_module(ge.PKG_NAME + ".ops")


@pytest.fixture(scope="module")
def hip(pkg):
    return import_module(ge.PKG_NAME + ".hip")


# ---- products: m x n chooses the kernel (a few tokens: strips; else the tile), k the number of stages of 128 columns, fewer and more than the rings hold ----
@pytest.mark.parametrize("stages", [1, 2, 3, 4, 5, 7])
@pytest.mark.parametrize("m,n", [(3, 700), (5, 8203), (17, 700), (17, 33000), (100, 700), (33, 16385), (70, 16390), (33, 33000), (31, 20001), (8385, 842), (390, 16390)])
def test_stages(ops, m, n, stages):
    k = stages * 128 - (stages * 37 + m) % 128
    a, w = int8_rows(ops, m, k, m), int8_rows(ops, n, k, n + 1)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    check_product(ops.int8_matmul(a, w), a, w)
    check_product(ops.int8_matmul(a, w, bias, torch.bfloat16), a, w, bias)


@pytest.mark.parametrize("m,n,k", [(40, 300, 9000), (33, 64, 1024), (64, 1024, 4096), (1, 20, 131071), (17, 64, 8192), (24, 257, 30000), (65, 1000, 14336), (130, 500, 5000), (257, 513, 4100), (300, 1500, 1025), (35, 1189, 6600), (142, 1000, 30000),
                                   (512, 1024, 10000), (2758, 66, 4352)])
def test_sums_in_parts(ops, m, n, k):
    """Few tiles and a long k: every part's sums meet, beside each of the epilogue's forms."""
    a, w = int8_rows(ops, m, k, m, extra=16), int8_rows(ops, n, k, n + 1)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    for t in NAMES.values():
        wide = torch.full((m + 1, n + 3), 3.0, dtype=t, device=DEV)
        check_product(ops.int8_matmul(a, w, bias, t, out=wide[:m, 1:n + 1]), a, w, bias)
        assert (wide[m] == 3).all() and (wide[:, 0] == 3).all() and (wide[:, n + 1:] == 3).all()
    x = torch.from_numpy(odd_rows(m, k, 5)).to(DEV)
    y = ops.int8_linear(x, w)
    assert torch.equal(y, ops.int8_matmul(ops.quantize_rows(x), w))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = ops.int8_linear(x, w)
    for i in range(3):
        x.copy_(torch.from_numpy(odd_rows(m, k, 6 + i)))
        g.replay()
        y = ops.int8_linear(x, w)
        torch.cuda.synchronize()
        assert torch.equal(z, y)


@pytest.mark.parametrize("m,n,k", [(1, 8203, 1500), (1, 16411, 2500), (2, 8203, 1537), (4, 9001, 2600), (5, 8203, 2560), (11, 8200, 5000), (16, 8193, 6016), (3, 8192, 4097), (30, 8100, 1100), (18, 300, 384)])
def test_strips(ops, m, n, k):
    a, w = int8_rows(ops, m, k, m, extra=32), int8_rows(ops, n, k, n + 1, extra=16)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    check_product(ops.int8_matmul(a, w), a, w)
    check_product(ops.int8_matmul(a, w, bias, torch.float16), a, w, bias)


@pytest.mark.parametrize("n,k", [(9001, 130), (9001, 8192), (9001, 8193), (20, 16384), (20, 16385), (32768, 300), (32769, 300), (5, 1)])
def test_one_token(ops, n, k):
    w = int8_rows(ops, n, k, 4)
    for t in NAMES.values():
        x = torch.from_numpy(odd_rows(1, k, k)).to(t).to(DEV)
        x = torch.where(torch.isfinite(x), x, torch.ones_like(x))
        a = ops.quantize_rows(x)
        y = ops.int8_linear(x, w, dtype=torch.float32)
        assert torch.equal(y, ops.int8_matmul(a, w))
        check_product(y, a, w)


@pytest.mark.parametrize("m,n,k", [(2, 100, 8192), (2, 100, 8193), (3, 100, 4096), (4, 100, 4097), (5, 100, 2048), (8, 33, 2049), (7, 700, 1), (2, 9001, 4096), (2, 9001, 4097), (4, 9001, 2048),
                                   (3, 9001, 2049), (8, 9001, 300), (6, 9001, 1000), (8, 32768, 130), (8, 32769, 130), (4, 16384, 130), (4, 16385, 130), (8, 8192, 130), (8, 8193, 130), (9, 100, 300)])
def test_a_few_tokens(ops, m, n, k):
    w = int8_rows(ops, n, k, 4)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    for t in NAMES.values():
        x = torch.from_numpy(odd_rows(m, k + 5, k)).to(t).to(DEV)
        x = torch.where(torch.isfinite(x), x, torch.ones_like(x))
        x[m - 1, 3 + k // 2] = float("nan")
        x[0, 4:] = 0 if m > 1 else x[0, 4:]
        for v in (x[:, 4:k + 4], x[:, 3:k + 3].contiguous()):
            wide = torch.full((m + 2, n + 3), 3.0, device=DEV)
            y = ops.int8_linear(v, w, bias, torch.float32, out=wide[1:m + 1, 2:n + 2])
            a = ops.quantize_rows(v)
            assert torch.equal(y.nan_to_num(7e30), ops.int8_matmul(a, w, bias).nan_to_num(7e30)) and bool(torch.isnan(y[m - 1]).all()) == bool(torch.isnan(v[m - 1]).any())          # (one column: the NaN lies beside one of the two views)
            check_product(y[:m - 1], ops.Int8Rows(a.codes[:m - 1], a.scale[:m - 1], k), w, bias)
            assert (wide[0] == 3).all() and (wide[m + 1] == 3).all() and (wide[:, :2] == 3).all() and (wide[:, n + 2:] == 3).all()


@pytest.mark.parametrize("rows,cols", [(3000, 700), (3000, 2048), (3000, 2049), (70, 5000), (70, 8192), (70, 8193), (64, 8192), (3, 9000), (2, 32768), (2, 32769), (3, 512), (3, 513), (5, 2049)])
def test_codes_of_rows_of_every_length(ops, rows, cols):
    for dtype in NAMES:
        x = torch.from_numpy(odd_rows(rows, cols + 1, rows + cols))
        if dtype == "f16":
            x.clamp_(-60000, 60000)
        x = x.to(NAMES[dtype])[:, 1:]
        got = ops.quantize_rows(x.to(DEV))
        q, s = codes_of(x.float().numpy())
        assert np.array_equal(got.scale.cpu().numpy(), s) and np.array_equal(got.codes.cpu().numpy()[:, :cols], q) and not got.codes[:, cols:].any()


@pytest.mark.parametrize("m,n,k", [(65536 + 130, 40, 70), (1, 262144 + 77, 130), (3, 262144 + 77, 130), (40, 262144 + 77, 130)])
def test_products_in_pieces(ops, m, n, k):
    a, w = int8_rows(ops, m, k, 1), int8_rows(ops, n, k, 2)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    check_product(ops.int8_matmul(a, w, bias), a, w, bias)


def test_more_rows_of_logits_than_a_launch_takes(ops):
    rows, vocab = 65535 + 1200, 9
    x = torch.from_numpy(rng(1).standard_normal((rows, vocab)).astype(np.float32)).to(DEV)
    t = targets_of(rows, vocab, 2, low=-1)
    got = ops.token_logprobs(x, t, 3)
    for lo, hi in ((0, 300), (65400, 65700), (rows - 300, rows)):
        check_rows(type(got)(*(v[lo:hi] for v in got)), x[lo:hi], t[lo:hi], 3)
    lp = torch.log_softmax(x.double(), 1)
    assert torch.allclose(got.top_logprobs[:, 0].double(), lp.max(1).values, rtol=0, atol=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 3001, 40000])
def test_nan_of_every_kind(ops, dtype, vocab):
    """Quiet and signalling NaN, of either sign, beside the largest logits: no alternative, and the others' order is what it is without them."""
    x = torch.from_numpy((rng(vocab).standard_normal((8, vocab)) * 3).astype(np.float32)).to(NAMES[dtype])
    whole, kinds = {"f32": (torch.int32, [0x7fc00000, 0x7f800001, -0x400000, -0x7fffff]), "f16": (torch.int16, [0x7e00, 0x7c01, -0x200, -0x3ff]), "bf16": (torch.int16, [0x7fc0, 0x7f81, -0x40, -0x7f])}[dtype]
    bits = x.view(whole)
    for r in range(8):
        for i, at in enumerate(torch.topk(x[r].float(), 12).indices.tolist()):
            if i % 2 and at ^ 1 < vocab:
                bits[r, at ^ 1] = kinds[(r + i) % 4]          # beside a large one, in its vector
        bits[r, r] = kinds[r % 4]
    assert torch.isnan(x).any(1).all()
    x = x.to(DEV)
    t = targets_of(8, vocab, 3)
    check_rows(ops.token_logprobs(x, t, 11), x, t, 11)


# ---- offsets that pass 32 bits: the last rows are what they are on their own ----
def test_results_past_32_bits(ops):
    m, n = 16800, 128256          # 2.15 G results
    a = ops.Int8Rows(torch.randint(-127, 128, (m, 128), dtype=torch.int8, device=DEV), torch.rand(m, device=DEV), 128)
    w = ops.Int8Rows(torch.randint(-127, 128, (n, 128), dtype=torch.int8, device=DEV), torch.rand(n, device=DEV), 128)
    y = ops.int8_matmul(a, w, None, torch.bfloat16)
    for lo in (0, 8000, m - 70):
        part = ops.Int8Rows(a.codes[lo:lo + 70], a.scale[lo:lo + 70], 128)
        assert torch.equal(y[lo:lo + 70], ops.int8_matmul(part, w, None, torch.bfloat16))
    part = ops.Int8Rows(a.codes[m - 5:], a.scale[m - 5:], 128)
    check_product(y[m - 5:], part, w)
    # rows of logits, and rows to be quantised, that start behind 2^31 elements
    t = torch.full((m,), 77, dtype=torch.int32, device=DEV)
    got = ops.token_logprobs(y, t, 2)
    for lo in (0, m - 3):
        check_rows(type(got)(*(v[lo:lo + 3] for v in got)), y[lo:lo + 3], t[lo:lo + 3], 2)
    q = ops.quantize_rows(y)
    last = ops.quantize_rows(y[m - 40:])
    assert torch.equal(q.codes[m - 40:], last.codes) and torch.equal(q.scale[m - 40:], last.scale)
    c, s = codes_of(y[m - 2:].float().cpu().numpy())
    assert np.array_equal(q.codes[m - 2:].cpu().numpy()[:, :n], c) and np.array_equal(q.scale[m - 2:].cpu().numpy(), s)


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_weights_past_32_bits(ops, m):
    n, k = 262000, 8200          # 2.18 GB of codes
    w = ops.Int8Rows(torch.randint(-127, 128, (n, 8320), dtype=torch.int8, device=DEV), torch.rand(n, device=DEV), k)
    w.codes[:, k:] = 0
    x = torch.randn(m, k, device=DEV)
    y = ops.int8_linear(x, w)
    for lo in (0, n - 300):
        part = ops.Int8Rows(w.codes[lo:lo + 300], w.scale[lo:lo + 300].clone(), k)
        assert torch.equal(y[:, lo:lo + 300], ops.int8_linear(x, part))
    check_product(y[:, n - 300:], ops.quantize_rows(x), ops.Int8Rows(w.codes[n - 300:], w.scale[n - 300:].clone(), k))


# ---- calls ----
def test_the_default_stream(ops, hip):
    """Stream NULL from C, with a workspace of the caller."""
    import ctypes as C
    L = hip.lib()
    m, n, k, vocab = 7, 300, 200, 300
    x = torch.from_numpy(odd_rows(m, k, 1)).to(DEV)
    w = int8_rows(ops, n, k, 2)
    nbytes, need = C.c_uint64(), C.c_uint64()
    assert L.gl3_int8_workspace(m, n, k, None, C.byref(nbytes)) == 0 and L.gl3_logprobs_workspace(m, vocab, 5, C.byref(need)) == 0
    ws = torch.empty(max(nbytes.value, need.value, 16), dtype=torch.uint8, device=DEV)
    y = torch.empty(m, n, device=DEV)
    t = torch.zeros(m, dtype=torch.int32, device=DEV)
    lp, rank, ids, values = torch.empty(m, device=DEV), torch.empty(m, dtype=torch.int32, device=DEV), torch.empty(m, 5, dtype=torch.int32, device=DEV), torch.empty(m, 5, device=DEV)
    torch.cuda.synchronize()
    assert L.gl3_int8_linear(0, None, x.data_ptr(), 0, k, w.codes.data_ptr(), w.ld, w.scale.data_ptr(), None, m, n, k, y.data_ptr(), 0, n, ws.data_ptr(), nbytes.value) == 0
    assert L.gl3_token_logprobs(0, None, y.data_ptr(), 0, m, vocab, n, t.data_ptr(), 5, lp.data_ptr(), rank.data_ptr(), None, ids.data_ptr(), values.data_ptr(), ws.data_ptr(), need.value) == 0
    torch.cuda.synchronize()
    check_product(y, ops.quantize_rows(x), w)
    want = ops.token_logprobs(y, t, 5)
    assert torch.equal(lp, want.logprob) and torch.equal(rank, want.rank) and torch.equal(ids, want.top_ids) and torch.equal(values, want.top_logprobs)


def test_rows_that_overlap_are_refused(ops, hip):
    """A broadcast row and sliding windows have a stride below a row's length."""
    w = int8_rows(ops, 10, 100, 1)
    x = torch.randn(1, 100, device=DEV)
    for bad in (x.expand(4, 100), torch.randn(400, device=DEV).as_strided((4, 100), (50, 1))):
        for call in (lambda: ops.quantize_rows(bad), lambda: ops.int8_linear(bad, w), lambda: ops.token_logprobs(bad)):
            with pytest.raises(hip.Gl3Error):
                call()
    with pytest.raises(hip.Gl3Error):
        ops.int8_linear(torch.randn(4, 100, device=DEV), w, dtype=torch.float32, out=torch.zeros(1, 10, device=DEV).expand(4, 10))
    assert ops.int8_linear(x, w).shape == (1, 10)


def test_two_graphs_with_workspaces_of_their_own(ops):
    """Replayed at the same time on two streams, each as it is alone."""
    w = int8_rows(ops, 3001, 768, 1)
    graphs, outs, xs = [], [], []
    for i in range(2):
        x = torch.from_numpy(odd_rows(60, 768, i)).to(DEV)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.token_logprobs(ops.int8_linear(x, w), None, 5)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.token_logprobs(ops.int8_linear(x, w), None, 5))
        graphs.append(g); xs.append(x)
    want = [ops.token_logprobs(ops.int8_linear(x, w), None, 5) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got.top_ids, ref.top_ids) and torch.equal(got.top_logprobs, ref.top_logprobs) and torch.equal(got.entropy, ref.entropy)


def test_no_gradient_is_lost_in_silence(ops, hip):
    w, x = int8_rows(ops, 10, 100, 1), torch.randn(4, 100, device=DEV)
    bias, out = torch.zeros(10, device=DEV, requires_grad=True), torch.zeros(4, 10, device=DEV, requires_grad=True)
    for call in (lambda: ops.int8_linear(x, w, bias), lambda: ops.int8_matmul(ops.quantize_rows(x), w, bias), lambda: ops.int8_linear(x, w, out=out),
                 lambda: ops.Int8Rows(w.codes, w.scale.clone().requires_grad_(), 100), lambda: ops.token_logprobs(out), lambda: ops.quantize_rows(out)):
        with pytest.raises(hip.Gl3Error):
            call()
    with torch.no_grad():
        assert torch.equal(ops.int8_linear(x, w, bias, out=out), ops.int8_linear(x, w))


def test_no_tangent_is_lost_in_silence(ops, hip):
    """Forward-mode derivatives, of every float input, also where gradients are off; and scales that require a gradient only after they have been wrapped."""
    from torch.autograd import forward_ad
    w, x, bias = int8_rows(ops, 10, 100, 1), torch.randn(4, 100, device=DEV), torch.zeros(10, device=DEV)
    a = ops.quantize_rows(x)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.quantize_rows(dual(x)), lambda: ops.int8_linear(dual(x), w), lambda: ops.int8_linear(x, w, dual(bias)), lambda: ops.int8_matmul(a, w, dual(bias)),
                     lambda: ops.token_logprobs(dual(x)), lambda: ops.int8_linear(x, w, out=dual(torch.zeros(4, 10, device=DEV))), lambda: ops.Int8Rows(w.codes, dual(w.scale), 100)):
            with pytest.raises(hip.Gl3Error):
                call()
            with torch.no_grad(), pytest.raises(hip.Gl3Error):
                call()
        assert torch.equal(ops.int8_linear(x, w), ops.int8_matmul(a, w))          # (nothing here has one)
    with pytest.raises(hip.Gl3Error):
        torch.func.jvp(lambda t: ops.token_logprobs(t).entropy, (x,), (x,))
    want = ops.int8_linear(x, w)
    for rows in (w, a):
        rows.scale.requires_grad_()
        with pytest.raises(hip.Gl3Error):
            ops.int8_matmul(a, w)
        with torch.no_grad():
            assert torch.equal(ops.int8_matmul(a, w), want)
        rows.scale.requires_grad_(False)
    w.scale.requires_grad_()
    with pytest.raises(hip.Gl3Error):
        ops.int8_linear(x, w)
    with torch.no_grad():
        assert torch.equal(ops.int8_linear(x, w), want)


def test_a_saved_tensor_that_is_written_is_noticed(ops):
    """out= is a write in place: a backward pass that has saved the tensor refuses it, as for torch's own."""
    w, x = int8_rows(ops, 10, 100, 1), torch.randn(4, 100, device=DEV)
    for call in (lambda out: ops.int8_linear(x, w, out=out), lambda out: ops.int8_matmul(ops.quantize_rows(x), w, out=out)):
        wide = torch.ones(6, 12, device=DEV)
        g = torch.ones(6, 12, device=DEV, requires_grad=True)
        y = (g * wide).sum()          # saves wide
        call(wide[1:5, 1:11])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        out = torch.zeros(4, 10, device=DEV)
        assert torch.equal(ops.int8_linear(x, w, out=out), ops.int8_linear(x, w))


def test_a_result_over_an_input_is_refused(ops, hip):
    """Results over x or the bias; columns of one buffer side by side are apart."""
    for m in (1, 3, 40, 300):
        buffer = torch.randn(m, 400, device=DEV)
        x = buffer[:, :128]
        w = int8_rows(ops, 128, 128, 1)
        want = ops.int8_linear(x.clone(), w)
        for out in (x, buffer[:, 100:228], buffer[:, :128]):
            with pytest.raises(hip.Gl3Error):
                ops.int8_linear(x, w, out=out)
        bias = buffer.view(-1)[200:328]
        with pytest.raises(hip.Gl3Error):
            ops.int8_linear(x.clone(), w, bias, out=buffer[:, 180:308])
        with pytest.raises(hip.Gl3Error):
            ops.int8_matmul(ops.quantize_rows(x), w, bias, out=buffer[:, 180:308])
        assert torch.equal(ops.int8_linear(x, w, out=buffer[:, 128:256]), want) and torch.equal(buffer[:, 128:256], want)
        assert torch.equal(ops.int8_linear(x, w, out=buffer[:, 272:400]), want)
        bias = buffer[m // 2, 128:256]          # beside the columns that are written
        want = ops.int8_linear(x, w, bias.clone())
        assert torch.equal(ops.int8_linear(x, w, bias, out=buffer[:, 256:384]), want)
    assert ops.int8_linear(buffer[:0, :128], w, out=buffer[:0, :128]).shape == (0, 128)


def test_a_pending_error_is_not_an_operators(ops, hip):
    """A failed HIP call of the thread that the program has dealt with: the operators behind it succeed and are right."""
    L = hip.lib()
    m, n, k, vocab = 20, 70, 300, 70000
    x, w, logits = torch.randn(m, k, device=DEV), int8_rows(ops, n, k, 1), torch.randn(3, vocab, device=DEV)
    want, scores = ops.int8_linear(x, w), ops.token_logprobs(logits, None, 4)
    y, ent, ids, values = torch.zeros(m, n, device=DEV), torch.zeros(3, device=DEV), torch.zeros(3, 4, dtype=torch.int32, device=DEV), torch.zeros(3, 4, device=DEV)
    codes, scale, ws = torch.zeros(m, 384, dtype=torch.int8, device=DEV), torch.zeros(m, device=DEV), torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    s = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    p = lambda t: t.data_ptr()
    calls = [lambda: L.gl3_quantize_rows(0, s, p(x), 0, m, k, k, p(codes), 384, p(scale)),
             lambda: L.gl3_int8_linear(0, s, p(x), 0, k, p(w.codes), w.ld, p(w.scale), None, m, n, k, p(y), 0, n, p(ws), ws.numel()),
             lambda: L.gl3_token_logprobs(0, s, p(logits), 0, 3, vocab, vocab, None, 4, None, None, p(ent), p(ids), p(values), p(ws), ws.numel())]
    try:
        for call in calls:
            assert L.hipSetDevice(1000) != 0          # pending until somebody asks
            assert call() == 0, L.gl3_last_error(None)
    finally:
        L.hipGetLastError()
    torch.cuda.synchronize()
    a = ops.quantize_rows(x)
    assert torch.equal(codes, a.codes) and torch.equal(scale, a.scale) and torch.equal(y, want)
    assert torch.equal(ent, scores.entropy) and torch.equal(ids, scores.top_ids) and torch.equal(values, scores.top_logprobs)
