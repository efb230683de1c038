"""Operators on device memory against plain restatements in 64 bits: codes and scales bit for bit, products and log probabilities within the
roundings that their definitions have."""
import math
import threading
from importlib import import_module

import numpy as np
import pytest
import torch

import __graft_entry__ as ge

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 2.0 ** -24            # half a step of float32
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}          # half the distance of subnormal numbers


@pytest.fixture(scope="module")
def ops(pkg):
    return import_module(ge.PKG_NAME + ".ops")


@pytest.fixture(scope="module")
def hip(pkg):
    return import_module(ge.PKG_NAME + ".hip")


def rng(seed):
    return np.random.default_rng(seed)


# ---- codes ------------------------------------------------------------------------------------------------------------------------------
def codes_of(x):
    """float32 rows -> codes and scales by the definition, in numpy's float32."""
    x = np.asarray(x, np.float32)
    a = np.abs(x).max(1)
    good = np.isfinite(x).all(1)
    live = good & (a >= np.float32(2.0 ** -100))
    safe = np.where(live, a, np.float32(1)).astype(np.float32)
    scale = np.where(live, safe / np.float32(127), np.float32(0)).astype(np.float32)
    scale[~good] = np.nan
    to_code = (np.float32(127) / safe).astype(np.float32)
    with np.errstate(all="ignore"):
        q = np.rint((np.where(live[:, None], x, 0) * to_code[:, None]).astype(np.float32)).clip(-127, 127)
    return q.astype(np.int8), scale


def odd_rows(rows, cols, seed):
    r = rng(seed)
    x = r.standard_normal((rows, cols)).astype(np.float32)
    x[:, r.integers(0, cols, max(1, cols // 200))] *= 25
    x *= np.exp2(r.integers(-20, 20, (rows, 1))).astype(np.float32)
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad,first", [(1, 1, 0, 0), (3, 127, 0, 0), (5, 128, 0, 0), (2, 129, 3, 0), (7, 1000, 0, 0), (4, 1001, 1, 1), (4, 4096, 0, 0), (9, 4096, 8, 3), (600, 130, 0, 0),
                                                  (33, 14336, 0, 0), (2, 20011, 5, 5), (1, 131071, 0, 0)])
def test_codes(ops, dtype, rows, cols, pad, first):
    wide = torch.from_numpy(odd_rows(rows, first + cols + pad, rows * 1000 + cols))
    if dtype == "f16":
        wide.clamp_(-60000, 60000)
    wide = wide.to(NAMES[dtype]).to(DEV)
    x = wide[:, first:first + cols]
    got = ops.quantize_rows(x)
    q, s = codes_of(x.float().cpu().numpy())
    assert got.cols == cols and got.codes.shape == (rows, -(-cols // 128) * 128)
    assert np.array_equal(got.scale.cpu().numpy(), s)
    assert np.array_equal(got.codes.cpu().numpy()[:, :cols], q) and not got.codes[:, cols:].any()
    assert abs(int(q.max())) <= 127 and int(np.abs(q.astype(np.int32)).max()) == 127


def test_codes_of_odd_values(ops):
    x = odd_rows(12, 300, 5)
    x[1] = 0
    x[2] = 0; x[2, 7] = -0.0; x[2, 9] = 2.0 ** -101
    x[3] = 0; x[3, 299] = 2.0 ** -100
    x[4, 5] = np.nan
    x[5, 299] = -np.inf
    x[6] = np.float32(3.4e38)
    x[7] *= np.float32(1e38) / np.abs(x[7]).max(); x[7, 3] = np.float32(-3.4028235e38)
    x[8] = 1.0; x[8, ::2] = -1.0
    x[9] = np.arange(300) * np.float32(0.5) / 149.5 * 127        # halves between codes
    x[10] = 1e-45
    got = ops.quantize_rows(torch.from_numpy(x).to(DEV))
    q, s = codes_of(x)
    assert np.array_equal(got.scale.cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(got.codes.cpu().numpy()[:, :300], q)
    assert np.isnan(s[4]) and np.isnan(s[5]) and s[1] == s[2] == s[10] == 0 and s[3] > 0
    for t in (torch.float16, torch.bfloat16):
        y = torch.from_numpy(x[:6]).to(t)
        got = ops.quantize_rows(y.to(DEV))
        q, s = codes_of(y.float().numpy())
        assert np.array_equal(got.scale.cpu().numpy(), s, equal_nan=True) and np.array_equal(got.codes.cpu().numpy()[:, :300], q)


def test_codes_leave_what_is_beside_them(hip):
    """Wider rows of codes: bytes behind the block, rows behind the last and the scale behind them stay."""
    L = hip.lib()
    x = torch.from_numpy(odd_rows(5, 200, 1)).to(DEV)
    codes = torch.full((7, 400), 77, dtype=torch.int8, device=DEV)
    scale = torch.full((7,), -5.0, device=DEV)
    assert L.gl3_quantize_rows(0, torch.cuda.current_stream().cuda_stream, x.data_ptr(), 0, 5, 200, 200, codes.data_ptr(), 400, scale.data_ptr()) == 0
    q, s = codes_of(x.cpu().numpy())
    c = codes.cpu().numpy()
    assert np.array_equal(c[:5, :200], q) and not c[:5, 200:256].any() and (c[:5, 256:] == 77).all() and (c[5:] == 77).all()
    assert np.array_equal(scale[:5].cpu().numpy(), s) and (scale[5:] == -5).all()


# ---- products ---------------------------------------------------------------------------------------------------------------------------
def int8_rows(ops, rows, cols, seed, extra=0, extreme=False):
    r = rng(seed)
    ld = -(-cols // 128) * 128
    c = np.zeros((rows, ld + extra), np.int8)
    c[:, :cols] = -128 if extreme else r.integers(-127, 128, (rows, cols))
    if extra:
        c[:, ld:] = 99          # behind the block: not the operator's
    s = (r.random(rows) * 0.01 + 1e-4).astype(np.float32)
    return ops.Int8Rows(torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV), cols)


def product64(a, w, bias):
    """The result before its last rounding, and what the float32 roundings before it amount to at most."""
    qa, qw = a.codes[:, :a.cols].cpu().numpy().astype(np.float64), w.codes[:, :w.cols].cpu().numpy().astype(np.float64)
    p = (qa @ qw.T) * a.scale.cpu().numpy().astype(np.float64)[:, None] * w.scale.cpu().numpy().astype(np.float64)          # (integers below 2^53: the sum is exact)
    tol = 3 * EPS * 1.001 * np.abs(p)          # int32 -> float32, times a scale, times the other
    if bias is not None:
        p = p + bias.cpu().numpy().astype(np.float64)
        tol = tol + EPS * (np.abs(p) + tol)
    return p, tol


def check_product(y, a, w, bias=None):
    p, tol = product64(a, w, bias)
    t = y.dtype
    if t != torch.float32:
        tol = tol + HALF_STEP[t] * (np.abs(p) + tol) + LEAST[t]
    err = np.abs(y.double().cpu().numpy() - p)
    assert y.shape == p.shape and (err <= tol).all(), float((err - tol).max())


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 7, 127), (2, 33, 128), (3, 1000, 129), (4, 257, 500), (5, 4096, 640), (8, 100, 1100), (9, 511, 4096), (15, 64, 256), (16, 96, 1024), (17, 130, 1000),
          (31, 2050, 384), (32, 300, 2560), (33, 65, 200), (48, 1024, 896), (63, 63, 63), (64, 512, 768), (65, 129, 1024), (100, 1300, 333), (127, 640, 512), (128, 256, 128), (129, 257, 257),
          (200, 4100, 512), (257, 1000, 1536), (300, 72, 4096), (511, 2049, 130), (1, 5000, 4096), (1, 3, 14336), (2, 4099, 2048), (1, 17, 131071), (20, 40, 131071), (130, 130, 20000)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ops, m, n, k):
    a, w = int8_rows(ops, m, k, m), int8_rows(ops, n, k, n + 1)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    check_product(ops.int8_matmul(a, w), a, w)
    check_product(ops.int8_matmul(a, w, bias, torch.bfloat16), a, w, bias)
    check_product(ops.int8_matmul(a, w, bias, torch.float16), a, w, bias)


@pytest.mark.parametrize("m,n", [(1, 40), (16, 40), (40, 40), (150, 300), (300, 300)])
def test_sums_that_fill_32_bits(ops, m, n):
    a, w = int8_rows(ops, m, 131071, 1, extreme=True), int8_rows(ops, n, 131071, 2, extreme=True)
    y = ops.int8_matmul(a, w)
    check_product(y, a, w)
    assert (y > 0).all()


@pytest.mark.parametrize("m,n,k", [(1, 700, 900), (4, 300, 130), (12, 90, 2000), (40, 333, 700), (140, 400, 1000), (520, 300, 300)])
def test_strides_and_what_lies_beside_the_result(ops, m, n, k):
    """Wider rows of codes on both sides, a result inside a wider buffer: nothing beside it changes."""
    a, w = int8_rows(ops, m, k, 7, extra=128 + 16), int8_rows(ops, n, k, 8, extra=48)
    for t in NAMES.values():
        wide = torch.full((m + 2, n + 5), 3.0, dtype=t, device=DEV)
        y = ops.int8_matmul(a, w, None, t, out=wide[1:m + 1, 2:n + 2])
        check_product(y, a, w)
        assert (wide[0] == 3).all() and (wide[m + 1] == 3).all() and (wide[:, :2] == 3).all() and (wide[:, n + 2:] == 3).all()
    some = ops.int8_matmul(ops.Int8Rows(a.codes[:m], a.scale, k), ops.Int8Rows(w.codes[5:77], w.scale[5:77].clone(), k))
    assert torch.equal(some, ops.int8_matmul(a, w)[:, 5:77])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 300, 130), (1, 2048, 2048), (1, 513, 14336), (1, 40, 131071), (2, 700, 1100), (3, 64, 4096), (5, 1000, 999), (8, 128, 14336), (13, 500, 2560), (16, 33, 640), (17, 33, 640),
                                   (40, 1000, 1111), (150, 700, 2048), (300, 1500, 500)])
def test_linear_is_the_two_calls(ops, m, n, k, dtype):
    wide = torch.from_numpy(odd_rows(m, k + 3, m + k)).to(NAMES[dtype]).to(DEV)
    wide[:, :] = torch.where(torch.isfinite(wide), wide, torch.ones_like(wide))
    w = int8_rows(ops, n, k, 4)
    bias = torch.from_numpy(rng(3).standard_normal(n).astype(np.float32)).to(DEV)
    for x in (wide[:, :k].contiguous(), wide[:, 1:k + 1]):
        a = ops.quantize_rows(x)
        for t in NAMES.values():
            assert torch.equal(ops.int8_linear(x, w, bias, t), ops.int8_matmul(a, w, bias, t))
        assert ops.int8_linear(x, w).dtype == x.dtype
        check_product(ops.int8_linear(x, w, dtype=torch.float32), a, w)


@pytest.mark.parametrize("m", [1, 3, 20, 70, 300])
def test_a_spoiled_row_spoils_its_results_alone(ops, m):
    x = torch.from_numpy(odd_rows(m, 600, 2))
    x[0, 5] = math.inf
    if m > 2:
        x[2, 599] = math.nan
    w = torch.from_numpy(odd_rows(50, 600, 3)).to(DEV)
    w[7, 1] = math.nan
    wr = ops.quantize_rows(w)
    y = ops.int8_linear(x.to(DEV), wr).cpu()
    bad = torch.zeros(m, 50, dtype=torch.bool)
    bad[0] = True
    bad[:, 7] = True
    if m > 2:
        bad[2] = True
    assert torch.equal(torch.isnan(y), bad)
    clean = x.clone(); clean[0] = 0
    if m > 2:
        clean[2] = 0
    assert torch.equal(ops.int8_linear(clean.to(DEV), wr).cpu()[~bad], y[~bad])
    zero = ops.int8_linear(torch.zeros(m, 600, device=DEV), wr).cpu()
    assert (zero[:, :7] == 0).all()


def test_a_row_does_not_depend_on_the_rows_beside_it(ops):
    """A token's results are the same bits alone and in any batch."""
    w = int8_rows(ops, 777, 1500, 9)
    x = torch.from_numpy(odd_rows(260, 1500, 10)).to(DEV)
    whole = ops.int8_linear(x, w)
    for lo, hi in ((0, 1), (3, 5), (10, 18), (0, 16), (100, 133), (1, 66), (60, 260)):
        assert torch.equal(ops.int8_linear(x[lo:hi], w), whole[lo:hi])


# ---- log probabilities --------------------------------------------------------------------------------------------------------------------
def row64(x, t, top):
    """One row by the definition, in 64 bits: logprob, rank, entropy, ids, log probabilities, and the bounds of the float32 evaluation's error."""
    x = np.asarray(x, np.float64)
    V = x.size
    bad = bool((np.isnan(x) | (x == np.inf)).any())
    # order: falling logit, lower id first; NaN and -inf are no alternatives
    usable = np.where(np.isnan(x) | (x == -np.inf))[0].size < V
    cand = np.where(~np.isnan(x) & (x > -np.inf))[0]
    order = cand[np.lexsort((cand, -x[cand]))]
    ids = np.full(top, -1)
    ids[:min(top, order.size)] = order[:top]
    if bad:
        lse = np.nan
    elif not usable:
        lse = -np.inf
    else:
        m = x.max()
        d = x - m
        e = np.exp(d)
        S = e.sum()
        lse = m + math.log(S)
    lp = np.full(V, np.nan) if bad else np.full(V, -np.inf) if lse == -np.inf else d - math.log(S)          # (logits of 1e38 swallow the logarithm)
    if bad:
        H = np.nan
    elif lse == -np.inf:
        H = 0.0
    else:
        p = e / S
        H = float(-(p[p > 0] * lp[p > 0]).sum())
    rank = 0
    if 0 <= t < V and not np.isnan(x[t]):
        rank = 1 + int((x > x[t]).sum() + ((x == x[t]) & (np.arange(V) < t)).sum())
    logprob = 0.0 if t < 0 else np.nan if t >= V else lp[t]
    values = np.where(ids >= 0, lp[ids], -np.inf)
    if bad or lse == -np.inf:
        return logprob, rank, H, ids, values, 0.0, 0.0
    # One term e^d: d rounded (|d| eps), turned into a power of two (the factor and the product: 2 |d| eps), the exponential 2 steps: 4 |d| + 4 half
    # steps.  Sums: at least 64 chains of V / 64 additions, joined by up to 64 more (which scale each side by one more e^d of at most log V + 20).
    fin = p > 0
    spread = float((p[fin] * np.abs(d[fin])).sum())
    rel = EPS * (4 * spread + 4 + V / 64 + 64 + 8 * (math.log(V) + 20))
    tol_lse = rel + EPS * (2 * abs(m) + 4 * abs(math.log(S)) + 2 * abs(lse))
    tol_H = rel * (2 + 2 * spread) + 4 * EPS * (abs(math.log(S)) + spread)
    return logprob, rank, H, ids, values, tol_lse, tol_H


def check_rows(got, logits, targets, top):
    x = logits.float().cpu().numpy()
    t = targets.cpu().numpy() if targets is not None else np.full(x.shape[0], -1)
    for r in range(x.shape[0]):
        logprob, rank, H, ids, values, tol, tol_h = row64(x[r], int(t[r]), top)
        if targets is not None:
            assert int(got.rank[r]) == rank, (r, int(got.rank[r]), rank)
            g = float(got.logprob[r])
            assert (math.isnan(g) and math.isnan(logprob)) or g == logprob or abs(g - logprob) <= tol + 2 * EPS * abs(logprob), (r, g, logprob, tol)
        if got.entropy is not None:
            g = float(got.entropy[r])
            assert (math.isnan(g) and math.isnan(H)) or abs(g - H) <= tol_h, (r, g, H, tol_h)
        if top:
            assert np.array_equal(got.top_ids[r].cpu().numpy(), ids), (r, got.top_ids[r], ids)
            g = got.top_logprobs[r].double().cpu().numpy()
            same = (np.isnan(g) & np.isnan(values)) | (g == values)
            with np.errstate(invalid="ignore"):
                assert (same | (np.abs(g - values) <= tol + 2 * EPS * np.abs(values))).all(), (r, g, values)


def logits_of(rows, vocab, dtype, seed, sigma=3.0, pad=0, first=0):
    r = rng(seed)
    x = r.standard_normal((rows, first + vocab + pad)) * sigma
    x[:, r.integers(0, first + vocab + pad, 5)] += 9
    return torch.from_numpy(x.astype(np.float32)).to(NAMES[dtype]).to(DEV)[:, first:first + vocab]


def targets_of(rows, vocab, seed, low=0):
    return torch.from_numpy(rng(seed).integers(low, vocab, rows).astype(np.int32)).to(DEV)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top,pad,first", [(1, 1, 1, 0, 0), (1, 1, 64, 0, 0), (3, 2, 5, 1, 1), (2, 63, 64, 0, 0), (4, 64, 64, 3, 2), (5, 65, 3, 0, 0), (9, 1003, 3, 0, 0), (8, 1003, 20, 5, 3),
                                                       (3, 4096, 0, 0, 0), (2, 8191, 10, 2, 1), (7, 32064, 20, 8, 0), (1, 50257, 64, 0, 0), (2, 128256, 5, 0, 0), (1, 151936, 20, 7, 5), (40, 3001, 33, 1, 0),
                                                       (300, 700, 7, 0, 0), (1500, 130, 2, 0, 0)])
def test_logprobs(ops, rows, vocab, top, pad, first, dtype):
    x = logits_of(rows, vocab, dtype, rows * 7 + vocab, pad=pad, first=first)
    t = targets_of(rows, vocab, 3, low=-1)
    t[0] = int(x[0].float().argmax())
    check_rows(ops.token_logprobs(x, t, top), x, t, top)


def test_logprobs_parts_alone(ops):
    """Every output is what it is whether the others are asked for or not."""
    x, t = logits_of(6, 9001, "f32", 1), targets_of(6, 9001, 2)
    full = ops.token_logprobs(x, t, 11)
    only = ops.token_logprobs(x, t, 0, entropy=False)
    assert only.entropy is None and only.top_ids is None and torch.equal(only.logprob, full.logprob) and torch.equal(only.rank, full.rank)
    only = ops.token_logprobs(x, None, 0)
    assert only.logprob is None and only.rank is None and torch.equal(only.entropy, full.entropy)
    only = ops.token_logprobs(x, None, 11, entropy=False)
    assert torch.equal(only.top_ids, full.top_ids) and torch.equal(only.top_logprobs, full.top_logprobs)
    nothing = ops.token_logprobs(x, None, 0, entropy=False)
    assert all(v is None for v in nothing)
    for lo, hi in ((0, 1), (2, 6)):
        part = ops.token_logprobs(x[lo:hi], t[lo:hi].clone(), 11)
        assert torch.equal(part.top_ids, full.top_ids[lo:hi]) and torch.equal(part.rank, full.rank[lo:hi])
        check_rows(part, x[lo:hi], t[lo:hi], 11)


@pytest.mark.parametrize("vocab", [5, 129, 3000, 70001])
def test_ties_go_to_the_lowest_id(ops, vocab):
    r = rng(vocab)
    x = r.integers(-2, 3, (12, vocab)).astype(np.float32)
    x[1] = 0; x[2] = -0.0; x[2, ::3] = 0.0
    x[3] = np.arange(vocab)                  # every token better than the ones before it
    x[4] = -np.arange(vocab)
    x[5, :] = -np.inf; x[5, vocab // 2:] = 1
    x[6] = 1; x[6, -1] = 2
    x[7] = 1; x[7, 0] = 2
    t = targets_of(12, vocab, 4)
    t[8], t[9] = 0, vocab - 1
    for dtype in NAMES:
        y = torch.from_numpy(x).to(NAMES[dtype]).to(DEV)
        if dtype != "f32":
            y[3:5].clamp_(-2000, 2000)
        check_rows(ops.token_logprobs(y, t, 21), y, t, 21)


@pytest.mark.parametrize("vocab", [7, 300, 5003, 40000])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masks(ops, vocab, dtype):
    r = rng(vocab)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[dtype]
    x = (r.standard_normal((16, vocab)) * 2).astype(np.float32)
    x[0] = -np.inf                                         # nothing left
    x[1] = -np.inf; x[1, vocab - 1] = 0.5                  # one token left
    x[2, r.random(vocab) < 0.9] = -np.inf
    x[3] = low                                             # masked with the type's lowest value instead
    x[4] = low; x[4, vocab // 3] = -1
    x[5, 0] = np.inf
    x[6, vocab // 2] = np.nan
    x[7] = np.nan
    x[8] = -np.inf; x[8, 0] = np.nan
    x[9] = np.inf
    x[10] *= 100 if dtype == "f16" else 1e30               # one token holds it all
    x[11] = 7.25
    x[12, :vocab // 2] = -np.inf
    x[13, vocab // 2:] = -np.inf
    x[14] = x[14] * 0.01 - 9000
    y = torch.from_numpy(x).to(NAMES[dtype]).to(DEV)
    t = targets_of(16, vocab, 6)
    t[1] = vocab - 1; t[5] = 0; t[6] = vocab // 2; t[12] = 0; t[15] = vocab          # the last: no such token
    check_rows(ops.token_logprobs(y, t, 9), y, t, 9)
    t = torch.full((16,), -7, dtype=torch.int32, device=DEV)
    got = ops.token_logprobs(y, t, 2)
    assert (got.logprob == 0).all() and (got.rank == 0).all()
    t[:] = 2 ** 31 - 1
    got = ops.token_logprobs(y, t, 2)
    assert torch.isnan(got.logprob).all() and (got.rank == 0).all()


def test_certain_rows_keep_small_entropies(ops):
    """Entropies far below 1: no cancellation against the size of the logits."""
    x = torch.full((3, 5000), -30.0)
    x[0, 17], x[1, 17], x[2, 4999] = 0.0, 60.0, -18.0
    x = x.to(DEV)
    got = ops.token_logprobs(x, torch.tensor([17, 17, 4999], dtype=torch.int32, device=DEV), 2)
    check_rows(got, x, torch.tensor([17, 17, 4999]), 2)
    assert float(got.entropy[1]) < 1e-30 and float(got.logprob[1]) == 0.0


# ---- as programs use them -------------------------------------------------------------------------------------------------------------------
def test_hidden_rows_to_log_probabilities(ops):
    """A head in 8 bits and what is read from its logits, on a stream of its own, against 64 bits all the way."""
    W = torch.from_numpy(rng(1).standard_normal((4001, 512)).astype(np.float32) * 0.05).to(DEV)
    s = torch.cuda.Stream()
    for m in (1, 5, 70, 200):
        x = torch.from_numpy(rng(m).standard_normal((m, 512)).astype(np.float32)).to(DEV)
        t = targets_of(m, 4001, m)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            w = ops.quantize_rows(W)
            logits = ops.int8_linear(x, w)
            got = ops.token_logprobs(logits, t, 8)
        torch.cuda.current_stream().wait_stream(s)
        check_product(logits, ops.quantize_rows(x), w)
        check_rows(got, logits, t, 8)


def test_captured_and_replayed(ops):
    """The run of them in a graph: replays with other inputs, with eager work of the same operators between them."""
    w = int8_rows(ops, 3001, 768, 1)
    for m in (1, 6, 40, 150):
        x, t = torch.zeros(m, 768, device=DEV), torch.zeros(m, dtype=torch.int32, device=DEV)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.token_logprobs(ops.int8_linear(x, w), t, 5)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            logits = ops.int8_linear(x, w)
            got = ops.token_logprobs(logits, t, 5)
        for i in range(4):
            x.copy_(torch.from_numpy(odd_rows(m, 768, i)))
            t.copy_(targets_of(m, 3001, i))
            g.replay()
            want_logits = ops.int8_linear(x, w)
            want = ops.token_logprobs(want_logits, t, 5)
            torch.cuda.synchronize()
            assert torch.equal(logits, want_logits)
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_two_threads(ops):
    """Calls at the same time, each on a stream of its own."""
    w = int8_rows(ops, 2000, 640, 1)
    xs = [torch.from_numpy(odd_rows(3 + 30 * i, 640, i)).to(DEV) for i in range(4)]
    want = [ops.token_logprobs(ops.int8_linear(x, w), None, 4) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = ops.token_logprobs(ops.int8_linear(xs[i], w), None, 4)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(got.top_ids, want[i].top_ids) and torch.equal(got.top_logprobs, want[i].top_logprobs) and torch.equal(got.entropy, want[i].entropy)):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong


def test_empty(ops):
    w = int8_rows(ops, 10, 100, 1)
    assert ops.quantize_rows(torch.zeros(0, 100, device=DEV)).codes.shape == (0, 128)
    assert ops.int8_linear(torch.zeros(0, 100, device=DEV), w).shape == (0, 10)
    assert ops.int8_matmul(w, ops.Int8Rows(w.codes[:0], w.scale[:0], 100)).shape == (10, 0)
    got = ops.token_logprobs(torch.zeros(0, 9, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), 3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)


def test_refusals(ops, hip):
    x = torch.zeros(4, 100, device=DEV)
    w = int8_rows(ops, 10, 100, 1)
    for call in (lambda: ops.quantize_rows(x.t()), lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(x[0]), lambda: ops.quantize_rows(torch.zeros(3, 0, device=DEV)),
                 lambda: ops.int8_linear(x[:, :99], w), lambda: ops.int8_linear(x, w, torch.zeros(9, device=DEV)), lambda: ops.int8_linear(x, w, torch.zeros(10)),
                 lambda: ops.int8_linear(x, w, None, torch.float64), lambda: ops.int8_linear(x, w, None, out=torch.zeros(4, 11, device=DEV)),
                 lambda: ops.int8_linear(x, ops.Int8Rows(w.codes[:, :100], w.scale, 100)), lambda: ops.int8_linear(x, ops.Int8Rows(w.codes, w.scale[:9], 100)),
                 lambda: ops.int8_linear(x, ops.Int8Rows(w.codes.cpu(), w.scale, 100)), lambda: ops.int8_linear(x, ops.Int8Rows(w.codes.float(), w.scale, 100)),
                 lambda: ops.int8_linear(x.clone().requires_grad_(), w), lambda: ops.token_logprobs(x, torch.zeros(4, dtype=torch.int64, device=DEV)),
                 lambda: ops.token_logprobs(x, torch.zeros(3, dtype=torch.int32, device=DEV)), lambda: ops.token_logprobs(x, top=65), lambda: ops.token_logprobs(x, top=-1),
                 lambda: ops.token_logprobs(x.t()), lambda: ops.token_logprobs(x[:, :0])):
        with pytest.raises(hip.Gl3Error):
            call()
    wide = torch.zeros(10, 128 + 8, dtype=torch.int8, device=DEV)          # rows of codes that do not start on 16 bytes
    with pytest.raises(hip.Gl3Error):
        ops.int8_linear(x, ops.Int8Rows(wide[:, :128], w.scale, 100))
    L = hip.lib()
    assert L.gl3_quantize_rows(99, None, x.data_ptr(), 0, 4, 100, 100, w.codes.data_ptr(), 128, w.scale.data_ptr()) == hip.E_ARG and b"device" in L.gl3_last_error(None)
    with torch.no_grad():
        assert ops.int8_linear(x.clone().requires_grad_(), w).shape == (4, 10)
