"""Scores of given tokens (gl3_forward_score) against the logits that the same plans hand out, and the output head in 8-bit integers
(GL3_FLAG_INT8_HEAD) against its definition and against the head it replaces."""
import math
import os
import subprocess
from importlib import import_module

import numpy as np
import pytest

import __graft_entry__ as ge
import test_kugadra_gpu as kugadra
import test_noditar_gpu as noditar
from test_ops_gpu import codes_of, row64

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
RUN = os.path.join(ge.ROOT, "tools", "gl3_run")


@pytest.fixture(scope="module")
def hy(pkg):
    return import_module(ge.PKG_NAME + ".hybrid")


@pytest.fixture(scope="module")
def plans(pkg):
    return import_module(ge.PKG_NAME + ".plan")


@pytest.fixture(scope="module")
def hip(pkg):
    return import_module(ge.PKG_NAME + ".hip")


def check(score, logits, targets, top):
    """score: dict of gl3_forward_score; logits: the same rows' logits, float32."""
    for r, x in enumerate(logits):
        t = -1 if targets is None else int(targets[r])
        logprob, rank, H, ids, values, tol, tol_h = row64(x, t, top)
        if targets is not None:
            assert score["ranks"][r] == rank and abs(float(score["logprobs"][r]) - logprob) <= tol + 2 * EPS * abs(logprob), (r, score["logprobs"][r], logprob)
        assert abs(float(score["entropies"][r]) - H) <= tol_h
        if top:
            assert np.array_equal(score["top_ids"][r], ids)
            with np.errstate(invalid="ignore"):
                assert ((score["top_logprobs"][r] == values) | (np.abs(score["top_logprobs"][r] - values) <= tol + 2 * EPS * np.abs(values))).all()


@pytest.mark.parametrize("name", ["tiny-llama", "tiny-qwen3"])
def test_block_quantised_plans(pkg, plans, name):
    if name not in pkg.synth.CONFIGS:
        pytest.skip("no such configuration")
    model = pkg.synth.make_numpy(pkg.synth.CONFIGS[name], seed=3)
    vocab = model.cfg.vocab
    toks = np.asarray(pkg.javarand.bench_tokens(vocab, 13), np.int32)
    plan = plans.HipMasterPlan(model)
    logits = np.stack([plan.forward_decode(int(t), p) for p, t in enumerate(toks)])
    plan.freeTornadoExecutionPlan()
    plan = plans.HipMasterPlan.initializeTornadoVMPlan(model, prefill_batch_size=4)
    for want, top in ((np.arange(12), 5), ([0, 5, 6, 12], 0), ([12], 64), ([], 3)):
        want = np.asarray(want, np.int32)
        targets = np.where(want + 1 < toks.size, toks[np.minimum(want + 1, toks.size - 1)], -1)
        got = plan.score(toks, 0, want, targets, top)
        check(got, logits[want], targets, top)
        got = plan.score(toks, 0, want, None, top)
        assert got["logprobs"] is None and got["ranks"] is None
        check(got, logits[want], None, top)
    assert np.array_equal(plan.forward_decode(int(toks[0]), 0), logits[0])
    plan.freeTornadoExecutionPlan()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("int8", [False, True])
def test_layer_list_plans(hy, tmp_path, dtype, int8):
    """Prompts longer than a portion and than a group of wanted rows, single tokens behind them, two slots."""
    m = noditar.Model(hy, tmp_path, noditar.config([noditar.att(), noditar.ssm(), noditar.lat()]), 5)
    toks = noditar.tokens_for(m.cfg, 75)
    kw = dict(dtype=dtype, max_batch=16, ctx=128, n_seqs=2, int8_head=int8)
    a, b = m.plan(**kw), m.plan(**kw)
    sa, sb = a.acquire(), b.acquire()
    want = [0, 3, 15, 16, 17, 40] + list(range(45, 74))
    targets = [int(toks[i + 1]) for i in want]
    logits = a.step(sa, toks[:74], 0, want)
    check(b.score(sb, toks[:74], 0, want, targets, 7), logits, targets, 7)
    for i in range(74, 75):
        logits = a.step(sa, toks[i:i + 1], i, [0])
        check(b.score(sb, toks[i:i + 1], i, [0], [-1], 20), logits, [-1], 20)
    other = b.acquire()
    check(b.score(other, toks[:20], 0, [19], [3], 2), a.step(a.acquire(), toks[:20], 0, [19]), [3], 2)


def test_refused(hy, hip, plans, pkg, tmp_path):
    m = noditar.Model(hy, tmp_path, noditar.config([noditar.att()]), 6)
    plan = m.plan(max_batch=8, ctx=64)
    seq = plan.acquire()
    vocab = m.cfg["vocab"]
    for kw in (dict(targets=[vocab]), dict(top=65), dict(top=-1), dict(targets=[1, 2]), dict(want=[4]), dict(want=[1, 1], targets=[0, 0])):
        a = dict(want=[3], targets=[1], top=2)
        a.update(kw)
        with pytest.raises(hip.Gl3Error):
            plan.score(seq, [1, 2, 3, 4], 0, a["want"], a["targets"], a["top"])
    L = hip.lib()
    t, w, f, i = np.arange(4, dtype=np.int32), np.zeros(1, np.int32), np.zeros(4, np.float32), np.zeros(4, np.int32)
    p = lambda x: x.ctypes.data
    assert L.gl3_forward_score(plan._ctx, seq, p(t), 4, 0, p(w), 1, p(i), 0, p(f), None, None, None, None) == hip.E_ARG          # no ranks
    assert L.gl3_forward_score(plan._ctx, seq, p(t), 4, 0, p(w), 1, None, 2, None, None, None, p(i), None) == hip.E_ARG           # no top_logprobs
    assert L.gl3_forward_score(None, seq, p(t), 4, 0, p(w), 1, None, 0, None, None, None, None, None) == hip.E_ARG
    check(plan.score(seq, [1, 2, 3, 4], 0, [3], [1], 2), plan.step(seq, [1, 2, 3, 4], 0, [3]), [1], 2)          # the slot is as before the refusals
    model = pkg.synth.make_numpy(pkg.synth.CONFIGS["tiny-llama"], seed=3)
    q = plans.HipMasterPlan(model)
    with pytest.raises(hip.Gl3Error):
        q.score([1, 2], 0, [1], [model.cfg.vocab], 0)
    with pytest.raises(hip.Gl3Error):
        q.score([1, 2], 0, [1, 0], [1, 1], 0)
    q.freeTornadoExecutionPlan()


def unit_head(width):
    """The first `width` rows of the head pick single columns of its input, so a float32 plan's first logits ARE that input."""
    def tweak(w):
        w["head"][:width] = np.eye(width)
    return tweak


def test_the_int8_head_is_its_definition(hy, tmp_path):
    cfg = noditar.config([noditar.att(), noditar.ssm()], width=104, vocab=311)
    m = noditar.Model(hy, tmp_path, cfg, 7, unit_head(104))
    toks = noditar.tokens_for(cfg, 20)
    f, q = m.plan("float32", max_batch=32, ctx=64), m.plan("float32", max_batch=32, ctx=64, int8_head=True)
    want = [3, 7, 19]
    x = f.step(f.acquire(), toks, 0, want)[:, :104]
    got = q.step(q.acquire(), toks, 0, want).astype(np.float64)
    cx, sx = codes_of(x)
    cw, sw = codes_of(np.asarray(m.w["head"], np.float32))
    p = (cx.astype(np.float64) @ cw.astype(np.float64).T) * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    assert (np.abs(got - p) <= 3 * EPS * 1.001 * np.abs(p)).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_int8_head_beside_the_head_it_replaces(hy, tmp_path, dtype):
    """Whole prompts, single tokens behind them, more rows than four, a soft cap, a tied head: logits differ by what two roundings to 8 bits do at most."""
    for make, cfg in ((noditar, noditar.config([noditar.att(), noditar.lat()], width=104, vocab=211)), (kugadra, kugadra.config([kugadra.lig(), kugadra.lat()], cap=11.0)),
                      (noditar, noditar.config([noditar.ssm()], width=136, vocab=190))):
        m = make.Model(hy, tmp_path, cfg, 8 + cfg["width"])
        toks = np.random.default_rng(3).integers(0, cfg["vocab"], 30).astype(np.int32)
        a, b = (hy.HybridPlan.from_dir(m.dir, dtype=dtype, max_batch=16, ctx=64, int8_head=i) for i in (False, True))
        sa, sb = a.acquire(), b.acquire()
        want = list(range(0, 25, 2))
        pairs = [(a.step(sa, toks[:25], 0, want), b.step(sb, toks[:25], 0, want))]
        for i in range(25, 30):
            pairs.append((a.step(sa, toks[i:i + 1], i, [0]), b.step(sb, toks[i:i + 1], i, [0])))
        head = np.asarray(m.w.get("head", m.w["embed"]), np.float64)          # (a tied head: the embedding)
        W = head.shape[1]
        cap = cfg.get("logit_softcap")
        for x, y in pairs:
            # A normed row has at most sqrt(W) x its largest weight in one place and sqrt(W) x as much in all, so a step of its codes is at most that / 127:
            # |dy| <= sum_k |w_k| step_x / 2 + |h|_1 step_w / 2 + W step_x step_w / 4, with |h|_1 <= W x the largest norm weight; bfloat16 rows add 2^-8 of |h|.
            g = float(np.abs(np.asarray(m.w["final.norm"], np.float64)).max())
            step_x, step_w = math.sqrt(W) * g / 127, np.abs(head).max(1) / 127
            bound = np.abs(head).sum(1) * step_x / 2 + W * g * step_w / 2 + W * step_x * step_w / 4
            assert (np.abs(x.astype(np.float64) - y) <= bound * 1.001 + 1e-3).all()          # (a soft cap has slope 1 at most)
            rms = math.sqrt(float(((x - y) ** 2).mean() / (x ** 2).mean()))
            assert rms < 0.03, rms          # two roundings of uniform error 1 / sqrt(12) of a step, steps about 1 / 40 of a deviation
            if cap:
                assert np.abs(y).max() <= cap
        assert len(b.generate(list(map(int, toks[:5])), 4)) == 4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_tokens_drawn_from_an_int8_head(hy, tmp_path, dtype):
    """Greedy tokens, tokens drawn all but coldly and the scores' first alternative are the largest of the logits that a step hands out."""
    m = noditar.Model(hy, tmp_path, noditar.config([noditar.att(), noditar.ssm()], width=104, vocab=311), 12)
    toks = noditar.tokens_for(m.cfg, 12)
    plans_ = [m.plan(dtype, max_batch=16, ctx=64, int8_head=True) for _ in range(4)]
    step, greedy, cold, score = plans_
    ss, sc = step.acquire(), score.acquire()
    for i, t in enumerate(toks):
        best = int(np.argmax(step.step(ss, [t], i, [0])[0]))
        assert greedy.forward_decode_sample(int(t), i, 0.0, 0.95, 0.5) == best
        assert cold.forward_decode_sample(int(t), i, 1e-4, 0.95, 0.5) == best
        assert score.score(sc, [t], i, [0], None, 1)["top_ids"][0, 0] == best


def test_the_run_tool_scores(hy, plans, pkg, tmp_path):
    m = noditar.Model(hy, tmp_path, noditar.config([noditar.att(), noditar.ssm()]), 9)
    toks = noditar.tokens_for(m.cfg, 12)
    for flags, kw in (([], {}), (["--f32"], dict(dtype="float32")), (["--int8-head"], dict(int8_head=True))):
        plan = m.plan(**dict(dict(dtype="bfloat16", max_batch=512, ctx=64), **kw))
        want = plan.score(plan.acquire(), toks[:-1], 0, list(range(11)), toks[1:], 3)
        out = subprocess.run([RUN, "-m", m.dir, "--ids", ",".join(map(str, toks)), "--score", "--top", "3", "-n", "64"] + flags, capture_output=True, text=True, timeout=120)
        assert out.returncode == 0, out.stderr
        lines = out.stdout.strip().split("\n")
        assert len(lines) == 12
        for i, line in enumerate(lines[:-1]):
            v = line.split()
            assert [int(v[0]), int(v[1]), int(v[3])] == [i + 1, toks[i + 1], want["ranks"][i]]
            assert abs(float(v[2]) - want["logprobs"][i]) < 2e-6 and abs(float(v[4]) - want["entropies"][i]) < 2e-6
            assert [int(c.split(":")[0]) for c in v[5:]] == list(want["top_ids"][i])
        total = float(np.sum(want["logprobs"].astype(np.float64)))
        assert abs(float(lines[-1].split()[1].rstrip(",")) - total) < 1e-5 and abs(float(lines[-1].split()[3]) - math.exp(-total / 11)) < 1e-4 * math.exp(-total / 11)
    assert subprocess.run([RUN, "-m", m.dir, "--ids", "1", "--score"], capture_output=True, timeout=120).returncode == 2
    assert subprocess.run([RUN, "-m", m.dir, "--ids", "1,2", "--score", "--top", "65"], capture_output=True, timeout=120).returncode == 2
