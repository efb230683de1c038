"""Scores of every GGUF family, type and transport against the logits of the same plans; the 8-bit head of every layer-list design against its definition, a logits'
multiplier among them."""
import threading
from importlib import import_module

import numpy as np
import pytest

import __graft_entry__ as ge
import test_kosusun_gpu as kosusun
import test_tutedra_gpu as tutedra
import test_vonulix_gpu as vonulix
import test_ziginex_gpu as ziginex
from test_ops_gpu import codes_of
from test_score_gpu import EPS, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hy(pkg):
    return import_module(ge.PKG_NAME + ".hybrid")


@pytest.fixture(scope="module")
def plans(pkg):
    return import_module(ge.PKG_NAME + ".plan")


@pytest.fixture(scope="module")
def hip(pkg):
    return import_module(ge.PKG_NAME + ".hip")


F16, Q4_0, Q8_0 = 1, 2, 8


def wanted(toks, want):
    return np.where(want + 1 < toks.size, toks[np.minimum(want + 1, toks.size - 1)], -1)


@pytest.mark.parametrize("name,wtype,flag,batch", [("tiny-qwen2", Q8_0, None, 4), ("tiny-granite", Q8_0, None, 4), ("tiny-phi3", Q8_0, None, 4), ("tiny-devstral", Q8_0, None, 4), ("tiny-qwen2moe", Q8_0, None, 1),
                                                   ("tiny-llama", F16, None, 4), ("tiny-llama", Q4_0, None, 4), ("tiny-granite", F16, None, 1), ("tiny-llama", Q8_0, "FLAG_F32_ACTIVATION", 4),
                                                   ("tiny-llama", F16, "FLAG_SCALAR_DOT", 1), ("tiny-llama", Q8_0, "FLAG_NO_GRAPH", 1), ("tiny-llama-tied", Q8_0, None, 4)])
def test_scores_of_a_plan(pkg, plans, hip, name, wtype, flag, batch):
    model = pkg.synth.make_numpy(pkg.synth.CONFIGS[name], wtype=wtype, seed=3)
    toks = np.asarray(pkg.javarand.bench_tokens(model.cfg.vocab, 11), np.int32)
    flags = getattr(hip, flag) if flag else 0
    plan = plans.HipMasterPlan(model, flags=flags)
    logits = np.stack([plan.forward_decode(int(t), p) for p, t in enumerate(toks)])
    plan.freeTornadoExecutionPlan()
    plan = plans.HipMasterPlan(model, prefill_batch_size=batch, flags=flags)
    for want, top in ((np.arange(10), 5), ([0, 4, 5, 10], 0), ([10], 64)):
        want = np.asarray(want, np.int32)
        targets = wanted(toks, want)
        check(plan.score(toks, 0, want, targets, top), logits[want], targets, top)
    assert np.array_equal(plan.forward_decode(int(toks[0]), 0), logits[0])
    plan.freeTornadoExecutionPlan()


@pytest.mark.parametrize("name,wtype", [("mid-llama", Q8_0), ("tiny-llama", Q4_0)])
def test_scores_of_two_ranks(pkg, plans, hip, name, wtype):
    """Every rank has the whole row of logits, and so the same scores."""
    model = pkg.synth.make_numpy(pkg.synth.CONFIGS[name], wtype=wtype, seed=17)
    toks = np.asarray(pkg.javarand.bench_tokens(model.cfg.vocab, 4), np.int32)
    want = np.arange(4, dtype=np.int32)
    group = plans.make_local_group(2)
    logits, scores, errors = [None] * 2, [None] * 2, [None] * 2

    def rank(r):
        try:
            plan = plans.HipMasterPlan(model, tp_rank=r, tp_size=2, local_group=group)
            logits[r] = np.stack([plan.forward_decode(int(t), p) for p, t in enumerate(toks)])
            scores[r] = plan.score(toks, 0, want, wanted(toks, want), 7)
            plan.freeTornadoExecutionPlan()
        except Exception as e:   # noqa: BLE001
            errors[r] = e
    threads = [threading.Thread(target=rank, args=(r,), daemon=True) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert errors == [None, None] and not any(t.is_alive() for t in threads)
    hip.lib().gl3_local_group_destroy(group)
    assert np.array_equal(logits[0], logits[1])
    for r in range(2):
        check(scores[r], logits[0], wanted(toks, want), 7)


def unit_rows(cfg, w):
    """The first rows of the head pick single columns of its input, so a float32 plan's first logits ARE that input (a tied head: of the embedding)."""
    head = w["head"] if "head" in w else w["embed"]
    head[:cfg["width"]] = np.eye(cfg["width"])


DESIGNS = [("kosusun", kosusun, lambda: kosusun.config([kosusun.par(), kosusun.mls()], logit_scale=0.37)), ("kosusun x 5", kosusun, lambda: kosusun.config([kosusun.par()], logit_scale=5.0)),
           ("vonulix", vonulix, lambda: vonulix.config([vonulix.layer(), vonulix.layer()])), ("tutedra", tutedra, lambda: tutedra.config([tutedra.hgrn(), tutedra.att()])),
           ("ziginex", ziginex, lambda: ziginex.config([ziginex.par(), ziginex.lat()]))]


@pytest.mark.parametrize("name,design,config", DESIGNS, ids=[d[0] for d in DESIGNS])
def test_the_int8_head_of_a_design(hy, tmp_path, name, design, config):
    cfg = config()
    W = cfg["width"]
    m = design.Model(hy, tmp_path, cfg, 7, unit_rows)
    head = np.asarray(m.w["head"] if "head" in m.w else m.w["embed"], np.float32)
    toks = np.random.default_rng(5).integers(0, cfg["vocab"], 24).astype(np.int32)
    f, q = (m.plan("float32", max_batch=32, ctx=64, int8_head=i) for i in (False, True))
    sf, sq = f.acquire(), q.acquire()
    cw, sw = codes_of(head)
    steps = [(toks[:20], 0, [0, 3, 7, 18, 19])] + [(toks[i:i + 1], i, [0]) for i in range(20, 24)]
    for t, pos, want in steps:
        x = f.step(sf, t, pos, want)[:, :W]
        got = q.step(sq, t, pos, want).astype(np.float64)
        cx, sx = codes_of(x)
        p = (cx.astype(np.float64) @ cw.astype(np.float64).T) * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
        assert (np.abs(got - p) <= 3 * EPS * 1.001 * np.abs(p)).all()
    scores = q.score(sq, toks[:20], 0, [2, 19], [1, -1], 3)
    check(scores, q.step(sq, toks[:20], 0, [2, 19]), [1, -1], 3)
