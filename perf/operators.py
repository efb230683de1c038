"""Performance cases of the operators on the caller's device memory: products in 8-bit integers and log probabilities of tokens.

Three kinds of case.  "linear": y = x W^T (+ bias) of float rows with int8 weights (one scale per channel); the rows are quantised inside
the call (one scale per token).  "shared": rows are quantised once and several products read the codes, as projections of one activation
do.  "logprobs": log probability and rank of a given token per row of logits, the row's entropy and its most probable tokens.

The definition of the quantiser is in float32 numbers, so that a code is the same wherever it is computed: a = max |x|, scale = a / 127,
code = rint(x * (127 / a)), every operation rounded to float32.
"""
import math

import torch

own = False
DEVICE = "cuda"
CODE_BLOCK = 128             # rows of codes end on a multiple of this many, zeros behind the last column
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST_PRODUCT = 512 * 4096 * 128256
LARGEST_LOGITS = 512 * 128256


def linear(name, m, k, n, x, y, bias=False):
    case = {"kind": "linear", "m": m, "k": k, "n": n, "x": x, "y": y, "bias": bias}
    return dict(case, name=name) if name else case


def shared(name, m, k, n, outputs, x, y, bias=False):
    """`n` rows for the first product and `n2` for each of the others (queries; keys and values)."""
    case = {"kind": "shared", "m": m, "k": k, "n": n[0], "n2": n[1], "outputs": outputs, "x": x, "y": y, "bias": bias}
    return dict(case, name=name) if name else case


def logprobs(name, rows, vocab, top, x, pad=0, masked=0.0):
    """pad: elements between rows; masked: share of every row's tokens that a grammar or a mask has set to -inf."""
    case = {"kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "x": x, "pad": pad, "masked": masked}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one projection of one token of a small model: the smallest call, launch and latency
        linear("linear-token-2048", 1, 2048, 2048, "bf16", "f32"),
        # logits of one token in the benchmark's vocabulary: all weights once
        linear("linear-token-head", 1, 4096, 128256, "f32", "f32"),
        # logits of a static batch of 32 sequences, the largest vocabulary
        linear("linear-batch32-head", 32, 2560, 151936, "f32", "f32"),
        # logits of every token of the benchmark's prompt (scoring): the largest product
        linear("linear-prompt-head", 512, 4096, 128256, "bf16", "f32"),
        # odd everything: ragged columns and rows, biases, half precision
        linear("linear-ragged", 77, 1100, 8199, "f16", "f16", True),
        # queries, keys and values of four tokens that wait together
        shared("shared-qkv-4", 4, 2560, (4096, 1024), 3, "bf16", "bf16", True),
        # gate and up of a long ragged prompt
        shared("shared-gate-up-2041", 2041, 4096, (14336, 14336), 2, "bf16", "bf16"),
        # the log probabilities a chat server returns with one token
        logprobs("logprobs-token", 1, 128256, 20, "f32"),
        # ... with the tokens of 32 sequences
        logprobs("logprobs-batch32", 32, 151936, 5, "f32"),
        # scoring of the benchmark's prompt
        logprobs("logprobs-prompt", 512, 128256, 5, "f32"),
        # answers under a grammar: most tokens masked, rows behind each other in a wider buffer
        logprobs("logprobs-masked", 1500, 32064, 20, "bf16", 7, 0.9),
        # a small vocabulary with an odd row length
        logprobs("logprobs-1003", 7, 1003, 3, "f16"),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "shared", "logprobs", "logprobs"])
    if kind == "logprobs":
        while True:
            rows, vocab = log_int(rng, 1, 2048), log_int(rng, 500, 160000)
            if rows * vocab <= LARGEST_LOGITS:
                break
        return logprobs(None, rows, vocab, rng.choice([0, 1, 2, 5, 10, 20, 33, 64]), rng.choice(["f32", "f32", "bf16", "f16"]), rng.choice([0, 0, 1, 24]),
                        rng.choice([0.0, 0.0, 0.0, 0.5, 0.99]))
    types = rng.choice([("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "f16")])
    if kind == "linear":
        while True:
            m, k, n = log_int(rng, 1, 2048), log_int(rng, 256, 14336), log_int(rng, 256, 151936)
            if m * k * n <= LARGEST_PRODUCT and k * n <= 151936 * 4096:
                break
        return linear(None, m, k, n, *types, rng.random() < 0.3)
    while True:
        m, k, n, n2, outputs = log_int(rng, 1, 2048), log_int(rng, 256, 8192), log_int(rng, 256, 16384), log_int(rng, 256, 16384), rng.randint(2, 3)
        if m * k * (n + (outputs - 1) * n2) <= LARGEST_PRODUCT:
            break
    return shared(None, m, k, (n, n2), outputs, *types, rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def activations(m, k, dtype, g):
    """Normed rows: unit scale, one column in 200 twenty times as large."""
    x = torch.randn(m, k, generator=g, device=DEVICE)
    loud = torch.rand(k, generator=g, device=DEVICE) < 0.005
    return (x * (1.0 + 19.0 * loud)).to(dtype)


def channel_weights(n, k, g):
    """Codes [n, k rounded up to CODE_BLOCK] and scales [n] of a normal matrix whose largest entry of a row is about four deviations."""
    codes = torch.zeros(n, -(-k // CODE_BLOCK) * CODE_BLOCK, dtype=torch.int8, device=DEVICE)
    step = max(1, (1 << 27) // k)
    for r in range(0, n, step):
        part = torch.randn(min(step, n - r), k, generator=g, device=DEVICE)
        codes[r:r + step, :k] = (part * 32.0).round_().clamp_(-127, 127)
    scale = (0.02 / 32.0) * (1.0 + 0.5 * torch.rand(n, generator=g, device=DEVICE))
    return codes, scale


def widths(case):
    return [case["n"]] if case["kind"] == "linear" else [case["n"]] + [case["n2"]] * (case["outputs"] - 1)


def prepare(case, seed):
    g = generator(seed)
    if case["kind"] == "logprobs":
        return prepare_logprobs(case, g)
    m, k = case["m"], case["k"]
    state = {"case": case, "x": activations(m, k, TYPES[case["x"]], g)}
    state["weights"] = [channel_weights(n, k, g) for n in widths(case)]
    state["bias"] = [0.1 * torch.randn(n, generator=g, device=DEVICE) if case["bias"] else None for n in widths(case)]
    if own:
        ops = product()
        state["ops"] = ops
        state["rows"] = [ops.Int8Rows(codes, scale, k) for codes, scale in state["weights"]]
    return state


def prepare_logprobs(case, g):
    rows, vocab = case["rows"], case["vocab"]
    buffer = torch.empty(rows, vocab + case["pad"], dtype=TYPES[case["x"]], device=DEVICE)
    for r in range(0, rows, 128):          # a wide bulk and some tokens far above it, from certain rows to undecided ones
        n = min(128, rows - r)
        part = torch.randn(n, vocab + case["pad"], generator=g, device=DEVICE) * 2.0
        hot = torch.randint(0, vocab, (n, 8), generator=g, device=DEVICE)
        part.scatter_(1, hot, 6.0 + 12.0 * torch.rand(n, 8, generator=g, device=DEVICE))
        if case["masked"]:
            part[torch.rand(n, vocab + case["pad"], generator=g, device=DEVICE) < case["masked"]] = -math.inf
        buffer[r:r + n] = part.to(buffer.dtype)
    logits = buffer[:, :vocab]
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
    best = torch.stack([row.argmax() for row in logits]) if rows <= 64 else logits.argmax(1)
    targets = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.5, best, targets).to(torch.int32)
    if rows >= 4:          # the last token of a prompt has none behind it; a mask may leave nothing
        targets[rows - 1] = -1
        if case["masked"]:
            logits[rows // 2] = -math.inf
    state = {"case": case, "logits": logits, "targets": targets}
    if own:
        state["ops"] = product()
    return state


def product():
    import importlib
    ge = importlib.import_module("__graft_entry__")
    ge.load_package()
    return importlib.import_module(ge.PKG_NAME + ".ops")


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"linear": own_linear, "shared": own_shared, "logprobs": own_logprobs}[case["kind"]](state, case)
    return {"linear": plain_products, "shared": plain_products, "logprobs": plain_logprobs}[case["kind"]](state, case)


def own_linear(state, case):
    return [state["ops"].int8_linear(state["x"], state["rows"][0], state["bias"][0], TYPES[case["y"]])]


def own_shared(state, case):
    ops = state["ops"]
    rows = ops.quantize_rows(state["x"])
    return [ops.int8_matmul(rows, w, b, TYPES[case["y"]]) for w, b in zip(state["rows"], state["bias"])]


def own_logprobs(state, case):
    out = state["ops"].token_logprobs(state["logits"], state["targets"], case["top"])
    return result(out.logprob, out.rank, out.entropy, out.top_ids, out.top_logprobs)


def result(logprob, rank, entropy, ids, top_logprobs):
    out = {"logprob": logprob, "rank": rank, "entropy": entropy}
    if ids is not None and ids.shape[1]:
        out.update(top_ids=ids, top_logprobs=top_logprobs)
    return out


def plain_products(state, case):
    x = state["x"].float()
    a = x.abs().amax(1, keepdim=True)
    most = torch.full_like(a, 127.0)          # (a number there would be divided by as its rounded inverse)
    scale, to_code = a / most, most / a
    codes = (x * to_code).round().clamp(-127, 127)
    out = []
    for (w, w_scale), bias in zip(state["weights"], state["bias"]):
        y = (codes @ w[:, :case["k"]].float().t()) * scale * w_scale
        if bias is not None:
            y = y + bias
        out.append(y.to(TYPES[case["y"]]))
    return out


def plain_logprobs(state, case):
    x, t = state["logits"].float(), state["targets"].long()
    vocab = case["vocab"]
    top = x.amax(1, keepdim=True)
    none = top == -math.inf
    d = x - torch.where(none, torch.zeros_like(top), top)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    entropy = torch.where(none, torch.zeros_like(s), log_s - torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1, keepdim=True) / s)
    lse = top + log_s
    given = (t >= 0).unsqueeze(1)
    at = t.clamp(min=0).unsqueeze(1)
    xt = x.gather(1, at)
    minus = torch.full_like(xt, -math.inf)
    logprob = torch.where(given, torch.where(none, minus, xt - lse), torch.zeros_like(xt))
    before = torch.arange(vocab, device=DEVICE).unsqueeze(0) < at
    rank = torch.where(given, 1 + ((x > xt) | ((x == xt) & before)).sum(1, keepdim=True), torch.zeros_like(at))
    ids = values = None
    if case["top"]:
        # one whole number per token that orders as (logit, lowest id first)
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        keys = (order << 32) | (0x7FFFFFFF - torch.arange(vocab, device=DEVICE))
        k = min(case["top"], vocab)
        ids = 0x7FFFFFFF - (torch.topk(keys, k, dim=1).values & 0x7FFFFFFF)
        values = x.gather(1, ids)
        ids = torch.where(values == -math.inf, torch.full_like(ids, -1), ids).to(torch.int32)
        values = torch.where(values == -math.inf, values, values - lse)
        if k < case["top"]:
            fill = (x.shape[0], case["top"] - k)
            ids = torch.cat([ids, ids.new_full(fill, -1)], 1)
            values = torch.cat([values, values.new_full(fill, -math.inf)], 1)
    return result(logprob.squeeze(1), rank.squeeze(1).to(torch.int32), entropy.squeeze(1), ids, values)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------
def size(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    if case["kind"] == "logprobs":
        cells = case["rows"] * case["vocab"]
        # per logit: its distance to the largest, the exponential, and the two sums
        return {"bytes": cells * size(case["x"]) + case["rows"] * (16 + 8 * case["top"]), "flops": 5 * cells}
    m, k, n = case["m"], case["k"], sum(widths(case))
    return {"bytes": m * k * size(case["x"]) + n * k + n * (8 if case["bias"] else 4) + m * n * size(case["y"]), "flops": 2 * m * k * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    return exact_logprobs(state, case) if case["kind"] == "logprobs" else exact_products(state, case)


def exact_products(state, case):
    x = state["x"].double()
    peak = x.abs().max(1).values
    scale = (peak / torch.full_like(peak, 127.0)).float().double()             # float32 numbers by definition
    to_code = (torch.full_like(peak, 127.0) / peak).float().double()
    codes = (x * to_code[:, None]).float().double().round_().clamp_(-127, 127)
    out = []
    for (w, w_scale), bias in zip(state["weights"], state["bias"]):
        parts = []
        for r in range(0, w.shape[0], 16384):
            y = torch.matmul(codes, w[r:r + 16384, :case["k"]].double().t())
            y = y * torch.outer(scale, w_scale[r:r + 16384].double())
            parts.append(y if bias is None else y + bias[r:r + 16384].double())
        out.append(torch.cat(parts, 1))
    return out


def exact_logprobs(state, case):
    logprob, rank, entropy, ids, values = [], [], [], [], []
    for row, t in zip(state["logits"], state["targets"].tolist()):
        x = row.double()
        order = torch.sort(x, descending=True, stable=True) if case["top"] or t >= 0 else None
        lse = torch.logsumexp(x, 0)
        nothing = bool(x.max() == -math.inf)
        lp = x - lse if not nothing else torch.full_like(x, -math.inf)
        kept = lp[lp > -math.inf]
        entropy.append(float(-(kept.exp() * kept).sum()) if not nothing else 0.0)
        logprob.append(float(lp[t]) if t >= 0 else 0.0)
        rank.append(int((order.indices == t).nonzero()[0]) + 1 if t >= 0 else 0)
        if case["top"]:
            first = order.indices[:case["top"]]
            first = first[x[first] > -math.inf]
            fill = case["top"] - first.numel()
            ids.append(torch.cat([first, first.new_full((fill,), -1)]))
            values.append(torch.cat([lp[first], lp.new_full((fill,), -math.inf)]))
    make = lambda v, dtype: torch.tensor(v, dtype=dtype, device=DEVICE)
    return result(make(logprob, torch.float64), make(rank, torch.int32), make(entropy, torch.float64),
                  torch.stack(ids).to(torch.int32) if ids else None, torch.stack(values) if ids else None)
