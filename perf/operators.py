"""What the operators on rows of scores are measured on: the product in 8-bit integers that makes the scores, the log
probabilities of given ids with entropy and top alternatives, and distillation from a teacher's top logits.

A row holds one query's (or token's) scores over n candidates: an index's vectors or a vocabulary's tokens.  Batches of
1,000, rows of 960 values, pools of 100,000 candidates and lists of 10 neighbors are those of bench.py's workloads; the
other sizes are generic.

`own` is set from outside: False computes the plain form in torch, True calls the package.
"""

import torch

own = False

FLOATS = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1}


def _scores(name, m, k, n, queries, out, bias=False):
    return dict(what="scores", name=name, m=m, k=k, n=n, queries=queries, out=out, bias=bias)


def _log_probs(name, m, n, dtype, t, top, masked=False, pad=0, backward=False, temperature=1.0):
    return dict(what="log_probs", name=name, m=m, n=n, dtype=dtype, t=t, top=top, masked=masked, pad=pad,
                backward=backward, temperature=temperature)


def _distill(name, m, n, dtype, k, form, ragged=False, pad=0, temperature=1.0):
    return dict(what="distill", name=name, m=m, n=n, dtype=dtype, k=k, form=form, ragged=ragged, pad=pad,
                temperature=temperature)


def listed():
    return [
        # one query's state against a vocabulary's (or pool's) rows: what a service waits for, token by token
        _scores("score_one", m=1, k=1024, n=32_000, queries="bfloat16", out="bfloat16"),
        # a few requests at once, their states already quantized by the step before
        _scores("score_few", m=24, k=2048, n=50_000, queries="int8", out="float16"),
        # nothing even: a ragged batch over a small pool, 32-bit scores that rank as squared distances
        _scores("score_odd", m=333, k=1001, n=5_003, queries="float32", out="float32", bias=True),
        # bench.py's batch of 1,000 queries of 960 values, scored against a pool of 100,000 rows
        _scores("score_pool", m=1000, k=960, n=100_000, queries="float16", out="float16", bias=True),
        # a training batch's hidden states through a wide layer: bound by the matrix cores
        _scores("score_large", m=8192, k=4096, n=16_384, queries="bfloat16", out="bfloat16"),
        # one generated token: its log probability, the entropy and 20 alternatives
        _log_probs("logp_one", m=1, n=128_000, dtype="bfloat16", t=1, top=20),
        # constrained decoding over a padded vocabulary: a third of the ids masked, a row with nothing left
        _log_probs("logp_masked", m=333, n=50_021, dtype="float32", t=4, top=5, masked=True, pad=43, temperature=0.7),
        # scoring of sequences offline: the log probability of every given token and its alternatives
        _log_probs("logp_batch", m=2048, n=128_000, dtype="bfloat16", t=1, top=20),
        # a policy's training step: log probability and entropy, and the gradient of both
        _log_probs("logp_train", m=4096, n=32_000, dtype="bfloat16", t=1, top=0, backward=True),
        # a few rows distilled at a time: both directions in one call, 32-bit logits
        _distill("distill_few", m=16, n=32_000, dtype="float32", k=10, form="step", temperature=2.0),
        # a query encoder distilled from searches: lists of 10 neighbors, padded with -1; forward, then backward
        _distill("distill_search", m=1000, n=100_003, dtype="float16", k=10, form="apart", ragged=True, pad=5),
        # a training batch distilled from a larger model's 64 best tokens: loss and gradient
        _distill("distill_large", m=4096, n=128_000, dtype="bfloat16", k=64, form="step", temperature=2.0),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    what = rng.choice(["scores", "scores", "log_probs", "distill"])
    if what == "scores":
        m, k, n = _log(rng, 1, 8192), _log(rng, 32, 8192), _log(rng, 500, 100_000)
        while m * n > 100_000_000 or m * n * k > 500_000_000_000:
            m = (m + 1) // 2
        if rng.random() < 0.6:
            k = max(32, k // 32 * 32)
        case = _scores("", m, k, n, rng.choice(["int8", "float32", "float16", "bfloat16", "bfloat16"]),
                       rng.choice(["float32", "float16", "bfloat16", "bfloat16"]), rng.random() < 0.3)
    else:
        m, n = _log(rng, 1, 8192), _log(rng, 1000, 256_000)
        while m * n > 200_000_000:
            m = (m + 1) // 2
        if rng.random() < 0.5:
            n = n // 64 * 64
        dtype, pad = rng.choice(["float32", "float16", "bfloat16", "bfloat16"]), rng.choice([0, 0, rng.randrange(1, 100)])
        temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
        if what == "log_probs":
            case = _log_probs("", m, n, dtype, _log(rng, 1, 16), rng.choice([0, 1, 5, 20, 64]), rng.random() < 0.3, pad,
                              rng.random() < 0.4, temperature)
        else:
            case = _distill("", m, n, dtype, _log(rng, 1, 256), rng.choice(["step", "step", "apart"]),
                            rng.random() < 0.4, pad, temperature)
    del case["name"]
    return case


# -------------------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _loss_scale(case):
    """16-bit floats are trained with a scaled loss, so that small gradients do not vanish."""
    return 4096.0 if case["dtype"] == "float16" else 1.0


def _distinct(g, m, n, k):
    """k distinct ids under n for each of m rows."""
    start = torch.randint(0, n, (m, 1), generator=g, device="cuda")
    step = 1 + torch.randint(0, n // k, (m, 1), generator=g, device="cuda")
    return (start + step * torch.arange(k, device="cuda")) % n


def _codes(x):
    """Rows in 8 bits: scale = max |x| / 127 and the whole numbers nearest to x / scale, both rounded to 32 bits first."""
    x = x.float()
    scale = x.abs().amax(1) / 127
    return torch.round(x / torch.where(scale > 0, scale, 1)[:, None]), scale


def _rows_of_logits(case, g):
    """Rows of m x n logits (the first n of n + pad columns), as a model's: a broad bulk, made block by block."""
    m, n = case["m"], case["n"]
    full = torch.empty((m, n + case["pad"]), dtype=FLOATS[case["dtype"]], device="cuda")
    for a in range(0, m, 512):
        b = min(m, a + 512)
        full[a:b] = 2.5 * torch.randn((b - a, n + case["pad"]), generator=g, device="cuda")
    return full[:, :n]


def prepare(case, seed):
    g = _gen(seed)
    m, n, state = case["m"], case["n"], {"case": case}
    if case["what"] == "scores":
        k = case["k"]
        x = torch.randn((m, k), generator=g, device="cuda") * (0.5 + _rand(g, m, 1))
        x[:, :: max(1, k // 8)] *= 4  # a few outlying values a row
        rows = torch.empty((n, k), dtype=torch.int8, device="cuda")
        state["row_scales"] = torch.empty(n, device="cuda")
        for a in range(0, n, 8192):
            b = min(n, a + 8192)
            c, state["row_scales"][a:b] = _codes(torch.randn((b - a, k), generator=g, device="cuda"))
            rows[a:b] = c.to(torch.int8)
        state["rows"] = rows
        state["bias"] = -0.5 * k * _rand(g, n) if case["bias"] else None
        if case["queries"] == "int8":
            c, state["query_scales"] = _codes(x)
            state["queries"] = c.to(torch.int8)
        else:
            state["queries"], state["query_scales"] = x.to(FLOATS[case["queries"]]), None
        return state
    state["logits"] = x = _rows_of_logits(case, g)
    if case["what"] == "log_probs":
        ids = _distinct(g, m, n, case["t"])
        # given tokens are likely ones, as generated or taught text is
        x.scatter_(1, ids, (x.gather(1, ids).float() + 6 + 4 * _rand(g, m, case["t"])).to(x.dtype))
        if case["masked"]:
            for a in range(0, m, 512):
                b = min(m, a + 512)
                x[a:b].masked_fill_(_rand(g, b - a, n) < 0.33, float("-inf"))
            x[m // 2] = float("-inf")
        state["ids"] = ids
        if case["backward"]:
            scale = _loss_scale(case) / m
            state["grad_log_probs"] = torch.randn((m, case["t"]), generator=g, device="cuda") * scale
            state["grad_entropy"] = torch.full((m,), -0.01 * scale, device="cuda")
        return state
    k = case["k"]
    ids = _distinct(g, m, n, k)
    teacher = (2 * torch.randn((m, k), generator=g, device="cuda")).sort(1, descending=True).values + 9
    # the student has learned part of it
    x.scatter_(1, ids, (x.gather(1, ids).float() + 0.6 * teacher * _rand(g, m, k)).to(x.dtype))
    if case["ragged"]:  # a search that found fewer: padded with -1, one row with nothing
        found = torch.randint(1, k + 1, (m, 1), generator=g, device="cuda")
        found[m // 2] = 0
        ids[torch.arange(k, device="cuda") >= found] = -1
    state["ids"], state["teacher"] = ids, teacher
    state["grad_loss"] = (0.5 + _rand(g, m)) * (_loss_scale(case) / m)
    return state


# -------------------------------------------------------------------------------------------------------------- passes


def _plain_top(x, z, lse, top):
    """The `top` largest of each row by (value, lowest id): whole keys of a value's order and its place."""
    bits = (x.float() + 0.0).view(torch.int32)  # -0 and 0 are one value
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    place = torch.arange(z.shape[1], device=z.device)
    keys = (order << 32) | (0x7FFFFFFF - place)
    ids = 0x7FFFFFFF - (keys.topk(top, dim=1).values & 0x7FFFFFFF)
    best = z.gather(1, ids)
    nothing = best == float("-inf")
    return torch.where(nothing, best, best - lse[:, None]), ids.masked_fill(nothing, -1)


def _plain_softmax(x, temperature):
    """z = x / temperature, its log-sum-exp and probabilities; a row with nothing has no probability anywhere."""
    z = x.float() / temperature
    top = z.amax(1)
    top = torch.where(top == float("-inf"), 0, top)
    e = torch.exp(z - top[:, None])
    s = e.sum(1)
    return z, top + torch.log(s), e / torch.where(s > 0, s, 1)[:, None]


def _plain(state):
    case = state["case"]
    if case["what"] == "scores":
        if case["queries"] == "int8":
            a, scales = state["queries"].float(), state["query_scales"]
        else:
            a, scales = _codes(state["queries"])
        out = a @ state["rows"].float().T
        out *= scales[:, None]
        out *= state["row_scales"]
        if state["bias"] is not None:
            out += state["bias"]
        return out.to(FLOATS[case["out"]])
    x, ids, t = state["logits"], state["ids"], case["temperature"]
    z, lse, p = _plain_softmax(x, t)
    if case["what"] == "log_probs":
        given = z.gather(1, ids)
        logp = torch.where(given == float("-inf"), given, given - lse[:, None])
        entropy = -(p * torch.where(p > 0, z - lse[:, None], 0)).sum(1)
        out = [logp, entropy, lse]
        if case["top"]:
            out += _plain_top(x, z, lse, case["top"])
        if case["backward"]:
            gl, gh = state["grad_log_probs"], state["grad_entropy"]
            grad = -p * (gl.sum(1)[:, None] + gh[:, None] * (torch.where(p > 0, z - lse[:, None], 0) + entropy[:, None]))
            grad.scatter_add_(1, ids, gl)
            out.append((grad / t).to(x.dtype))
        return out
    listed_ = ids >= 0
    some = listed_.any(1)
    teacher = torch.where(listed_, state["teacher"] / t, float("-inf"))
    w = torch.exp(teacher - torch.where(some, teacher.amax(1), 0)[:, None])
    q = w / torch.where(some, w.sum(1), 1)[:, None]
    at = ids.clamp_min(0)
    loss = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1)) - z.gather(1, at) + lse[:, None]), 0).sum(1)
    grad = p.scatter_add_(1, at, -q) * (torch.where(some, state["grad_loss"], 0) / t)[:, None]
    return loss, grad.to(x.dtype)


def _package(state):
    import octex_amd

    case = state["case"]
    if case["what"] == "scores":
        return octex_amd.int8_scores(state["queries"], state["rows"], state["row_scales"], bias=state["bias"],
                                     query_scales=state["query_scales"], dtype=case["out"])
    x, ids, t = state["logits"], state["ids"], case["temperature"]
    if case["what"] == "log_probs":
        r = octex_amd.log_probs(x, ids, top=case["top"], temperature=t)
        out = [r.log_probs, r.entropy, r.lse]
        if case["top"]:
            out += [r.top_log_probs, r.top_ids]
        if case["backward"]:
            out.append(octex_amd.log_probs_backward(state["grad_log_probs"], state["grad_entropy"], x, ids, r.lse,
                                                    r.entropy, temperature=t))
        return out
    if case["form"] == "step":
        return octex_amd.distill_step(state["grad_loss"], x, ids, state["teacher"], temperature=t)
    loss, lse = octex_amd.distill(x, ids, state["teacher"], temperature=t)
    return loss, octex_amd.distill_backward(state["grad_loss"], x, ids, state["teacher"], lse, temperature=t)


def run(state):
    return _package(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ what a pass is held against


def work(case):
    """Every input read once and every output written once.  An exponential, its sum and its weighted sum are taken as 6
    operations a logit, a gradient as 4 more."""
    m, n = case["m"], case["n"]
    if case["what"] == "scores":
        k = case["k"]
        bytes_ = m * k * SIZES[case["queries"]] + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * SIZES[case["out"]]
        return {"bytes": bytes_ + (4 * m if case["queries"] == "int8" else 0), "flops": 2.0 * m * n * k}
    rows = m * n * SIZES[case["dtype"]]
    if case["what"] == "log_probs":
        back = 1 if case["backward"] else 0
        return {"bytes": rows * (1 + back) + m * (12 * case["t"] + 8 + 12 * case["top"] + back * (4 * case["t"] + 4)),
                "flops": (6.0 + 4.0 * back) * m * n}
    return {"bytes": 2 * rows + m * (12 * case["k"] + 8), "flops": 10.0 * m * n}


def _exact_scores(case, state):
    rows, out = state["rows"].double(), []
    if case["queries"] == "int8":
        codes, scales = state["queries"].double(), state["query_scales"].double()
    else:  # 8-bit codes are defined by 32-bit quotients; everything after them is in 64 bits
        x = state["queries"].to(torch.float32)
        top = torch.maximum(x.max(1).values, -x.min(1).values)
        s32 = top / torch.full_like(top, 127)
        codes = torch.where(s32[:, None] > 0, (x / s32[:, None]).double(), 0).round()
        scales = s32.double()
    per_row = state["row_scales"].double()
    for a in range(0, len(codes), 1024):
        y = torch.mm(codes[a : a + 1024], rows.t()) * (scales[a : a + 1024, None] * per_row[None, :])
        out.append(y if state["bias"] is None else y + state["bias"].double()[None, :])
    return torch.cat(out)


def _exact_log_probs(case, state, a, b):
    x, ids = state["logits"][a:b].double() / case["temperature"], state["ids"][a:b]
    empty = torch.isinf(x).all(1, keepdim=True)
    lse = torch.logsumexp(x, 1, keepdim=True)
    logp = torch.where(torch.isinf(x), float("-inf"), x - torch.where(empty, 0, lse))
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0).sum(1, keepdim=True)
    out = [logp.gather(1, ids), entropy[:, 0], lse[:, 0]]
    if case["top"]:  # ids by the places of the values, equal ones in their order
        at = torch.sort(state["logits"][a:b], dim=1, descending=True, stable=True).indices[:, : case["top"]]
        best = logp.gather(1, at)
        out += [best, torch.where(torch.isinf(best), -1, at)]
    if case["backward"]:
        gl, gh = state["grad_log_probs"][a:b].double(), state["grad_entropy"][a:b].double()
        one = torch.zeros_like(x)
        for j in range(ids.shape[1]):
            one[torch.arange(b - a, device=x.device), ids[:, j]] += gl[:, j]
        inner = torch.where(p > 0, logp + entropy, 0)
        out.append((one - gl.sum(1, keepdim=True) * p - gh[:, None] * p * inner) / case["temperature"])
    return out


def _exact_distill(case, state, a, b):
    x, ids, t = state["logits"][a:b].double() / case["temperature"], state["ids"][a:b], case["temperature"]
    logp = torch.log_softmax(x, 1)
    grad, loss = logp.exp(), torch.zeros(b - a, dtype=torch.float64, device=x.device)
    teacher = (state["teacher"][a:b].double() / t).masked_fill(ids < 0, float("-inf"))
    any_ = (ids >= 0).any(1)
    logq = torch.log_softmax(torch.where(any_[:, None], teacher, 0), 1)
    row = torch.arange(b - a, device=x.device)
    for j in range(ids.shape[1]):
        keep = ids[:, j] >= 0
        q = torch.where(keep, logq[:, j].exp(), 0)
        at = torch.where(keep, ids[:, j], 0)
        loss += torch.where(q > 0, q * (logq[:, j] - logp[row, at]), 0)
        grad[row, at] -= q
    grad *= (state["grad_loss"][a:b].double() * any_ / t)[:, None]
    return loss, grad


def exact(case, seed):
    state = prepare(case, seed)
    if case["what"] == "scores":
        return _exact_scores(case, state)
    one = _exact_log_probs if case["what"] == "log_probs" else _exact_distill
    step = max(1, 32_000_000 // case["n"])
    parts = [one(case, state, a, min(case["m"], a + step)) for a in range(0, case["m"], step)]
    return type(parts[0])(torch.cat(p) for p in zip(*parts))
