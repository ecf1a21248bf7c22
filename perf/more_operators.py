"""What the operators at both ends of a model's training step are measured on: rows of a table by ids and the table's gradient,
a policy's clipped loss from rows of logits, and the balance of rows over experts.

A table holds a vocabulary's embeddings or an index's vectors (then ids are a search's neighbors, padded with -1).  Batches of
1,000, lists of 10, pools of 100,000 rows and rows of 960 values are those of bench.py's workloads; the other sizes are
generic.

`own` is set from outside: False computes the plain form in torch, True calls the package.
"""

import math

import torch

own = False

FLOATS = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1}


def _embed(name, m, n, d, table, out, t=1, scale=1.0, padded=False, zipf=True):
    return dict(what="embed", name=name, m=m, n=n, d=d, table=table, out=out, t=t, scale=scale, padded=padded, zipf=zipf)


def _gradient(name, m, n, d, grad, out, scale=1.0, padded=False, zipf=True, pad=0):
    return dict(what="gradient", name=name, m=m, n=n, d=d, grad=grad, out=out, scale=scale, padded=padded, zipf=zipf, pad=pad)


def _policy(name, m, n, dtype, form, kl=0.0, entropy=0.0, masked=False, padding=0.0, pad=0, temperature=1.0, high=0.2):
    return dict(what="policy", name=name, m=m, n=n, dtype=dtype, form=form, kl=kl, entropy=entropy, masked=masked,
                padding=padding, pad=pad, temperature=temperature, low=0.2, high=high)


def _balance(name, m, e, k, dtype, form, z=0.0, padding=0.0, dropped=False, pad=0):
    return dict(what="balance", name=name, m=m, e=e, k=k, dtype=dtype, form=form, z=z, padding=padding, dropped=dropped,
                pad=pad)


def listed():
    return [
        # one token on its way into a model, as a service has it at every step
        _embed("embed_one", m=1, n=32_000, d=1024, table="bfloat16", out="bfloat16", scale=32.0),
        # what a reader is given of a search: 10 neighbors of 1,000 queries from 8-bit rows, some lists short
        _embed("embed_neighbors", m=1000, t=10, n=100_000, d=960, table="int8", out="bfloat16", padded=True, zipf=False),
        # prompts of a training batch through a large vocabulary
        _embed("embed_prompts", m=32_768, n=128_000, d=4096, table="bfloat16", out="bfloat16", scale=64.0),
        # a short text's gradient
        _gradient("gradient_few", m=512, n=32_000, d=1024, grad="bfloat16", out="bfloat16", scale=32.0),
        # nothing even: rows apart, padding among the ids, 32 bits
        _gradient("gradient_odd", m=5_003, n=50_021, d=1001, grad="float32", out="float32", padded=True, pad=7),
        # a training batch's gradient: a few tokens have a large share of it
        _gradient("gradient_large", m=32_768, n=128_000, d=4096, grad="bfloat16", out="bfloat16", scale=64.0),
        # a few tokens of a policy, both directions in one call
        _policy("policy_few", m=16, n=32_000, dtype="float32", form="step"),
        # constrained actions over a padded vocabulary, prompts among the rows; forward, then backward, with every term
        _policy("policy_masked", m=333, n=50_021, dtype="float16", form="apart", kl=0.05, entropy=0.01, masked=True,
                padding=0.25, pad=43, temperature=0.7, high=0.28),
        # a policy's training batch, held to a reference model
        _policy("policy_large", m=4096, n=128_000, dtype="bfloat16", form="step", kl=0.02),
        # a small batch's router
        _balance("balance_few", m=64, e=8, k=2, dtype="float32", form="step"),
        # uneven experts, rows left out and choices dropped, forward, then backward
        _balance("balance_odd", m=5_003, e=60, k=4, dtype="float16", form="apart", z=0.1, padding=0.2, dropped=True, pad=4),
        # a training batch over many experts
        _balance("balance_large", m=131_072, e=256, k=8, dtype="bfloat16", form="step", z=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    what = rng.choice(["embed", "gradient", "policy", "balance"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    pad = rng.choice([0, 0, rng.randrange(1, 100)])
    if what in ("embed", "gradient"):
        m, n, d = _log(rng, 1, 65_536), _log(rng, 1000, 256_000), _log(rng, 64, 8192)
        if rng.random() < 0.6:
            d = d // 64 * 64
        while m * d > 134_000_000:
            m = (m + 1) // 2
        while n * d > 250_000_000:
            n = (n + 1) // 2
        scale, padded, zipf = rng.choice([1.0, 0.25, d**0.5]), rng.random() < 0.4, rng.random() < 0.6
        if what == "embed":
            table = rng.choice(["int8", dtype])
            case = _embed("", m, n, d, table, dtype, rng.choice([1, 1, 1 + rng.randrange(10)]), scale, padded, zipf)
            case["m"] = max(1, m // case["t"])
        else:
            case = _gradient("", m, n, d, dtype, rng.choice([dtype, "float32"]), scale, padded, zipf, pad)
    elif what == "policy":
        m, n = _log(rng, 1, 8192), _log(rng, 1000, 256_000)
        while m * n > 200_000_000:
            m = (m + 1) // 2
        case = _policy("", m, n, dtype, rng.choice(["step", "step", "apart"]), rng.choice([0.0, 0.02]),
                       rng.choice([0.0, 0.01]), rng.random() < 0.3, rng.choice([0.0, 0.0, 0.3]), pad,
                       rng.choice([1.0, 1.0, 0.7]), rng.choice([0.2, 0.28]))
    else:
        m, e = _log(rng, 1, 131_072), _log(rng, 4, 1024)
        while m * e > 32_000_000:
            m = (m + 1) // 2
        case = _balance("", m, e, min(e, _log(rng, 1, 16)), dtype, rng.choice(["step", "step", "apart"]),
                        rng.choice([0.0, 0.1]), rng.choice([0.0, 0.3]), rng.random() < 0.3, pad)
    del case["name"]
    return case


# -------------------------------------------------------------------------------------------------------------- inputs


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _randn(g, m, n, dtype, scale=1.0, pad=0):
    """Normal values, the first n of n + pad columns, made block by block."""
    full = torch.empty((m, n + pad), dtype=dtype, device="cuda")
    step = max(1, 32_000_000 // (n + pad))
    for a in range(0, m, step):
        b = min(m, a + step)
        full[a:b] = scale * torch.randn((b - a, n + pad), generator=g, device="cuda")
    return full[:, :n]


def _loss_scale(dtype):
    """16-bit floats are trained with a scaled loss, so that small gradients do not vanish."""
    return 4096.0 if dtype == "float16" else 1.0


def _table_ids(case, g, count):
    """Ids of a table's rows: as text's tokens are (the share of the i-th commonest falls as 1 / i), or all alike."""
    n, u = case["n"], _rand(g, count)
    if case["zipf"]:
        rank = (torch.exp(u.double() * math.log(n + 1)) - 1).long().clamp(0, n - 1)
        ids = torch.randperm(n, generator=g, device="cuda")[rank]
    else:
        ids = (u.double() * n).long().clamp(0, n - 1)
    if case["padded"]:
        ids[_rand(g, count) < 0.1] = -1
    return ids


def _prepare_policy(case, g, state):
    m, n, t = case["m"], case["n"], case["temperature"]
    state["logits"] = x = _randn(g, m, n, FLOATS[case["dtype"]], 2.5, case["pad"])
    ids = torch.randint(0, n, (m, 1), generator=g, device="cuda")
    likely = (x.gather(1, ids).float() + 6 + 4 * _rand(g, m, 1)).to(x.dtype)  # tokens that were sampled are likely ones
    x.scatter_(1, ids, likely)
    if case["masked"]:
        for a in range(0, m, 512):
            b = min(m, a + 512)
            x[a:b].masked_fill_(_rand(g, b - a, n) < 0.33, float("-inf"))
        x.scatter_(1, ids, likely)
    now = torch.empty(m, device="cuda")
    step = max(1, 32_000_000 // n)
    for a in range(0, m, step):
        z = x[a : a + step].float() / t
        now[a : a + step] = z.gather(1, ids[a : a + step])[:, 0] - torch.logsumexp(z, 1)
    # the policy has moved since its tokens were sampled; ratios at the clip's very border, where the gradient jumps, are moved
    moved = 0.15 * torch.randn(m, generator=g, device="cuda")
    for border in (math.log(1 - case["low"]), math.log(1 + case["high"])):
        moved = torch.where((moved - border).abs() < 2e-3, border + 4e-3, moved)
    state["old"] = now - moved
    state["reference"] = now + 0.2 * torch.randn(m, generator=g, device="cuda") if case["kl"] else None
    state["advantages"] = torch.randn(m, generator=g, device="cuda")
    ids = ids[:, 0]
    left = int(case["padding"] * m)  # a prompt's tokens stand in front
    ids[:left] = -1
    if left and case["masked"]:
        x[0] = float("-inf")
    state["ids"] = ids
    state["grad_loss"] = torch.full((m,), _loss_scale(case["dtype"]) / max(1, m - left), device="cuda")
    return state


def _prepare_balance(case, g, state):
    m, e, k = case["m"], case["e"], case["k"]
    x = _randn(g, m, e, FLOATS[case["dtype"]], 1.0, case["pad"])
    x += torch.randn(e, generator=g, device="cuda").to(x.dtype)  # some experts are liked better
    experts = x.float().topk(k, dim=1).indices
    if case["dropped"]:  # choices that found their expert full
        experts[_rand(g, m, k) < 0.1] = -1
    experts[: int(case["padding"] * m)] = -1
    state["logits"], state["experts"] = x, experts
    state["grad_loss"] = torch.tensor(_loss_scale(case["dtype"]), device="cuda")
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["what"] == "policy":
        return _prepare_policy(case, g, state)
    if case["what"] == "balance":
        return _prepare_balance(case, g, state)
    m, n, d = case["m"], case["n"], case["d"]
    if case["what"] == "gradient":
        state["ids"] = _table_ids(case, g, m)
        state["grad"] = _randn(g, m, d, FLOATS[case["grad"]], 0.01 * _loss_scale(case["grad"]) ** 0.5, case["pad"])
        return state
    state["ids"] = _table_ids(case, g, m * case["t"]).view((m, case["t"]) if case["t"] > 1 else (m,))
    if case["table"] == "int8":
        state["table"] = torch.randint(-127, 128, (n, d), generator=g, device="cuda", dtype=torch.int8)
        state["row_scales"] = (0.5 + _rand(g, n)) / 127
    else:
        state["table"], state["row_scales"] = _randn(g, n, d, FLOATS[case["table"]], 0.05), None
    return state


# -------------------------------------------------------------------------------------------------------------- passes


def _plain_embed(state):
    case, ids = state["case"], state["ids"]
    at = ids.clamp_min(0)
    rows = state["table"][at].float()
    if state["row_scales"] is None:
        rows = rows * case["scale"]
    else:
        rows = rows * (state["row_scales"][at] * case["scale"])[..., None]
    return torch.where((ids >= 0)[..., None], rows, 0).to(FLOATS[case["out"]])


def _plain_gradient(state):
    case, ids, grad = state["case"], state["ids"], state["grad"]
    kept = torch.where((ids >= 0)[:, None], grad.float(), 0)
    out = torch.zeros((case["n"], case["d"]), device="cuda").index_add_(0, ids.clamp_min(0), kept)
    return (out * case["scale"]).to(FLOATS[case["out"]])


def _plain_softmax(x, temperature=1.0):
    """z = x / temperature, its log-sum-exp and probabilities; a row with nothing has no probability anywhere."""
    z = x.float() / temperature
    top = z.amax(1)
    top = torch.where(top == float("-inf"), 0, top)
    e = torch.exp(z - top[:, None])
    s = e.sum(1)
    return z, top + torch.log(s), e / torch.where(s > 0, s, 1)[:, None]


def _plain_policy(state):
    case, x, ids = state["case"], state["logits"], state["ids"]
    listed_ = ids >= 0
    at = ids.clamp_min(0)[:, None]
    z, lse, p = _plain_softmax(x, case["temperature"])
    log_p = torch.where(p > 0, z - lse[:, None], 0)
    entropy = -(p * log_p).sum(1)
    now = z.gather(1, at)[:, 0] - lse
    now = torch.where(listed_, now, 0)
    a = state["advantages"]
    ratio = torch.exp(now - state["old"])
    kept = ratio.clamp(1 - case["low"], 1 + case["high"])
    loss = -torch.minimum(ratio * a, kept * a)
    slope = torch.where(ratio * a <= kept * a, -ratio * a, 0)
    if case["kl"]:
        far = state["reference"] - now
        loss = loss + case["kl"] * (torch.expm1(far) - far)
        slope = slope - case["kl"] * torch.expm1(far)
    loss = loss - case["entropy"] * entropy
    g = torch.where(listed_, state["grad_loss"] / case["temperature"], 0)[:, None]
    grad = p * (case["entropy"] * (log_p + entropy[:, None]) - slope[:, None])
    grad.scatter_add_(1, at, slope[:, None])
    grad = torch.where(listed_[:, None], grad * g, 0)
    return [torch.where(listed_, v, 0) for v in (loss, now, entropy, lse)] + [grad.to(x.dtype)]


def _plain_balance(state):
    case, x, experts = state["case"], state["logits"], state["experts"]
    e = case["e"]
    counted = (experts >= 0).any(1)
    rows = counted.sum().clamp_min(1)
    counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    counts.scatter_add_(0, torch.where(experts >= 0, experts, e).view(-1), torch.ones_like(experts).view(-1))
    counts = counts[:e]
    f = counts.float() / counts.sum().clamp_min(1)
    _, lse, p = _plain_softmax(x)
    p, lse = torch.where(counted[:, None], p, 0), torch.where(counted, lse, 0)
    probs = p.sum(0) / rows
    loss = e * (f * probs).sum() + case["z"] * (lse * lse).sum() / rows
    grad = p * (e * (f - (p @ f)[:, None]) + 2 * case["z"] * lse[:, None]) * (state["grad_loss"] / rows)
    return loss, counts, probs, lse, grad.to(x.dtype)


PLAIN = {"embed": _plain_embed, "gradient": _plain_gradient, "policy": _plain_policy, "balance": _plain_balance}


def _package(state):
    import octex_amd

    case = state["case"]
    if case["what"] == "embed":
        return octex_amd.embed(state["table"], state["ids"], row_scales=state["row_scales"], scale=case["scale"],
                               dtype=case["out"])
    if case["what"] == "gradient":
        return octex_amd.embed_backward(state["grad"], state["ids"], case["n"], scale=case["scale"], dtype=case["out"])
    if case["what"] == "policy":
        args = (state["logits"], state["ids"], state["old"], state["advantages"])
        how = dict(ref_log_probs=state["reference"], clip=(case["low"], case["high"]), kl=case["kl"],
                   entropy=case["entropy"], temperature=case["temperature"])
        if case["form"] == "step":
            r, grad = octex_amd.policy_step(state["grad_loss"], *args, **how)
        else:
            r = octex_amd.policy_loss(*args, **how)
            grad = octex_amd.policy_loss_backward(state["grad_loss"], *args, r, **how)
        return [r.loss, r.log_probs, r.entropy, r.lse, grad]
    args, how = (state["logits"], state["experts"]), dict(weight=1.0, z_weight=case["z"])
    if case["form"] == "step":
        r, grad = octex_amd.balance_step(state["grad_loss"], *args, **how)
    else:
        r = octex_amd.balance_loss(*args, **how)
        grad = octex_amd.balance_loss_backward(state["grad_loss"], *args, r, **how)
    return r.loss, r.counts, r.probs, r.lse, grad


def run(state):
    return _package(state) if own else PLAIN[state["case"]["what"]](state)


# ------------------------------------------------------------------------------------------ what a pass is held against


def work(case):
    """Every input read once and every output written once; of a table, as many rows as there are ids.  An exponential, its
    sum and its weighted sum are taken as 6 operations a logit, a gradient as 4 more."""
    if case["what"] == "embed":
        ids, size = case["m"] * case["t"], SIZES[case["table"]]
        row = case["d"] * size + (4 if size == 1 else 0)
        return {"bytes": 8 * ids + min(ids, case["n"]) * row + ids * case["d"] * SIZES[case["out"]],
                "flops": 1.0 * ids * case["d"]}
    if case["what"] == "gradient":
        m, n, d = case["m"], case["n"], case["d"]
        return {"bytes": 8 * m + m * d * SIZES[case["grad"]] + n * d * SIZES[case["out"]], "flops": 1.0 * m * d}
    if case["what"] == "policy":
        m, row = case["m"], case["n"] * SIZES[case["dtype"]]
        read = m - int(case["padding"] * m)
        return {"bytes": (read + m) * row + m * (8 + 4 * (8 if case["kl"] else 7)), "flops": 10.0 * read * case["n"]}
    m, e, k = case["m"], case["e"], case["k"]
    read = m - int(case["padding"] * m)
    return {"bytes": (read + m) * e * SIZES[case["dtype"]] + 8 * m * k + 4 * m + 12 * e, "flops": 10.0 * read * e}


def _exact_embed(case, state):
    out = torch.empty((*state["ids"].shape, case["d"]), dtype=torch.float64, device="cuda").view(-1, case["d"])
    ids = state["ids"].reshape(-1)
    for a in range(0, len(ids), 8192):
        i = ids[a : a + 8192]
        rows = torch.index_select(state["table"], 0, torch.where(i < 0, 0, i)).to(torch.float64) * case["scale"]
        if state["row_scales"] is not None:
            rows *= state["row_scales"].double()[torch.where(i < 0, 0, i)].unsqueeze(1)
        rows[i < 0] = 0.0
        out[a : a + 8192] = rows
    return out.view(*state["ids"].shape, case["d"])


def _exact_gradient(case, state):
    keep = torch.nonzero(state["ids"] >= 0)[:, 0]
    out = torch.zeros((case["n"], case["d"]), dtype=torch.float64, device="cuda")
    for a in range(0, len(keep), 8192):
        at = keep[a : a + 8192]
        out.index_put_((state["ids"][at],), state["grad"][at].double() * case["scale"], accumulate=True)
    return out


def _exact_policy(case, state, a, b):
    t, ids = case["temperature"], state["ids"][a:b]
    use = torch.nonzero(ids >= 0)[:, 0]
    logp = torch.log_softmax(state["logits"][a:b][use].double() / t, 1)
    p, row, chosen = logp.exp(), torch.arange(len(use), device="cuda"), ids[use]
    weighted = torch.where(p > 0, logp, 0)
    entropy = -(p * weighted).sum(1)
    now = logp[row, chosen]
    adv = state["advantages"][a:b][use].double()
    ratio = (now - state["old"][a:b][use].double()).exp()
    low, high = 1 - case["low"], 1 + case["high"]
    bound = torch.where(adv < 0, low, high)
    clipped = torch.where(adv < 0, ratio < low, ratio > high)
    loss = -adv * torch.where(clipped, bound, ratio) - case["entropy"] * entropy
    slope = torch.where(clipped, 0, -adv * ratio)
    if case["kl"]:
        d = state["reference"][a:b][use].double() - now
        loss += case["kl"] * (d.exp() - 1 - d)
        slope += case["kl"] * (1 - d.exp())
    grad = -slope[:, None] * p + case["entropy"] * p * (weighted + entropy[:, None])
    grad[row, chosen] += slope
    grad *= state["grad_loss"][a:b][use].double()[:, None] / t
    x = state["logits"][a:b][use].double() / t
    out = [loss, now, entropy, torch.logsumexp(x, 1), grad]
    return [torch.zeros((b - a, *v.shape[1:]), dtype=torch.float64, device="cuda").index_copy_(0, use, v) for v in out]


def _exact_balance(case, state):
    e, experts = case["e"], state["experts"]
    use = torch.nonzero(experts.max(1).values >= 0)[:, 0]
    rows = max(1, len(use))
    counts = torch.bincount(experts[experts >= 0], minlength=e)
    f = counts.double() / max(1, int(counts.sum()))
    x = state["logits"][use].double()
    p, lse = torch.softmax(x, 1), torch.logsumexp(x, 1)
    probs = p.sum(0) / rows
    loss = e * torch.dot(f, probs) + case["z"] * lse.square().sum() / rows
    inner = f[None, :] - torch.mv(p, f)[:, None]
    grad = torch.zeros(state["logits"].shape, dtype=torch.float64, device="cuda")
    grad[use] = p * (e * inner + 2 * case["z"] * lse[:, None]) * (state["grad_loss"].double() / rows)
    return loss, counts, probs, torch.zeros(case["m"], dtype=torch.float64, device="cuda").index_copy_(0, use, lse), grad


def exact(case, seed):
    state = prepare(case, seed)
    if case["what"] == "policy":
        step = max(1, 32_000_000 // case["n"])
        parts = [_exact_policy(case, state, a, min(case["m"], a + step)) for a in range(0, case["m"], step)]
        return [torch.cat(p) for p in zip(*parts)]
    return {"embed": _exact_embed, "gradient": _exact_gradient, "balance": _exact_balance}[case["what"]](case, state)
