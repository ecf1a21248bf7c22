"""The operators at both ends of a training step together, as one step of a routed query encoder; and their C entries with outputs
and workspaces between guard bytes.

Bounds, derived before the first run: 32-bit logits h . v of d values are off by (d + 4) E of sum |h| |v|, which with the sums'
own error is that of a log probability, D; a probability or ratio is off by 2 D of itself and a gradient's terms by 4 D of
theirs; each of the products and sums behind (over columns, then over a token's places) adds E of the sum of sizes a step."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from operators64 import E, TYPES, close, gen, padded, randn, softmax64, sum_error  # noqa: E402
from test_gpu_balance import Rows as BalanceRows  # noqa: E402
from test_gpu_policy import Rows as PolicyRows  # noqa: E402
from test_gpu_scores_outputs import Guarded, O, S, call, check, sized, whole  # noqa: E402, F401
from test_gpu_tables import ids_of, table_of  # noqa: E402


@pytest.mark.parametrize("batch,length,n,d,pool,experts,k", [(3, 5, 40, 24, 60, 4, 1), (40, 33, 900, 48, 700, 16, 2),
                                                             (60, 40, 90, 32, 5000, 8, 2)])
def test_a_step_of_a_routed_query_encoder(O, batch, length, n, d, pool, experts, k):  # noqa: F811
    """Tokens through a table; a router over experts, whose choices are its own best; a policy over a pool of rows; back to the
    table's gradient.  Short queries are padded."""
    g = gen(batch)
    scale, kl, weight, z = d**0.5, 0.05, 0.5, 0.1
    table, router, rows = 0.1 * randn(g, n, d), randn(g, d, experts) / d**0.5, randn(g, pool, d) / d**0.5
    tokens = torch.randint(0, n, (batch, length), generator=g, device="cuda")
    left = torch.randint(1, length + 1, (batch, 1), generator=g, device="cuda")
    tokens[torch.arange(length, device="cuda")[None] >= left] = -1
    used = (tokens >= 0).view(-1)
    m = batch * length

    h = O.embed(table, tokens, scale=scale).view(m, d)
    routed, scores = h @ router, h @ rows.T
    chosen = O.log_probs(routed, tokens.view(-1, 1), top=k).top_ids
    chosen[~used] = -1
    ids = torch.randint(0, pool, (m,), generator=g, device="cuda")
    ids[~used] = -1
    lse, log_p, p = softmax64(scores)
    now = log_p.gather(1, ids.clamp_min(0)[:, None])[:, 0]
    moved = 0.1 * randn(g, m)  # inside the bounds of 0.5 and 2
    old, ref, adv = (now - moved).float(), (now + 0.2 * randn(g, m)).float(), randn(g, m)
    each = torch.full((m,), 1.0 / int(used.sum()), device="cuda")
    policy, d_scores = O.policy_step(each, scores, ids, old, adv, ref_log_probs=ref, clip=(0.5, 1.0), kl=kl)
    balance, d_routed = O.balance_step(None, routed, chosen, weight=weight, z_weight=z)
    d_h = (d_scores @ rows + d_routed @ router.T).view(batch, length, d)
    got = O.embed_backward(d_h, tokens, n, scale=scale)

    # the same in 64 bits, by torch's own differentiation
    leaf = table.double().requires_grad_()
    h64 = torch.where(used[:, None], leaf[tokens.view(-1).clamp_min(0)] * scale, 0.0)
    x, q = h64 @ rows.double().T, h64 @ router.double()
    lp = torch.log_softmax(x, 1).gather(1, ids.clamp_min(0)[:, None])[:, 0]
    ratio, far = (lp - old.double()).exp(), ref.double() - lp
    assert ((ratio > 0.5) & (ratio < 2))[used].all()
    losses = -ratio * adv.double() + kl * (far.exp() - 1 - far)
    counts = torch.bincount(chosen[used].view(-1), minlength=experts).double()
    probs = torch.softmax(q, 1)[used].mean(0)
    evenness = weight * experts * (counts / counts.sum() * probs).sum() + z * torch.logsumexp(q, 1)[used].square().mean()
    (torch.where(used, losses, 0.0).sum() / used.sum() + evenness).backward()

    with torch.no_grad():
        near = ((d + 4) * E * (h64.abs() @ rows.double().abs().T).max() + sum_error(pool) + 16 * E * (1 + lse.abs().max())).item()
        near_routed = ((d + 4) * E * (h64.abs() @ router.double().abs()).max() + sum_error(experts) + 16 * E * 8).item()
        one = torch.zeros_like(p).scatter_(1, ids.clamp_min(0)[:, None], 1.0)
        slope = ((ratio * adv).abs() + kl * (far.exp() + 1)) * each
        size = torch.where(used[:, None], slope[:, None] * (one + p), 0.0) @ rows.double().abs()
        steps = (pool + experts + d + 40) * E
        tol = (4 * near + steps) * size
        pr, f = torch.softmax(q, 1), counts / counts.sum()
        l = torch.logsumexp(q, 1).abs()[:, None]
        part = pr * (weight * experts * (f + pr @ f[:, None]) + 2 * z * (l + 1)) / used.sum()
        size_routed = torch.where(used[:, None], part, 0.0) @ router.double().abs().T
        tol = tol + (4 * near_routed + steps) * size_routed
        at = torch.where(used, tokens.view(-1), n)
        over = lambda v: torch.zeros((n + 1, d), dtype=torch.float64, device="cuda").index_add_(0, at, v)[:n] * scale
        most = torch.bincount(at, minlength=n + 1)[:n].max().item()
        bound = over(tol) + (most + 4) * E * over(size + size_routed)
        close(got, leaf.grad, bound + 1e-30, "the table's gradient")
        close(policy.loss[used], losses[used], (4 * near + 8 * E) * ((ratio * adv).abs() + kl * (far.exp() + 1 + far.abs()))[used],
              "the policy's loss")
        close(balance.loss, evenness, (4 * near_routed + (m / 1024 + 80) * E) * (evenness + 2 * z * l.max()), "the balance's loss")
        assert torch.equal(balance.counts.double(), counts) and int(balance.rows) == int(used.sum())
        assert (policy.loss[~used] == 0).all() and (d_routed[~used] == 0).all() and (d_scores[~used] == 0).all()


@pytest.mark.parametrize("d", [1, 3, 8, 13, 64, 65, 513, 1001])
@pytest.mark.parametrize("kind", ["int8", *TYPES])
def test_rows_between_guard_bytes(O, S, d, kind):  # noqa: F811
    g = gen(d)
    table, scales = table_of(g, 50, d, kind)
    for m in (1, 6, 130):
        ids = ids_of(g, m, 50, "any")[:, None]
        for dtype in TYPES:
            want = O.embed(table, ids[:, 0], row_scales=scales, scale=0.37, dtype=dtype)
            for pad, odd in ((0, 1), (1, 0), (13, 3)):
                out = Guarded((m, d), TYPES[dtype], pad, odd)
                call(S, "octexEmbed", whole(S, table), None if scales is None else scales.data_ptr(), whole(S, ids), 0.37,
                     out.matrix(S))
                check([("rows", out, want)])


@pytest.mark.parametrize("m,n,d", [(1, 1, 1), (40, 300, 7), (700, 90, 65), (1500, 301, 13), (9000, 2000, 264), (20_000, 40, 1001),
                                   (70_000, 5000, 24), (600_000, 3000, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_between_guard_bytes(O, S, m, n, d, dtype):  # noqa: F811
    g = gen(m)
    grad, ids = randn(g, m, d).to(TYPES[dtype]), ids_of(g, m, n, "common")
    want = O.embed_backward(grad, ids, n, scale=0.37)
    column = ids[:, None]
    for pad, odd in ((0, 1), (1, 0), (13, 3)):
        out = Guarded((n, d), TYPES[dtype], pad, odd)
        sized(S, "octexEmbedBackward", whole(S, grad), whole(S, column), 0.37, 0, out.matrix(S))
        check([("gradient", out, want)])
        out = Guarded((n, d), TYPES[dtype], pad, odd)
        out.t.fill_(1.0)
        sized(S, "octexEmbedBackward", whole(S, grad), whole(S, column), 0.37, 1, out.matrix(S))
        check([("added gradient", out, O.embed_backward(grad, ids, scale=0.37, add_to=torch.ones_like(want)))])


@pytest.mark.parametrize("m,n", [(3, 3), (7, 9), (5, 3001), (2100, 5), (2100, 701), (2100, 3001), (300, 20_011), (20, 60_003),
                                 (600, 40_001), (3, 65_537), (2, 200_003)])
@pytest.mark.parametrize("dtype", TYPES)
def test_policies_between_guard_bytes(O, S, m, n, dtype):  # noqa: F811
    r = PolicyRows(m, n, dtype)
    want, grad = O.policy_step(r.grad_loss, *r.args, **r.how)
    apart = O.policy_loss(*r.args, **r.how)
    back = O.policy_loss_backward(r.grad_loss, *r.args, apart, **r.how)
    column = r.ids[:, None]
    x = padded(r.x, 3)
    args = (whole(S, x), whole(S, column), r.T, r.old.data_ptr(), r.adv.data_ptr(), r.ref.data_ptr(), 1 - r.clip[0], 1 + r.clip[1],
            r.kl, r.entropy)
    for pad, odd in ((0, 1), (1, 0), (13, 3)):
        out, dx = [Guarded((m,)) for _ in range(4)], Guarded((m, n), TYPES[dtype], pad, odd)
        sized(S, "octexPolicyLossStep", *args, r.grad_loss.data_ptr(), *[v.at for v in out], dx.matrix(S))
        check([*zip(want._fields, out, want), ("gradient", dx, grad)])
        out, dx = [Guarded((m,)) for _ in range(4)], Guarded((m, n), TYPES[dtype], pad, odd)
        sized(S, "octexPolicyLoss", *args, *[v.at for v in out])
        call(S, "octexPolicyLossBackward", *args, r.grad_loss.data_ptr(), *[v.at for v in out[1:]], dx.matrix(S))
        check([*zip(apart._fields, out, apart), ("gradient", dx, back)])


@pytest.mark.parametrize("m,e,k", [(1, 1, 1), (7, 3, 2), (300, 60, 4), (4000, 257, 8), (900, 1300, 2), (40_000, 24, 2),
                                   (33_000, 500, 1), (3000, 2048, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_balances_between_guard_bytes(O, S, m, e, k, dtype):  # noqa: F811
    r = BalanceRows(m, e, k, dtype)
    want, grad = O.balance_step(r.grad_loss, r.x, r.experts, **r.how)
    back = O.balance_loss_backward(r.grad_loss, r.x, r.experts, want, **r.how)
    x = padded(r.x, 3)
    for pad, odd in ((0, 1), (1, 0), (13, 3)):
        out = [Guarded((1,)), Guarded((e,), torch.int64), Guarded((1,), torch.int64), Guarded((e,)), Guarded((m,))]
        dx, apart = Guarded((m, e), TYPES[dtype], pad, odd), Guarded((m, e), TYPES[dtype], pad, odd)
        sized(S, "octexBalanceLoss", whole(S, x), whole(S, r.experts), r.weight, r.z, *[v.at for v in out],
              r.grad_loss.data_ptr(), dx.matrix(S))
        call(S, "octexBalanceLossBackward", whole(S, x), whole(S, r.experts), r.weight, r.z, out[1].at, out[2].at,
             r.grad_loss.data_ptr(), apart.matrix(S))
        check([*zip(want._fields, out, [v.reshape(-1) if v.ndim == 0 else v for v in want]), ("gradient", dx, grad),
               ("gradient apart", apart, back)])
