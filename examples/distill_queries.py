"""A query encoder taught by a search: the operators on rows of scores beside an octex index.

The index holds vectors; a teacher knows each training query's own vector and searches its nearest rows.  A student sees
only features of the query and learns, from the search's neighbors and distances, to score the rows as the teacher does:

    scores   = octex.int8_scores(student's vectors, 8-bit rows, bias = -|row|^2 / 2)   # ranks as squared distances
    loss, g  = octex.distill_step(weights, scores, neighbors, -distances / 2)          # q over the neighbors, p over all rows
    r        = octex.log_probs(scores, ids of the nearest rows, top=5)                 # how sure it is, and of what

    PYTHONPATH=. python examples/distill_queries.py [--steps 200]
"""

import argparse

import torch

import octex_amd as octex


def main(steps=200, n=20_000, dim=64, features=96, batch=256, k=10, temperature=4.0, rate=0.02, seed=0, quiet=False):
    """Trains the student; returns the first and the last mean loss, and the share of held-out queries whose nearest row is
    the student's likeliest before and after."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    centers = 3 * rand(50, dim)
    rows = centers[torch.randint(50, (n,), generator=g, device="cuda")] + rand(n, dim)
    torch.cuda.synchronize()  # a build does not wait for its dataset's producer
    index, _ = octex.build_in_memory(rows.half(), copies=40, list_len=32, table_len=32, log_buckets=14, member_lists=True)

    codes, scales = octex.quantize_rows(rows)
    rows8 = codes.float() * scales[:, None]  # what the codes stand for
    bias = -0.5 * (rows8 * rows8).sum(1)
    mixing = rand(features, dim) / features**0.5  # from a query's features to its vector: what the student has to learn
    weights = (mixing + 0.5 * rand(features, dim) / features**0.5).requires_grad_(False)

    def draw(m):
        vectors = centers[torch.randint(50, (m,), generator=g, device="cuda")] + rand(m, dim)
        return vectors @ torch.linalg.pinv(mixing), vectors

    def nearest(test):
        feats, vectors = test
        _, ids = index.search(vectors, k=1)
        scores = octex.int8_scores(feats @ weights, codes, scales, bias=bias)
        r = octex.log_probs(scores, ids, top=5, temperature=temperature)
        return r, (r.top_ids[:, :1] == ids).float().mean().item()

    test = draw(500)
    before = nearest(test)[1]
    losses = []
    for step in range(steps):
        feats, vectors = draw(batch)
        distances, neighbors = index.search(vectors, k=k)
        scores = octex.int8_scores(feats @ weights, codes, scales, bias=bias)
        # -|x - q|^2 / 2 is the score less a term of the query alone, which the teacher's softmax does not see
        loss, grad = octex.distill_step(torch.full((batch,), 1.0 / batch, device="cuda"), scores, neighbors, -0.5 * distances,
                                        temperature=temperature)
        weights -= rate * feats.t() @ (grad @ rows8)  # the scores' gradient passes the quantization as if it were not there
        losses.append(loss.mean().item())
        if not quiet and step % 20 == 0:
            print(f"step {step:4d}  loss {losses[-1]:.4f}", flush=True)
    r, after = nearest(test)
    if not quiet:
        print(f"nearest row likeliest: {before:.3f} before, {after:.3f} after; its mean log probability "
              f"{r.log_probs.mean().item():.3f}, entropy {r.entropy.mean().item():.3f}")
    return losses[0], losses[-1], before, after


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=200)
    main(steps=p.parse_args().steps)
