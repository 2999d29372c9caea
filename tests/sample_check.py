"""The sampler's definition in 64 bits, one row at a time on the host."""
import math

import numpy as np

STEP = 2.0 ** -40  # the unit the weights are summed in, of the largest


def kept_weights(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(weights in index order, 0 for the entries that are not kept; how far the filters are from
    keeping another set, relative). None where there is nothing to choose."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return None
    margin = 1.0
    w = np.where(x == top, 1.0, 0.0)
    if not temperature > 0:
        w[:] = 0.0
        w[int(np.argmax(x))] = 1.0
        return w, margin
    if np.isfinite(top):
        with np.errstate(over="ignore", invalid="ignore"):
            w = np.where(np.isfinite(x), np.exp((x - top) / temperature), 0.0)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[np.isfinite(x[order]) | (x[order] == np.inf)]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        run = np.cumsum(w[order])
        share = float(top_p) * run[-1]
        n = min(len(order), 1 + int((run < share).sum()))
        margin = min(margin, float(np.abs(run - share).min() / run[-1])) if share > 0 else margin
        order = order[:n]
    if min_p > 0:
        q = min(float(min_p), 1.0)
        others = w[order][w[order] < 1.0]
        if len(others):
            margin = min(margin, float(np.abs(others / q - 1.0).min()))
        order = order[w[order] >= q]
    keep = np.zeros_like(w)
    keep[order] = w[order]
    return keep, margin


def slack_of(vocab):
    """A weight is off by its power's last place (2^-22 at most) and half a unit (STEP / 2) of the
    largest; the sums of `vocab` weights by as much."""
    return 2.0 ** -22 + vocab * STEP


def off_borders(logits, params):
    """The parameters without the shares and least weights whose border is too near to a sum or a weight
    to say which side is right."""
    params = {n: v.clone() for n, v in params.items()}
    for r in range(len(logits)):
        got = kept_weights(logits[r], **{n: v[r].item() for n, v in params.items()})
        if got is not None and got[1] <= 2 * slack_of(len(logits[r])):
            params["top_p"][r], params["min_p"][r] = 1.0, 0.0
    return params


def check_row(logits, token, logprob, uniform=0.0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, label=""):
    """The token's own stretch of the running weight holds u, and its logprob is that stretch's.

    Where a border of it is nearer to u than the sums are exact (slack_of), either side is right. The
    filters' own borders have to be further than that from any sum: asserted."""
    got = kept_weights(logits, temperature, top_k, top_p, min_p)
    token = int(token)
    if got is None:
        assert token in (-1, 0xffffffff) and logprob == -math.inf, label
        return
    w, margin = got
    slack = slack_of(len(w))
    assert margin > 2 * slack, f"{label}: inputs on a border of the filters ({margin})"
    assert 0 <= token < len(w) and w[token] > 0, f"{label}: token {token} is not kept"
    u = 0.0 if not uniform > 0 else min(float(uniform), 1.0)
    run = np.cumsum(w)
    total = run[-1]
    low, high = (run[token] - w[token]) / total, run[token] / total
    assert low - slack <= u <= high + slack, f"{label}: u {u} outside [{low}, {high}] of token {token}"
    want = math.log(w[token] / total)
    tol = 2 * slack + STEP / w[token] + 2.0 ** -23 * abs(want)
    assert abs(logprob - want) <= tol, f"{label}: logprob {logprob}, {want} expected"
