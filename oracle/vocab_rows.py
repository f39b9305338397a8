"""Plain 64-bit numpy forms of the operators on rows of logits, for the tests (nothing in the shipped package imports them).

The reference has no fused form of either: its sampler takes softmax and top-k of logits (backend.py:2260-2494), its
policy-gradient loss the log-probability of a token (rl_autograd.py:518-524).  Written from the formulas of the C interface.
"""
from __future__ import annotations

import numpy as np

F64 = np.float64
LEAST_REST = 2.0 ** -18   # what the roundings of a list in 32 bits can leave of a distribution


def log_softmax(x, temperature=1.0):
    """(log p, m, L) of rows x; rows of nothing but -inf give -inf throughout, NaN and +inf spoil their row."""
    x = np.asarray(x, F64)
    with np.errstate(all="ignore"):
        m = np.max(np.where(np.isnan(x), -np.inf, x), axis=1, keepdims=True)
        bad = np.isnan(x).any(1, keepdims=True) | (m == np.inf)
        d = np.where(x == -np.inf, -np.inf, (x - m) / temperature)
        total = np.log(np.sum(np.exp(d), axis=1, keepdims=True))
        lp = np.where(x == -np.inf, -np.inf, d - total)
    lp = np.where(bad, np.nan, lp)
    return lp, m[:, 0], np.where(bad, np.nan, total)[:, 0]


def entropy(lp):
    with np.errstate(all="ignore"):
        h = -np.sum(np.where(lp == -np.inf, 0.0, np.exp(lp) * lp), axis=1)
    return h


def order(x):
    """Unsigned keys in the order of the alternatives: NaN largest, -0 beside +0."""
    u = (np.ascontiguousarray(x, np.float32) + np.float32(0)).view(np.uint32)
    k = np.where(u >> 31, ~u, u | np.uint32(0x80000000))
    return np.where(np.isnan(x), np.uint32(0xFFFFFFFF), k)


def top(x, count):
    """Indices of the `count` largest of each row, equal ones by the lower index."""
    return np.argsort(-order(x).astype(np.int64), axis=1, kind="stable")[:, :count].astype(np.int32)


def token_logprobs(x, ids, temperature=1.0):
    """(logprob, entropy, log p, m, L)"""
    lp, m, total = log_softmax(x, temperature)
    has = (ids >= 0) & (ids < x.shape[1])
    got = np.where(has, np.take_along_axis(lp, np.where(has, ids, 0)[:, None].astype(np.int64), 1)[:, 0], 0.0)
    return got, entropy(lp), lp, m, total


def token_logprobs_backward(x, ids, dlogprob, dentropy, temperature=1.0):
    """(d logits, size): size bounds the terms that it is the difference of."""
    lp, m, _ = log_softmax(x, temperature)
    h = entropy(lp)[:, None]
    has = (ids >= 0) & (ids < x.shape[1])
    a = np.where(has, dlogprob if dlogprob is not None else 0.0, 0.0)[:, None].astype(F64)
    b = (np.zeros(len(x)) if dentropy is None else np.asarray(dentropy, F64))[:, None]
    onehot = np.zeros(lp.shape)
    onehot[np.flatnonzero(has), ids[has]] = 1.0
    with np.errstate(all="ignore"):
        p = np.exp(lp)
        finite = np.where(lp == -np.inf, 0.0, lp)
        g = (a * (onehot - p) - b * p * (finite + h)) / temperature
        size = (np.abs(a) * (onehot + p) + np.abs(b) * p * (np.abs(finite) + h + 1.0)) / temperature
    still = ((a == 0) & (b == 0)) | (np.asarray(x) == -np.inf).all(1, keepdims=True)
    return np.where(still, 0.0, g), np.where(still, 0.0, size), lp


def teacher(ids, t, vocab, temperature=1.0, rest=False):
    """(in use, q, ln q, r, row takes part); r of LEAST_REST and less is none."""
    used = (ids >= 0) & (ids < vocab)
    with np.errstate(all="ignore"):
        t = np.where(used, np.asarray(t, F64), -np.inf)
        m = np.max(t, axis=1, keepdims=True)
        row = m[:, 0] != -np.inf
        if rest:
            log_q = t
        else:
            d = np.where(t == -np.inf, -np.inf, (t - np.where(row[:, None], m, 0.0)) / temperature)
            log_q = d - np.log(np.sum(np.exp(d), axis=1, keepdims=True))
            log_q = np.where(t == -np.inf, -np.inf, log_q)
        q = np.where(row[:, None], np.exp(log_q), 0.0)
        left = 1.0 - q.sum(1)
        left = np.where(row & ~(left <= LEAST_REST), left, 0.0) if rest else np.zeros(len(t))
    return used, q, log_q, left, row


def distill(x, ids, t, row_scale=None, dloss=1.0, temperature=1.0, rest=False):
    """loss, row_loss, d logits, and for bounds of their errors: the sizes of the terms of both, ln p, ln p_rest, and `share`, the
    logarithm of an unlisted token's part of p_rest.  p_rest may be no number of 64 bits: its logarithm and the shares are formed
    from the unlisted logits alone."""
    n, v = x.shape
    lp, m, total = log_softmax(x, temperature)
    used, q, log_q, left, row = teacher(ids, t, v, temperature, rest)
    at = np.where(used, ids, 0).astype(np.int64)
    with np.errstate(all="ignore"):
        p = np.exp(lp)
        mass, listed = np.zeros((n, v)), np.zeros((n, v), bool)
        rows = np.arange(n)[:, None].repeat(ids.shape[1], 1)
        np.add.at(mass, (rows[used], at[used]), q[used])
        listed[rows[used], at[used]] = True
        share, m_out, total_out = log_softmax(np.where(listed, -np.inf, np.asarray(x, F64)), temperature)
        log_rest = np.where(m_out == -np.inf, -np.inf, (m_out - m) / temperature + total_out - total)
        part = np.exp(share)
        some = used & (q > 0)
        slot_lp = np.take_along_axis(lp, at, 1)
        row_loss = np.where(some, q * (log_q - slot_lp), 0.0).sum(1)
        size = np.where(some, q * (np.abs(log_q) + np.abs(slot_lp)), 0.0).sum(1) + 1.0
        has = left > 0
        row_loss = row_loss + np.where(has, left * (np.log(left) - log_rest), 0.0)
        size = size + np.where(has, np.abs(np.log(left)) + np.abs(log_rest), 0.0)
        row_loss = np.where(row, row_loss, 0.0)
        weight = np.full(n, 1.0 / n) if row_scale is None else np.asarray(row_scale, F64)
        take = weight != 0
        loss = np.sum(weight[take] * row_loss[take])
        full = (q.sum(1) + left)[:, None]
        has = (has & (m_out != -np.inf))[:, None]
        s = (dloss * weight / temperature)[:, None]
        g = s * (p * full - mass - np.where(has, left[:, None] * part, 0.0))
        gsize = np.abs(s) * (p * full + mass + np.where(has, (left[:, None] + 0.1) * part, 0.0))
    still = (~take | ~row | (np.asarray(x) == -np.inf).all(1) | (s[:, 0] == 0))[:, None]
    return {"loss": loss, "row_loss": row_loss, "loss_size": size, "dlogits": np.where(still, 0.0, g),
            "size": np.where(still, 0.0, gsize), "lp": lp, "log_rest": log_rest, "share": share,
            "weight": weight}
