"""Choices from rows of scores, from their definitions, in 64 bits (numpy)."""
import math

import numpy as np

BIG = float(np.finfo(np.float32).max)


def to_bits(x, dtype):
    """fp32 values as the array of `dtype` that holds them rounded, and those rounded values as float64."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x, x.astype(np.float64)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float64)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r[np.isnan(x)] = 0x7FC0
    return r, from_bits(r, dtype)


def from_bits(a, dtype):
    if dtype == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def storage(dtype):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[dtype]


HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step among the smallest numbers


def adjust(x, history=None, lengths=None, first=None, rep=None, presence=None, frequency=None, offsets=None, ids=None, values=None,
           masks=None, mask_row=None, xadj=None, adjncy=None, states=None):
    """(rows of adjusted logits, a bound of the fp32 rounding errors made on the way, before the last rounding)."""
    rows, columns = x.shape
    out, size = x.astype(np.float64).copy(), np.abs(np.where(np.isfinite(x), x, 0.0))
    for r in range(rows):
        y = out[r]
        if history is not None:
            n = history.shape[1] if lengths is None else min(int(lengths[r]), history.shape[1])
            h, at = history[r, :n].astype(np.int64), np.arange(n)
            ok = h < columns
            seen = np.unique(h[ok])
            if rep is not None and seen.size:
                p = float(rep[r])
                y[seen] = np.where(y[seen] > 0, y[seen] / p, y[seen] * p)
                size[r][seen] = np.maximum(size[r][seen], np.abs(y[seen]))
            counted = ok & (at >= (0 if first is None else int(first[r])))
            c, k = np.unique(h[counted], return_counts=True)
            cost = (0.0 if presence is None else float(presence[r])) + (0.0 if frequency is None else float(frequency[r])) * k
            y[c] -= cost
            size[r][c] += np.abs(cost)
        if offsets is not None:
            lo, hi = min(int(offsets[r]), len(ids)), min(int(offsets[r + 1]), len(ids))
            for i in range(lo, hi):
                if ids[i] < columns:
                    y[ids[i]] += float(values[i])
                    size[r][ids[i]] += abs(float(values[i]))
        if masks is not None:
            m = r if mask_row is None else int(mask_row[r])
            if mask_row is None and masks.shape[0] == 1:
                m = 0
            if m != 0xFFFFFFFF:
                bits = np.unpackbits(masks[m].view(np.uint8), bitorder="little")[:columns] if m < masks.shape[0] else np.zeros(columns)
                y[bits == 0] = -np.inf
        if states is not None:
            v, stay = int(states[r]), np.zeros(columns, bool)
            if v < len(xadj) - 1:
                near = adjncy[xadj[v]:xadj[v + 1]]
                stay[near[near < columns]] = True
            y[~stay] = -np.inf
    # a quotient, a product, a sum, a difference, a handful of sums of biases: each off by at most 2^-24 of the largest term
    return out, size * 8 * 2.0 ** -24


def order_of(x):
    """Columns that are there, largest first, equal ones by column, and their values."""
    z = np.minimum(np.where(np.isnan(x), -np.inf, x), BIG)
    there = np.flatnonzero(z > -np.inf)
    o = there[np.argsort(-z[there], kind="stable")]
    return o, z[o]


def draw(x, t=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(id, logarithm of its probability, how many stay) of one row; the id is None for a row with nothing to draw."""
    o, z = order_of(x)
    if o.size == 0:
        return None, -math.inf, 0
    if not t > 0:
        return int(o[0]), 0.0, 1
    w = np.exp((z - z[0]) / t)
    n = o.size if not top_k else min(o.size, int(top_k))
    cum = np.cumsum(w[:n])
    if top_p < 1:
        n = min(n, 1 + int(np.searchsorted(cum, max(top_p, 0.0) * cum[-1], side="left")))
    if min_p > 0:
        n = min(n, max(1, int(np.count_nonzero(w >= min_p))))
    at = min(n - 1, int(np.searchsorted(cum[:n], u * cum[n - 1], side="right")))
    return int(o[at]), float((z[at] - z[0]) / t - math.log(cum[n - 1])), n


def philox_uniform(orc, seed, walker, step):
    x, y = [int(v) for v in orc.philox([walker & 0xFFFFFFFF, step, 0, 6], [seed & 0xFFFFFFFF, seed >> 32])[:2]]
    return ((x >> 5) * 2.0 ** 26 + (y >> 6)) * 2.0 ** -53


def _open(x):
    return np.where(np.isnan(x), -np.inf, np.minimum(x, BIG))


def scores(x, sigmoid):
    z = _open(x)
    if sigmoid:
        with np.errstate(over="ignore"):
            return np.where(z == -np.inf, 0.0, 1.0 / (1.0 + np.exp(-z)))
    top = np.max(z, axis=1, keepdims=True)
    e = np.exp(np.where(z == -np.inf, -np.inf, z - np.where(np.isfinite(top), top, 0.0)))
    total = e.sum(1, keepdims=True)
    return e / np.where(total > 0, total, 1.0)


def shares(x, ids, sigmoid):
    """Scores of the chosen over their sum, from their logarithms."""
    z = _open(x)
    l = z if not sigmoid else np.where(z == -np.inf, -np.inf, np.minimum(z, 0.0) - np.log1p(np.exp(-np.abs(np.where(np.isfinite(z), z, 0.0)))))
    c = np.where(ids < x.shape[1], np.take_along_axis(l, np.minimum(ids, x.shape[1] - 1).astype(np.int64), 1), -np.inf)
    top = c.max(1, keepdims=True)
    e = np.exp(np.where(c == -np.inf, -np.inf, c - np.where(np.isfinite(top), top, 0.0)))
    total = e.sum(1, keepdims=True)
    return e / np.where(total > 0, total, 1.0)


def route(x, k, sigmoid=False, bias=None, groups=1, kept=1, top2=False, renormalise=True, scale=1.0):
    rows, E = x.shape
    z, s = _open(x), scores(x, sigmoid)
    choice = s + (0.0 if bias is None else bias.astype(np.float64))
    if bias is None and not (groups > 1 and top2):
        choice = z  # both scores ascend with the logit
    choice = np.where(z == -np.inf, -np.inf, choice)
    ids = np.full((rows, k), 0xFFFFFFFF, np.uint32)
    for r in range(rows):
        c = choice[r].copy()
        if groups > 1 and kept < groups:
            worth = []
            for g in range(groups):
                part = np.sort(c[g * (E // groups):(g + 1) * (E // groups)])[::-1]
                part = part[part > -np.inf]
                worth.append(-np.inf if part.size == 0 else part[0] + part[1] if top2 and part.size > 1 else part[0])
            stay = np.argsort(-np.array(worth), kind="stable")[:kept]
            for g in range(groups):
                if g not in stay:
                    c[g * (E // groups):(g + 1) * (E // groups)] = -np.inf
        o = np.argsort(-c, kind="stable")
        o = o[c[o] > -np.inf][:k]
        ids[r, :o.size] = o
    if renormalise:
        w = shares(x, ids, sigmoid)
    else:
        w = np.where(ids < E, np.take_along_axis(s, np.minimum(ids, E - 1).astype(np.int64), 1), 0.0)
    return ids, w * scale, np.bincount(ids[ids < E].astype(np.int64), minlength=E).astype(np.uint32)


def route_backward(x, ids, dw, sigmoid=False, renormalise=True, scale=1.0):
    rows, E = x.shape
    s, out = scores(x, sigmoid), np.zeros((rows, E))
    there = (ids < E) & (np.take_along_axis(_open(x), np.minimum(ids, E - 1).astype(np.int64), 1) > -np.inf)
    g = np.where(there, dw.astype(np.float64) * scale, 0.0)
    at = np.minimum(ids, E - 1).astype(np.int64)
    sc = np.where(there, np.take_along_axis(s, at, 1), 0.0)
    if renormalise:
        p = shares(x, ids, sigmoid)
        d = p * (g - (g * p).sum(1, keepdims=True))
        if sigmoid:
            d *= 1.0 - sc
    elif sigmoid:
        d = g * sc * (1.0 - sc)
    else:
        d = g * sc
        out -= s * d.sum(1, keepdims=True)
    for r in range(rows):
        np.add.at(out[r], at[r][there[r]], d[r][there[r]])
    return out
