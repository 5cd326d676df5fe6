"""Plain 64-bit forms of the selection operators, for the tests: routing to experts
and its gradient, beam selection and reordering, eviction from a cache.  Loops
over rows, from the definitions in include/mflat.h."""
import numpy as np
import torch

NEG = -np.inf
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# half a step of each type, relative to the value
HALF = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def scores(x, score):
    """Scores of one token's logits; -inf and NaN weigh nothing, +inf takes all."""
    x = np.where(np.isnan(x), NEG, x)
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return x, 1.0 / (1.0 + np.exp(-x))
    m = x.max(initial=NEG)
    if m == NEG:
        return x, np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        e = np.where(x == m, 1.0, np.where(x == NEG, 0.0, np.exp(x - m)))
    return x, e / e.sum()


def best(key, k):
    """Indices of the k largest keys above -inf, ties to the lowest, -1 padded."""
    order = np.lexsort((np.arange(len(key)), -key))[:k]
    out = np.full(k, -1)
    order = order[key[order] > NEG]
    out[:len(order)] = order
    return out


def quotients(x, score):
    """s_i / sum s over the chosen logits, from their logarithms."""
    if score == "softmax":
        ls = np.where(x == np.inf, 0.0, x if not np.isinf(x).any() else NEG)
    else:
        ls = -np.logaddexp(0.0, -x)
    e = np.exp(ls - ls.max())
    return e / e.sum()


def route(x, k, score, bias=None, mask=None, renormalise=False, scale=1.0, groups=1, kept=1, top=1):
    x, bias = f64(x), f64(bias)
    t, n = x.shape
    ids, w = np.full((t, k), -1), np.zeros((t, k))
    for i in range(t):
        if mask is not None and not mask[i]:
            continue
        xi, s = scores(x[i], score)
        b = np.zeros(n) if bias is None else np.where(np.isnan(bias), NEG, bias)
        sums = np.where(xi == NEG, NEG, s + b)
        key = xi if bias is None else sums
        if groups > 1:
            rank = np.full(groups, NEG)
            for g in range(groups):
                at = slice(g * n // groups, (g + 1) * n // groups)
                v = np.sort((key if bias is None and top == 1 else sums)[at][key[at] > NEG])[::-1][:top]
                if len(v):
                    rank[g] = v.sum()
            open_ = np.lexsort((np.arange(groups), -rank))[:kept]
            key = np.where(np.isin(np.arange(n) // (n // groups), open_), key, NEG)
        ids[i] = best(key, k)
        c = ids[i][ids[i] >= 0]
        if len(c):
            w[i, :len(c)] = scale * (quotients(xi[c], score) if renormalise else s[c])
    return ids, w


def lists(ids, experts):
    flat = ids.reshape(-1)
    at = np.flatnonzero(flat >= 0)
    order = at[np.argsort(flat[at], kind="stable")]
    start = np.searchsorted(flat[order], np.arange(experts + 1))
    return start, order


def route_grad(x, ids, g, score, renormalise=False, scale=1.0):
    """The gradient, and what the absolute values of its terms add up to: a difference
    is as far off as its two terms are, however small it is (with one expert w = 1,
    and g - g w has nothing left).  Differences check the formulas (the GPU tests)."""
    x, g = f64(x), f64(g)
    out, size = np.zeros_like(x), np.zeros_like(x)
    for t in range(x.shape[0]):
        xi, p = scores(x[t], score)
        use = np.array([j for j, e in enumerate(ids[t]) if 0 <= e < x.shape[1] and xi[e] > NEG], dtype=int)
        if not len(use):
            continue
        i, gi = np.asarray(ids[t])[use], g[t][use]
        with np.errstate(over="ignore"):
            rest = 1.0 / (1.0 + np.exp(xi))         # 1 - sigmoid(x)
        for to, s, gj in ((out, -1, gi), (size, 1, np.abs(gi))):
            if renormalise:
                w = quotients(xi[i], score)
                v = w * (gj + s * (gj * w).sum()) * (rest[i] if score == "sigmoid" else 1)
                np.add.at(to[t], i, v)
            elif score == "softmax":
                np.add.at(to[t], i, gj)
                to[t] = p * (to[t] + s * (gj * p[i]).sum())
            else:
                np.add.at(to[t], i, gj * p[i] * rest[i])
    return scale * out, abs(scale) * size


def beam(x, cum, k, finished=None, eos=-1):
    x, cum = f64(x), f64(cum)
    b, w, v = x.shape
    parents, tokens, out = np.full((b, k), -1), np.full((b, k), -1), np.full((b, k), NEG)
    for i in range(b):
        key = np.full((w, v), NEG)
        for j in range(w):
            if not np.isfinite(cum[i, j]):
                continue
            if finished is not None and finished[i, j]:
                key[j, eos] = cum[i, j]
                continue
            xi = np.where(np.isnan(x[i, j]), NEG, x[i, j])
            m = xi.max()
            if m == NEG:
                continue
            with np.errstate(invalid="ignore"):
                d = np.where(xi == m, 0.0, np.where(xi == NEG, NEG, xi - m))
            key[j] = cum[i, j] + (d - np.log(np.exp(d).sum()))
        at = best(key.ravel(), k)
        ok = at >= 0
        parents[i, ok], tokens[i, ok] = at[ok] // v, at[ok] % v
        out[i, ok] = key.ravel()[at[ok]]
    return parents, tokens, out


def reorder(rows, parents):
    """rows [outer][batch][beams][...]: torch tensor; a new one."""
    out = rows.clone()
    for b, line in enumerate(parents):
        for i, j in enumerate(line):
            if 0 <= j < len(line):
                out[:, b, i] = rows[:, b, j]
    return out


def evict(lens, seen, acc, pos, budget, recent, sink, weights=None, rows=None, group=1):
    """(new lens, acc', source slot of every slot below the new length) per (b, h).
    weights [b][heads * group][queries][slots]."""
    b, h, cap = acc.shape
    acc, out_lens, total, source = f64(acc), [], np.zeros((b, h, cap), np.float32), {}
    w = f64(weights)
    for i in range(b):
        n = min(max(int(lens[i]), 0), cap)
        m = min(n, budget)
        out_lens.append(m)
        for j in range(h):
            s = acc[i, j, :n].copy()
            if w is not None:
                q = w.shape[2] if rows is None else min(max(int(rows[i]), 0), w.shape[2])
                s += w[i, j * group:(j + 1) * group, :q, :n].sum((0, 1))
            total[i, j, :n] = s.astype(np.float32)
            p = pos[i, j, :n].astype(np.int64)
            fixed = (p < sink) | (p >= int(seen[i]) - recent)
            a = total[i, j, :n].astype(np.float64)
            a = np.where(fixed, 0.0, a)         # the protected are equals
            worth = np.where(np.isnan(a), -3.0, np.where(a == NEG, -2.0, np.where(a == np.inf, 2.0, 0.0)))
            order = np.lexsort((np.arange(n), -np.where(np.isfinite(a), a, 0.0), -worth, ~fixed))
            keep = np.zeros(n, bool)
            keep[order[:m]] = True
            at = np.arange(m)
            at[~keep[:m]] = m + np.flatnonzero(keep[m:])
            source[i, j] = at
    return np.array(out_lens), total, source
