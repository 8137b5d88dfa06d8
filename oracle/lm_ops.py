"""TEST INFRASTRUCTURE (oracle) -- not part of the product path.

The language-model operators (`stablehlo.custom_call` of the `rx.` targets, reactant.jl_amd/csrc/rx_lm.h) in numpy with
64-bit arithmetic, written from their formulas with plain loops over tokens and sequences.  They have no counterpart in the
reference; closed forms and differences pin them (tests/test_lm_operators.py)."""
import re

import numpy as np


def parse_config(text):
    """`{key = value : type, ..}` -> dict of numbers and strings."""
    out = {}
    for key, string, number in re.findall(r'(\w+)\s*=\s*(?:"([^"]*)"|([-+0-9.eE]+)(?:\s*:\s*\w+)?)', text):
        out[key] = string if not number else (float(number) if re.search(r"[.eE]", number) else int(number))
    return out


def embedding(table, ids, scale=1.0):
    ids = np.asarray(ids)
    flat = ids.reshape(-1)
    out = np.zeros((flat.size, table.shape[1]))
    for t, i in enumerate(flat):
        if 0 <= i < table.shape[0]:
            out[t] = np.float64(scale) * table[i]
    return out.reshape(ids.shape + (table.shape[1],))


def embedding_grad(dy, ids, rows, scale=1.0):
    width = dy.shape[-1]
    out = np.zeros((rows, width))
    for row, i in zip(dy.reshape(-1, width), np.asarray(ids).reshape(-1)):
        if 0 <= i < rows:
            out[i] += row
    return out * scale


def rotate(x, cos, sin, rotation):
    """x [heads, D] by the angles of one position, as products of complex numbers."""
    x = np.array(x, dtype=np.float64)
    half = len(cos)
    if rotation == "none":
        return x
    first = np.arange(half) * 2 if rotation == "pairs" else np.arange(half)
    second = first + (1 if rotation == "pairs" else half)
    z = (x[:, first] + 1j * x[:, second]) * (np.asarray(cos, dtype=np.float64) + 1j * np.asarray(sin, dtype=np.float64))
    x[:, first], x[:, second] = z.real, z.imag
    return x


def _slot(cache, page, slot, layout):
    return cache[page, slot] if layout == "slots" else cache[page, :, slot]


def _page_size(cache, layout):
    return cache.shape[1] if layout == "slots" else cache.shape[2]


def kv_append(q, k, v, cos, sin, position, sequence, pages, k_cache, v_cache, rotation="halves", layout="slots"):
    k_cache, v_cache = np.array(k_cache, dtype=np.float64), np.array(v_cache, dtype=np.float64)
    out = np.zeros(q.shape)
    size = _page_size(k_cache, layout)
    limit = pages.shape[1] * size
    if rotation != "none" and cos.shape[1]:
        limit = min(limit, cos.shape[0])
    for t in range(q.shape[0]):
        p, s = int(position[t]), int(sequence[t])
        if not (0 <= p < limit and 0 <= s < pages.shape[0]):
            continue
        c, d = (cos[p], sin[p]) if p < cos.shape[0] else (cos[:0].reshape(-1), sin[:0].reshape(-1))
        out[t] = rotate(q[t], c, d, rotation)
        page = int(pages[s, p // size])
        if 0 <= page < k_cache.shape[0]:
            _slot(k_cache, page, p % size, layout)[...] = rotate(k[t], c, d, rotation)
            _slot(v_cache, page, p % size, layout)[...] = v[t]
    return out, k_cache, v_cache


def paged_attention(q, k_cache, v_cache, pages, lengths, scale=None, window=0, layout="slots"):
    """(out, lse, sum of weights times |v|): the last for error bounds."""
    b, hq, d = q.shape
    size = _page_size(k_cache, layout)
    hk = k_cache.shape[2] if layout == "slots" else k_cache.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, lse, mag = np.zeros((b, hq, v_cache.shape[3])), np.full((b, hq), -np.inf), np.zeros((b, hq, v_cache.shape[3]))
    for s in range(b):
        n = min(max(int(lengths[s]), 0), pages.shape[1] * size)
        there = [j for j in range(max(0, n - window) if window else 0, n) if 0 <= pages[s, j // size] < k_cache.shape[0]]
        if not there:
            continue
        k = np.stack([_slot(k_cache, int(pages[s, j // size]), j % size, layout) for j in there]).astype(np.float64)   # [n, hk, d]
        v = np.stack([_slot(v_cache, int(pages[s, j // size]), j % size, layout) for j in there]).astype(np.float64)
        for h in range(hq):
            x = scale * (k[:, h // (hq // hk)] @ q[s, h].astype(np.float64))
            e = np.exp(x - x.max())
            w = e / e.sum()
            out[s, h] = w @ v[:, h // (hq // hk)]
            mag[s, h] = w @ np.abs(v[:, h // (hq // hk)])
            lse[s, h] = x.max() + np.log(e.sum())
    return out, lse, mag


def token_logprobs(logits, targets, top=0):
    x = np.asarray(logits, dtype=np.float64)
    shape, v = x.shape[:-1], x.shape[-1]
    x, y = x.reshape(-1, v), np.asarray(targets).reshape(-1)
    n = x.shape[0]
    logprob, lse, entropy = np.zeros(n), np.zeros(n), np.zeros(n)
    values, ids = np.zeros((n, top)), np.zeros((n, top), dtype=np.int32)
    for t in range(n):
        m = x[t].max()
        if m == -np.inf:
            lse[t], entropy[t] = -np.inf, 0.0
            logprob[t] = -np.inf if 0 <= y[t] < v else 0.0
            values[t], ids[t] = -np.inf, np.arange(top)
            continue
        with np.errstate(invalid="ignore"):
            e = np.exp(x[t] - m)
            lse[t] = m + np.log(e.sum())
            p = e / e.sum()
            entropy[t] = -(p[p > 0] * (x[t][p > 0] - lse[t])).sum() if not np.isnan(m) else np.nan
            if 0 <= y[t] < v:
                logprob[t] = x[t, y[t]] - lse[t]
        order = np.argsort(-np.where(np.isnan(x[t]), np.inf, x[t]), kind="stable")   # equal values by index
        nan = np.flatnonzero(np.isnan(x[t]))
        order = np.concatenate([nan, order[~np.isin(order, nan)]])                    # NaN counts as the largest
        ids[t] = order[:top]
        with np.errstate(invalid="ignore"):
            values[t] = x[t, ids[t]] - lse[t]
    res = [a.reshape(shape) for a in (logprob, lse, entropy)]
    return res + ([values.reshape(shape + (top,)), ids.reshape(shape + (top,))] if top else [])


def token_logprobs_grad(logits, targets, lse, entropy, d_logprob, d_entropy):
    x = np.asarray(logits, dtype=np.float64)
    v = x.shape[-1]
    flat, y = x.reshape(-1, v), np.asarray(targets).reshape(-1)
    l, h, g, e = (np.asarray(a, dtype=np.float64).reshape(-1) for a in (lse, entropy, d_logprob, d_entropy))
    out = np.zeros(flat.shape)
    for t in range(flat.shape[0]):
        if l[t] > -np.inf:
            z = flat[t] - l[t]
            p = np.exp(z)
            counts = 0 <= y[t] < v
            some = p > 0
            out[t, some] = -p[some] * ((g[t] if counts else 0.0) + e[t] * (z[some] + h[t]))
            if counts:
                out[t, y[t]] += g[t]
        elif 0 <= y[t] < v:
            out[t, y[t]] += g[t]
    return out.reshape(x.shape)


def evaluate(target, arrays, config):
    """Results of one custom_call on numpy arrays (numbers)."""
    if target == "rx.embedding":
        return [embedding(*arrays, scale=config.get("scale", 1.0))]
    if target == "rx.kv_append":
        return list(kv_append(*arrays, **config))
    if target == "rx.paged_attention":
        return list(paged_attention(*arrays, **config)[:2])
    if target == "rx.token_logprobs":
        return token_logprobs(*arrays, top=config.get("top", 0))
    if target == "rx.token_logprobs_grad":
        return [token_logprobs_grad(*arrays)]
    raise NotImplementedError("custom_call @%s" % target)
