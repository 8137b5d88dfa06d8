"""Language-model operators on the GPU against their formulas in 64 bits (oracle/lm_ops.py).

Bounds, with u the unit roundoff of a type (2^-24, 2^-11, 2^-8 for f32, f16, bf16; every rounding is off by at most u of its
value) and U that of f32:
  embedding      one product in f32, rounded: equal
  embedding_grad n terms summed in f32, times the scale: (n + 1) U of the sum of magnitudes, then u of the result
  append         two products and a sum in f32: 3 U of the magnitudes, then u of the result
  attention      scores are sums of D products: off by s = (D + 2) U scale |q|.|k|; weights by 2 s relative, and u where they
                 are rounded to the cache's type for the product with the values (in the weights and in their sum: 2 u); sums
                 over n positions, rescaled by exponentials (8 U each time the maximum grows, at most n times, but by a common
                 factor of weights and sum): (n + 16) U; then u of the result
  logprobs       sums of exponentials in chains of at most V / 64 + 64 terms, exponentials off by (|x - m| + 4) U: below
                 (V / 64 + 64 + 40 + 4) U of the sums
  gradient       p is off by (|x - lse| + 4) 2 U of p (x - lse rounds, the exponential rounds), the terms around it by 4 U of theirs
"""
import importlib

import numpy as np
import pytest

from _loader import load_pkg
from _harness import gpu_run
from oracle import lm_ops as L
from oracle import stablehlo_interp as I

load_pkg()
P = importlib.import_module("reactant_jl_amd.lm_programs")
pytestmark = pytest.mark.gpu
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
UF = U["f32"]
# results below the smallest normal number of a type are rounded to a fixed step
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}


def rounded(a, dt):
    return I.Tensor(I._round_to(np.asarray(a), dt), dt)


def close(got, ref, bound, dt="f32"):
    got, ref = np.asarray(got, dtype=np.float64), np.asarray(ref, dtype=np.float64)
    assert got.shape == ref.shape
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        ok = same | (np.abs(got - ref) <= bound + U[dt] * np.abs(ref) + TINY[dt])
    assert ok.all(), "%d of %d beyond the bound, first at %s: %r for %r" % ((~ok).sum(), ok.size, np.argwhere(~ok)[0], got[~ok][0], ref[~ok][0])


# ----------------------------------------------------------------------------
# embedding
# ----------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,rows,width,dt,idt,scale", [
    (1, 1, 1, "f32", "i32", 1.0), (37, 100, 64, "bf16", "i32", 32.0), (300, 1000, 33, "f16", "i64", 0.37), (5, 7, 1001, "bf16", "i64", 1.7), (129, 50, 260, "f32", "i32", 3.0),
])
def test_embedding(rx, client, tokens, rows, width, dt, idt, scale):
    rng = np.random.default_rng(tokens)
    table = rounded(rng.normal(size=(rows, width)), dt)
    ids = rng.integers(-2, rows + 2, size=tokens)
    ids[0] = rows - 1
    if idt == "i64" and tokens > 2:
        ids[1], ids[2] = 2 ** 32, -2 ** 40        # whole numbers whose low words are rows
    out, _ = gpu_run(rx, client, P.embedding(tokens, rows, width, dt=dt, ids=idt, scale=scale), [table, I.Tensor(ids, idt)])
    ref = np.zeros((tokens, width), dtype=np.float32)
    there = (ids >= 0) & (ids < rows)
    ref[there] = table.a[ids[there]].astype(np.float32) * np.float32(scale)
    assert np.array_equal(out[0].a, rounded(ref, dt).a)


GRADS = [
    (1, 1, 1, "f32", None, "i32", "any"), (40, 100, 64, "bf16", "f32", "i32", "any"), (513, 77, 100, "f32", None, "i32", "text"), (600, 37, 33, "f16", None, "i64", "any"),
    (700, 50, 24, "bf16", None, "i32", "one"), (0, 5, 8, "f32", None, "i32", "any"), (64, 9, 130, "f16", "f32", "i32", "none"), (3000, 20000, 40, "bf16", "f32", "i32", "text"),
    (5000, 300, 72, "f32", None, "i64", "text"), (20000, 1500, 16, "bf16", "f32", "i32", "text"), (20000, 40, 8, "f32", None, "i32", "one"),
]


@pytest.mark.parametrize("tokens,rows,width,dt,out,idt,how", GRADS)
def test_embedding_grad(rx, client, tokens, rows, width, dt, out, idt, how):
    rng = np.random.default_rng(rows)
    dy = rounded(rng.normal(size=(tokens, width)), dt)
    ids = rng.integers(-1, rows + 1, size=tokens)
    if how == "text":                              # a few rows have most tokens
        ids = np.minimum((rows ** rng.random(tokens)).astype(np.int64) - 1, rows - 1)
        ids[rng.random(tokens) < 0.02] = -1
    elif how == "one":
        ids[:] = rows - 3
        ids[::7] = rows - 2
    elif how == "none":
        ids[:] = -1
    text = P.embedding_grad(tokens, rows, width, dt=dt, out=out, ids=idt, scale=1.5)
    args = [dy, I.Tensor(ids, idt)]
    got, exe = gpu_run(rx, client, text, args)
    again, _ = gpu_run(rx, client, text, args, exe)
    assert np.array_equal(got[0].a, again[0].a)    # the same bits every run
    n = np.bincount(ids[(ids >= 0) & (ids < rows)], minlength=rows)
    mag = L.embedding_grad(np.abs(dy.a.astype(np.float64)), ids, rows, 1.5)
    close(got[0].a, L.embedding_grad(dy.a.astype(np.float64), ids, rows, 1.5), (n[:, None] + 1) * UF * mag, out or dt)
    assert np.all(got[0].a[n == 0] == 0)


def test_embedding_grad_order_of_tokens(rx, client):
    """A row's terms are summed as they come or in chunks of them, never in an order that a run chooses: exact in f32 where no
    partial sum rounds, in any order; and equal sums for a permutation of the tokens within what rounding allows."""
    rng = np.random.default_rng(5)
    tokens, rows, width = 9000, 11, 12
    dy = rng.integers(-500, 500, size=(tokens, width)).astype(np.float64)          # sums below 2^24
    ids = rng.integers(0, rows, size=tokens)
    got, _ = gpu_run(rx, client, P.embedding_grad(tokens, rows, width, dt="f32"), [I.Tensor(dy, "f32"), I.Tensor(ids, "i32")])
    assert np.array_equal(got[0].a, L.embedding_grad(dy, ids, rows))


# ----------------------------------------------------------------------------
# paged cache
# ----------------------------------------------------------------------------
def cache(rng, dt, pages, size, heads, dim, layout):
    return rounded(rng.normal(size=P.cache_shape(pages, size, heads, dim, layout)), dt)


def append_case(rng, tokens, seqs, hq, hk, d, dv, pages, size, cols, positions, r, dt, layout, idt):
    q, k, v = (rounded(rng.normal(size=(tokens, h, n)), dt) for h, n in ((hq, d), (hk, d), (hk, dv)))
    angle = rng.uniform(-3, 3, size=(positions, r // 2))
    table = rng.permutation(pages)[:seqs * cols].reshape(seqs, cols) if seqs * cols <= pages else rng.integers(0, pages, size=(seqs, cols))
    slots = [(s, p) for s in range(seqs) for p in range(min(cols * size, positions))]
    chosen = [slots[i] for i in rng.permutation(len(slots))[:tokens]]
    seq, pos = np.array([c[0] for c in chosen]), np.array([c[1] for c in chosen])
    kc, vc = cache(rng, dt, pages, size, hk, d, layout), cache(rng, dt, pages, size, hk, dv, layout)
    return [q, k, v, I.Tensor(np.cos(angle), "f32"), I.Tensor(np.sin(angle), "f32"), I.Tensor(pos, idt), I.Tensor(seq, idt), I.Tensor(table, idt), kc, vc]


APPENDS = [
    (1, 1, 1, 1, 2, 2, 1, 1, 1, 1, 2, "f32", "halves", "slots", "i32"), (3, 2, 8, 2, 64, 64, 20, 16, 4, 64, 64, "bf16", "halves", "slots", "i32"),
    (50, 5, 6, 3, 80, 48, 40, 24, 4, 60, 40, "f16", "pairs", "heads", "i64"), (29, 3, 4, 4, 33, 17, 9, 5, 3, 15, 32, "f32", "halves", "heads", "i32"),
    (200, 4, 16, 8, 128, 128, 40, 16, 5, 80, 128, "bf16", "pairs", "slots", "i32"), (20, 2, 2, 1, 256, 256, 60, 1, 30, 30, 128, "f16", "halves", "heads", "i32"),
    (7, 2, 3, 1, 96, 96, 12, 7, 6, 42, 96, "f32", "pairs", "slots", "i64"),
]


@pytest.mark.parametrize("tokens,seqs,hq,hk,d,dv,pages,size,cols,positions,r,dt,rotation,layout,idt", APPENDS)
def test_append(rx, client, tokens, seqs, hq, hk, d, dv, pages, size, cols, positions, r, dt, rotation, layout, idt):
    rng = np.random.default_rng(tokens)
    args = append_case(rng, tokens, seqs, hq, hk, d, dv, pages, size, cols, positions, r, dt, layout, idt)
    if tokens >= 20:                                # padding, positions and sequences that do not exist, pages outside the cache
        args[5].a[2], args[5].a[5], args[6].a[7], args[6].a[11] = -1, positions, seqs, -1
        args[7].a[0, 0], args[7].a[-1, -1] = pages, -1
    text = P.kv_append(tokens, seqs, hq, hk, d, pages, size, cols, positions, dt=dt, rotary_dim=r, rotation=rotation, layout=layout, ids=idt, value_dim=dv)
    got, _ = gpu_run(rx, client, text, args)
    a = [t.a for t in args]
    q, kc, vc = L.kv_append(*a, rotation=rotation, layout=layout)
    mag = L.kv_append(*[np.abs(t) for t in a[:5]], *a[5:], rotation="none", layout=layout)
    close(got[0].a, q, 3 * UF * 4 * np.abs(a[0]).max(), dt)
    close(got[1].a, kc, 3 * UF * 4 * np.abs(a[1]).max(), dt)
    assert np.array_equal(got[2].a, vc.astype(got[2].a.dtype))
    untouched = np.all(mag[1] == a[8], axis=-1)
    assert np.array_equal(got[1].a[untouched], a[8][untouched])


def test_append_without_rotation_copies_bits(rx, client):
    rng = np.random.default_rng(3)
    args = append_case(rng, 9, 2, 4, 2, 24, 24, 8, 4, 3, 12, 24, "bf16", "slots", "i32")
    got, _ = gpu_run(rx, client, P.kv_append(9, 2, 4, 2, 24, 8, 4, 3, 12, rotation="none"), args)
    q, kc, vc = L.kv_append(*[t.a for t in args], rotation="none")
    assert np.array_equal(got[0].a, q) and np.array_equal(got[1].a, kc) and np.array_equal(got[2].a, vc)


def test_append_donated_and_not(rx, client):
    """Donated caches are updated where they are; otherwise the arguments keep their contents."""
    rng = np.random.default_rng(4)
    args = append_case(rng, 9, 2, 4, 2, 24, 24, 8, 4, 3, 12, 24, "f32", "slots", "i32")
    thunk = rx.compile(P.kv_append(9, 2, 4, 2, 24, 8, 4, 3, 12, dt="f32"))
    dev = [rx.to_rarray(t.a.T, t.dt) for t in args]
    kept = thunk(*dev)
    assert np.array_equal(dev[8].to_array().T, args[8].a) and np.array_equal(dev[9].to_array().T, args[9].a)
    at = [d.data.buffer.unsafe_pointer() for d in dev[8:]]
    out = thunk(*dev, donated=[False] * 8 + [True, True])
    assert [o.data.buffer.unsafe_pointer() for o in out[1:]] == at and dev[8].donated
    for a, b in zip(kept, out):
        assert np.array_equal(a.to_array(), b.to_array())
    # one array given as both caches: each result is its own
    both = rx.to_rarray(args[8].a.T, "f32")
    out = thunk(*dev[:8], both, both, donated=[False] * 8 + [True, True])
    ref = L.kv_append(*[t.a for t in args[:9]], args[8].a)
    assert np.array_equal(out[2].to_array().T, ref[2].astype(np.float32))
    close(out[1].to_array().T, ref[1], 12 * UF * np.abs(args[1].a).max())


def attention_case(rng, lengths, hq, hk, d, dv, pages, size, cols, dt, layout, idt="i32"):
    b = len(lengths)
    q = rounded(rng.normal(size=(b, hq, d)), dt)
    kc, vc = cache(rng, dt, pages, size, hk, d, layout), cache(rng, dt, pages, size, hk, dv, layout)
    table = np.full((b, cols), -5, dtype=np.int64)
    used = np.zeros((pages, size), dtype=bool)
    order = rng.permutation(pages)
    at = 0
    for s, n in enumerate(lengths):
        need = min(-(-max(n, 0) // size), cols)
        table[s, :need] = order[at:at + need]
        for j in range(min(max(n, 0), cols * size)):
            used[table[s, j // size], j % size] = True
        at += need
        if need < cols:
            table[s, need:] = rng.choice([-1, pages, pages + 7, 0], size=cols - need)      # not looked at
    # what no sequence holds is not a number
    for c in (kc, vc):
        rows = c.a if layout == "slots" else c.a.transpose(0, 2, 1, 3)
        rows[~used] = np.nan
    return [q, kc, vc, I.Tensor(table, idt), I.Tensor(np.array(lengths), idt)]


def attention_bound(args, scale, lse, mag, dt, n):
    q, k = args[0].a.astype(np.float64), np.abs(np.nan_to_num(args[1].a.astype(np.float64))).max()
    s = (q.shape[2] + 2) * UF * scale * np.abs(q).sum(-1).max() * k
    return mag * (2 * U[dt] * (dt != "f32") + 2 * s + (n + 16) * UF), s + (n + 16) * UF * 2


ATTENTION = [
    ([1], 1, 1, 1, 1, 1, 1, "f32", "slots", 0, "i32"), ([0, 1, 2, 15, 16, 17], 8, 2, 64, 64, 16, 2, "bf16", "slots", 0, "i32"),
    ([33, 0, 64, 31], 4, 4, 128, 128, 32, 2, "f16", "heads", 0, "i64"), ([100, 7], 12, 12, 80, 80, 24, 5, "f32", "slots", 0, "i32"),
    ([513, 300, 77], 16, 1, 128, 128, 16, 40, "bf16", "heads", 0, "i32"), ([90, 200], 6, 2, 33, 17, 5, 40, "f16", "slots", 0, "i32"),
    ([70, 3, 129], 40, 2, 96, 64, 1, 130, "bf16", "slots", 0, "i32"), ([257], 7, 1, 256, 256, 64, 5, "bf16", "heads", 0, "i32"),
    ([200, 64, 3], 8, 2, 64, 128, 16, 13, "f32", "heads", 50, "i32"), ([1000, 2000, 1], 8, 8, 64, 64, 128, 16, "bf16", "slots", 65, "i64"),
    ([-3, 40, 5], 4, 2, 64, 64, 16, 2, "bf16", "slots", 0, "i32"), ([5000], 32, 8, 128, 128, 16, 313, "bf16", "slots", 0, "i32"),
    ([3000, 10], 64, 2, 192, 192, 48, 63, "f16", "heads", 0, "i32"), ([4100, 40], 34, 2, 80, 80, 16, 300, "f32", "slots", 0, "i32"), ([40] * 70, 4, 2, 16, 8, 8, 5, "bf16", "slots", 1, "i32"),
]


@pytest.mark.parametrize("lengths,hq,hk,d,dv,size,cols,dt,layout,window,idt", ATTENTION)
def test_attention(rx, client, lengths, hq, hk, d, dv, size, cols, dt, layout, window, idt):
    rng = np.random.default_rng(sum(lengths) + hq)
    pages = sum(-(-max(n, 0) // size) for n in lengths) + 2
    args = attention_case(rng, lengths, hq, hk, d, dv, pages, size, cols, dt, layout, idt)
    text = P.paged_attention(len(lengths), hq, hk, d, pages, size, cols, dt=dt, window=window, layout=layout, ids=idt, value_dim=dv, lse=True)
    got, _ = gpu_run(rx, client, text, args)
    out, lse, mag = L.paged_attention(*[t.a for t in args], window=window, layout=layout)
    bound, lse_bound = attention_bound(args, d ** -0.5, lse, mag, dt, max(lengths))
    close(got[0].a, out, bound, dt)
    close(got[1].a, lse, lse_bound)
    empty = np.array(lengths) <= 0
    assert np.all(got[0].a[empty] == 0) and np.all(got[1].a[empty] == -np.inf)


def test_attention_of_scores_far_apart(rx, client):
    """Scores from -1e4 to 1e4: the largest decides, nothing overflows; pages in use that do not exist are left out."""
    rng = np.random.default_rng(8)
    args = attention_case(rng, [300, 300], 8, 2, 64, 64, 40, 16, 20, "f32", "slots")
    args[0].a *= 1e4
    args[3].a[1, 3], args[3].a[1, 7] = -1, 40
    args[3].a[0, 0] = args[3].a[0, 1]                 # two places of a sequence on one page
    got, _ = gpu_run(rx, client, P.paged_attention(2, 8, 2, 64, 40, 16, 20, dt="f32", lse=True, scale=0.25), args)
    out, lse, mag = L.paged_attention(*[t.a for t in args], scale=0.25)
    s = 66 * UF * 0.25 * np.abs(args[0].a).sum(-1).max() * np.abs(np.nan_to_num(args[1].a)).max()
    close(got[1].a, lse, s + 1e-3)
    close(got[0].a, out, 2 * s * mag + 400 * UF * mag)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_attention_of_equal_keys_is_the_mean(rx, client, dt):
    """All weights equal: the mean of the values, which whole numbers give exactly in any split."""
    rng = np.random.default_rng(9)
    n, pages = 2048, 140
    args = attention_case(rng, [n, 64], 8, 2, 32, 32, pages, 16, 128, dt, "slots")
    args[1].a[...] = 0.5
    args[2].a[...] = np.round(np.nan_to_num(args[2].a) * 2)
    got, _ = gpu_run(rx, client, P.paged_attention(2, 8, 2, 32, pages, 16, 128, dt=dt), args)
    out, _, _ = L.paged_attention(*[t.a for t in args])
    assert np.array_equal(got[0].a, rounded(out, dt).a)


# ----------------------------------------------------------------------------
# token log probabilities
# ----------------------------------------------------------------------------
LOGITS = [
    (1, 1, 1, "f32", "i32"), (4, 100, 5, "bf16", "i32"), (3, 1001, 64, "f16", "i64"), (2, 7, 7, "f32", "i32"), (5, 32000, 20, "bf16", "i32"), (2, 50021, 3, "f32", "i32"),
    (1, 131072, 20, "bf16", "i32"), (70, 513, 0, "f16", "i32"), (9, 4096, 1, "f32", "i64"), (300, 1000, 5, "bf16", "i32"), (1, 300001, 10, "f16", "i32"), (600, 2051, 0, "bf16", "i32"),
]


def logits_case(rng, n, v, dt):
    x = rng.normal(size=(n, v)) * 3
    if v > 5:
        x[:, rng.permutation(v)[:v // 5]] = -np.inf
    if n > 2 and v > 1:
        x[1] = -np.inf                                 # nothing left
        x[2, :] = 0.5                                  # all alike: ties
        x[2, v // 2] = -np.inf
    y = rng.integers(0, v, size=n)
    if n > 3:
        y[3], y[0] = -1, v
    return rounded(x, dt), y


@pytest.mark.parametrize("n,v,top,dt,idt", LOGITS)
def test_token_logprobs(rx, client, n, v, top, dt, idt):
    rng = np.random.default_rng(v)
    x, y = logits_case(rng, n, v, dt)
    got, _ = gpu_run(rx, client, P.token_logprobs(n, v, top=top, dt=dt, ids=idt), [x, I.Tensor(y, idt)])
    ref = L.token_logprobs(x.a, y, top)
    e = (v / 64 + 64 + 44) * UF
    size = np.where(np.isfinite(ref[1]), np.abs(ref[1]), 0) * UF
    close(got[1].a, ref[1], e + 2 * size)
    close(got[0].a, ref[0], e + 3 * size)
    close(got[2].a, ref[2], 2 * e * (1 + np.abs(ref[2])) + 4 * size)
    if top:
        assert np.array_equal(got[4].a, ref[4])
        close(got[3].a, ref[3], (e + 3 * size)[:, None])


def test_token_logprobs_of_sorted_rows(rx, client):
    """The largest values next to one another, first and last, and rows with one value repeated."""
    v = 20000
    x = np.stack([np.linspace(-5, 5, v), np.linspace(5, -5, v), np.repeat(np.arange(v // 100), 100) * 0.01, np.zeros(v), np.where(np.arange(v) % 3 == 0, -0.0, 0.0)])
    x = rounded(x, "bf16")
    got, _ = gpu_run(rx, client, P.token_logprobs(5, v, top=64), [x, I.Tensor(np.arange(5), "i32")])
    assert np.array_equal(got[4].a, L.token_logprobs(x.a, np.arange(5), 64)[4])


def test_token_logprobs_of_special_values(rx, client):
    x = np.zeros((4, 300))
    x[0, 7] = np.nan
    x[1, 7], x[1, 9] = np.inf, 3.0
    x[2] = -np.inf
    x[2, 299] = -3e38
    x[3, :] = 3e38
    x = I.Tensor(x, "f32")
    got, _ = gpu_run(rx, client, P.token_logprobs(4, 300, top=2, dt="f32"), [x, I.Tensor([3, 3, 299, 3], "i32")])
    logprob, lse, ent, values, ids = [t.a for t in got]
    assert np.isnan(logprob[0]) and np.isnan(lse[0]) and np.isnan(ent[0]) and ids[0, 0] == 7 and ids[0, 1] == 0
    assert lse[1] == np.inf or np.isnan(lse[1])
    assert ids[1, 0] == 7 and ids[1, 1] == 9
    assert logprob[2] == 0 and ent[2] == 0 and values[2, 0] == 0 and np.array_equal(ids[2], [299, 0])
    assert lse[3] == np.float32(3e38) and np.array_equal(ids[3], [0, 1]) and abs(ent[3] - np.log(300)) < 1e-5


@pytest.mark.parametrize("n,v,dt,idt", [(1, 1, "f32", "i32"), (4, 100, "bf16", "i32"), (5, 1001, "f16", "i64"), (3, 50021, "bf16", "i32"), (6, 4096, "f32", "i32"), (200, 37, "bf16", "i32")])
def test_token_logprobs_grad(rx, client, n, v, dt, idt):
    rng = np.random.default_rng(v)
    x, y = logits_case(rng, n, v, dt)
    lse, ent = [a.astype(np.float32) for a in L.token_logprobs(x.a, y)[1:3]]
    g, h = rng.normal(size=n).astype(np.float32), rng.normal(size=n).astype(np.float32)
    args = [x, I.Tensor(y, idt)] + [I.Tensor(a, "f32") for a in (lse, ent, g, h)]
    got, _ = gpu_run(rx, client, P.token_logprobs_grad(n, v, dt=dt, ids=idt), args)
    ref = L.token_logprobs_grad(x.a, y, lse, ent, g, h)
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(np.isfinite(lse)[:, None] & np.isfinite(x.a), x.a.astype(np.float64) - lse[:, None], -1e3)
    p = np.exp(z)
    inner = np.abs(g)[:, None] + np.abs(h)[:, None] * (np.abs(z) + np.abs(ent)[:, None])
    bound = p * inner * ((np.abs(z) + 4) * 2 + np.abs(x.a).max(where=np.isfinite(x.a), initial=0) + 4) * UF + 4 * UF * np.abs(g)[:, None] * (np.arange(v) == y[:, None])
    close(got[0].a, ref, bound + 2.0 ** -126, dt)
    assert np.all(got[0].a[1] == 0) if n > 2 and v > 1 and not 0 <= y[1] < v else True


# ----------------------------------------------------------------------------
# together
# ----------------------------------------------------------------------------
def tie_gap(logits_row, k):
    s = np.sort(logits_row)[::-1]
    return np.abs(np.diff(s[:k + 1])).min()


@pytest.mark.parametrize("dt,layout,rotation", [("f32", "slots", "halves"), ("f32", "heads", "pairs")])
def test_decode_steps(rx, client, dt, layout, rotation):
    """Three tokens of three sequences, one of which ends early, through two layers: caches stay on the device, donated from
    step to step, against the interpreter's caches."""
    b, vocab, width, hq, hk, d, hidden, pages, size, cols, positions = 3, 101, 64, 8, 2, 32, 96, 14, 4, 4, 16
    text, types, cache_results = P.decode_step(b, vocab, width, hq, hk, d, hidden, pages, size, cols, positions, layers=2, top=3, dt=dt, layout=layout, rotation=rotation)
    rng = np.random.default_rng(11)
    values = [rng.normal(size=s) * (s[0] ** -0.5 if len(s) == 2 else 1.0) if t != "i32" else np.zeros(s) for s, t in types]
    angle = np.arange(positions)[:, None] * 10.0 ** -(np.arange(d // 2) / 4)[None, :]
    values[4], values[5] = np.cos(angle), np.sin(angle)
    values[3] = rng.permutation(pages)[:b * cols].reshape(b, cols)
    cache_args = [k for k, (s, t) in enumerate(types) if len(s) == 4]
    args = [rounded(v, t) if t != "i32" else I.Tensor(v, t) for v, (s, t) in zip(values, types)]
    thunk = rx.compile(text)
    dev = [rx.to_rarray(a.a.T, a.dt) for a in args]
    for step in range(3):
        pos = np.array([step, 5 + step, step if step < 2 else -1])
        for k, v in enumerate((rng.integers(0, vocab, b), rng.integers(0, vocab, b), pos)):
            args[k] = I.Tensor(v, "i32")
            dev[k] = rx.to_rarray(v.astype(np.int32))
        out = thunk(*dev, donated=[k in cache_args for k in range(len(dev))])
        ref = I.run_text(text, args, hifi=True)
        for k, r in zip(cache_args, cache_results):
            dev[k], args[k] = out[r], ref[r]
        for r in range(5):
            if r != 4:
                assert np.allclose(out[r].to_array().T, ref[r].a, atol=2e-4, rtol=2e-4), (step, r)
        assert np.array_equal(out[4].to_array().T, ref[4].a)
        for r in cache_results:
            assert np.allclose(out[r].to_array().T, ref[r].a, atol=1e-4, rtol=1e-4)


def test_a_model_of_one_table(rx, client):
    """Loss and gradient through lookup, product, log probabilities and entropy, against differences of the loss in 64 bits."""
    tokens, vocab, width, weight = 19, 23, 8, 0.1
    rng = np.random.default_rng(12)
    table = I.Tensor(rng.normal(size=(vocab, width)), "f32")
    ids, targets = rng.integers(0, vocab, tokens), rng.integers(0, vocab, tokens)
    ids[3], targets[5] = -1, -1

    def loss(t):
        h = L.embedding(t, ids)
        lp, _, ent = L.token_logprobs(h @ t.T, targets)
        return -(lp + weight * ent).sum() / tokens
    got, _ = gpu_run(rx, client, P.tied_head_step(tokens, vocab, width, entropy_weight=weight), [table, I.Tensor(ids, "i32"), I.Tensor(targets, "i32")])
    t = table.a.astype(np.float64)
    assert abs(float(got[0].a) - loss(t)) < 1e-5
    for _ in range(12):
        i, j = rng.integers(0, vocab), rng.integers(0, width)
        step = np.zeros_like(t)
        step[i, j] = 1e-4
        assert abs(got[1].a[i, j] - (loss(t + step) - loss(t - step)) / 2e-4) < 2e-5
