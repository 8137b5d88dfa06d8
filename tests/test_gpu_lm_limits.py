"""Language-model operators at what their numbers can hold: ties, values that are no numbers, infinities, large logits.  Bounds as
in test_gpu_lm_operators.py."""
import importlib

import numpy as np
import pytest

from _loader import load_pkg
from _harness import gpu_run
from oracle import lm_ops as L
from oracle import stablehlo_interp as I
import test_gpu_lm_operators as T

load_pkg()
P = importlib.import_module("reactant_jl_amd.lm_programs")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v,top", [(600, 9001, 20), (3, 40000, 64), (520, 40000, 1)])
def test_equal_logits_come_in_their_order_in_every_run(rx, client, n, v, top):
    """More equal elements than LDS holds in every row: a constant, a mask that leaves fewer than are asked for, two values in turn;
    whole rows and split ones."""
    x = np.zeros((n, v))
    x[1::3] = -np.inf
    for t in range(1, n, 3):
        x[t, np.random.default_rng(t).permutation(v)[:t % 5]] = 1.0
    x[2::3, ::2] = 1.0
    x = T.rounded(x, "bf16")
    exe = rx.xla_compile(client, P.token_logprobs(n, v, top=top))
    bufs = [rx.Buffer.from_host(client, np.frombuffer(x.to_bytes(), dtype=np.uint16).reshape(x.shape), "bf16"), rx.Buffer.from_host(client, np.zeros(n, np.int32), "i32")]
    want = L.token_logprobs(x.a, np.zeros(n, np.int32), top)[4]
    for _ in range(20):
        assert np.array_equal(exe.execute_sharded(bufs)[4].synced_buffer().to_host(), want)


@pytest.mark.parametrize("n,v,top,dt", [(4, 5, 5, "f32"), (4, 300, 2, "bf16"), (3, 1, 1, "f16"), (5, 64, 64, "f32"), (4, 70001, 20, "bf16"), (600, 1001, 7, "f16")])
def test_alternatives_of_rows_that_are_no_numbers(rx, client, n, v, top, dt):
    """NaN ranks first, in the order of the indices, wherever it stands: at the row's start, everywhere, at its end; all alternatives there are."""
    x = np.random.default_rng(v).normal(size=(n, v))
    x[0, 0] = np.nan
    x[1, :] = np.nan
    x[2, -1] = x[2, 0] = np.nan
    if n > 3:
        x[3, v // 2], x[3, 0] = np.nan, np.inf
    x = T.rounded(x, dt)
    got = [t.a for t in gpu_run(rx, client, P.token_logprobs(n, v, top=top, dt=dt), [x, I.Tensor(np.zeros(n), "i32")])[0]]
    want = L.token_logprobs(x.a, np.zeros(n, int), top)
    assert np.array_equal(got[4], want[4])
    no_number = np.isnan(x.a).any(1)
    for out in got[:3]:
        assert np.array_equal(np.isnan(out), no_number)
    assert np.isnan(got[3][no_number]).all() and not np.isnan(got[3][~no_number]).any()


@pytest.mark.parametrize("lengths,hq,hk,d,size,dt,layout", [
    ([5, 0, 70], 4, 2, 64, 16, "bf16", "slots"), ([3000, 40, 0, 1], 8, 1, 128, 16, "f16", "heads"), ([900, 33], 3, 3, 40, 7, "f32", "slots"), ([6000], 8, 2, 64, 64, "f32", "heads"),
    ([64] * 70, 24, 1, 32, 16, "bf16", "slots"),
])
def test_attention_of_what_is_no_number(rx, client, lengths, hq, hk, d, size, dt, layout):
    """A query with NaN, keys in use with NaN, and scores that are all -inf give NaN, in sequences of one part and of many; other
    heads and sequences keep their bits, and empty ones their zeros."""
    rng = np.random.default_rng(d)
    b = len(lengths)
    cols, pages = -(-max(lengths) // size) + 1, sum(-(-n // size) for n in lengths) + 2
    args = T.attention_case(rng, lengths, hq, hk, d, d, pages, size, cols, dt, layout)
    text = P.paged_attention(b, hq, hk, d, pages, size, cols, dt=dt, layout=layout, lse=True)
    clean, exe = gpu_run(rx, client, text, args)
    full = [s for s in range(b) if lengths[s]]

    def others_keep(got, sequence, heads):
        same = np.ones((b, hq), bool)
        same[sequence, heads] = False
        assert np.array_equal(got[0].a[same], clean[0].a[same]) and np.array_equal(got[1].a[same], clean[1].a[same])
    for s in {full[0], full[-1]}:
        q = args[0].a.copy()
        q[s, 1, 3] = np.nan                                             # every score of one head
        got, _ = gpu_run(rx, client, text, [I.Tensor(q, dt)] + args[1:], exe)
        assert np.isnan(got[0].a[s, 1]).all() and np.isnan(got[1].a[s, 1])
        others_keep(got, s, [1])
        at = rng.integers(0, lengths[s])                                # one key of one head
        k = args[1].a.copy()
        page, slot = args[3].a[s, at // size], at % size
        k[(page, slot, 0) if layout == "slots" else (page, 0, slot)] = np.nan
        got, _ = gpu_run(rx, client, text, [args[0], I.Tensor(k, dt)] + args[2:], exe)
        assert np.isnan(got[0].a[s, :hq // hk]).all() and np.isnan(got[1].a[s, :hq // hk]).all()
        others_keep(got, s, range(hq // hk))
        q = args[0].a.copy()
        q[s, 0] = 0.0
        q[s, 0, 0] = -np.inf                                            # all scores -inf: a sum of nothing
        k = args[1].a.copy()
        k[..., 0] = np.where(np.isnan(k[..., 0]), np.nan, 1.0)
        got, _ = gpu_run(rx, client, text, [I.Tensor(q, dt), I.Tensor(k, dt)] + args[2:], exe)
        assert np.isnan(got[0].a[s, 0]).all() and got[1].a[s, 0] == -np.inf
    for s in range(b):
        if not lengths[s]:
            assert np.all(clean[0].a[s] == 0) and np.all(clean[1].a[s] == -np.inf)


def test_attention_of_a_few_scores_of_minus_infinity(rx, client):
    """Positions whose scores are -inf among others count nothing, wherever the first finite one stands."""
    n, pages = 300, 20
    rng = np.random.default_rng(4)
    args = T.attention_case(rng, [n, 31], 4, 2, 64, 64, pages + 2, 16, 20, "f32", "heads")
    k = args[1].a
    k[..., 0] = np.where(np.isnan(k[..., 0]), np.nan, 1.0)
    finite = [5, 40, 299], [30]
    for s, js in enumerate(finite):
        for j in js:
            k[args[3].a[s, j // 16], :, j % 16] = 0.0
    args[0].a[:, :, 0] = -3.0e38                                        # times 1.0 and the scale's 8 beyond f32
    text = P.paged_attention(2, 4, 2, 64, pages + 2, 16, 20, dt="f32", layout="heads", lse=True, scale=8.0)
    got, _ = gpu_run(rx, client, text, args)
    v = args[2].a
    for s, js in enumerate(finite):                                     # scores of 0: their mean
        rows = np.stack([v[args[3].a[s, j // 16], :, j % 16] for j in js]).astype(np.float64)
        for h in range(4):
            assert np.all(np.abs(got[0].a[s, h] - rows[:, h // 2].mean(0)) <= 8 * T.UF * np.abs(rows[:, h // 2]).max(0))
            assert abs(got[1].a[s, h] - np.log(len(js))) <= 4 * T.UF


@pytest.mark.parametrize("n,v,top,dt,around", [(5, 1000, 5, "f32", 3.0e4), (5, 1000, 5, "f32", -3.0e4), (4, 33000, 20, "f16", 4.0e4), (3, 70001, 3, "bf16", 1.0e4), (600, 777, 1, "f32", 1.0e6), (4, 5000, 0, "f32", 5.0e3)])
def test_log_probabilities_of_large_logits(rx, client, n, v, top, dt, around):
    """A log probability is a difference of logits less the log of a sum of moderate size, whatever the logits' own magnitude: off by
    the sum's error (as for small logits) and roundings of the difference and of that log; the log of the sum of exponentials
    itself by those and its own rounding."""
    rng = np.random.default_rng(v)
    x = T.rounded(around + rng.normal(size=(n, v)) * 3, dt)
    y = np.argmax(x.a, 1)
    got = [t.a.astype(np.float64) for t in gpu_run(rx, client, P.token_logprobs(n, v, top=top, dt=dt), [x, I.Tensor(y, "i32")])[0]]
    want = L.token_logprobs(x.a, y, top)
    e = (v / 64 + 64 + 44) * T.UF
    below = want[1] - x.a.max(1)                                        # log of the sum of e^(x - max)
    error = e + 4 * T.UF * (np.abs(below) + 1)
    assert np.all(np.abs(got[1] - want[1]) <= error + T.UF * np.abs(want[1]))
    assert np.all(np.abs(got[0] - want[0]) <= error)
    assert np.all(np.abs(got[2] - want[2]) <= 2 * e * (1 + np.abs(want[2])) + 4 * T.UF * (np.abs(want[2]) + 1))
    if top:
        assert np.array_equal(got[4], want[4])
        far = x.a.max(1, keepdims=True) - np.take_along_axis(x.a, want[4], 1)
        assert np.all(np.abs(got[3] - want[3]) <= error[:, None] + 4 * T.UF * far)


def test_rows_with_plus_infinity_have_no_probabilities(rx, client):
    x = np.zeros((3, 5000))
    x[0, 7] = x[1, 0] = np.inf
    got = [t.a for t in gpu_run(rx, client, P.token_logprobs(3, 5000, top=3, dt="f32"), [I.Tensor(x, "f32"), I.Tensor([7, 3, 3], "i32")])[0]]
    for out in got[:4]:
        assert np.isnan(out[:2]).all() and not np.isnan(out[2]).any()
    assert np.array_equal(got[4], [[7, 0, 1], [0, 1, 2], [0, 1, 2]])


@pytest.mark.parametrize("lengths,hq,hk,d,dt", [([64, 7, 2], 8, 2, 64, "bf16"), ([64, 7, 2], 8, 2, 64, "f16"), ([40], 16, 1, 128, "bf16"), ([7, 2], 24, 1, 128, "f16")])
def test_attention_weights_are_not_rounded_to_the_caches_type(rx, client, lengths, hq, hk, d, dt):
    """Values of 1 and -1 under nearly equal weights: results near zero, of which an error of the weights is a large part.  The weights
    enter the product as two 16-bit numbers, off by u of u of themselves; scores and sums are off as in test_gpu_lm_operators.py.  Weights
    rounded once, in the formula, do not meet the bound."""
    rng = np.random.default_rng(d + hq)
    b, size, scale = len(lengths), 16, 0.005
    cols, pages = -(-max(lengths) // size) + 1, sum(-(-n // size) for n in lengths) + 2
    args = T.attention_case(rng, lengths, hq, hk, d, d, pages, size, cols, dt, "slots")
    args[2].a[...] = np.where(np.isnan(args[2].a), np.nan, np.sign(args[2].a))
    got, _ = gpu_run(rx, client, P.paged_attention(b, hq, hk, d, pages, size, cols, dt=dt, scale=scale), args)
    a = [t.a for t in args]
    ref, lse, mag = L.paged_attention(*a, scale=scale)
    q, k = a[0].astype(np.float64), np.abs(np.nan_to_num(a[1].astype(np.float64))).max()
    s = (d + 2) * T.UF * scale * np.abs(q).sum(-1).max() * k
    bound = mag * (T.U[dt] ** 2 + 2 * s + (max(lengths) + 16) * T.UF) + T.U[dt] * np.abs(ref)
    assert np.all(np.abs(got[0].a.astype(np.float64) - ref) <= bound)
    worst = 0.0
    for j, n in enumerate(lengths):                                     # the mistake, in the formula
        rows = [(a[3][j, t // size], t % size) for t in range(n)]
        keys, vals = (np.stack([c[r] for r in rows]).astype(np.float64) for c in a[1:3])
        for h in range(hq):
            x = scale * keys[:, h // (hq // hk)] @ q[j, h]
            p = np.exp(x - x.max())
            wrong = (T.rounded(p, dt).a.astype(np.float64) @ vals[:, h // (hq // hk)]) / p.sum()
            worst = max(worst, (np.abs(wrong - ref[j, h]) / bound[j, h]).max())
    assert worst > 1


@pytest.mark.parametrize("n,v,top", [(40, 500, 3), (6, 30001, 20), (600, 4099, 0)])
def test_logits_of_every_size(rx, client, n, v, top):
    """Rows whose maximum lies anywhere from -3e38 to 3e38, others far below it or equal to it, whole and split among workgroups."""
    rng = np.random.default_rng(n)
    sizes = np.array([-np.inf, -3e38, -1e31, -1e29, -4e10, -1e9 - 64, -1e9, -1e8 - 8, -1e8, -1e8 + 8, -5e7 - 4, -5e7, -5e7 + 4, -50.0, 0.0, 5.0, 1e5, 5e7 - 4, 5e7, 5e7 + 4, 1e8 - 8, 1e8, 1e8 + 8,
                      1e9, 1e9 + 64, 4e10, 1e29, 2e30, 3e38])
    x = np.empty((n, v))
    for t in range(n):
        high = 1 + t % (len(sizes) - 1)
        x[t] = sizes[rng.integers(0, high + 1, size=v)] if t % 3 else sizes[rng.integers(max(0, high - 2), high)]
        x[t, rng.integers(0, v, size=1 + t % 4)] = sizes[high]
    x = I.Tensor(x.astype(np.float32).astype(np.float64), "f32")
    y = rng.integers(0, v, n)
    got = [t.a.astype(np.float64) for t in gpu_run(rx, client, P.token_logprobs(n, v, top=top, dt="f32"), [x, I.Tensor(y, "i32")])[0]]
    want = L.token_logprobs(x.a, y, top)
    # (64 bits are not enough for x - lse here: differences from the maximum, less the log of their sum)
    big = x.a.astype(np.float64)
    far = big - big.max(1, keepdims=True)
    below = np.log(np.exp(far).sum(1))
    logprob = (far - below[:, None])[np.arange(n), y]
    e = (v / 64 + 64 + 44) * T.UF
    assert np.all(np.abs(got[1] - (big.max(1) + below)) <= e + 4 * T.UF * (np.abs(below) + 1) + T.UF * np.abs(want[1]))

    def near(a, b):
        with np.errstate(invalid="ignore", over="ignore"):
            return (a == b) | (np.abs(a - b) <= e + 8 * T.UF * (np.abs(b) + 20)) | (np.isneginf(a) & (b < -3.4e38))
    assert near(got[0], logprob).all()
    p = np.exp(far) / np.exp(far).sum(1, keepdims=True)
    entropy = below - np.where(p > 0, p * np.maximum(far, -1e300), 0.0).sum(1)
    assert np.all(np.abs(got[2] - entropy) <= 2 * e * (1 + np.abs(entropy)) + 8 * T.UF * (np.abs(entropy) + 1))
    if top:
        assert np.array_equal(got[4], want[4]) and near(got[3], np.take_along_axis(far, want[4], 1) - below[:, None]).all()


@pytest.mark.parametrize("pages,cols,seqs,positions,hq", [(0, 4, 2, 64, 8), (10, 0, 2, 64, 8), (10, 4, 0, 64, 8), (10, 4, 2, 0, 8), (10, 4, 2, 64, 0)])
def test_append_where_there_is_nothing(rx, client, pages, cols, seqs, positions, hq):
    """No pages, no page table, no sequences, no angles, no query heads: everything is padding but in the last one."""
    rng = np.random.default_rng(1)
    q, k, v = (T.rounded(rng.normal(size=(3, h, 64)), "f32") for h in (hq, 2, 2))
    angle = rng.uniform(-3, 3, size=(positions, 32))
    table = I.Tensor(rng.permutation(10)[:seqs * cols].reshape(seqs, cols), "i32")
    caches = [T.rounded(rng.normal(size=(pages, 16, 2, 64)), "f32") for _ in range(2)]
    args = [q, k, v, I.Tensor(np.cos(angle), "f32"), I.Tensor(np.sin(angle), "f32"), I.Tensor([0, 5, 17], "i32"), I.Tensor([0, 1, 0], "i32"), table] + caches
    thunk = rx.compile(P.kv_append(3, seqs, hq, 2, 64, pages, 16, cols, positions, dt="f32"))
    want = L.kv_append(*[t.a for t in args])
    for donated in (None, [False] * 8 + [True] * 2):
        out = thunk(*[rx.to_rarray(t.a.T, t.dt) for t in args], donated=donated)
        for got, ref in zip(out, want):
            got = got.to_array().T
            assert got.shape == ref.shape and np.all(np.abs(got - ref) <= 3 * T.UF * 8)
    res = [rx.Buffer.uninitialized(client, t.shape, "f32") for t in (q, *caches)]
    thunk.exec.execute_no_alloc([rx.Buffer.from_host(client, t.a, t.dt) for t in args], res)
    client.default_device().synchronize()
    for got, ref in zip(res, want):
        assert np.all(np.abs(got.to_host() - ref) <= 3 * T.UF * 8)


@pytest.mark.parametrize("pages,cols", [(0, 4), (10, 0), (0, 0)])
def test_attention_where_there_is_nothing(rx, client, pages, cols):
    q = T.rounded(np.random.default_rng(2).normal(size=(3, 8, 64)), "bf16")
    cache = I.Tensor(np.ones((pages, 16, 2, 64)), "bf16")
    got, _ = gpu_run(rx, client, P.paged_attention(3, 8, 2, 64, pages, 16, cols, lse=True), [q, cache, cache, I.Tensor(np.zeros((3, cols)), "i32"), I.Tensor([0, 5, 64], "i32")])
    assert np.all(got[0].a == 0) and np.all(got[1].a == -np.inf)
