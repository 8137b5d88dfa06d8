"""Modules that update a cache and do other things with it, on the GPU against the interpreter's 64-bit evaluation of the same text.
A rotated element is two products and a sum in f32: off by 3 * 2^-24 of the magnitudes, below 8 here; everything else is exact."""
import numpy as np
import pytest

from _loader import load_pkg
from oracle import stablehlo_interp as I
import test_lm_updates as M

load_pkg()
pytestmark = pytest.mark.gpu
BOUND = 3 * 2.0 ** -24 * 8


def values(text, seed=1):
    """Arguments in the order of the module's: every token's slot is its own, whatever the append."""
    rng = np.random.default_rng(seed)
    angle = rng.uniform(-3, 3, size=(M.POSITIONS, M.D // 2))
    out = [I.Tensor(rng.normal(size=s), "f32") for s in ([M.T, M.HQ, M.D], [M.T, M.HK, M.D], [M.T, M.HK, M.D])]
    out += [I.Tensor(np.cos(angle), "f32"), I.Tensor(np.sin(angle), "f32"), I.Tensor([4, 3, -1], "i32"), I.Tensor([0, 1, 1], "i32"),
            I.Tensor(rng.permutation(M.PAGES)[:M.B * M.COLS].reshape(M.B, M.COLS), "i32")]
    if "%arg10" in text:
        out.append(I.Tensor([9, 15, 0], "i32"))                        # the second append's positions
    return out + [I.Tensor(rng.normal(size=M.CACHE), "f32") for _ in range(2)]


def close(got, want):
    assert got.shape == want.shape and np.all(np.abs(got.astype(np.float64) - want) <= BOUND)


def check(rx, client, text):
    """With the caches kept, with them donated, and without allocations: the same results, and arguments that are not donated stay."""
    args = values(text)
    want = [t.a for t in I.run_text(text, args, hifi=True)]
    thunk = rx.compile(text)
    for donated in (False, True, True):
        dev = [rx.to_rarray(a.a.T, a.dt) for a in args]
        out = thunk(*dev, donated=[False] * (len(dev) - 2) + [True] * 2 if donated else None)
        for got, ref in zip(out, want):
            close(got.to_array().T, ref)
        for d, a in zip(dev, args):
            assert d.donated or np.array_equal(d.to_array().T, a.a)
    bufs = [rx.Buffer.from_host(client, a.a, a.dt) for a in args]
    res = [rx.Buffer.uninitialized(client, ref.shape, "f32") for ref in want]
    for _ in range(3):
        thunk.exec.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        for got, ref in zip(res, want):
            close(got.to_host(), ref)
        for b, a in zip(bufs, args):
            assert np.array_equal(b.to_host(), a.a)


@pytest.mark.parametrize("name", sorted(M.TEMPORARIES))
def test_appends_to_temporaries(rx, client, name):
    check(rx, client, M.TEMPORARIES[name])


@pytest.mark.parametrize("reader", ["sqrt", "negate"])
def test_a_reduction_of_the_cache_before_an_append(rx, client, reader):
    text = M.reduce_then_append(reader)
    args = values(text)
    want = [t.a for t in I.run_text(text, args, hifi=True)]
    thunk = rx.compile(text)
    n = args[8].a.size
    for donated in (False, True):
        dev = [rx.to_rarray(a.a.T, a.dt) for a in args]
        out = thunk(*dev, donated=[False] * 8 + [True] * 2 if donated else None)
        for got, ref in zip(out[:3], want):
            close(got.to_array().T, ref)
        # squares and their sum in f32: n + 1 roundings of 2^-24 at most, then the reader's
        assert abs(float(out[3].to_array()) - float(want[3])) <= (n + 3) * 2.0 ** -24 * abs(float(want[3]))
    bufs = [rx.Buffer.from_host(client, a.a, a.dt) for a in args]
    res = [rx.Buffer.uninitialized(client, ref.shape, "f32") for ref in want]
    for _ in range(2):
        thunk.exec.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        close(res[1].to_host(), want[1])
        assert abs(float(res[3].to_host()) - float(want[3])) <= (n + 3) * 2.0 ** -24 * abs(float(want[3]))


def test_a_reduction_of_a_product_before_its_update(rx, client):
    text = M.reduce_then_update()
    rng = np.random.default_rng(2)
    args = [I.Tensor(rng.integers(-3, 4, size=s).astype(np.float64), "f32") for s in ([64, 32], [32, 32])] + [I.Tensor(np.full((8, 32), 1000.0), "f32")]
    m = args[0].a.astype(np.float64) @ args[1].a                       # whole numbers: exact, and so is the sum of their squares
    want = m.copy()
    want[16:24] = 1000.0
    got = [o.to_array().T for o in rx.compile(text)(*[rx.to_rarray(a.a.T, a.dt) for a in args])]
    assert np.array_equal(got[0], want) and abs(float(got[1]) - np.sqrt((m * m).sum())) <= 2.0 ** -22 * np.sqrt((m * m).sum())
