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
