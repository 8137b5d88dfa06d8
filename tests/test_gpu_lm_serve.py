"""Norms, caches of 8 bits and drafted tokens on the GPU against their formulas in 64 bits (oracle/lm_ops.py).

Bounds, with u the unit roundoff of a type and U that of f32 (as in test_gpu_lm_operators.py):
  norm         squares are summed in chains of at most 32 terms and joined in a tree of at most 16 steps: (32 + 16 + 2) U relative, half
               of it in the root; the division, the root and its reciprocal, two products: 5 U; together below 32 U of y, then u of the result
  8 bits       the scale is off by 33 U relative (that of y, and its division); a number is the value over the scale, rounded: half a step, 2^-4 of
               it for f8E4M3FN (2^-10 below its normal numbers) and 1/2 for i8, and 34 U of the value before that
  norm_grad    with u = h r, g = dy weight: r and u off by 32 U, mean(g u) by 32 + 50 + 4 U of mean |g u|; dx by 64 U |r g| + 160 U |r u| mean |g u|
               + 2 U |dh|; dweight sums n rows' terms, each off by 34 U: (n + 36) U of the sum of magnitudes
  write        in f32: the same operations give the same bits, in numpy as on the GPU
  attention    scores: sums of D products, a scale of the key and one of the softmax, queries split to 2^-24: s = (D + 5) U scale |q| |k|; weights by 2 s
               relative, a product with the value's scale (U), and by w where they are split into bf16 or f16 numbers: two leave 2^-16 (f16: 2^-22),
               three 2^-24; sums over n positions: (n + 16) U; then u of the result
"""
import importlib

import numpy as np
import pytest

from _loader import load_pkg
from _harness import gpu_run
from oracle import lm_ops as L
from oracle import lowfloat as LF
from oracle import stablehlo_interp as I
import test_gpu_lm_operators as T

load_pkg()
P = importlib.import_module("reactant_jl_amd.lm_programs")
pytestmark = pytest.mark.gpu
UF = T.UF
EIGHT = ("f8E4M3FN", "i8")


def same_bits(a, b):
    a, b = np.asarray(a), np.asarray(b)
    return a.shape == b.shape and bool(np.all((a == b) | ((a != a) & (b != b))))


def close_to_numbers(codes, scale, y, dt, slack):
    """Numbers of 8 bits against the values y that they stand for."""
    with np.errstate(invalid="ignore"):
        off = np.abs(codes.astype(np.float64) * scale[..., None] - y)
        half = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * scale[..., None]) if dt == "f8E4M3FN" else 0.5 * scale[..., None]
        ok = (off <= half + slack) | (np.isnan(scale)[..., None] & (codes == 0))
    assert ok.all(), "%d of %d beyond the bound, first at %s" % ((~ok).sum(), ok.size, np.argwhere(~ok)[0])


# ----------------------------------------------------------------------------
# norms
# ----------------------------------------------------------------------------
NORMS = [
    (1, 1, "f32", None, True), (3, 64, "bf16", "f8E4M3FN", True), (5, 1001, "f32", "i8", True), (7, 100, "f16", None, False), (2, 8192, "bf16", "f8E4M3FN", True), (300, 260, "f32", "f8E4M3FN", False),
    (3, 8193, "bf16", "i8", True), (2, 32768, "f16", "f8E4M3FN", True), (1, 32767, "f32", None, True), (9, 1024, "bf16", None, True), (4, 1025, "f16", "i8", False), (1030, 512, "bf16", "f8E4M3FN", True),
    (6, 7, "bf16", "i8", True), (48, 4096, "bf16", "f8E4M3FN", True), (2, 20000, "f32", "f8E4M3FN", True),
]


@pytest.mark.parametrize("rows,width,dt,out,residual", NORMS)
def test_norm(rx, client, rows, width, dt, out, residual):
    rng = np.random.default_rng(rows + width)
    x, res, w = (T.rounded(a, dt) for a in (rng.normal(size=(rows, width)), rng.normal(size=(rows, width)) * 3, 1 + 0.2 * rng.normal(size=width)))
    if rows > 4:
        x.a[1], res.a[1] = 0, 0                                  # a row of zeros
        x.a[2] = 0 if residual else 1e-3
        res.a[2], res.a[2, 0] = 0, 0.25                          # one element
        x.a[3], res.a[3] = 1e-4, -1e-4                           # below eps
    got, exe = gpu_run(rx, client, P.rms_norm(rows, width, dt=dt, out=out, residual=residual), [x, res, w] if residual else [x, w])
    got = [g.a for g in got]
    ref = L.rms_norm(x.a, res.a if residual else None, w.a, out=out)
    y = L.rms_norm(x.a, None if not residual else res.a, w.a)[-1]
    if residual:
        assert np.array_equal(got[0], T.rounded(x.a.astype(np.float32) + res.a.astype(np.float32), dt).a)
        got, ref = got[1:], ref[1:]
    if out is None:
        T.close(got[0], y, 33 * UF * np.abs(y), dt)
        return
    # (a row's largest number may be another of two that differ by a rounding: the scale by theirs)
    T.close(got[1], ref[1], 33 * UF * np.abs(ref[1]))
    close_to_numbers(got[0], got[1].astype(np.float64), y, out, 34 * UF * np.abs(y).max(-1, keepdims=True))
    with np.errstate(invalid="ignore"):
        assert np.all(np.abs(got[0].astype(np.float64)).max(-1) == (L.LARGEST[out] if rows <= 4 else np.where(np.abs(y).max(-1) > 0, L.LARGEST[out], 0)))


def test_norm_of_special_values(rx, client):
    """Infinities and NaN stay in their rows; tiny numbers and a weight of zero."""
    x = np.ones((6, 200))
    x[0, 3], x[1, 5], x[2, 7], x[3] = np.nan, np.inf, -np.inf, 1e-38
    w = np.ones(200)
    for dt in ("f32", "bf16"):
        a, b = T.rounded(x, dt), T.rounded(w, dt)
        y, scale = (g.a for g in gpu_run(rx, client, P.rms_norm(6, 200, dt=dt, out="f8E4M3FN", residual=False), [a, b])[0])
        assert np.isnan(scale[:3]).all() and np.all(y[:3] == 0)
        assert np.all(y[4:] == 448) and np.allclose(scale[4:], 1 / 448, rtol=1e-6)
        # a row of 1e-35 has the scale of 2^-100: 0.00566 steps of 2^-9 are 2.9 of them
        assert scale[3] == np.float32(2.0 ** -100) / np.float32(448) and np.all(y[3] == 3 * 2.0 ** -9)
        y, = (g.a for g in gpu_run(rx, client, P.rms_norm(6, 200, dt=dt, residual=False), [a, b])[0])
        assert np.isnan(y[0]).all() and np.all(np.isnan(y[1]) | (y[1] == 0)) and np.allclose(y[4:], 1, rtol=2 ** -7)
    w[:] = 0
    y, scale = (g.a for g in gpu_run(rx, client, P.rms_norm(6, 200, dt="f32", out="i8", residual=False), [T.rounded(x, "f32"), T.rounded(w, "f32")])[0])
    assert np.all(y == 0) and np.all(scale[3:] == np.float32(2.0 ** -100) / np.float32(127))


@pytest.mark.parametrize("width", [8193, 20000, 32768])
def test_norm_of_wide_rows_in_f32(rx, client, width):
    """A lane's 32 squares, 6 steps of a wavefront and 4 that join sixteen of them: (32 + 10 + 2) U of the mean, half of it in the root, and 5 U
    of the division, the root, its reciprocal and two products.  Magnitudes over many powers of two, and equal ones, whose roundings agree."""
    rng = np.random.default_rng(width)
    x = np.exp(rng.uniform(-8, 8, size=(4, width)))
    x[1], x[2] = 1 / 3, np.sort(x[2])
    x, w = T.rounded(x, "f32"), T.rounded(1 + 0.2 * rng.normal(size=width), "f32")
    got, _ = gpu_run(rx, client, P.rms_norm(4, width, dt="f32", residual=False), [x, w])
    y = L.rms_norm(x.a, None, w.a)[0]
    assert np.all(np.abs(got[0].a - y) <= 27 * UF * np.abs(y))


GRADS = [(1, 1, "f32", "f32", True), (513, 1001, "f32", "f32", False), (40, 64, "bf16", "bf16", True), (7, 8192, "f16", "f32", True), (3, 8193, "f32", "f32", True), (2, 32768, "bf16", "f32", False),
         (0, 100, "f32", "f32", True), (5000, 96, "bf16", "f32", True), (1300, 1040, "f16", "f16", True), (5, 20011, "f32", "f32", True)]


@pytest.mark.parametrize("rows,width,dt,out,residual", GRADS)
def test_norm_grad(rx, client, rows, width, dt, out, residual):
    rng = np.random.default_rng(rows + width)
    h, dy, dh, w = (T.rounded(a, dt) for a in (rng.normal(size=(rows, width)) * 2, rng.normal(size=(rows, width)), rng.normal(size=(rows, width)), 1 + 0.2 * rng.normal(size=width)))
    text, args = P.rms_norm_grad(rows, width, dt=dt, out=out, residual=residual), [h, w, dy] + ([dh] if residual else [])
    got, exe = gpu_run(rx, client, text, args)
    again, _ = gpu_run(rx, client, text, args, exe)
    assert all(np.array_equal(a.a, b.a) for a, b in zip(got, again))            # the same bits every run
    dx, dw = L.rms_norm_grad(h.a, w.a, dy.a, dh.a if residual else None)
    a, b = np.abs(h.a.astype(np.float64)), np.abs(dy.a.astype(np.float64))
    r = 1 / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-6) if rows else np.zeros((0, 1))
    g, u = b * np.abs(w.a), a * r
    bound = 64 * UF * r * g + 160 * UF * r * u * ((g * u).mean(-1, keepdims=True) if rows else 0) + 2 * UF * (np.abs(dh.a) if residual else 0)
    T.close(got[0].a, dx, bound, dt)
    T.close(got[1].a, dw, (rows + 36) * UF * (b * u).sum(0), out)


# ----------------------------------------------------------------------------
# caches
# ----------------------------------------------------------------------------
def stored(rng, dt, pages, size, heads, dim, layout):
    """(numbers, scales or None)"""
    shape = P.cache_shape(pages, size, heads, dim, layout)
    if dt not in EIGHT:
        return T.rounded(rng.normal(size=shape), dt), None
    x = rng.integers(-127, 128, size=shape) if dt == "i8" else LF.round_e4m3fn(rng.normal(size=shape).astype(np.float32) * 60)
    return I.Tensor(x, dt), I.Tensor(rng.uniform(0.5, 2, size=(pages, heads, size)) / 60, "f32")


def write_case(rng, tokens, seqs, hq, hk, d, dv, pages, size, cols, positions, r, axes, dt, cache, layout, idt):
    args = T.append_case(rng, tokens, seqs, hq, hk, d, dv, pages, size, cols, cols * size, r, dt, layout, idt)
    angle = rng.uniform(-3, 3, size=(positions, r // 2))
    (kc, ks), (vc, vs) = (stored(rng, cache, pages, size, hk, n, layout) for n in (d, dv))
    args[3], args[4] = I.Tensor(np.cos(angle), "f32"), I.Tensor(np.sin(angle), "f32")
    args = args[:5] + [I.Tensor(rng.integers(0, positions, size=(axes, tokens)), idt)] + args[5:8] + [kc, vc]
    return args + ([ks, vs] if ks is not None else [])


def turned(x, cos, sin, angle, axis, rotation):
    """In f32, operation by operation."""
    x, half = np.asarray(x, dtype=np.float32), cos.shape[1]
    if rotation == "none" or not half:
        return x
    rows = np.asarray(angle)[axis].T                             # [token, pair]
    c, s = (np.asarray(m, dtype=np.float32)[rows, np.arange(half)][:, None, :] for m in (cos, sin))
    first = np.arange(half) * 2 if rotation == "pairs" else np.arange(half)
    second = first + (1 if rotation == "pairs" else half)
    y = x.copy()
    y[..., first], y[..., second] = x[..., first] * c - x[..., second] * s, x[..., second] * c + x[..., first] * s
    return y


def numbers(y, dt):
    """(numbers, scales) in f32, operation by operation."""
    y = np.asarray(y, dtype=np.float32)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(y).all(-1)
        scale = np.where(bad, np.float32(np.nan), np.maximum(np.abs(y).max(-1), np.float32(2.0 ** -100)) / np.float32(L.LARGEST[dt])).astype(np.float32)
        z = np.where(bad[..., None], np.float32(0), y / scale[..., None]).astype(np.float32)
    return (np.rint(z) if dt == "i8" else LF.round_e4m3fn(np.clip(z, -448, 448))), scale


WRITES = [
    (1, 1, 1, 1, 2, 2, 1, 1, 1, 1, 2, [1], "f32", "i8", "halves", "slots", "i32"), (3, 2, 8, 2, 64, 64, 20, 16, 4, 64, 64, [32], "bf16", "f8E4M3FN", "halves", "slots", "i32"),
    (50, 5, 6, 3, 80, 48, 40, 24, 4, 60, 40, [4, 16], "f16", "f16", "pairs", "heads", "i64"), (29, 3, 4, 4, 33, 17, 9, 5, 3, 15, 32, [0, 9, 7], "f32", "f8E4M3FN", "halves", "heads", "i32"),
    (200, 4, 16, 8, 128, 128, 40, 16, 5, 80, 128, [16, 24, 24], "bf16", "i8", "pairs", "slots", "i32"), (20, 2, 2, 1, 256, 256, 60, 1, 30, 30, 128, [64], "f16", "f8E4M3FN", "halves", "heads", "i32"),
    (7, 2, 3, 1, 96, 96, 12, 7, 6, 42, 96, [20, 10, 10, 8], "f32", "f32", "pairs", "slots", "i64"), (2100, 3, 5, 3, 64, 64, 140, 16, 45, 100, 64, [8, 12, 12], "bf16", "f8E4M3FN", "halves", "slots", "i32"),
    (2060, 2, 4, 2, 72, 40, 270, 16, 130, 300, 48, [24], "bf16", "bf16", "halves", "heads", "i32"), (40, 3, 4, 2, 256, 32, 30, 16, 10, 50, 256, [128], "f32", "i8", "pairs", "heads", "i32"),
    (2050, 2, 3, 1, 100, 100, 140, 16, 70, 90, 34, [17], "f16", "i8", "halves", "slots", "i64"), (30, 2, 2, 2, 64, 64, 20, 16, 8, 9, 0, None, "bf16", "f8E4M3FN", "halves", "slots", "i32"),
]


def check_write(got, args, axis, dt, cache, rotation, layout):
    """Against the same operations in f32, and the caches' other places as they were."""
    a = [t.a for t in args]
    q, k, v, cos, sin, angle, position, sequence, pages = a[:9]
    size = a[9].shape[1 if layout == "slots" else 2]
    known = (position >= 0) & (position < pages.shape[1] * size) & (sequence >= 0) & (sequence < pages.shape[0])
    if rotation != "none" and cos.shape[1]:
        known &= ((angle >= 0) & (angle < cos.shape[0])).all(0)
    rows = np.clip(angle, 0, max(0, cos.shape[0] - 1))
    want_q = np.where(known[:, None, None], turned(q, cos, sin, rows, axis, rotation), np.float32(0))
    assert same_bits(got[0], T.rounded(want_q, dt).a)
    page = np.where(known, pages[np.where(known, sequence, 0), np.where(known, position, 0) // size], -1)
    keep = (page >= 0) & (page < a[9].shape[0])
    at, slot = page[keep], (position % size)[keep]
    want = [np.array(t, copy=True) for t in a[9:]]
    for n, new in enumerate((turned(k, cos, sin, rows, axis, rotation), np.asarray(v, dtype=np.float32))):
        if cache in EIGHT:
            new, scale = numbers(new, cache)
            want[2 + n][at, :, slot] = scale[keep]
        else:
            new = T.rounded(new, dt).a
        if layout == "slots":
            want[n][at, slot] = new[keep]
        else:
            want[n][at, :, slot] = new[keep]
    for g, w in zip(got[1:], want):
        assert same_bits(g, w)


@pytest.mark.parametrize("tokens,seqs,hq,hk,d,dv,pages,size,cols,positions,r,sections,dt,cache,rotation,layout,idt", WRITES)
def test_write(rx, client, tokens, seqs, hq, hk, d, dv, pages, size, cols, positions, r, sections, dt, cache, rotation, layout, idt):
    rng = np.random.default_rng(tokens + d)
    axes = len(sections) if sections else 1
    args = write_case(rng, tokens, seqs, hq, hk, d, dv, pages, size, cols, positions, r, axes, dt, cache, layout, idt)
    if tokens >= 20:                                # padding, positions, sequences and rows that do not exist, pages outside the cache, special values
        angle, position, sequence, table = (args[k].a for k in (5, 6, 7, 8))
        position[2], position[5], sequence[7], sequence[11], angle[-1, 13], angle[0, 15] = -1, cols * size, seqs, -1, positions, -1
        table[0, 0], table[-1, -1] = pages, -1
        args[1].a[3, 0, 0], args[2].a[4, -1, -1], args[1].a[6], args[2].a[8] = np.inf, np.nan, 0, 0
    text = P.kv_write(tokens, seqs, hq, hk, d, pages, size, cols, positions, dt=dt, cache=cache, sections=sections, rotary_dim=r, rotation=rotation, layout=layout, ids=idt, value_dim=dv)
    got, _ = gpu_run(rx, client, text, args)
    check_write([g.a for g in got], args, np.repeat(np.arange(axes), sections if sections else [r // 2]), dt, cache, rotation, layout)


def test_write_without_rotation(rx, client):
    rng = np.random.default_rng(3)
    args = write_case(rng, 9, 2, 4, 2, 24, 24, 8, 4, 3, 12, 24, 1, "bf16", "f8E4M3FN", "slots", "i32")
    args[5].a[:] = -7                                # rows of angles that nothing reads
    got, _ = gpu_run(rx, client, P.kv_write(9, 2, 4, 2, 24, 8, 4, 3, 12, cache="f8E4M3FN", rotation="none"), args)
    check_write([g.a for g in got], args, np.zeros(12, int), "bf16", "f8E4M3FN", "none", "slots")


def test_numbers_stand_for_their_values(rx, client):
    """Written numbers times their scales against keys and values in 64 bits: half a step of the type, and what f32 leaves of the rotation."""
    rng = np.random.default_rng(4)
    for cache in EIGHT:
        args = write_case(rng, 40, 1, 4, 2, 64, 64, 3, 16, 3, 60, 64, 2, "f32", cache, "slots", "i32")
        got, _ = gpu_run(rx, client, P.kv_write(40, 1, 4, 2, 64, 3, 16, 3, 60, dt="f32", cache=cache, sections=[20, 12]), args)
        raw = L.kv_write(*[t.a for t in args[:9]], np.zeros((3, 16, 2, 64)), np.zeros((3, 16, 2, 64)), sections="20,12")
        for n in (1, 2):
            y, scale = raw[n], got[n + 2].a.astype(np.float64).transpose(0, 2, 1)
            at = np.abs(y).sum(-1) > 0
            close_to_numbers(got[n].a[at], scale[at], y[at], cache, 4 * UF * 2 * np.abs(y[at]).max(-1, keepdims=True))


MOVES = [(1, 1, 1, 1, 1, 1, 1, 1, "f32", "slots", "i32"), (6, 5, 2, 64, 64, 16, 4, 40, "f8E4M3FN", "slots", "i32"), (5, 16, 3, 80, 48, 24, 3, 40, "f16", "heads", "i64"), (4, 17, 2, 33, 17, 5, 9, 30, "i8", "heads", "i32"),
         (3, 40, 1, 128, 128, 16, 8, 100, "bf16", "slots", "i32"), (70, 7, 8, 128, 128, 16, 3, 20, "f8E4M3FN", "heads", "i32"), (2, 64, 2, 256, 100, 1, 200, 100, "f32", "slots", "i64"), (9, 33, 1, 20, 20, 7, 12, 50, "i8", "slots", "i32")]


@pytest.mark.parametrize("seqs,steps,hk,d,dv,size,cols,longest,cache,layout,idt", MOVES)
def test_move(rx, client, seqs, steps, hk, d, dv, size, cols, longest, cache, layout, idt):
    rng = np.random.default_rng(seqs + steps)
    pages = seqs * cols + 2
    table = rng.permutation(pages)[:seqs * cols].reshape(seqs, cols)
    lengths = rng.integers(0, min(longest, max(1, cols * size - steps)), size=seqs)
    path = rng.integers(-1, steps + 3, size=(seqs, steps))            # forwards and backwards, the same source twice, slots that are moved from and to
    if seqs > 3:
        lengths[0], lengths[1], table[2, 1] = -1, cols * size - 2, pages + 1
        path[3] = rng.permutation(steps)                              # exchanged among themselves
        path[1, -1] = 2 ** 31 - 1
    (kc, ks), (vc, vs) = (stored(rng, cache, pages, size, hk, n, layout) for n in (d, dv))
    args = [I.Tensor(lengths, idt), I.Tensor(path, idt), I.Tensor(table, idt), kc, vc] + ([ks, vs] if ks is not None else [])
    got, _ = gpu_run(rx, client, P.kv_move(seqs, steps, hk, d, pages, size, cols, cache=cache, layout=layout, ids=idt, value_dim=dv), args)
    for g, want in zip(got, L.kv_move(*[t.a for t in args], layout=layout)):
        assert np.array_equal(g.a, want)


def test_donated_and_not(rx, client):
    """Donated caches and scales are updated where they are; otherwise the arguments keep their contents; the same without allocations."""
    rng = np.random.default_rng(5)
    args = write_case(rng, 9, 2, 4, 2, 24, 24, 8, 4, 3, 12, 24, 1, "f32", "i8", "slots", "i32")
    axis = np.zeros(12, int)
    thunk = rx.compile(P.kv_write(9, 2, 4, 2, 24, 8, 4, 3, 12, dt="f32", cache="i8"))
    dev = [rx.to_rarray(t.a.T, t.dt) for t in args]
    kept = thunk(*dev)
    assert all(np.array_equal(x.to_array().T, t.a) for x, t in zip(dev, args))
    check_write([o.to_array().T for o in kept], args, axis, "f32", "i8", "halves", "slots")
    bufs = [rx.Buffer.from_host(client, np.ascontiguousarray(t.a), t.dt) for t in args]
    res = [rx.Buffer.uninitialized(client, t.shape, t.dt) for t in [args[0]] + args[9:]]
    for _ in range(3):
        thunk.exec.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        check_write([r.to_host() for r in res], args, axis, "f32", "i8", "halves", "slots")
        assert all(np.array_equal(b.to_host(), t.a) for b, t in zip(bufs[9:], args[9:]))
    at = [d.data.buffer.unsafe_pointer() for d in dev[9:]]
    out = thunk(*dev, donated=[False] * 9 + [True] * 4)
    assert [o.data.buffer.unsafe_pointer() for o in out[1:]] == at and dev[9].donated
    for a, b in zip(kept, out):
        assert np.array_equal(a.to_array(), b.to_array())


# ----------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------
def tree(rng, b, n):
    """Masks of random trees; some tokens see nothing of the tree, not even themselves."""
    mask = np.zeros((b, n, n), dtype=bool)
    for s in range(b):
        for i in range(n):
            parent = int(rng.integers(-1, i)) if i else -1
            if parent >= 0:
                mask[s, i] = mask[s, parent]
            mask[s, i, i] = True
        mask[s, rng.integers(0, n)] &= rng.random() < 0.5
    return mask


def attention_case(rng, lengths, n, hq, hk, d, dv, size, cols, dt, cache, layout, idt="i32"):
    b = len(lengths)
    pages = sum(min(-(-(max(m, -n) + n) // size), cols) for m in lengths) + 2
    q = T.rounded(rng.normal(size=(b, n, hq, d)), dt)
    (kc, ks), (vc, vs) = (stored(rng, cache, pages, size, hk, m, layout) for m in (d, dv))
    table = np.full((b, cols), -5, dtype=np.int64)
    used = np.zeros((pages, size), dtype=bool)
    order, at = rng.permutation(pages), 0
    for s, m in enumerate(lengths):
        total = min(m + n, cols * size) if m >= 0 else 0
        need = -(-total // size)
        table[s, :need] = order[at:at + need]
        for j in range(total):
            used[table[s, j // size], j % size] = True
        at += need
        if need < cols:
            table[s, need:] = rng.choice([-1, pages, pages + 7, 0], size=cols - need)      # not looked at
    # what no sequence holds is not a number
    for c in (kc, vc):
        if cache != "i8":
            rows = c.a if layout == "slots" else c.a.transpose(0, 2, 1, 3)
            rows[~used] = np.nan
    for c in (ks, vs):
        if c is not None:
            c.a.transpose(0, 2, 1)[~used] = np.nan
    return [q, kc, vc, I.Tensor(table, idt), I.Tensor(np.array(lengths), idt)], ([ks, vs] if ks is not None else [])


def attention_bound(args, scales, scale, mag, dt, cache, n):
    q, k = args[0].a.astype(np.float64), np.abs(np.nan_to_num(args[1].a.astype(np.float64))).max()
    if scales:
        k *= np.nan_to_num(scales[0].a).max()
    s = (q.shape[3] + 5) * UF * scale * np.abs(q).sum(-1).max() * k
    split = 0 if dt == "f32" and not scales else 2.0 ** -24 if dt == "f32" else 2.0 ** -22 if dt == "f16" and not scales else 2.0 ** -16
    return mag * (2 * split + 2 * s + (n + 17) * UF), s + (n + 16) * UF * 2


def check_tree(rx, client, args, scales, mask, n, hq, hk, d, dv, size, cols, dt, cache, layout, window, idt="i32", scale=None):
    b, pages = args[0].shape[0], args[1].shape[0]
    how = False if mask is None else True if mask.ndim == 3 else "shared"
    text = P.tree_attention(b, n, hq, hk, d, pages, size, cols, dt=dt, cache=cache, mask=how, window=window, layout=layout, ids=idt, value_dim=dv, lse=True, scale=scale)
    full = args + ([I.Tensor(mask, "i1")] if mask is not None else []) + scales
    got, exe = gpu_run(rx, client, text, full)
    out, lse, mag = L.tree_attention(*[t.a for t in args], mask, *([t.a for t in scales] or [None, None]), window=window, layout=layout, scale=scale)
    bound, lse_bound = attention_bound(args, scales, d ** -0.5 if scale is None else abs(scale), mag, dt, cache, cols * size)
    T.close(got[0].a, out, bound, dt)
    T.close(got[1].a, lse, lse_bound)
    empty = lse == -np.inf
    assert np.all(got[0].a[empty] == 0) and np.all(got[1].a[empty] == -np.inf)
    return got, exe, full


TREES = [
    # few rows: the wavefronts share the positions
    ([0], 1, 1, 1, 1, 1, 1, 1, "f32", "f32", "slots", 0, "i32", "none"), ([0, 1, 2, 15, 16, 17, -1], 3, 4, 2, 64, 64, 16, 3, "bf16", "bf16", "slots", 0, "i32", "tree"),
    ([33, 0, 64, 31], 4, 4, 4, 128, 128, 32, 3, "f16", "f16", "heads", 0, "i64", "shared"), ([100, 7], 1, 12, 12, 80, 80, 24, 5, "f32", "f32", "slots", 0, "i32", "none"),
    ([513, 300, 77, -1], 2, 16, 1, 128, 128, 16, 40, "bf16", "f8E4M3FN", "heads", 0, "i32", "tree"), ([90, 200], 5, 6, 2, 33, 17, 5, 45, "f16", "f16", "slots", 0, "i32", "tree"),
    ([70, 3, 129], 1, 8, 2, 96, 64, 1, 130, "bf16", "i8", "slots", 0, "i32", "none"), ([257], 7, 4, 1, 256, 256, 64, 5, "bf16", "f8E4M3FN", "heads", 0, "i32", "tree"),
    ([200, 64, 3], 4, 8, 2, 64, 128, 16, 13, "f32", "i8", "heads", 50, "i32", "tree"), ([1000, 2000, 1], 1, 8, 8, 64, 64, 128, 16, "bf16", "f8E4M3FN", "slots", 65, "i64", "none"),
    ([5000], 1, 32, 8, 128, 128, 16, 313, "bf16", "f8E4M3FN", "slots", 0, "i32", "none"), ([300, 299], 8, 4, 1, 100, 36, 12, 30, "f32", "f8E4M3FN", "slots", 0, "i32", "shared"),
    ([40] * 70, 2, 4, 2, 16, 8, 8, 6, "bf16", "bf16", "slots", 2, "i32", "none"), ([77, 500], 1, 20, 1, 72, 72, 16, 40, "f16", "i8", "heads", 0, "i32", "none"),
    ([6000, 3], 6, 4, 1, 64, 64, 16, 377, "f16", "f8E4M3FN", "slots", 0, "i32", "tree"),
    # many rows: they share keys and values
    ([100, 0, 31, -1], 16, 8, 2, 64, 64, 16, 10, "bf16", "bf16", "slots", 0, "i32", "tree"), ([300, 5], 33, 4, 4, 128, 128, 24, 20, "f16", "f16", "heads", 0, "i32", "tree"),
    ([1000, 500, 64], 64, 16, 2, 128, 128, 16, 80, "bf16", "f8E4M3FN", "slots", 0, "i32", "tree"), ([200, 90], 40, 2, 1, 33, 17, 5, 60, "f16", "f16", "slots", 0, "i64", "tree"),
    ([64, 260], 64, 4, 2, 80, 80, 16, 30, "f32", "f32", "slots", 0, "i32", "shared"), ([129], 50, 4, 4, 256, 256, 16, 20, "bf16", "bf16", "heads", 100, "i32", "tree"),
    ([200], 35, 2, 2, 256, 200, 16, 20, "f32", "f32", "slots", 0, "i32", "tree"), ([400, 0], 70, 8, 1, 96, 64, 1, 500, "f16", "i8", "slots", 0, "i32", "none"),
    ([3000], 34, 8, 4, 64, 64, 16, 200, "bf16", "i8", "heads", 64, "i32", "tree"), ([100, 41, 900], 16, 12, 4, 128, 40, 48, 30, "f32", "f8E4M3FN", "heads", 0, "i32", "tree"),
    ([20] * 40, 37, 1, 1, 20, 20, 8, 8, "f32", "i8", "slots", 0, "i32", "none"), ([500, 100], 200, 2, 1, 64, 64, 32, 24, "bf16", "bf16", "slots", 0, "i32", "none"), ([64], 300, 1, 1, 100, 100, 12, 40, "f16", "f8E4M3FN", "heads", 301, "i32", "shared"),
    ([12000, 4], 40, 2, 2, 64, 64, 16, 760, "bf16", "f8E4M3FN", "heads", 0, "i32", "tree"),
    # the largest stages in LDS, and rows of no whole 16 bytes
    ([90, 3], 40, 2, 1, 256, 256, 16, 10, "f32", "f32", "heads", 0, "i32", "tree"), ([77], 70, 2, 1, 255, 250, 16, 10, "f32", "f32", "slots", 0, "i32", "none"),
    ([60, 200], 36, 2, 2, 256, 256, 8, 30, "f16", "f16", "slots", 0, "i32", "tree"), ([50], 33, 3, 1, 250, 255, 16, 6, "f32", "i8", "heads", 40, "i32", "none"),
]


@pytest.mark.parametrize("lengths,n,hq,hk,d,dv,size,cols,dt,cache,layout,window,idt,how", TREES)
def test_tree_attention(rx, client, lengths, n, hq, hk, d, dv, size, cols, dt, cache, layout, window, idt, how):
    rng = np.random.default_rng(abs(sum(lengths)) + n + hq)
    args, scales = attention_case(rng, lengths, n, hq, hk, d, dv, size, cols, dt, cache, layout, idt)
    mask = None if how == "none" else tree(rng, len(lengths), n) if how == "tree" else tree(rng, 1, n)[0]
    got, exe, full = check_tree(rx, client, args, scales, mask, n, hq, hk, d, dv, size, cols, dt, cache, layout, window, idt)
    again, _ = gpu_run(rx, client, "", full, exe)
    assert all(np.array_equal(x.a, y.a) for x, y in zip(got, again))            # the same bits every run


@pytest.mark.parametrize("n,d,cache,size", [(20, 64, "bf16", 1), (20, 33, "bf16", 1), (20, 64, "f8E4M3FN", 3), (4, 64, "i8", 1)])
def test_more_positions_than_a_block_of_pages(rx, client, n, d, cache, size):
    """Positions whose page entries are brought to LDS several times."""
    rng = np.random.default_rng(n + d)
    lengths = [2500 * size, 1024 * size, 1010 * size]
    cols = 2500 + n
    args, scales = attention_case(rng, lengths, n, 4, 1, d, d, size, cols, "bf16", cache, "slots")
    args[3].a[0, 1500], args[3].a[2, 100] = -1, args[1].shape[0]
    check_tree(rx, client, args, scales, tree(rng, 3, n), n, 4, 1, d, d, size, cols, "bf16", cache, "slots", 0)


@pytest.mark.parametrize("dt,cache,layout,window", [("bf16", "bf16", "slots", 0), ("f16", "i8", "heads", 0), ("bf16", "f8E4M3FN", "slots", 1030)])
def test_the_most_drafted_tokens(rx, client, dt, cache, layout, window):
    """1024 tokens of a prompt, causal, behind none, a few and many positions; the last sequence's end lies beyond the page table."""
    rng = np.random.default_rng(18)
    n, hq, hk, d, size, cols = 1024, 2, 1, 64, 16, 80
    args, scales = attention_case(rng, [0, 37, 256, 300, -1], n, hq, hk, d, d, size, cols, dt, cache, layout)
    check_tree(rx, client, args, scales, None, n, hq, hk, d, d, size, cols, dt, cache, layout, window)


@pytest.mark.parametrize("n,hq", [(6, 4), (24, 4)])
@pytest.mark.parametrize("dt,cache", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8E4M3FN")])
def test_special_values_that_a_token_does_not_see(rx, client, n, hq, dt, cache):
    """Infinities and NaN in the keys and values of drafted tokens: those that see them have them, the others are as without them."""
    rng = np.random.default_rng(7)
    args, scales = attention_case(rng, [70, 0, 33], n, hq, 2, 64, 64, 16, 8, dt, cache, "slots")
    mask = np.broadcast_to(np.eye(n, dtype=bool), (3, n, n)).copy()
    mask[1, 2] = False                                                          # nothing left: zeros
    clean = check_tree(rx, client, args, scales, mask, n, hq, 2, 64, 64, 16, 8, dt, cache, "slots", 0)[0]
    table, lengths = args[3].a, args[4].a

    def at(s, j):
        p = int(lengths[s]) + j
        return int(table[s, p // 16]), p % 16
    for s in range(3):
        args[1].a[at(s, 1)] = np.nan
        args[2].a[at(s, 3)] = np.nan
        args[2].a[at(s, 4)][0, 5] = np.nan if cache in EIGHT else np.inf
        if scales:
            scales[1].a[at(s, 5)[0], :, at(s, 5)[1]] = np.inf
    b, pages = 3, args[1].shape[0]
    text = P.tree_attention(b, n, hq, 2, 64, pages, 16, 8, dt=dt, cache=cache, mask=True)
    got, _ = gpu_run(rx, client, text, args + [I.Tensor(mask, "i1")] + scales)
    out, ref = got[0].a, clean[0].a
    assert np.isnan(out[:, 1]).all() and np.isnan(out[:, 3]).all()
    assert not np.isfinite(out[:, 4, :hq // 2, 5]).any() and np.array_equal(np.delete(out[:, 4], 5, -1), np.delete(ref[:, 4], 5, -1)) and np.array_equal(out[:, 4, hq // 2:], ref[:, 4, hq // 2:])
    rest = [i for i in range(n) if i not in (1, 3, 4) + ((5,) if scales else ())]
    assert np.array_equal(out[:, rest], ref[:, rest])
    assert not scales or not np.isfinite(out[:, 5]).any()


@pytest.mark.parametrize("n", [3, 20])
@pytest.mark.parametrize("d,dt,scale", [(80, "bf16", None), (72, "f16", 0.2), (40, "bf16", -0.1), (100, "f32", None), (20, "f32", -0.3), (33, "f16", None)])
def test_infinite_keys_have_no_weight(rx, client, n, d, dt, scale):
    """Infinities in a key's last dimensions that make its scores -inf, among the positions before the drafted tokens and among those:
    weights of zero.  Heads whose keys are no whole fragments."""
    rng = np.random.default_rng(d + n)
    hq, hk, size, cols, lengths = 4, 2, 16, 8, [70, 0, 33]
    args, scales = attention_case(rng, lengths, n, hq, hk, d, d, size, cols, dt, dt, "slots")
    last = 4 if dt == "f32" else 8                                          # dimensions of 16 bytes
    args[0].a[..., -last:] = np.abs(args[0].a[..., -last:]) + 0.5           # one sign for every query
    args[0] = T.rounded(args[0].a, dt)
    mask = tree(rng, 3, n)
    finite = [I.Tensor(np.array(a.a), a.dt) for a in args]
    table = args[3].a
    for s, j, dim in ((0, 5, d - 1), (0, 50, d - last), (0, 71, d - 2), (1, 1, d - 1), (2, 20, d - 3), (2, 34, d - 1)):
        args[1].a[table[s, j // size], j % size, :, dim] = np.inf if scale is not None and scale < 0 else -np.inf
    text = P.tree_attention(3, n, hq, hk, d, args[1].shape[0], size, cols, dt=dt, mask=True, lse=True, scale=scale)
    got, _ = gpu_run(rx, client, text, args + [I.Tensor(mask, "i1")])
    with np.errstate(invalid="ignore"):
        out, lse, mag = L.tree_attention(*(t.a for t in args), mask, scale=scale)
    assert np.isfinite(out[0]).all() and np.isfinite(out[2]).all()
    lse[np.isnan(lse)] = -np.inf                                            # a token of the second sequence may see that key alone
    bound, lse_bound = attention_bound(finite, scales, d ** -0.5 if scale is None else abs(scale), mag, dt, dt, cols * size)
    T.close(got[0].a, out, bound, dt)
    T.close(got[1].a, lse, lse_bound)


@pytest.mark.parametrize("n", [2, 20])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dt,cache,power", [("f16", "f16", 18), ("f16", "f16", 20), ("f16", "f16", 21), ("f16", "f16", 24), ("f16", "f16", 25), ("f16", "f16", 26), ("f16", "f16", 27), ("f16", "f16", 100),
                                            ("bf16", "bf16", 21), ("bf16", "bf16", 33), ("bf16", "bf16", 40), ("f32", "f32", 33), ("f32", "f32", 100), ("bf16", "i8", 25), ("f16", "f8E4M3FN", 40)])
def test_large_finite_scores(rx, client, n, sign, dt, cache, power):
    """Scores of about 2^power (their logarithms to base 2): the largest of them has all of the weight, or shares it with its equals.
    One dimension, of whole numbers, so that products are exact; others are further from the largest than f32 rounds it.  The sum of
    exponentials is then their number, and lse is off by five roundings before its own: the factor's, its product's, those of the shift
    of f16 weights and of the sum's logarithm, which are added to it, and that of ln 2."""
    rng = np.random.default_rng(power + n)
    hq, hk, d, size, cols, lengths = 4, 2, 64, 16, 160, [2500, 40, 3]
    args, scales = attention_case(rng, lengths, n, hq, hk, d, d, size, cols, dt, cache, "slots")
    bits = {"f16": 11, "f32": 11, "bf16": 8, "i8": 7, "f8E4M3FN": 4}
    for t, b in ((args[0], bits[dt]), (args[1], bits[cache])):
        t.a[...] = 0
        t.a[..., 9] = rng.integers(2 ** (b - 1), 2 ** b, size=t.a.shape[:-1])
    args[0].a[..., 9] *= rng.choice([-1, 1], size=args[0].shape[:-1])
    for t in scales[:1]:
        t.a[...] = 1
    scale = sign * 1.3 * 2.0 ** (power + 1 - bits[dt] - bits[cache])       # (products with it are rounded)
    mask = tree(rng, 3, n)
    text = P.tree_attention(3, n, hq, hk, d, args[1].shape[0], size, cols, dt=dt, cache=cache, mask=True, lse=True, scale=scale)
    got, exe = gpu_run(rx, client, text, args + [I.Tensor(mask, "i1")] + scales)
    out, lse, mag = L.tree_attention(*(t.a for t in args), mask, *(scales and [t.a for t in scales] or [None, None]), scale=scale)
    split = 0 if dt == "f32" and not scales else 2.0 ** -22 if dt == "f16" and not scales else 2.0 ** -16
    T.close(got[0].a, out, mag * (2 * split + (cols * size + 17) * UF), dt)
    with np.errstate(invalid="ignore"):
        T.close(got[1].a, lse, 5 * UF * np.abs(lse) + (cols * size + 16) * 2 * UF)


@pytest.mark.parametrize("n", [2, 20])
def test_queries_beyond_the_largest_of_bf16(rx, client, n):
    """Queries in f32 up to its largest number over caches of 8 bits: their parts in bf16 are finite, and scores with small scales of keys ordinary."""
    rng = np.random.default_rng(n)
    hq, hk, d, size, cols = 4, 2, 64, 16, 8
    args, scales = attention_case(rng, [70, 3, 0], n, hq, hk, d, d, size, cols, "f32", "f8E4M3FN", "slots")
    args[0].a[...] = 0
    args[0].a[..., 40] = rng.choice([-1, 1], size=args[0].shape[:-1]) * np.where(rng.random(args[0].shape[:-1]) < 0.5, np.float64(np.finfo(np.float32).max), 3.395e38)
    args[0] = T.rounded(args[0].a, "f32")
    args[1].a[...] = LF.round_e4m3fn(rng.uniform(-1, 1, size=args[1].shape).astype(np.float32))    # (no product beyond f32)
    scales[0].a[...] = 2.0 ** -123
    mask = tree(rng, 3, n)
    check_tree(rx, client, args, scales, mask, n, hq, hk, d, d, size, cols, "f32", "f8E4M3FN", "slots", 0, scale=0.5)


def test_scores_far_apart_and_pages_that_do_not_exist(rx, client):
    rng = np.random.default_rng(8)
    for n in (5, 20):
        args, scales = attention_case(rng, [300, 280], n, 8, 2, 64, 64, 16, 25, "f32", "f32", "slots")
        args[0].a *= 1e4
        args[3].a[1, 3], args[3].a[1, 7], args[3].a[0, 18] = -1, args[1].shape[0], -1    # of the prefix, and of drafted tokens
        args[3].a[0, 0] = args[3].a[0, 1]                                                 # two places of a sequence on one page
        mask = tree(rng, 2, n)
        text = P.tree_attention(2, n, 8, 2, 64, args[1].shape[0], 16, 25, dt="f32", lse=True, scale=-0.25)
        got, _ = gpu_run(rx, client, text, args + [I.Tensor(mask, "i1")])
        out, lse, mag = L.tree_attention(*[t.a for t in args], mask, scale=-0.25)
        s = 69 * UF * 0.25 * np.abs(args[0].a).sum(-1).max() * np.abs(np.nan_to_num(args[1].a)).max()
        T.close(got[1].a, lse, s + 400 * UF)
        T.close(got[0].a, out, 2 * s * mag + 420 * UF * mag)


def test_lengths_at_the_page_tables_end(rx, client):
    """Drafted tokens beyond the page table are left out; lengths beyond it are the table's; the sequence of -1 sees nothing."""
    rng = np.random.default_rng(9)
    for n in (4, 40):
        args, scales = attention_case(rng, [62, 64, 30, -1], n, 4, 2, 64, 64, 16, 4, "f32", "f32", "heads")
        check_tree(rx, client, args, scales, tree(rng, 4, n), n, 4, 2, 64, 64, 16, 4, "f32", "f32", "heads", 0)
        args[4] = I.Tensor(np.array([62, 10 ** 6, 30, -2 ** 31]), "i32")
        check_tree(rx, client, args, scales, None, n, 4, 2, 64, 64, 16, 4, "f32", "f32", "heads", 0)


def test_no_pages_sequences_or_heads_of_the_cache(rx, client):
    q = T.rounded(np.ones((2, 3, 4, 8)), "f32")
    for pages, cols in ((0, 0), (0, 5), (3, 0)):
        c = I.Tensor(np.zeros((pages, 4, 2, 8)), "f32")
        got, _ = gpu_run(rx, client, P.tree_attention(2, 3, 4, 2, 8, pages, 4, cols, dt="f32", mask=False, lse=True), [q, c, c, I.Tensor(np.zeros((2, cols)), "i32"), I.Tensor([7, 0], "i32")])
        assert np.all(got[0].a == 0) and np.all(got[1].a == -np.inf)


@pytest.mark.parametrize("n", [2, 33])
def test_many_uneven_sequences(rx, client, n):
    """Stretches that end inside of sequences, hold several, and start others; the same bits in every run, and with small temporaries."""
    rng = np.random.default_rng(n)
    b, hq, hk, d, size = 90, 4, 2, 64, 16
    lengths = np.round(700 ** rng.random(b)).astype(int)
    lengths[rng.integers(0, b, size=9)] = -1
    cols = -(-(lengths.max() + n) // size) + 1
    args, scales = attention_case(rng, lengths.tolist(), n, hq, hk, d, d, size, cols, "bf16", "f8E4M3FN", "slots")
    mask = tree(rng, b, n)
    got, exe, full = check_tree(rx, client, args, scales, mask, n, hq, hk, d, d, size, cols, "bf16", "f8E4M3FN", "slots", 0)
    for _ in range(10):
        again, _ = gpu_run(rx, client, "", full, exe)
        assert np.array_equal(again[0].a, got[0].a) and np.array_equal(again[1].a, got[1].a)
    bufs = [rx.Buffer.from_host(client, np.frombuffer(a.to_bytes(), dtype=rx._STORAGE[a.dt]).reshape(a.shape), a.dt) for a in full]
    res = [rx.Buffer.uninitialized(client, (b, n, hq, d), "bf16"), rx.Buffer.uninitialized(client, (b, n, hq), "f32")]
    out, lse, mag = L.tree_attention(*[t.a for t in args], mask, *[t.a for t in scales])
    bound, lse_bound = attention_bound(args, scales, d ** -0.5, mag, "bf16", "f8E4M3FN", cols * size)
    for _ in range(2):
        exe.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        T.close(rx.decode(res[0].to_host(), "bf16"), out, bound, "bf16")
        T.close(res[1].to_host(), lse, lse_bound)


def test_partial_results_fit_calls_without_allocations(rx, client):
    """Long sequences of many rows, whose parts take more than the library's scratch array in the usual plan."""
    rng = np.random.default_rng(10)
    n, hq, hk, d, size, cols = 64, 16, 2, 128, 16, 260
    args, scales = attention_case(rng, [4000, 100], n, hq, hk, d, d, size, cols, "bf16", "bf16", "slots")
    _, exe, full = check_tree(rx, client, args, scales, None, n, hq, hk, d, d, size, cols, "bf16", "bf16", "slots", 0)
    bufs = [rx.Buffer.from_host(client, np.frombuffer(a.to_bytes(), dtype=rx._STORAGE[a.dt]).reshape(a.shape), a.dt) for a in full]
    res = [rx.Buffer.uninitialized(client, (2, n, hq, d), "bf16"), rx.Buffer.uninitialized(client, (2, n, hq), "f32")]
    out, lse, mag = L.tree_attention(*[t.a for t in args])
    bound, lse_bound = attention_bound(args, scales, d ** -0.5, mag, "bf16", "bf16", cols * size)
    grad = rx.xla_compile(client, P.rms_norm_grad(3000, 4096, dt="bf16"))
    h, dy, w = (T.rounded(rng.normal(size=s), "bf16") for s in ((3000, 4096), (3000, 4096), 4096))
    gbufs = [rx.Buffer.from_host(client, np.frombuffer(a.to_bytes(), dtype=np.uint16).reshape(a.shape), "bf16") for a in (h, w, dy, h)]
    gres = [rx.Buffer.uninitialized(client, (3000, 4096), "bf16"), rx.Buffer.uninitialized(client, (4096,), "f32")]
    _, dw = L.rms_norm_grad(h.a, w.a, dy.a)
    r = 1 / np.sqrt((h.a.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
    for _ in range(2):
        exe.execute_no_alloc(bufs, res)
        grad.execute_no_alloc(gbufs, gres)
        client.default_device().synchronize()
        T.close(rx.decode(res[0].to_host(), "bf16"), out, bound, "bf16")
        T.close(res[1].to_host(), lse, lse_bound)
        T.close(gres[1].to_host(), dw, (3000 + 36) * UF * (np.abs(dy.a.astype(np.float64) * h.a) * r).sum(0))


def test_cache_of_more_than_2_to_the_31_numbers(rx, client):
    """Written to the last pages of caches of 2.4e9 numbers of 8 bits, read back by the attention, and moved."""
    hq, hk, d, size, pages, n = 8, 8, 128, 16, 146000, 40
    rng = np.random.default_rng(2)
    q, k, v = (T.rounded(rng.normal(size=(n, h, d)), "bf16") for h in (hq, hk, hk))
    none, table = I.Tensor(np.zeros((64, 0)), "f32"), I.Tensor([[pages - 1, pages - 2, pages - 70000, 5]], "i32")
    pos, zero = I.Tensor(np.arange(n), "i32"), I.Tensor(np.zeros(n), "i32")
    write = rx.compile(P.kv_write(n, 1, hq, hk, d, pages, size, 4, 64, rotary_dim=0, cache="f8E4M3FN"))
    dev = [rx.to_rarray(t.a.T, t.dt) for t in (q, k, v, none, none, I.Tensor(np.zeros((1, n)), "i32"), pos, zero, table)]

    def array(shape, dt):
        return rx.ConcreteRArray(rx.AsyncBuffer(rx.Buffer.uninitialized(client, shape, dt)), shape[::-1], dt)
    caches = [array((pages, size, hk, d), "f8E4M3FN") for _ in range(2)] + [array((pages, hk, size), "f32") for _ in range(2)]
    out = write(*dev, *caches, donated=[False] * 9 + [True] * 4)
    small = []
    for x in (k.a, v.a):
        codes, scale = numbers(x, "f8E4M3FN")
        c, s = np.zeros((3, size, hk, d)), np.zeros((3, hk, size))
        c.reshape(-1, hk, d)[:n] = codes
        s.transpose(0, 2, 1).reshape(-1, hk)
        for j in range(n):
            s[j // size, :, j % size] = scale[j]
        small.append((c, s))
    at = I.Tensor([n - 8], "i32")
    last = I.Tensor(q.a[None, -8:], "bf16")
    attend = rx.compile(P.tree_attention(1, 8, hq, hk, d, pages, size, 4, cache="f8E4M3FN", mask=False, lse=True))
    got = attend(rx.to_rarray(last.a.T, "bf16"), out[1], out[2], dev[8], rx.to_rarray(at.a.astype(np.int32)), out[3], out[4])
    (kc, ks), (vc, vs) = small
    ref, lse, mag = L.tree_attention(last.a, kc, vc, np.array([[0, 1, 2]]), at.a, None, ks, vs)
    bound, lse_bound = attention_bound([last, I.Tensor(kc, "f32")], [I.Tensor(ks, "f32")], d ** -0.5, mag, "bf16", "f8E4M3FN", n)
    T.close(got[0].to_array().T, ref, bound, "bf16")
    T.close(got[1].to_array().T, lse, lse_bound)
    path = np.array([[5, 0, 7]], dtype=np.int32)
    move = rx.compile(P.kv_move(1, 3, hk, d, pages, size, 4, cache="f8E4M3FN"))
    out2 = move(rx.to_rarray(at.a.astype(np.int32)), rx.to_rarray(path.T), dev[8], *out[1:], donated=[False] * 3 + [True] * 4)
    kc, vc, ks, vs = L.kv_move(at.a, path, np.array([[0, 1, 2]]), kc, vc, ks, vs)
    got = attend(rx.to_rarray(last.a.T, "bf16"), out2[0], out2[1], dev[8], rx.to_rarray(at.a.astype(np.int32)), out2[2], out2[3])
    ref, lse, mag = L.tree_attention(last.a, kc, vc, np.array([[0, 1, 2]]), at.a, None, ks, vs)
    T.close(got[0].to_array().T, ref, bound + attention_bound([last, I.Tensor(kc, "f32")], [I.Tensor(ks, "f32")], d ** -0.5, mag, "bf16", "f8E4M3FN", n)[0], "bf16")


def test_scores_of_a_factor_of_zero(rx, client):
    """All weights alike: the mean of the values that a token sees, masked ones left out."""
    rng = np.random.default_rng(14)
    for n, cache in ((3, "bf16"), (40, "bf16"), (3, "i8"), (40, "f8E4M3FN")):
        args, scales = attention_case(rng, [70, 0], n, 4, 2, 64, 64, 16, 8, "bf16", cache, "slots")
        check_tree(rx, client, args, scales, tree(rng, 2, n), n, 4, 2, 64, 64, 16, 8, "bf16", cache, "slots", 0, scale=0.0)


def test_norms_of_other_ranks(rx, client):
    """Rows in several dimensions, and one row alone."""
    rng = np.random.default_rng(15)
    text = P.rms_norm(6, 40, dt="f32", out="i8")
    x, res, w = (T.rounded(rng.normal(size=s), "f32") for s in ((6, 40), (6, 40), 40))
    flat = [g.a for g in gpu_run(rx, client, text, [x, res, w])[0]]
    deep = text.replace("tensor<6x40x", "tensor<2x3x40x").replace("tensor<6xf32>", "tensor<2x3xf32>")
    got = [g.a for g in gpu_run(rx, client, deep, [I.Tensor(x.a.reshape(2, 3, 40), "f32"), I.Tensor(res.a.reshape(2, 3, 40), "f32"), w])[0]]
    assert [g.shape for g in got] == [(2, 3, 40), (2, 3, 40), (2, 3)] and all(np.array_equal(g.reshape(f.shape), f) for g, f in zip(got, flat))
    one = text.replace("tensor<6x40x", "tensor<40x").replace("tensor<6xf32>", "tensor<f32>")
    got = [g.a for g in gpu_run(rx, client, one, [I.Tensor(x.a[2], "f32"), I.Tensor(res.a[2], "f32"), w])[0]]
    assert got[2].shape == () and np.array_equal(got[1], flat[1][2]) and got[2] == flat[2][2]
    grad = P.rms_norm_grad(6, 40, dt="f32")
    args = [x, w, res, res]
    dx, dw = (g.a for g in gpu_run(rx, client, grad, args)[0])
    deep = [I.Tensor(a.a.reshape(3, 2, 40), "f32") if a.a.ndim == 2 else a for a in args]
    got = [g.a for g in gpu_run(rx, client, grad.replace("tensor<6x40x", "tensor<3x2x40x"), deep)[0]]
    assert np.array_equal(got[0].reshape(6, 40), dx) and np.array_equal(got[1], dw)


def test_one_array_given_twice(rx, client):
    """The same array as both caches, and as both scales: every result is its own."""
    rng = np.random.default_rng(16)
    args = write_case(rng, 9, 2, 4, 2, 24, 24, 8, 4, 3, 12, 24, 1, "f32", "i8", "slots", "i32")
    args[10], args[12] = args[9], args[11]
    thunk = rx.compile(P.kv_write(9, 2, 4, 2, 24, 8, 4, 3, 12, dt="f32", cache="i8"))
    dev = [rx.to_rarray(t.a.T, t.dt) for t in args[:9]]
    cache, scale = rx.to_rarray(args[9].a.T, "i8"), rx.to_rarray(args[11].a.T, "f32")
    out = thunk(*dev, cache, cache, scale, scale, donated=[False] * 9 + [True] * 4)
    check_write([o.to_array().T for o in out], args, np.zeros(12, int), "f32", "i8", "halves", "slots")


def test_moves_without_pages(rx, client):
    for pages, cols in ((0, 3), (2, 0)):
        c = I.Tensor(np.arange(pages * 8.0).reshape(pages, 4, 1, 2), "f32")
        got, _ = gpu_run(rx, client, P.kv_move(2, 3, 1, 2, pages, 4, cols, cache="f32"), [I.Tensor([1, 0], "i32"), I.Tensor([[2, 1, 0]] * 2, "i32"), I.Tensor(np.zeros((2, cols)), "i32"), c, c])
        assert all(np.array_equal(g.a, c.a) for g in got)


# ----------------------------------------------------------------------------
# together
# ----------------------------------------------------------------------------
def verify_values(rng, text, types, eight, b, n, pages, cols, positions, d):
    values = []
    for s, t in types:
        if t == "f8E4M3FN" and len(s) == 2:
            values.append(LF.round_e4m3fn(rng.normal(size=s).astype(np.float32) * 50))          # weights, with a factor
        elif t in EIGHT:
            values.append(np.zeros(s))
        elif t == "f32" and s == []:
            values.append(np.float32(1 / (50 * 8)))
        else:
            values.append(rng.normal(size=s) * (s[1] ** -0.5 if len(s) == 2 else 1.0) if t != "i32" else np.zeros(s))
    angle = np.arange(positions)[:, None] * 10.0 ** -(np.arange(d // 2) / 4)[None, :]
    values[6], values[7] = np.cos(angle), np.sin(angle)
    values[5] = rng.permutation(pages)[:b * cols].reshape(b, cols)
    return [T.rounded(v, t) if t not in ("i32", "i1", "i8") else I.Tensor(v, t) for v, (s, t) in zip(values, types)]


@pytest.mark.parametrize("layout,rotation,axes", [("slots", "halves", 1), ("heads", "pairs", 3)])
def test_verify_steps(rx, client, layout, rotation, axes):
    """Two steps of drafted trees of three sequences, the accepted branch moved together between them, through two layers in f32:
    caches stay on the device, donated from call to call, against the interpreter's.  As for the decoding steps of
    test_gpu_lm_operators.py, whose chain of products this is."""
    b, n, vocab, width, hq, hk, d, hidden, pages, size, cols, positions = 3, 4, 101, 64, 8, 2, 32, 96, 20, 4, 5, 20
    text, types, cache_results = P.verify_step(b, n, vocab, width, hq, hk, d, hidden, pages, size, cols, positions, layers=2, axes=axes, top=3, dt="f32", cache="f32", products="f32",
                                               layout=layout, rotation=rotation)
    move_text = P.kv_move(b, 3, hk, d, pages, size, cols, cache="f32", layout=layout)
    rng = np.random.default_rng(11)
    args = verify_values(rng, text, types, False, b, n, pages, cols, positions, d)
    cache_args = [k for k, (s, t) in enumerate(types) if len(s) == 4]
    thunk, move = rx.compile(text), rx.compile(move_text)
    dev = [rx.to_rarray(a.a.T, a.dt) for a in args]
    lengths = np.array([5, 0, -1])
    for step in range(2):
        mask = tree(rng, b, n)
        depth = mask.sum(-1) - 1
        angle = np.stack([np.clip(lengths[:, None] + depth + a, 0, positions - 1) for a in range(axes)])
        for k, v in enumerate((rng.integers(0, vocab, (b, n)), rng.integers(0, vocab, (b, n)), angle, lengths)):
            args[k] = I.Tensor(v, "i32")
        args[4] = I.Tensor(mask, "i1")
        for k in range(5):
            dev[k] = rx.to_rarray(args[k].a.T, args[k].dt)
        out = thunk(*dev, donated=[k in cache_args for k in range(len(dev))])
        ref = I.run_text(text, args, hifi=True)
        for k, r in zip(cache_args, cache_results):
            dev[k], args[k] = out[r], ref[r]
        live = np.repeat(lengths >= 0, n)
        for r in range(4):
            assert np.allclose(out[r].to_array().T[live], ref[r].a[live], atol=2e-4, rtol=2e-4), (step, r)
        assert np.array_equal(out[4].to_array().T[live], ref[4].a[live])
        for r in cache_results:
            assert np.allclose(out[r].to_array().T, ref[r].a, atol=1e-4, rtol=1e-4)
        path = np.array([[0, 2, 3], [1, 3, -1], [0, 1, 2]])
        for k in range(0, 4, 2):
            pair = cache_args[k:k + 2]
            moved = move(dev[3], rx.to_rarray(path.T.astype(np.int32)), dev[5], *(dev[c] for c in pair), donated=[False] * 3 + [True] * 2)
            want = L.kv_move(lengths, path, args[5].a, *(args[c].a for c in pair), layout=layout)
            for c, m, w in zip(pair, moved, want):
                dev[c], args[c] = m, I.Tensor(w, "f32")
                assert np.allclose(m.to_array().T, w, atol=1e-4, rtol=1e-4)
        lengths = np.array([8, 2, -1])


def test_a_step_in_8_bits(rx, client):
    """Norm, product, write, attention and move in 8 bits, each on the device's own results of the one before."""
    rng = np.random.default_rng(12)
    b, n, width, hq, hk, d, pages, size, cols = 3, 6, 256, 8, 2, 64, 12, 16, 3
    t = b * n
    x, res, w = (T.rounded(a, "bf16") for a in (rng.normal(size=(t, width)), rng.normal(size=(t, width)), np.ones(width)))
    h, y, s = gpu_run(rx, client, P.rms_norm(t, width, out="f8E4M3FN"), [x, res, w])[0]
    exact = L.rms_norm(x.a, res.a, w.a)[1]
    close_to_numbers(y.a, s.a.astype(np.float64), exact, "f8E4M3FN", 34 * UF * np.abs(exact).max(-1, keepdims=True))
    # q, k and v by one product in 8 bits, with its scales
    out = (hq + 2 * hk) * d
    weight, factor = I.Tensor(LF.round_e4m3fn(rng.normal(size=(out, width)).astype(np.float32) * 50), "f8E4M3FN"), np.float32(1 / (50 * 16))
    m = P._Text()
    ya, sa, wa = m.arg([t, width], "f8E4M3FN"), m.arg([t], "f32"), m.arg([out, width], "f8E4M3FN")
    f = m.binary("multiply", m.dot(ya, wa, (1, 1), "f32"), m.spread(sa, [0], [t, out]))
    f = m.convert(m.binary("multiply", f, m.constant("%.9e" % factor, [t, out], "f32")), "bf16")
    qkv = gpu_run(rx, client, m.module("product", [f]), [y, s, weight])[0][0]
    prod = (y.a.astype(np.float64) @ weight.a.T.astype(np.float64)) * s.a[:, None].astype(np.float64) * np.float64(factor)
    size_of = (np.abs(y.a.astype(np.float64)) @ np.abs(weight.a.T.astype(np.float64))) * s.a[:, None] * factor
    T.close(qkv.a, prod, (width + 4) * UF * size_of, "bf16")
    q, k, v = (I.Tensor(p.reshape(t, -1, d), "bf16") for p in np.split(qkv.a, [hq * d, (hq + hk) * d], 1))
    # written behind 20, 3 and no positions
    lengths = np.array([20, 3, 0])
    angle = rng.uniform(-3, 3, size=(40, d // 2))
    mask = tree(rng, b, n)
    position = (lengths[:, None] + np.arange(n)).reshape(-1)
    rows = (lengths[:, None] + mask.sum(-1)).reshape(1, -1)
    table = rng.permutation(pages)[:b * cols].reshape(b, cols)
    (kc, ks), (vc, vs) = (stored(rng, "f8E4M3FN", pages, size, hk, d, "slots") for _ in range(2))
    args = [q, k, v, I.Tensor(np.cos(angle), "f32"), I.Tensor(np.sin(angle), "f32"), I.Tensor(rows, "i32"), I.Tensor(position, "i32"), I.Tensor(np.repeat(np.arange(b), n), "i32"), I.Tensor(table, "i32"), kc, vc, ks, vs]
    q2, kc, vc, ks, vs = gpu_run(rx, client, P.kv_write(t, b, hq, hk, d, pages, size, cols, 40, cache="f8E4M3FN"), args)[0]
    check_write([g.a for g in (q2, kc, vc, ks, vs)], args, np.zeros(d // 2, int), "bf16", "f8E4M3FN", "halves", "slots")
    query = I.Tensor(q2.a.reshape(b, n, hq, d), "bf16")
    check_tree(rx, client, [query, kc, vc, I.Tensor(table, "i32"), I.Tensor(lengths, "i32")], [ks, vs], mask, n, hq, hk, d, d, size, cols, "bf16", "f8E4M3FN", "slots", 0)
    path = np.array([[0, 3, 5], [2, -1, -1], [0, 1, 4]])
    margs = [I.Tensor(lengths, "i32"), I.Tensor(path, "i32"), I.Tensor(table, "i32"), kc, vc, ks, vs]
    moved = gpu_run(rx, client, P.kv_move(b, 3, hk, d, pages, size, cols, cache="f8E4M3FN"), margs)[0]
    assert all(np.array_equal(g.a, w) for g, w in zip(moved, L.kv_move(*[a.a for a in margs])))
    # the next token over the accepted branch
    check_tree(rx, client, [I.Tensor(query.a[:, :1], "bf16"), moved[0], moved[1], I.Tensor(table, "i32"), I.Tensor(lengths + [3, 1, 3], "i32")], list(moved[2:]), None, 1, hq, hk, d, d, size, cols, "bf16",
               "f8E4M3FN", "slots", 0)


def test_a_whole_step_in_8_bits_runs(rx, client):
    """One module in 8 bits: the same bits every run, probabilities that are some, scales and numbers written where they belong alone."""
    b, n, vocab, width, hq, hk, d, hidden, pages, size, cols, positions = 2, 3, 101, 64, 8, 2, 32, 96, 9, 4, 4, 16
    text, types, cache_results = P.verify_step(b, n, vocab, width, hq, hk, d, hidden, pages, size, cols, positions, layers=2, top=3)
    rng = np.random.default_rng(13)
    args = verify_values(rng, text, types, True, b, n, pages, cols, positions, d)
    mask = tree(rng, b, n)
    lengths = np.array([5, 0])
    for k, v in enumerate((rng.integers(0, vocab, (b, n)), rng.integers(0, vocab, (b, n)), (lengths[:, None] + mask.sum(-1) - 1).clip(0)[None], lengths)):
        args[k] = I.Tensor(v, "i32")
    args[4] = I.Tensor(mask, "i1")
    got, exe = gpu_run(rx, client, text, args)
    again, _ = gpu_run(rx, client, text, args, exe)
    assert all(same_bits(x.a, y.a) for x, y in zip(got, again))
    logprob, lse, entropy = (g.a for g in got[:3])
    assert np.all(logprob <= 0) and np.isfinite(lse).all() and np.all((entropy >= 0) & (entropy <= np.log(vocab) + 1e-5))
    written = np.zeros((pages, size), dtype=bool)
    for s in range(b):
        for j in range(n):
            p = lengths[s] + j
            written[args[5].a[s, p // size], p % size] = True
    caches = [k for k, (s, t) in enumerate(types) if len(s) == 4 or (len(s) == 3 and t == "f32")]
    for k, r in zip(caches, cache_results):
        new, old = got[r].a, args[k].a
        if new.ndim == 3:
            new, old = new.transpose(0, 2, 1), old.transpose(0, 2, 1)
        assert same_bits(new[~written], old[~written]) and np.isfinite(new[written]).all()
        assert np.any(new[written] != old[written])


class Near:
    """Numbers v in 64 bits, and e, what the device's may be off by."""

    def __init__(self, v, e=0.0):
        self.v = np.asarray(v, dtype=np.float64)
        self.e = np.broadcast_to(np.asarray(e, dtype=np.float64), self.v.shape)

    def rounds(self, n):
        """After n roundings to f32."""
        return Near(self.v, self.e + n * UF * (np.abs(self.v) + self.e))

    def __add__(self, o):
        return Near(self.v + o.v, self.e + o.e).rounds(1)

    def __mul__(self, o):
        return Near(self.v * o.v, self.e * np.abs(o.v) + np.abs(self.v) * o.e + self.e * o.e).rounds(1)

    def __getitem__(self, i):
        return Near(self.v[i], self.e[i])

    def reshape(self, *s):
        return Near(self.v.reshape(*s), self.e.reshape(*s))

    def product(self, w):
        """With rows of w that hold few numbers beside zeros: their products and sums."""
        a, b = np.abs(self.v) + self.e, np.abs(w)
        return Near(self.v @ w.T, self.e @ b.T + ((w != 0).sum(1) + 4) * UF * (a @ b.T))

    def normed(self, w):
        """The root is off by half of what the mean of the squares is, relative to it; of a row no longer than a wavefront, whose sum takes 6 steps,
        (1 + 6 + 2) / 2 + 5 U more."""
        a, mean = np.abs(self.v), (self.v ** 2).mean(-1, keepdims=True) + 1e-6
        off = (2 * a * self.e + self.e ** 2).mean(-1, keepdims=True) / mean
        assert np.all(off < 0.5)
        r, y = mean ** -0.5, self.v * mean ** -0.5 * w
        return Near(y, self.e * r * np.abs(w) * (1 + off) + np.abs(y) * (off + 10 * UF))

    def quantized(self, dt):
        """(numbers, scales): numbers go either way where their values lie next to a border."""
        top = np.abs(self.v).max(-1)
        scale = Near(np.maximum(top, 2.0 ** -100) / L.LARGEST[dt], self.e.max(-1) / L.LARGEST[dt]).rounds(1)
        z = self.v / scale.v[..., None]
        off = (self.e / scale.v[..., None] + np.abs(z) * (scale.e / (scale.v - scale.e))[..., None]) * 1.001 + UF * np.abs(z)

        def near(x):
            x = np.clip(x, -L.LARGEST[dt], L.LARGEST[dt])
            return np.rint(x) if dt == "i8" else LF.round_e4m3fn(x.astype(np.float32)).astype(np.float64)
        codes = near(z)
        return Near(codes, np.maximum(np.abs(near(z - off) - codes), np.abs(near(z + off) - codes))), scale


def assert_near(got, ref):
    got = np.asarray(got, dtype=np.float64)
    ok = np.abs(got - ref.v) <= ref.e
    assert got.shape == ref.v.shape and ok.all(), "%d of %d, first at %s: %r for %r, bound %r" % ((~ok).sum(), ok.size, np.argwhere(~ok)[0], got[~ok][0], ref.v[~ok][0], ref.e[~ok][0])


@pytest.mark.parametrize("seed,cache,products,layout,rotation,axes", [(17, "f8E4M3FN", "f8E4M3FN", "slots", "halves", 1), (3, "i8", "f8E4M3FN", "heads", "pairs", 3), (3, "f8E4M3FN", "i8", "heads", "halves", 2)])
def test_values_of_a_whole_step_in_8_bits(rx, client, seed, cache, products, layout, rotation, axes):
    """One module of two layers, f32 between its 8 bits, against the operators' definitions in 64 bits, with what every operation may be off
    by carried along: numbers that the device may round the other way count with their whole step.  Inputs that have next to none of those, so
    that the results' bounds are small."""
    b, n, vocab, width, hq, hk, d, hidden, pages, size, cols, positions = 2, 3, 101, 32, 4, 2, 16, 32, 9, 4, 4, 16
    t, half = b * n, d // 2
    text, types, cache_results = P.verify_step(b, n, vocab, width, hq, hk, d, hidden, pages, size, cols, positions, layers=2, axes=axes, top=3, dt="f32", cache=cache, products=products, layout=layout,
                                               rotation=rotation)
    rng = np.random.default_rng(seed)
    args = verify_values(rng, text, types, True, b, n, pages, cols, positions, d)
    for k, (s, dt) in enumerate(types[8:], 8):
        if len(s) == 2:                              # weights: three numbers of a row, so that roundings stay few
            x = np.zeros(s)
            for row in x:
                row[rng.permutation(s[1])[:3]] = rng.choice([-2, -1, 1, 2], size=3)
            args[k] = I.Tensor(x, dt)
        elif dt in EIGHT:                            # what the caches hold already, and its scales
            x = rng.normal(size=s) * 50
            args[k] = I.Tensor(np.rint(x.clip(-127, 127)) if dt == "i8" else LF.round_e4m3fn(x.astype(np.float32)), dt)
        elif len(s) == 3:
            args[k] = I.Tensor(rng.uniform(0.005, 0.015, size=s), "f32")
        elif not s:
            args[k] = I.Tensor(np.float32(rng.uniform(0.05, 0.1)), "f32")
    mask, lengths = tree(rng, b, n), np.array([5, 0])
    depth = mask.sum(-1)
    angle = np.stack([(lengths[:, None] + depth + 2 * a) % positions for a in range(axes)])
    args[8] = T.rounded(rng.normal(size=(vocab, width)), "f32")
    for k, v in enumerate((rng.integers(0, vocab, (b, n)), rng.integers(0, vocab, (b, n)), angle, lengths)):
        args[k] = I.Tensor(v, "i32")
    args[4] = I.Tensor(mask, "i1")
    got = [g.a for g in gpu_run(rx, client, text, args)[0]]
    a = [np.asarray(x.a, dtype=np.float64) if x.dt not in ("i32", "i1") else x.a for x in args]
    tokens, targets, table, cos, sin, given = a[0].reshape(-1), a[1].reshape(-1), a[5], a[6], a[7], iter(a[8:])
    position = (lengths[:, None] + np.arange(n)).reshape(-1)
    page, slot = table[np.arange(t) // n, position // size], position % size
    axis = np.repeat(np.arange(axes), [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1))
    c, s = (Near(m[angle.reshape(axes, t)[axis].T, np.arange(half)][:, None]) for m in (cos, sin))
    first = np.arange(half) * (2 if rotation == "pairs" else 1)
    second = first + (1 if rotation == "pairs" else half)

    def rotated(x):
        p, q = x[..., first], x[..., second]
        minus, plus = p * c + q * Near(-s.v), q * c + p * s
        v, e = np.zeros(x.v.shape), np.zeros(x.v.shape)
        v[..., first], e[..., first], v[..., second], e[..., second] = minus.v, minus.e, plus.v, plus.e
        return Near(v, e)

    def attended(q, caches, scales):
        out_v, out_e = np.zeros((t, hq, d)), np.zeros((t, hq, d))
        for i in range(t):
            before = lengths[i // n]
            at = np.concatenate([np.arange(before), before + np.flatnonzero(mask[i // n, i % n])])
            if not len(at):
                continue
            pg, sl = table[i // n, at // size], at % size
            for h in range(hq):
                g = h // (hq // hk)
                k, v = (rows[pg, sl, g] * Near(sc.v[pg, g, sl][:, None], sc.e[pg, g, sl][:, None]) for rows, sc in zip(caches, scales))
                x, ax = k.v @ q.v[i, h], np.abs(k.v) + k.e
                off = (k.e @ np.abs(q.v[i, h]) + ax @ q.e[i, h] + (d + 5) * UF * (ax @ np.abs(q.v[i, h]))) * d ** -0.5
                w = np.exp((x - x.max()) * d ** -0.5)
                w /= w.sum()
                more = np.expm1(2 * off.max()) + (len(at) + 17) * UF + 2.0 ** -23
                out_v[i, h], out_e[i, h] = w @ v.v, (1 + more) * (w @ v.e) + more * (w @ np.abs(v.v))
        return Near(out_v, out_e)

    x, late = Near(next(given)[tokens]), None
    for layer in range(2):
        w1, wq, wk, wv, wo, w2, gate, up, down = (next(given) for _ in range(9))
        factors = [Near(next(given)) for _ in range(5)]
        kc, vc, ks, vs = (next(given) for _ in range(4))
        x = x if late is None else late + x
        codes, scale = x.normed(w1).quantized(products)
        q, k, v = ((codes.product(w) * scale[:, None] * f).reshape(t, -1, d) for w, f in zip((wq, wk, wv), factors))
        held, held_scales = [], []
        for r, (old, old_scale, new) in enumerate(((kc, ks, rotated(k)), (vc, vs, v))):
            number, sc = new.quantized(cache)
            rows, scales = old if layout == "slots" else old.transpose(0, 2, 1, 3), old_scale
            now, now_scale = Near(rows.copy(), np.zeros(rows.shape)), Near(scales.copy(), np.zeros(scales.shape))
            now.e, now_scale.e = np.array(now.e), np.array(now_scale.e)
            now.v[page, slot], now.e[page, slot], now_scale.v[page, :, slot], now_scale.e[page, :, slot] = number.v, number.e, sc.v, sc.e
            device = got[cache_results[4 * layer + r]]
            assert_near(device if layout == "slots" else device.transpose(0, 2, 1, 3), now)
            assert_near(got[cache_results[4 * layer + 2 + r]], now_scale)
            held.append(now)
            held_scales.append(now_scale)
        x = attended(rotated(q), held, held_scales).reshape(t, hq * d).product(wo) + x
        codes, scale = x.normed(w2).quantized(products)
        y, z = (codes.product(w) * scale[:, None] * f for w, f in zip((gate, up), factors[3:]))
        sig = 1 / (1 + np.exp(-y.v))                 # (its slope is at most 1/4; the exponential and the quotient in f32)
        late = (y * Near(sig, y.e / 4 + 8 * UF * sig) * z).product(down)
    logits = (late + x).normed(next(given)).product(next(given))
    off = logits.e.max(-1) + (vocab / 64 + 108) * UF
    top = logits.v.max(-1, keepdims=True)
    lse = np.log(np.exp(logits.v - top).sum(-1)) + top[:, 0]
    assert off.max() < 0.01                          # (so that a wrong scale or product would show)
    assert_near(got[1], Near(lse, off + 4 * UF * np.abs(lse)))
    logp = logits.v - lse[:, None]
    assert_near(got[0], Near(logp[np.arange(t), targets], 2 * off + 4 * UF * np.abs(logp).max()))
    assert_near(got[3], Near(-np.sort(-logp, -1)[:, :3], (2 * off + 4 * UF * np.abs(logp).max())[:, None]))
