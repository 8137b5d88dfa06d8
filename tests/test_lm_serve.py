"""Norms, caches of 8 bits and drafted tokens without a device: the oracle's formulas against closed forms and differences, what
the importer refuses, and which launches a module becomes."""
import importlib
import os
import subprocess

import numpy as np
import pytest

from _loader import load_pkg, ROOT
from oracle import lm_ops as L
from oracle import stablehlo_interp as I
from test_lm_operators import swap, launches, copies

rx = load_pkg()
P = importlib.import_module("reactant_jl_amd.lm_programs")
HOSTCHECK = os.path.join(ROOT, "reactant.jl_amd", "csrc", "build", "rx_hostcheck_asan")


# ----------------------------------------------------------------------------
# the oracle
# ----------------------------------------------------------------------------
def test_norm_of_known_rows():
    h, y = L.rms_norm(np.array([[3.0, 0.0]]), np.array([[0.0, 4.0]]), np.array([1.0, 2.0]), eps=0.0)
    assert np.array_equal(h, [[3, 4]]) and np.allclose(y, [[3 / np.sqrt(12.5), 8 / np.sqrt(12.5)]])
    y, = L.rms_norm(np.full((1, 4), -7.0), None, np.ones(4))
    assert np.allclose(y, -1)


def test_gradient_of_the_norm_against_differences():
    rng = np.random.default_rng(0)
    h, w, dy, dh = rng.normal(size=(3, 5)), rng.normal(size=5), rng.normal(size=(3, 5)), rng.normal(size=(3, 5))

    def loss(h, w):
        return (dy * L.rms_norm(h, None, w, eps=0.3)[0]).sum() + (dh * h).sum()
    dx, dw = L.rms_norm_grad(h, w, dy, dh, eps=0.3)
    # central differences of steps of 1e-5 of a function whose third derivatives stay below about 100: 2e-9, rounding 1e-11 / 1e-5
    for t, j in np.ndindex(3, 5):
        step = np.zeros_like(h)
        step[t, j] = 1e-5
        assert abs(dx[t, j] - (loss(h + step, w) - loss(h - step, w)) / 2e-5) < 1e-7
    for j in range(5):
        step = np.zeros(5)
        step[j] = 1e-5
        assert abs(dw[j] - (loss(h, w + step) - loss(h, w - step)) / 2e-5) < 1e-7


def test_numbers_of_8_bits():
    y, scale = L.quantize([[0.0, 0.0], [1.0, -127.0], [2.0 ** -120, 0.0], [np.inf, 1.0], [np.nan, 2.0]], "i8")
    assert np.array_equal(scale[:2], [2.0 ** -100 / 127, 1.0]) and np.array_equal(y[:2], [[0, 0], [1, -127]]) and np.array_equal(y[2], [0, 0])
    assert np.isnan(scale[3:]).all() and np.all(y[3:] == 0)
    y, scale = L.quantize([[448.0 * 3, 3.0]], "f8E4M3FN")
    assert scale[0] == 3 and np.array_equal(y, [[448, 1]])


def test_axes_turn_their_sections():
    rng = np.random.default_rng(1)
    q, k, v = (rng.normal(size=(2, h, 8)) for h in (2, 1, 1))
    turn = np.arange(6)[:, None] * np.array([1.0, 0.5, 0.25, 0.125])[None, :]
    args = [q, k, v, np.cos(turn), np.sin(turn)]
    pages, cache = np.array([[1, 0]]), np.zeros((2, 4, 1, 8))
    angle = np.array([[3, 5], [1, 0], [4, 2]])
    out = L.kv_write(*args, angle, np.array([0, 6]), np.array([0, 0]), pages, cache, cache, sections="1,2,1")[:2]
    for t in range(2):
        rows = angle[[0, 1, 1, 2], t]
        c, s = np.cos(turn[rows, np.arange(4)]), np.sin(turn[rows, np.arange(4)])
        assert np.allclose(out[0][t], L.rotate(q[t], c, s, "halves"))
        assert np.allclose(out[1][[1, 0][t], [0, 2][t]], L.rotate(k[t], c, s, "halves"))
    # one axis that follows the position is rx.kv_append
    pos = np.array([3, 5])
    new = L.kv_write(*args, pos[None], pos, np.zeros(2, int), pages, cache, cache, rotation="pairs")
    old = L.kv_append(*args, pos, np.zeros(2, int), pages, cache, cache, rotation="pairs")
    assert all(np.array_equal(a, b) for a, b in zip(new, old))


def test_a_chain_of_drafted_tokens_is_dense_attention():
    rng = np.random.default_rng(2)
    n, before, hq, hk, d, size = 3, 5, 4, 2, 6, 4
    k, v, q = rng.normal(size=(2, 4, hk, d)), rng.normal(size=(2, 4, hk, d)), rng.normal(size=(2, n, hq, d))
    pages, lengths = np.array([[1, 0, -1], [0, -1, -1]]), np.array([before, -1])
    out, lse, _ = L.tree_attention(q, k, v, pages, lengths)
    assert np.all(out[1] == 0) and np.all(lse[1] == -np.inf)
    for i in range(n):      # one token at a time, each seeing one position more
        one, l1, _ = L.paged_attention(q[:1, i], k, v, pages[:1], np.array([before + i + 1]))
        assert np.allclose(out[0, i], one[0]) and np.allclose(lse[0, i], l1[0])
    out, lse, _ = L.tree_attention(q, k, v, pages, lengths, window=4)
    for i in range(n):
        one, l1, _ = L.paged_attention(q[:1, i], k, v, pages[:1], np.array([before + i + 1]), window=4)
        assert np.allclose(out[0, i], one[0]) and np.allclose(lse[0, i], l1[0])
    # siblings do not see one another: each as if it were alone
    mask = np.eye(n, dtype=bool)
    out, _, _ = L.tree_attention(q, k, v, pages, lengths, mask)
    for i in range(n):
        rows = [(int(pages[0, j // size]), j % size) for j in list(range(before)) + [before + i]]
        kk, vv = (np.stack([c[r] for r in rows]) for c in (k, v))
        for h in range(hq):
            x = kk[:, h // 2] @ q[0, i, h] / np.sqrt(d)
            assert np.allclose(out[0, i, h], np.exp(x - np.logaddexp.reduce(x)) @ vv[:, h // 2])
    assert np.all(L.tree_attention(q, k, v, pages, np.array([0, 0]), np.zeros((n, n)))[0] == 0)


def test_moves_take_what_was_there():
    c = np.arange(8.0).reshape(2, 4, 1, 1)
    s = np.arange(8.0).reshape(2, 1, 4)
    out = L.kv_move(np.array([2]), np.array([[1, 2, 0, -1, 3, 9]]), np.array([[1, 0]]), c, c, s, s)
    # positions 2..7 held 6 7 0 1 2 3: position 2 takes 3's, 3 takes 4's, 4 takes 2's, 6 takes 5's
    for o in out:
        assert np.array_equal(o.reshape(-1), [6, 1, 1, 3, 4, 5, 7, 0])


# ----------------------------------------------------------------------------
# refusals
# ----------------------------------------------------------------------------
NORM, NORM8, GRAD = P.rms_norm(3, 64), P.rms_norm(3, 64, out="f8E4M3FN"), P.rms_norm_grad(3, 64)
WRITE = P.kv_write(3, 2, 8, 2, 64, 10, 16, 4, 64, cache="i8", sections=[8, 12, 12])
PLAIN = P.kv_write(3, 2, 8, 2, 64, 10, 16, 4, 64)
MOVE, MOVE8 = P.kv_move(2, 5, 2, 64, 10, 16, 4), P.kv_move(2, 5, 2, 64, 10, 16, 4, cache="f8E4M3FN")
TREE, TREE8 = P.tree_attention(2, 5, 8, 2, 64, 10, 16, 4), P.tree_attention(2, 5, 8, 2, 64, 10, 16, 4, cache="i8")
REFUSED = {
    "norm of f64": (swap(NORM, ("bf16", "f64")), "must be f32, bf16 or f16"),
    "norm of nothing": (P.rms_norm(3, 0), "rows of 1 to 32768"),
    "rows too wide": (P.rms_norm(3, 32769), "rows of 1 to 32768"),
    "weight of another width": (swap(NORM, ("tensor<64xbf16>", "tensor<32xbf16>")), "the weight must be"),
    "weight of another type": (swap(NORM, ("tensor<64xbf16>", "tensor<64xf32>")), "the type of x"),
    "8 bits without scales": (swap(NORM, ("tensor<3x64xbf16>, tensor<3x64xbf16>) {", "tensor<3x64xbf16>, tensor<3x64xi8>) {"), ("-> (tensor<3x64xbf16>, tensor<3x64xbf16>)", "-> (tensor<3x64xbf16>, tensor<3x64xi8>)"),
                                   (" : tensor<3x64xbf16>, tensor<3x64xbf16>\n", " : tensor<3x64xbf16>, tensor<3x64xi8>\n")), "one result more"),
    "scales in bf16": (swap(NORM8, ("tensor<3xf32>", "tensor<3xbf16>")), "the scales must be f32"),
    "scales of another batch": (swap(NORM8, ("tensor<3xf32>", "tensor<1xf32>")), "the scales must be"),
    "result of e5m2": (swap(NORM8, ("f8E4M3FN", "f8E5M2")), "or be f8E4M3FN or i8"),
    "negative eps": (P.rms_norm(3, 64, eps=-1.0), "not negative"),
    "norm of one operand": (swap(P.rms_norm(3, 64, residual=False), ("(%arg0, %arg1)", "(%arg0)"), (" : (tensor<3x64xbf16>, tensor<64xbf16>) ->", " : (tensor<3x64xbf16>) ->")), "expected 2 to 3 operands, got 1"),
    "gradient of another shape": (swap(GRAD, ("%arg2: tensor<3x64xbf16>", "%arg2: tensor<4x64xbf16>"), (": (tensor<3x64xbf16>, tensor<64xbf16>, tensor<3x64xbf16>,", ": (tensor<3x64xbf16>, tensor<64xbf16>, tensor<4x64xbf16>,")), "h and dy"),
    "dweight in f16": (swap(GRAD, ("tensor<64xf32>", "tensor<64xf16>")), "the type of h, or be f32"),
    "axes without sections": (swap(WRITE, ('sections = "8,12,12"', 'rotation2 = "x"')), "unknown setting"),
    "sections left out": (swap(WRITE, (', sections = "8,12,12"', "")), "need the setting 'sections'"),
    "sections of another sum": (swap(WRITE, ("8,12,12", "8,12,13")), "must add up to the 32"),
    "sections of another number": (swap(WRITE, ("8,12,12", "20,12")), "one number for each of the 3"),
    "sections no numbers": (swap(WRITE, ("8,12,12", "8,,12")), "whole numbers with commas"),
    "sections below zero": (swap(WRITE, ("8,12,12", "-8,28,12")), "whole numbers with commas"),
    "five axes": (P.kv_write(3, 2, 8, 2, 64, 10, 16, 4, 64, sections=[7, 7, 7, 7, 4]), "one to four axes"),
    "8 bits without their scales": (swap(PLAIN, ("tensor<10x16x2x64xbf16>", "tensor<10x16x2x64xi8>")), "need k_scale"),
    "scales in another order": (swap(WRITE, ("tensor<10x2x16xf32>", "tensor<10x16x2xf32>")), "k_scale must be"),
    "scales of 16 bits": (swap(WRITE, ("tensor<10x16x2x64xi8>", "tensor<10x16x2x64xbf16>")), "scales belong to caches of 8 bits"),
    "cache of another type": (swap(PLAIN, ("tensor<10x16x2x64xbf16>", "tensor<10x16x2x64xf16>")), "the type of q"),
    "angle of one dimension": (swap(PLAIN, ("tensor<1x3xi32>", "tensor<3xi32>")), "angle must have 2 dimensions"),
    "angle of another batch": (swap(PLAIN, ("tensor<1x3xi32>", "tensor<1x4xi32>")), "angle must be"),
    "rotation beyond the head": (P.kv_write(3, 2, 8, 2, 64, 10, 16, 4, 64, rotary_dim=66), "exceed the head's"),
    "65 steps": (P.kv_move(2, 65, 2, 64, 10, 16, 4), "at most 64 steps"),
    "path of another batch": (swap(MOVE, ("tensor<2x5xi32>", "tensor<3x5xi32>")), "path must be"),
    "path of i64": (swap(MOVE, ("tensor<2x5xi32>", "tensor<2x5xi64>")), "must have one type"),
    "one scale": (swap(MOVE8, ("%arg5, %arg6)", "%arg5)"), (", tensor<10x2x16xf32>, tensor<10x2x16xf32>) ->", ", tensor<10x2x16xf32>) ->")), "belong together"),
    "caches of f64": (swap(MOVE, ("bf16", "f64")), "the caches must be f32"),
    "mask in i32": (swap(TREE, ("tensor<2x5x5xi1>", "tensor<2x5x5xi32>")), "the mask must be i1"),
    "mask of another size": (swap(TREE, ("tensor<2x5x5xi1>", "tensor<2x5x6xi1>")), "the mask must be"),
    "mask of one sequence": (swap(TREE, ("tensor<2x5x5xi1>", "tensor<1x5x5xi1>")), "the mask must be"),
    "window below the tree": (P.tree_attention(2, 5, 8, 2, 64, 10, 16, 4, window=4), "must hold the 5 drafted tokens"),
    "1025 drafted tokens": (P.tree_attention(2, 1025, 8, 2, 64, 10, 16, 4), "at most 1024"),
    "heads no multiple": (P.tree_attention(2, 5, 7, 2, 64, 10, 16, 4), "must be a multiple"),
    "heads of 257": (P.tree_attention(2, 5, 8, 2, 257, 10, 16, 4), "head dimensions from 1 to 256"),
    "result of another type": (swap(TREE8, ("-> tensor<2x5x8x64xbf16> {", "-> tensor<2x5x8x64xf32> {"), ("-> tensor<2x5x8x64xbf16>\n", "-> tensor<2x5x8x64xf32>\n"), (" : tensor<2x5x8x64xbf16>\n", " : tensor<2x5x8x64xf32>\n")), "the type of q"),
    "scale beyond f32": (P.tree_attention(2, 5, 8, 2, 64, 10, 16, 4, scale=3e38), "a number that f32 holds"),
    "drafted tokens in one dimension": (swap(TREE, ("tensor<2x5x8x64xbf16>", "tensor<10x8x64xbf16>")), "q must have 4 dimensions"),
}


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refusals(name):
    text, message = REFUSED[name]
    with pytest.raises(rx.ReactantInternalError) as e:
        rx.compile_offline(text)
    assert message in str(e.value)


# ----------------------------------------------------------------------------
# launches
# ----------------------------------------------------------------------------
def test_caches_and_scales_are_updated_in_place():
    assert launches(WRITE) == ["lm_kv_write"] and launches(MOVE8) == ["lm_kv_move"]
    for text, first in ((WRITE, 9), (MOVE8, 3)):
        plain = text
        for k in range(4):
            plain = plain.replace(" {tf.aliasing_output = %d : i32}" % (k + (first == 9)), "")
        assert len(copies(plain)) == 4                                  # copied: the arguments stay as they are


def test_nothing_to_do_is_no_launch():
    assert launches(P.rms_norm(0, 64)) == [] and launches(P.kv_write(0, 2, 8, 2, 64, 10, 16, 4, 64)) == [] and launches(P.kv_move(0, 5, 2, 64, 10, 16, 4)) == []
    assert launches(P.kv_move(2, 0, 2, 64, 10, 16, 4)) == [] and launches(P.tree_attention(0, 5, 8, 2, 64, 10, 16, 4)) == [] and launches(P.tree_attention(2, 0, 8, 2, 64, 10, 16, 4)) == []
    assert launches(P.rms_norm_grad(0, 64)) == ["lm_rms_norm_grad", "lm_rms_norm_weight"]      # zeros are written


def programs():
    mods = {"norm": NORM, "norm8": NORM8, "norm_odd": P.rms_norm(5, 1001, dt="f16", out="i8", residual=False), "norm_wide": P.rms_norm(2, 32767, dt="f32"), "norm_grad": GRAD,
            "norm_grad_wide": P.rms_norm_grad(3, 20000, dt="f32", residual=False), "write": WRITE, "write_plain": PLAIN,
            "write_odd": P.kv_write(30, 3, 4, 4, 33, 9, 5, 3, 15, dt="f32", cache="f8E4M3FN", rotary_dim=32, rotation="pairs", layout="heads", ids="i64", value_dim=17),
            "move": MOVE, "move8": MOVE8, "move_long": P.kv_move(3, 64, 1, 33, 9, 5, 3, cache="i8", ids="i64"), "tree": TREE, "tree8": TREE8,
            "tree_wide": P.tree_attention(3, 64, 64, 8, 128, 100, 24, 20, dt="f16", mask="shared", lse=True), "tree_f32": P.tree_attention(2, 9, 12, 12, 80, 30, 24, 9, dt="f32", mask=False, window=40),
            "tree_f32_8": P.tree_attention(2, 33, 8, 2, 256, 30, 24, 9, dt="f32", cache="f8E4M3FN", layout="heads", ids="i64"),
            "verify": P.verify_step(2, 3, 50, 32, 4, 2, 16, 48, 12, 4, 4, 64, layers=2)[0], "verify_f32": P.verify_step(2, 3, 50, 32, 4, 2, 16, 48, 12, 4, 4, 64, axes=3, dt="f32", cache="f32", products="f32")[0]}
    return mods


def test_host_code_under_sanitizers(tmp_path):
    if not os.path.exists(HOSTCHECK):
        pytest.skip("the sanitizer program is not built")
    files = []
    for name, text in programs().items():
        files.append(tmp_path / (name + ".mlir"))
        files[-1].write_text(text)
    for k, (text, _) in enumerate(REFUSED.values()):
        files.append(tmp_path / ("refused%d.mlir" % k))
        files[-1].write_text("// expect-error\n" + text)
    r = subprocess.run([HOSTCHECK] + [str(f) for f in files], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_interpreter_reads_the_calls():
    text = P.kv_move(1, 2, 1, 1, 1, 4, 1, cache="f32")
    c = np.arange(4.0).reshape(1, 4, 1, 1)
    out = I.run_text(text, [I.Tensor([1], "i32"), I.Tensor([[1, 0]], "i32"), I.Tensor([[0]], "i32"), I.Tensor(c, "f32"), I.Tensor(-c, "f32")])
    assert np.array_equal(out[0].a.reshape(-1), [0, 2, 1, 3]) and np.array_equal(out[1].a.reshape(-1), [0, -2, -1, -3])
    out = I.run_text(NORM8, [I.Tensor(np.ones((3, 64)), "bf16")] * 2 + [I.Tensor(np.ones(64), "bf16")])
    assert np.all(out[0].a == 2) and np.all(out[1].a == 448) and np.allclose(out[2].a, 1 / 448)


def test_programs_compile():
    for name in ("write_odd", "move_long", "tree_f32_8", "norm_wide", "verify"):
        assert launches(programs()[name])


def test_more_sequences_than_are_counted():
    with pytest.raises(rx.ReactantInternalError) as e:
        rx.compile_offline(P.tree_attention(65536, 1, 8, 2, 64, 10, 16, 4))
    assert "too many sequences or heads" in str(e.value)
