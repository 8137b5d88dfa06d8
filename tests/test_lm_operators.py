"""Language-model operators without a device: the oracle's formulas against closed forms and differences, what the importer
refuses, and which launches a module becomes."""
import importlib
import os
import subprocess

import numpy as np
import pytest

from _loader import load_pkg, ROOT
from oracle import lm_ops as L
from oracle import stablehlo_interp as I

rx = load_pkg()
P = importlib.import_module("reactant_jl_amd.lm_programs")
HOSTCHECK = os.path.join(ROOT, "reactant.jl_amd", "csrc", "build", "rx_hostcheck_asan")


# ----------------------------------------------------------------------------
# the oracle
# ----------------------------------------------------------------------------
def test_rotation_by_known_angles():
    x = np.arange(1.0, 7.0)[None, :]                                     # one head of 6: 4 rotated, 2 not
    quarter, none = np.array([0.0, 0.0]), np.array([1.0, 1.0])           # cosines and sines of 90 degrees
    assert np.allclose(L.rotate(x, quarter, none, "halves"), [[-3, -4, 1, 2, 5, 6]])
    assert np.allclose(L.rotate(x, quarter, none, "pairs"), [[-2, 1, -4, 3, 5, 6]])
    assert np.array_equal(L.rotate(x, quarter, none, "none"), x)


def test_scores_after_rotation_depend_on_the_distance():
    rng = np.random.default_rng(0)
    q, k = rng.normal(size=(1, 8)), rng.normal(size=(1, 8))
    freq = 10.0 ** -np.arange(4)

    def score(a, b, how):
        rows = [L.rotate(x, np.cos(p * freq), np.sin(p * freq), how) for x, p in ((q, a), (k, b))]
        return float((rows[0] * rows[1]).sum())
    for how in ("halves", "pairs"):
        assert np.isclose(score(9, 4, how), score(105, 100, how)) and not np.isclose(score(9, 4, how), score(9, 5, how))


def test_append_then_attend_is_dense_attention():
    rng = np.random.default_rng(1)
    n, hq, hk, d, size = 11, 4, 2, 6, 4
    q, k, v = rng.normal(size=(n, hq, d)), rng.normal(size=(n, hk, d)), rng.normal(size=(n, hk, d))
    angle = np.arange(16)[:, None] * np.array([1.0, 0.1, 0.01])[None, :]
    pages = np.array([[7, -1, -1, -1], [3, 0, 5, -1]], dtype=np.int32)
    for layout in ("slots", "heads"):
        empty = np.full((8, size, hk, d) if layout == "slots" else (8, hk, size, d), np.nan)
        q2, kc, vc = L.kv_append(q, k, v, np.cos(angle), np.sin(angle), np.arange(n), np.ones(n, int), pages, empty, empty, layout=layout)
        out, lse, _ = L.paged_attention(np.stack([q2[0], q2[-1]]), kc, vc, pages, np.array([0, n]), layout=layout)
        assert np.all(out[0] == 0) and np.all(lse[0] == -np.inf)
        for h in range(hq):
            rot = np.stack([L.rotate(k[j], np.cos(angle[j]), np.sin(angle[j]), "halves")[h // 2] for j in range(n)])
            x = rot @ q2[-1, h] / np.sqrt(d)
            assert np.isclose(lse[1, h], np.logaddexp.reduce(x))
            assert np.allclose(out[1, h], np.exp(x - lse[1, h]) @ v[:, h // 2])


def test_log_probabilities_of_known_distributions():
    v = 16
    lp, lse, ent, top, ids = L.token_logprobs(np.zeros((1, v)), [3], top=4)      # uniform: ties by index
    assert np.isclose(lp[0], -np.log(v)) and np.isclose(ent[0], np.log(v)) and np.array_equal(ids[0], [0, 1, 2, 3]) and np.allclose(top, -np.log(v))
    x = np.full((1, v), -np.inf)
    x[0, 5] = 2.0
    lp, lse, ent = L.token_logprobs(x, [5])
    assert lp[0] == 0 and lse[0] == 2 and ent[0] == 0
    lp, lse, ent = L.token_logprobs(x, [-1])
    assert lp[0] == 0
    lp, lse, ent, top, ids = L.token_logprobs(np.full((1, 4), -np.inf), [1], top=2)
    assert lp[0] == lse[0] == -np.inf and ent[0] == 0 and np.array_equal(ids[0], [0, 1])
    e = np.log([0.5, 0.25, 0.25])
    assert np.isclose(L.token_logprobs(e[None], [0])[2][0], 1.5 * np.log(2))


def test_gradients_against_differences():
    rng = np.random.default_rng(2)
    x, y = rng.normal(size=(3, 7)) * 2, np.array([2, 6, -1])
    x[1, 3] = -np.inf
    g, h = rng.normal(size=3), rng.normal(size=3)

    def loss(a):
        lp, _, ent = L.token_logprobs(a, y)
        return (g * lp + h * ent).sum()
    _, lse, ent = L.token_logprobs(x, y)
    grad = L.token_logprobs_grad(x, y, lse, ent, g, h)
    for t, j in np.ndindex(3, 7):
        if np.isinf(x[t, j]):
            assert grad[t, j] == 0
            continue
        step = np.zeros_like(x)
        step[t, j] = 1e-5
        # central differences of a function whose third derivatives stay below about 10: 1e-9, rounding 1e-11 / 1e-5
        assert abs(grad[t, j] - (loss(x + step) - loss(x - step)) / 2e-5) < 1e-7
    table, ids, dy = rng.normal(size=(5, 4)), np.array([1, -1, 1, 4, 9]), rng.normal(size=(5, 4))
    back = L.embedding_grad(dy, ids, 5, scale=3.0)                                 # linear: <dy, lookup(E)> = <grad, E>
    assert np.isclose((dy * L.embedding(table, ids, 3.0)).sum(), (back * table).sum()) and np.all(back[[0, 2, 3]] == 0)


def test_interpreter_reads_the_calls():
    text = P.embedding(3, 4, 2, dt="f32", scale=0.5)
    out = I.run_text(text, [I.Tensor(np.arange(8.0).reshape(4, 2), "f32"), I.Tensor(np.array([3, -1, 0]), "i32")])
    assert np.array_equal(out[0].a, [[3, 3.5], [0, 0], [0, 0.5]])


# ----------------------------------------------------------------------------
# refusals
# ----------------------------------------------------------------------------
def swap(text, *pairs):
    for a, b in pairs:
        assert a in text, a
        text = text.replace(a, b)
    return text


EMB, GRAD = P.embedding(5, 10, 8), P.embedding_grad(5, 10, 8)
APP = P.kv_append(3, 2, 8, 2, 64, 10, 16, 4, 64)
ATT = P.paged_attention(3, 8, 2, 64, 10, 16, 4)
LP, LPG = P.token_logprobs(4, 100, top=5), P.token_logprobs_grad(4, 100)
REFUSED = {
    "unknown target": (swap(EMB, ("rx.embedding", "rx.lookup")), "unknown target 'rx.lookup'"),
    "unknown setting": (swap(EMB, ("scale =", "factor =")), "unknown setting 'factor'"),
    "scale no number": (swap(EMB, ("scale = 1.00000000000000000e+00 : f64", 'scale = "x"')), "must be a finite number"),
    "setting twice": (swap(EMB, ("{scale", "{scale = 1.0 : f64, scale")), "given twice"),
    "config no dictionary": (swap(EMB, ("{scale = 1.00000000000000000e+00 : f64}", '"scale=1"')), "must be a dictionary"),
    "declared type differs": (swap(EMB, ("(%arg0, %arg1) {api_version = 4 : i32, backend_config = {scale = 1.00000000000000000e+00 : f64}} : (tensor<10x8xbf16>",
                                         "(%arg0, %arg1) {api_version = 4 : i32, backend_config = {scale = 1.00000000000000000e+00 : f64}} : (tensor<11x8xbf16>")), "declared"),
    "float ids": (swap(EMB, ("tensor<5xi32>", "tensor<5xf32>")), "must be i32 or i64"),
    "f64 table": (swap(EMB, ("bf16", "f64")), "must be f32, bf16 or f16"),
    "wrong rows": (swap(EMB, ("tensor<5x8xbf16>", "tensor<6x8xbf16>")), "the result must be tensor<5x8xbf16>"),
    "three operands": (swap(EMB, ("(%arg0, %arg1)", "(%arg0, %arg1, %arg1)"), (" : (tensor<10x8xbf16>, tensor<5xi32>) ->", " : (tensor<10x8xbf16>, tensor<5xi32>, tensor<5xi32>) ->")), "expected 2 operands"),
    "narrow gradient": (swap(P.embedding_grad(5, 10, 8, dt="f32"), ("tensor<10x8xf32>", "tensor<10x8xbf16>")), "type of dy, or be f32"),
    "rotation unknown": (swap(APP, ('"halves"', '"turns"')), "setting 'rotation' must be one of"),
    "layout unknown": (swap(APP, ('"slots"', '"rows"')), "setting 'layout' must be one of"),
    "rotation beyond the head": (P.kv_append(3, 2, 8, 2, 64, 10, 16, 4, 64, rotary_dim=66), "exceed the head's"),
    "cache of another layout": (swap(APP, ('"slots"', '"heads"')), "k must be"),
    "cache of another type": (swap(APP, ("tensor<10x16x2x64xbf16>", "tensor<10x16x2x64xf16>")), "the type of k"),
    "positions in another type": (swap(APP, ("tensor<2x4xi32>", "tensor<2x4xi64>")), "must have one type"),
    "heads of 257": (P.paged_attention(3, 8, 2, 257, 10, 16, 4), "head dimensions from 1 to 256"),
    "heads no multiple": (P.paged_attention(3, 7, 2, 64, 10, 16, 4), "must be a multiple"),
    "q wider than the cache": (swap(ATT, ("tensor<3x8x64xbf16>", "tensor<3x8x32xbf16>")), "same head dimension"),
    "page table of another batch": (swap(ATT, ("tensor<3x4xi32>", "tensor<4x4xi32>")), "the page table must be"),
    "lengths by head": (swap(ATT, ("tensor<3xi32>", "tensor<3x1xi32>")), "lengths must be"),
    "negative window": (P.paged_attention(3, 8, 2, 64, 10, 16, 4, window=-1), "must not be negative"),
    "lse in bf16": (swap(P.paged_attention(3, 8, 2, 64, 10, 16, 4, lse=True), ("tensor<3x8xf32>", "tensor<3x8xbf16>")), "lse must be f32"),
    "too many alternatives": (P.token_logprobs(4, 100, top=65), "at most 64"),
    "more alternatives than tokens": (P.token_logprobs(4, 3, top=4), "top must lie between"),
    "alternatives not asked for": (swap(LP, ("top = 5", "top = 0")), "three results are expected"),
    "part of an alternative": (swap(LP, ("top = 5 : i64", "top = 4.5 : f64")), "whole number"),
    "indices as i64": (swap(LP, ("tensor<4x5xi32>", "tensor<4x5xi64>")), "must be i32"),
    "empty vocabulary": (P.token_logprobs(4, 0), "need a vocabulary"),
    "targets per logit": (swap(LPG, ("tensor<4xi32>", "tensor<4x1xi32>")), "the targets must be"),
    "gradient of another type": (swap(LPG, ("-> tensor<4x100xbf16>", "-> tensor<4x100xf32>"), (" : tensor<4x100xbf16>\n", " : tensor<4x100xf32>\n")), "differ"),
    "entropy in bf16": (swap(LPG, ("%arg3: tensor<4xf32>", "%arg3: tensor<4xbf16>"), ("tensor<4xi32>, tensor<4xf32>, tensor<4xf32>,", "tensor<4xi32>, tensor<4xf32>, tensor<4xbf16>,")), "entropy must be f32"),
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
def launches(text):
    return [l.split("kind=")[1].split()[0] for l in rx.compile_offline(text).splitlines() if "kind=" in l]


def test_generic_form():
    text = P.token_logprobs(4, 100, top=5)
    line = [l for l in text.splitlines() if "custom_call" in l][0]
    generic = line.replace("stablehlo.custom_call @rx.token_logprobs(%arg0, %arg1) {", '"stablehlo.custom_call"(%arg0, %arg1) <{call_target_name = "rx.token_logprobs", has_side_effect = false, ')
    generic = generic.replace("}} : (", "}}> : (")
    assert launches(text.replace(line, generic)) == launches(text)


def copies(text):
    return [k for k in launches(text) if k.startswith("map")]


def test_caches_are_updated_in_place():
    assert copies(APP) == []                                            # arguments that the results may take over
    plain = swap(APP, (" {tf.aliasing_output = 1 : i32}", ""), (" {tf.aliasing_output = 2 : i32}", ""))
    assert len(copies(plain)) == 2                                      # copied: the arguments stay as they are
    assert len(copies(swap(APP, (" {tf.aliasing_output = 1 : i32}", "")))) == 1
    # an argument that a later kernel reads is copied
    later = swap(APP, ("    return %0#0, %0#1, %0#2 : ", "    %n = stablehlo.add %0#1, %arg8 : tensor<10x16x2x64xbf16>\n    return %n, %0#1, %0#2 : "),
                 ("-> (tensor<3x8x64xbf16>, tensor<10x16x2x64xbf16>, tensor<10x16x2x64xbf16>) {\n", "-> (tensor<10x16x2x64xbf16>, tensor<10x16x2x64xbf16>, tensor<10x16x2x64xbf16>) {\n"),
                 (" : tensor<3x8x64xbf16>, tensor<10x16x2x64xbf16>, tensor<10x16x2x64xbf16>\n", " : tensor<10x16x2x64xbf16>, tensor<10x16x2x64xbf16>, tensor<10x16x2x64xbf16>\n"))
    assert len(copies(later)) == 2                                      # the copy and the sum


def test_nothing_to_do_is_no_launch():
    assert launches(P.token_logprobs(0, 100, top=5)) == [] and launches(P.kv_append(0, 2, 8, 2, 64, 10, 16, 4, 64)) == []
    assert launches(P.embedding(7, 10, 0)) == [] and launches(P.embedding_grad(7, 0, 8)) == []
    assert launches(P.embedding_grad(0, 10, 8)) != []                   # zeros are written


def programs():
    mods = {"embedding": EMB, "embedding_odd": P.embedding(5, 10, 33, dt="f16", ids="i64"), "embedding_grad": GRAD, "append": APP, "attention": ATT, "logprobs": LP,
            "grad_large": P.embedding_grad(16384, 65536, 4096, out="f32"), "grad_i64": P.embedding_grad(3000, 1001, 77, dt="f16", ids="i64"),
            "append_heads": P.kv_append(3, 2, 8, 2, 80, 10, 24, 4, 64, rotary_dim=32, rotation="pairs", layout="heads", dt="f32", ids="i64"),
            "attention_long": P.paged_attention(8, 64, 8, 128, 20000, 64, 2048, layout="heads", lse=True),
            "attention_f32": P.paged_attention(7, 12, 12, 80, 1000, 24, 170, dt="f32", window=100),
            "logprobs_long": P.token_logprobs(4096, 131072, top=20), "logprobs_one": P.token_logprobs(1, 1, top=1, dt="f32"), "logprobs_grad": LPG,
            "decode": P.decode_step(3, 101, 64, 8, 2, 32, 96, 12, 16, 4, 64, layers=2)[0], "train": P.tied_head_step(7, 50, 32, entropy_weight=0.1)}
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
