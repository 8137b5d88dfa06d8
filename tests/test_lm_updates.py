"""Modules that update a cache and do other things with it, without a device: which buffers their plans update in place, and in
which order their launches run."""
import importlib
import os
import subprocess

import pytest

from _loader import load_pkg, ROOT

rx = load_pkg()
P = importlib.import_module("reactant_jl_amd.lm_programs")
HOSTCHECK = os.path.join(ROOT, "reactant.jl_amd", "csrc", "build", "rx_hostcheck_asan")

T, B, HQ, HK, D, PAGES, SIZE, COLS, POSITIONS = 3, 2, 4, 2, 32, 10, 4, 4, 16
CACHE = [PAGES, SIZE, HK, D]


def appends(text, q, k, v, cos, sin, position, sequence, pages, kc, vc, dt="f32"):
    return text.operator("rx.kv_append", [q, k, v, cos, sin, position, sequence, pages, kc, vc],
                         [([T, HQ, D], dt), (CACHE, dt), (CACHE, dt)], {"rotation": "halves", "layout": "slots"})


def arguments(text, aliases=(None, None), dt="f32", times=1):
    """The arguments of `times` appends (position apart) to one pair of caches: ([(q, k, v, cos, sin, position, sequence, pages)], k_cache, v_cache)."""
    first = [text.arg(s, t) for s, t in (([T, HQ, D], dt), ([T, HK, D], dt), ([T, HK, D], dt), ([POSITIONS, D // 2], "f32"), ([POSITIONS, D // 2], "f32"),
                                         ([T], "i32"), ([T], "i32"), ([B, COLS], "i32"))]
    more = [first[:5] + [text.arg([T], "i32")] + first[6:] for _ in range(times - 1)]
    kc, vc = (text.arg(CACHE, dt, a) for a in aliases)
    return [first] + more, kc, vc


def two_appends(dt="f32"):
    """(q, k, v, cos, sin, position, sequence, pages, second position, k_cache, v_cache) -> (q', k_cache', v_cache'), both appends' tokens in the caches."""
    x = P._Text()
    (a, b), kc, vc = arguments(x, (1, 2), dt, times=2)
    _, k1, v1 = appends(x, *a, kc, vc, dt=dt)
    return x.module("two_appends", appends(x, *b, k1, v1, dt=dt))


def append_to_computed(dt="f32"):
    """(.., k_cache, v_cache) -> (q', k_cache', v_cache') of the caches' negatives, appended to; and the keys' copy is a temporary of the module in the second."""
    x = P._Text()
    (a,), kc, vc = arguments(x, (None, None), dt)
    minus = [x.op("negate %s : (%s)" % (c, x.types[c]), CACHE, dt) for c in (kc, vc)]
    return x.module("append_to_computed", appends(x, *a, *minus, dt=dt))


def append_to_computed_inside(dt="f32"):
    """The appended caches are no results: their sum with the argument is."""
    x = P._Text()
    (a,), kc, vc = arguments(x, (None, None), dt)
    minus = [x.op("negate %s : (%s)" % (c, x.types[c]), CACHE, dt) for c in (kc, vc)]
    q, k1, v1 = appends(x, *a, *minus, dt=dt)
    return x.module("append_inside", [q, x.binary("add", k1, kc), x.binary("multiply", v1, v1)])


def appends_in_a_loop(times=3):
    """A `while` of `times` appends of the same tokens, each one position further, to caches that the results may take over."""
    q, kv, ang, one, table, cache = (P.tt(s, t) for s, t in (([T, HQ, D], "f32"), ([T, HK, D], "f32"), ([POSITIONS, D // 2], "f32"), ([T], "i32"), ([B, COLS], "i32"), (CACHE, "f32")))
    types = [q, kv, kv, ang, ang, one, one, table]
    params = ", ".join("%%arg%d: %s" % k for k in enumerate(types)) + ", %%arg8: %s {tf.aliasing_output = 0 : i32}, %%arg9: %s {tf.aliasing_output = 1 : i32}" % (cache, cache)
    call = P.custom_call("rx.kv_append", ["%arg0", "%arg1", "%arg2", "%arg3", "%arg4", "%p", "%arg6", "%arg7", "%k", "%v"], types + [cache, cache], [q, cache, cache],
                         {"rotation": "halves", "layout": "slots"}, "%n")
    return ("module @reactant_appends_in_a_loop {\n  func.func @main(%s) -> (%s, %s) {\n" % (params, cache, cache)
            + "    %zero = stablehlo.constant dense<0> : tensor<i32>\n    %one = stablehlo.constant dense<1> : tensor<i32>\n"
            + "    %%ones = stablehlo.constant dense<1> : %s\n    %%end = stablehlo.constant dense<%d> : tensor<i32>\n" % (one, times)
            + "    %%w:4 = stablehlo.while(%%i = %%zero, %%p = %%arg5, %%k = %%arg8, %%v = %%arg9) : tensor<i32>, %s, %s, %s\n" % (one, cache, cache)
            + "    cond {\n      %c = stablehlo.compare LT, %i, %end : (tensor<i32>, tensor<i32>) -> tensor<i1>\n      stablehlo.return %c : tensor<i1>\n    } do {\n"
            + call + "    %%p1 = stablehlo.add %%p, %%ones : %s\n    %%i1 = stablehlo.add %%i, %%one : tensor<i32>\n" % one
            + "      stablehlo.return %%i1, %%p1, %%n#1, %%n#2 : tensor<i32>, %s, %s, %s\n    }\n" % (one, cache, cache)
            + "    return %%w#2, %%w#3 : %s, %s\n  }\n}\n" % (cache, cache))


def reduce_then_append(reader="sqrt", dt="f32"):
    """(.., k_cache, v_cache) -> (q', k_cache', v_cache', sqrt of the sum of the keys' squares as they were): the reduction ends in its reader, which stands after the append."""
    x = P._Text()
    (a,), kc, vc = arguments(x, (1, 2), dt)
    total = x.op("reduce(%s init: %s) applies stablehlo.add across dimensions = [0, 1, 2, 3] : (%s, tensor<%s>)"
                 % (x.binary("multiply", kc, kc), x.constant("0.000000e+00", [], dt), x.types[kc], dt), [], dt)
    new = appends(x, *a, kc, vc, dt=dt)
    return x.module("reduce_then_append", new + [x.op("%s %s : (tensor<%s>)" % (reader, total, dt), [], dt)])


def reduce_then_update(dt="f32"):
    """The same with a range of a product: (a, b, u) -> (a b with u in its middle, the square root of the sum of the squares of a b)."""
    x = P._Text()
    a, b, u = x.arg([64, 32], dt), x.arg([32, 32], dt), x.arg([8, 32], dt)
    m = x.dot(a, b, (1, 0))
    total = x.op("reduce(%s init: %s) applies stablehlo.add across dimensions = [0, 1] : (%s, tensor<%s>)"
                 % (x.binary("multiply", m, m), x.constant("0.000000e+00", [], dt), x.types[m], dt), [], dt)
    at, zero = x.constant("16", [], "i32"), x.constant("0", [], "i32")
    new = x.op("dynamic_update_slice %s, %s, %s, %s : (%s, %s, tensor<i32>, tensor<i32>)" % (m, u, at, zero, x.types[m], x.types[u]), [64, 32], dt)
    return x.module("reduce_then_update", [new, x.op("sqrt %s : (tensor<%s>)" % (total, dt), [], dt)])


def report(text):
    lines = rx.compile_offline(text).splitlines()
    return [l.split("kind=")[1].split()[0] for l in lines if "kind=" in l], sorted(int(l.split("argument ")[1]) for l in lines if l.startswith("updated in place"))


def test_arguments_that_results_may_take_over_are_updated_in_place():
    kinds, updated = report(P.kv_append(T, B, HQ, HK, D, PAGES, SIZE, COLS, POSITIONS, dt="f32"))
    assert kinds == ["lm_kv_append"] and updated == [8, 9]


TEMPORARIES = {"two appends": two_appends(), "computed caches": append_to_computed(), "computed caches, no results": append_to_computed_inside(), "a loop of appends": appends_in_a_loop()}


@pytest.mark.parametrize("name", sorted(TEMPORARIES))
def test_a_temporary_is_no_argument_to_copy(name):
    """A temporary that an append updates has no contents of a caller's to save."""
    kinds, updated = report(TEMPORARIES[name])
    assert "lm_kv_append" in kinds and updated == []


def test_a_reduction_that_ends_in_a_later_kernel_reads_the_cache_as_it_was():
    """It runs where its reader does: an append before that place is to a copy."""
    kinds, updated = report(reduce_then_append())
    assert 9 in updated
    assert 8 not in updated or min(i for i, k in enumerate(kinds) if k.startswith("reduce")) < kinds.index("lm_kv_append")


def test_so_it_does_where_a_range_is_updated():
    """In the product's own memory (kind map_in_place: the range alone is written) only after the reduction has read it."""
    kinds, _ = report(reduce_then_update())
    assert "map_in_place" not in kinds or min(i for i, k in enumerate(kinds) if k.startswith("reduce")) < kinds.index("map_in_place")


@pytest.mark.parametrize("text", [P.embedding(3, 4, 8, scale=1e39), P.embedding_grad(3, 4, 8, scale=-4e38), P.paged_attention(2, 4, 2, 32, 10, 4, 4, scale=3e38)])
def test_a_factor_beyond_f32_is_refused(text):
    """It would be infinite in the kernel, and an infinity times zero no number."""
    with pytest.raises(rx.ReactantInternalError, match="number that f32 holds"):
        rx.compile_offline(text)
    rx.compile_offline(text.replace("e+38 :", "e+37 :"))


def test_host_code_under_sanitizers(tmp_path):
    if not os.path.exists(HOSTCHECK):
        pytest.skip("the sanitizer program is not built")
    files = []
    for k, text in enumerate([*TEMPORARIES.values(), reduce_then_append(), reduce_then_update()]):
        files.append(tmp_path / ("updates%d.mlir" % k))
        files[-1].write_text(text)
    r = subprocess.run([HOSTCHECK] + [str(f) for f in files], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
