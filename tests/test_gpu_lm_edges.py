"""Language-model operators where they can go wrong: offsets past 32 bits, masks that leave little or nothing, ties, splits over
many sequences, repeated runs, calls without allocations.  Bounds as in test_gpu_lm_operators.py."""
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


# ----------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------
def uneven(rng, b, longest):
    n = np.round(longest ** rng.random(b)).astype(int)
    n[rng.integers(0, b, size=max(1, b // 10))] = 0
    return n.tolist()


@pytest.mark.parametrize("lengths,hq,hk,d,dv,dt,layout", [
    ([20000], 1, 1, 64, 64, "f32", "slots"), ([20000], 1, 1, 33, 17, "bf16", "heads"), ([30001, 3, 0], 2, 2, 8, 8, "f16", "slots"), ([9000, 9000], 3, 1, 40, 24, "bf16", "slots"),
    ([25000], 5, 5, 16, 7, "f32", "heads"), ([1] * 40 + [12345], 8, 1, 128, 64, "bf16", "heads"),
])
def test_long_sequences_of_few_heads(rx, client, lengths, hq, hk, d, dv, dt, layout):
    """Many parts of few outputs: threads share the parts among them."""
    rng = np.random.default_rng(len(lengths) + d)
    size, b = 16, len(lengths)
    cols, pages = -(-max(lengths) // size) + 1, sum(-(-n // size) for n in lengths) + 2
    args = T.attention_case(rng, lengths, hq, hk, d, dv, pages, size, cols, dt, layout)
    text = P.paged_attention(b, hq, hk, d, pages, size, cols, dt=dt, layout=layout, lse=True, value_dim=dv)
    got, exe = gpu_run(rx, client, text, args)
    ref, lse, mag = L.paged_attention(*(t.a for t in args), layout=layout)
    bound, lse_bound = T.attention_bound(args, d ** -0.5, lse, mag, dt, cols * size)
    T.close(got[0].a, ref, bound, dt)
    T.close(got[1].a, lse, lse_bound)
    again, _ = gpu_run(rx, client, text, args, exe)
    assert all(np.array_equal(x.a, y.a) for x, y in zip(got, again))


@pytest.mark.parametrize("b,longest,hq,hk,d,size,dt,layout,window", [
    (130, 900, 4, 2, 64, 16, "bf16", "slots", 0), (70, 3000, 8, 8, 32, 7, "f16", "heads", 0), (200, 70, 2, 1, 128, 16, "f32", "slots", 0), (65, 2000, 6, 2, 48, 32, "bf16", "heads", 333),
    (9, 6000, 48, 1, 64, 64, "bf16", "slots", 0), (3, 9000, 24, 8, 256, 16, "bf16", "slots", 0),
])
def test_many_uneven_sequences(rx, client, b, longest, hq, hk, d, size, dt, layout, window):
    """Stretches that end inside of sequences, hold several, and start others; the same bits in every run."""
    rng = np.random.default_rng(b)
    lengths = uneven(rng, b, longest)
    cols = -(-max(lengths) // size) + 1
    pages = sum(-(-n // size) for n in lengths) + 2
    args = T.attention_case(rng, lengths, hq, hk, d, d, pages, size, cols, dt, layout)
    text = P.paged_attention(b, hq, hk, d, pages, size, cols, dt=dt, window=window, layout=layout, lse=True)
    got, exe = gpu_run(rx, client, text, args)
    out, lse, mag = L.paged_attention(*[t.a for t in args], window=window, layout=layout)
    bound, lse_bound = T.attention_bound(args, d ** -0.5, lse, mag, dt, max(lengths))
    T.close(got[0].a, out, bound, dt)
    T.close(got[1].a, lse, lse_bound)
    bufs = [rx.Buffer.from_host(client, np.frombuffer(a.to_bytes(), dtype=rx._STORAGE[a.dt]).reshape(a.shape), a.dt) for a in args]
    for _ in range(30):
        again = [r.synced_buffer().to_host() for r in exe.execute_sharded(bufs)]
        assert np.array_equal(I.Tensor.from_bytes(again[0].tobytes(), dt, out.shape).a, got[0].a) and np.array_equal(again[1], got[1].a)


def test_lengths_beyond_the_page_table(rx, client):
    rng = np.random.default_rng(1)
    args = T.attention_case(rng, [64, 30], 4, 2, 64, 64, 10, 16, 4, "f32", "slots")
    long = [*args[:4], I.Tensor(np.array([1000, 30]), "i32")]
    text = P.paged_attention(2, 4, 2, 64, 10, 16, 4, dt="f32")
    assert np.array_equal(gpu_run(rx, client, text, long)[0][0].a, gpu_run(rx, client, text, args)[0][0].a)


def test_cache_of_more_than_2_to_the_31_elements(rx, client):
    """Keys and values appended to the last pages of caches of 2.4e9 elements each, and read back by the attention."""
    hq, hk, d, size, pages, n = 8, 8, 128, 16, 146000, 40
    rng = np.random.default_rng(2)
    q, k, v = (T.rounded(rng.normal(size=(n, h, d)), "bf16") for h in (hq, hk, hk))
    angle = np.zeros((64, 0))
    table = I.Tensor(np.array([[pages - 1, pages - 2, pages - 70000, 5]]), "i32")
    pos = I.Tensor(np.arange(n), "i32")
    append = rx.compile(P.kv_append(n, 1, hq, hk, d, pages, size, 4, 64, rotary_dim=0))
    dev = [rx.to_rarray(t.a.T, t.dt) for t in (q, k, v, I.Tensor(angle, "f32"), I.Tensor(angle, "f32"), pos, I.Tensor(np.zeros(n), "i32"), table)]
    caches = [rx.ConcreteRArray(rx.AsyncBuffer(rx.Buffer.uninitialized(client, (pages, size, hk, d), "bf16")), (d, hk, size, pages), "bf16") for _ in range(2)]
    out = append(*dev, *caches, donated=[False] * 8 + [True, True])
    last = I.Tensor(q.a[-1:], "bf16")
    attend = rx.compile(P.paged_attention(1, hq, hk, d, pages, size, 4, lse=True))
    got = attend(rx.to_rarray(last.a.T, "bf16"), out[1], out[2], dev[7], rx.to_rarray(np.array([n], dtype=np.int32)))
    small = [np.zeros((3, size, hk, d)), np.zeros((3, size, hk, d))]
    for c, new in zip(small, (k.a, v.a)):
        c.reshape(-1, hk, d)[:n] = new
    ref, lse, mag = L.paged_attention(last.a, *small, np.array([[0, 1, 2]]), np.array([n]))
    bound, lse_bound = T.attention_bound([last, I.Tensor(small[0], "bf16")], d ** -0.5, lse, mag, "bf16", n)
    T.close(got[0].to_array().T, ref, bound, "bf16")
    T.close(got[1].to_array().T, lse, lse_bound)


def test_rows_of_a_table_of_more_than_2_to_the_31_elements(rx, client):
    rows, width = 600000, 4096
    rng = np.random.default_rng(3)
    table = rx.Buffer.uninitialized(client, (rows, width), "bf16")
    ids = np.array([rows - 1, 1, 524289, rows, 0])
    values = T.rounded(rng.normal(size=(5, width)), "bf16")
    for i, row in zip(ids, values.a):
        if i < rows:
            table.copy_from_host(rx.encode(row, "bf16"), int(i) * width * 2)
    exe = rx.xla_compile(client, P.embedding(5, rows, width, scale=2.0))
    got = exe.execute_sharded([table, rx.Buffer.from_host(client, ids.astype(np.int32), "i32")])[0].synced_buffer().to_host()
    ref = values.a * 2
    ref[3] = 0
    assert np.array_equal(rx.decode(got, "bf16"), ref)


# ----------------------------------------------------------------------------
# calls without allocations, and in place
# ----------------------------------------------------------------------------
def test_append_and_attend_without_allocations(rx, client):
    """The caller's result buffers receive the updated caches; the arguments stay; counters are left at zero for the next call."""
    rng = np.random.default_rng(4)
    args = T.append_case(rng, 9, 2, 4, 2, 32, 32, 80, 4, 30, 120, 32, "f32", "slots", "i32")
    exe = rx.xla_compile(client, P.kv_append(9, 2, 4, 2, 32, 80, 4, 30, 120, dt="f32"))
    bufs = [rx.Buffer.from_host(client, np.ascontiguousarray(t.a), t.dt) for t in args]
    res = [rx.Buffer.uninitialized(client, t.shape, "f32") for t in (args[0], args[8], args[9])]
    ref = L.kv_append(*[t.a for t in args])
    for _ in range(3):
        exe.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        for r, want in zip(res, ref):
            T.close(r.to_host(), want, 12 * T.UF * 4)
        assert np.array_equal(bufs[8].to_host(), args[8].a)
    att = rx.xla_compile(client, P.paged_attention(2, 4, 2, 32, 80, 4, 30, dt="f32"))
    q = T.rounded(rng.normal(size=(2, 4, 32)), "f32")
    lengths = np.array([120, 77], dtype=np.int32)
    abufs = [rx.Buffer.from_host(client, q.a, "f32"), res[1], res[2], bufs[7], rx.Buffer.from_host(client, lengths, "i32")]
    out = rx.Buffer.uninitialized(client, (2, 4, 32), "f32")
    want = att.execute_sharded(abufs)[0].synced_buffer().to_host()
    for _ in range(3):
        att.execute_no_alloc(abufs, [out])
        client.default_device().synchronize()
        assert np.array_equal(out.to_host(), want)
    o, lse, mag = L.paged_attention(q.a, res[1].to_host(), res[2].to_host(), args[7].a, lengths)
    T.close(want, o, T.attention_bound([q, I.Tensor(res[1].to_host(), "f32")], 32 ** -0.5, lse, mag, "f32", 120)[0])


def test_partial_results_fit_calls_without_allocations(rx, client):
    """Long sequences, and long rows of a table's gradient, whose partial results take more than the library's scratch array in
    the usual plan: calls without allocations share them among fewer workgroups."""
    rng = np.random.default_rng(8)
    lengths, hq, hk, d, size, cols = [8100, 5000, 7777, 3], 16, 2, 128, 16, 512
    args = T.attention_case(rng, lengths, hq, hk, d, d, 1400, size, cols, "bf16", "slots")
    exe = rx.xla_compile(client, P.paged_attention(4, hq, hk, d, 1400, size, cols, lse=True))
    bufs = [rx.Buffer.from_host(client, np.ascontiguousarray(rx.encode(t.a, "bf16") if t.dt == "bf16" else t.a), t.dt) for t in args]
    ref, lse, mag = L.paged_attention(*(t.a for t in args))
    bound, lse_bound = T.attention_bound(args, d ** -0.5, lse, mag, "bf16", cols * size)
    res = [rx.Buffer.uninitialized(client, (4, hq, d), "bf16"), rx.Buffer.uninitialized(client, (4, hq), "f32")]
    for _ in range(2):
        exe.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        T.close(rx.decode(res[0].to_host(), "bf16"), ref, bound, "bf16")
        T.close(res[1].to_host(), lse, lse_bound)
    tokens, rows, width = 1100, 5, 32768
    dy = rng.integers(-100, 100, size=(tokens, width)).astype(np.float32)          # sums that no order rounds
    ids = rng.integers(0, rows, size=tokens).astype(np.int32)
    exe = rx.xla_compile(client, P.embedding_grad(tokens, rows, width, dt="f32"))
    bufs, want = [rx.Buffer.from_host(client, dy, "f32"), rx.Buffer.from_host(client, ids, "i32")], L.embedding_grad(dy, ids, rows)
    res = [rx.Buffer.uninitialized(client, (rows, width), "f32")]
    for _ in range(2):
        exe.execute_no_alloc(bufs, res)
        client.default_device().synchronize()
        assert np.array_equal(res[0].to_host(), want)
    assert np.array_equal(exe.execute_sharded(bufs)[0].synced_buffer().to_host(), want)


@pytest.mark.parametrize("tokens", [512, 513, 768, 769])
@pytest.mark.parametrize("rows", [40, 4095, 4096])
def test_gradients_on_both_sides_of_the_sorted_list(rx, client, tokens, rows):
    rng = np.random.default_rng(tokens + rows)
    dy = rng.integers(-1000, 1000, size=(tokens, 72)).astype(np.float64)           # sums that no order rounds
    ids = np.minimum((rows ** rng.random(tokens)).astype(np.int64) - 1, rows - 1)
    got, _ = gpu_run(rx, client, P.embedding_grad(tokens, rows, 72, dt="f32"), [I.Tensor(dy, "f32"), I.Tensor(ids, "i32")])
    assert np.array_equal(got[0].a, L.embedding_grad(dy, ids, rows))


def test_append_to_an_array_returned_twice(rx, client):
    """Two results of one buffer: appending to the donated one leaves the other alone."""
    rng = np.random.default_rng(5)
    args = T.append_case(rng, 3, 1, 2, 1, 8, 8, 4, 4, 2, 8, 8, "f32", "slots", "i32")
    shape = "tensor<4x4x1x8xf32>"
    twice = rx.compile("module { func.func @main(%%a: %s) -> (%s, %s) { %%0 = stablehlo.negate %%a : %s\n return %%0, %%0 : %s, %s } }" % ((shape,) * 6))
    x, y = twice(rx.to_rarray(args[8].a.T, "f32"))
    thunk = rx.compile(P.kv_append(3, 1, 2, 1, 8, 4, 4, 2, 8, dt="f32"))
    dev = [rx.to_rarray(t.a.T, t.dt) for t in args]
    thunk(*dev[:8], x, dev[9], donated=[False] * 8 + [True, True])
    assert np.array_equal(y.to_array().T, -args[8].a)


def test_profiled_appends(rx, client):
    rng = np.random.default_rng(6)
    args = T.append_case(rng, 3, 1, 2, 1, 8, 8, 4, 4, 2, 8, 8, "f32", "slots", "i32")
    exe = rx.xla_compile(client, P.kv_append(3, 1, 2, 1, 8, 4, 4, 2, 8, dt="f32"))
    bufs = [rx.Buffer.from_host(client, np.ascontiguousarray(t.a), t.dt) for t in args]
    out, ms = exe.execute_timed(bufs)
    assert len(ms) == 1 and np.array_equal(bufs[8].to_host(), args[8].a)
    T.close(out[1].to_host(), L.kv_append(*[t.a for t in args])[1], 12 * T.UF * 4)


# ----------------------------------------------------------------------------
# log probabilities
# ----------------------------------------------------------------------------
def check_logprobs(rx, client, x, y, top, dt):
    n, v = x.shape
    got, _ = gpu_run(rx, client, P.token_logprobs(n, v, top=top, dt=dt), [x, I.Tensor(y, "i32")])
    ref = L.token_logprobs(x.a, y, top)
    e = (v / 64 + 64 + 44) * T.UF
    size = np.where(np.isfinite(ref[1]), np.abs(ref[1]), 0) * T.UF
    T.close(got[1].a, ref[1], e + 2 * size)
    T.close(got[0].a, ref[0], e + 3 * size)
    T.close(got[2].a, ref[2], 2 * e * (1 + np.abs(ref[2])) + 4 * size)
    assert np.array_equal(got[4].a, ref[4])
    T.close(got[3].a, ref[3], (e + 3 * size)[:, None])


@pytest.mark.parametrize("n", [3, 700])
@pytest.mark.parametrize("dt,low", [("f32", -np.inf), ("bf16", -np.inf), ("f32", np.finfo(np.float32).min), ("bf16", -3.3895313892515355e38), ("f16", -65504.0)])
def test_masks_that_leave_a_few_tokens(rx, client, n, dt, low):
    """Fewer tokens left than alternatives are asked for; masks of -inf and of a type's lowest value; rows split and whole."""
    v = 30011
    rng = np.random.default_rng(7)
    x = np.full((n, v), low)
    for t in range(n):
        left = rng.permutation(v)[:t % 7]
        x[t, left] = rng.normal(size=left.size)
    y = np.argmax(x, 1)
    check_logprobs(rx, client, T.rounded(x, dt), y, 20, dt)


@pytest.mark.parametrize("n", [2, 600])
def test_many_equal_maxima(rx, client, n):
    """More equal elements than any buffer holds, at the row's end, scattered, and in one thread's places; the lowest indices win."""
    v = 40000
    rng = np.random.default_rng(8)
    x = rng.normal(size=(n, v)).clip(-4, 4)
    x[0, v - 3000:] = 9.0
    x[1, rng.permutation(v)[:5000]] = 9.0
    if n > 2:
        x[2, 8::8192] = 7.0
        x[3, :] = -2.0
        x[4, ::2] = 5.0
        x[5, 4096:] = 6.0
        x[5, :30] = np.arange(30) * 0.125 + 6.5
    check_logprobs(rx, client, T.rounded(x, "bf16"), rng.integers(0, v, n), 33, "bf16")


def test_repeated_runs_give_the_same_bits(rx, client):
    rng = np.random.default_rng(9)
    x, y = T.logits_case(rng, 5, 120000, "bf16")
    exe = rx.xla_compile(client, P.token_logprobs(5, 120000, top=20))
    bufs = [rx.Buffer.from_host(client, np.frombuffer(x.to_bytes(), dtype=np.uint16).reshape(x.shape), "bf16"), rx.Buffer.from_host(client, y.astype(np.int32), "i32")]
    first = [r.synced_buffer().to_host() for r in exe.execute_sharded(bufs)]
    for _ in range(30):
        for a, b in zip(first, exe.execute_sharded(bufs)):
            assert np.array_equal(a.view(np.int32), b.synced_buffer().to_host().view(np.int32))
