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
