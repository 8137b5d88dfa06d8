"""Errors of executions that show after their call, on the GPU."""
import importlib

import numpy as np
import pytest

from _loader import load_pkg

load_pkg()
NN = importlib.import_module("reactant_jl_amd.nn_programs")
pytestmark = pytest.mark.gpu


def test_an_expired_wait_is_raised_by_the_call_that_takes_the_result(rx, monkeypatch):
    """The bound of the one-launch scan's waits is forced to zero polls from the host (every kernel still runs to its end): the call
    that is given the scan's result raises, and does not use it; the repeated scan has no such waits."""
    client = rx.Client()
    n = 1 << 24
    x = np.random.default_rng(3).normal(size=n).astype(np.float32)
    monkeypatch.setenv("RX_SCAN_SPIN_LIMIT", "0")
    scan = rx.compile(NN.cumulative([n], "f32", 0, "add", False), client)
    minus = rx.compile("module { func.func @main(%%a: %s {tf.aliasing_output = 0 : i32}) -> %s { %%0 = stablehlo.negate %%a : %s\n return %%0 : %s } }" % (("tensor<%dxf32>" % n,) * 4), client)
    assert scan.exec.waits and not minus.exec.waits
    arg = rx.to_rarray(x, client=client)
    with pytest.raises(rx.ReactantInternalError, match="bounded wait for another workgroup"):
        for _ in range(3):       # a run in which every slot happens to be there in time is possible, three in a row are not
            y = scan(arg)
            minus(y, donated=[True])
    assert not y.donated
    out = minus(scan(arg)).to_array()
    ref = -np.cumsum(x.astype(np.float64))
    assert np.all(np.abs(out - ref) <= 1e-5 * np.sqrt(n) * np.abs(ref).max())
