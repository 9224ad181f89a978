"""GPU tests of the block-scaled e4m3 operators where a call can go wrong
without an argument of it being unusual: two host threads at once, long sums,
rows near the ends of fp32, waits that run out."""

import ctypes
import threading

import numpy as np
import pytest

from tests import block128_ref as ref
from tests.helpers import stream_handle
from tests.test_block128_gpu import (BF16, CODE, F32, FILL, activations, addr, backward_inputs,
                                     check_backward, f64, on_gpu, run_backward, run_norm, up)

pytestmark = pytest.mark.gpu


# -------------------------------------------------------- two host threads


@pytest.mark.parametrize("op", ["norm", "gradient"])
def test_norms_of_different_widths_from_four_threads(cuda, cmb, op):
    """Threads call the norm, or its gradient, at two widths, each on a stream of
    its own: rows of both go through one kernel with different amounts of shared
    memory, and every call has to be taken and give what it gives alone.  (While
    a call set the kernel's limit to its own need, one wide call in 250 was
    refused.)"""
    rows, calls = 1500, 60000
    check = {"norm": cmb.lib.cmb_rmsnorm_e4m3_block128, "gradient": cmb.lib.cmb_rmsnorm_backward}[op]
    jobs = []
    for i in range(4):
        cols = (8192, 1032)[i % 2]
        rng = np.random.default_rng(i)
        x, r = (on_gpu(cuda, rng.normal(size=(rows, cols)), "bf16")[1] for _ in range(2))
        w = on_gpu(cuda, np.ones((1, cols)), "bf16")[1]
        out, rstd = cuda.zeros_like(x), cuda.ones(rows, device="cuda")
        stream = cuda.cuda.Stream()
        s = ctypes.c_void_p(stream.cuda_stream)
        if op == "norm":
            args = (addr(x), cols, None, 0, BF16, addr(w), BF16, ctypes.c_float(1e-5), rows, cols,
                    None, 0, addr(out), cols, None, 0, None, 0, None, s)
        else:
            args = (addr(x), cols, addr(r), cols, None, 0, BF16, addr(w), BF16, addr(rstd), rows,
                    cols, addr(out), cols, None, None, 0, s)
        cuda.cuda.synchronize()
        assert check(*args) == 0
        cuda.cuda.synchronize()
        jobs.append((args, out, out.clone(), stream, (x, r, w, rstd)))
        out.zero_()
    cuda.cuda.synchronize()
    refused, start = [0] * 4, threading.Barrier(4)

    def run(i):
        args, _, _, stream, _ = jobs[i]
        start.wait()
        for k in range(calls):
            refused[i] += check(*args) != 0
            if k % 10 == 9:
                stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    cuda.cuda.synchronize()
    assert refused == [0] * 4
    assert all(cuda.equal(out, alone) for _, out, alone, _, _ in jobs)


# ------------------------------------------------ rows near the ends of fp32


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(3, 300), (5, 8192), (600, 4096), (900, 1031)])
def test_gradient_of_rows_whose_rstd_squared_is_past_fp32(cuda, cmb, rows, cols, kind, residual):
    """Rows of 1e-20 and of 1e15 beside ordinary ones, eps = 0: rstd is 1e20, its
    square is not a number of fp32, and dx (of 1e20 times dy) is."""
    rng = np.random.default_rng(cols)
    size = np.array([1e-20, 1.0, 1e15, 3e-20, 1e-19])[np.arange(rows) % 5][:, None]
    _, dy = on_gpu(cuda, rng.normal(size=(rows, cols)), kind)
    _, h = on_gpu(cuda, rng.normal(size=(rows, cols)) * size, kind)
    dh = on_gpu(cuda, rng.normal(size=(rows, cols)) / size, kind)[1] if residual else None
    _, w = on_gpu(cuda, 1 + 0.1 * rng.normal(size=(1, cols)), "f32")
    rstd = (1 / h.double().square().mean(dim=1).sqrt()).float()
    assert float(rstd.max()) > 2.0 ** 64
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, kind, "f32")
    assert cuda.isfinite(dx).all()
    check_backward(dx, grad, f64(dy), f64(h), f64(dh) if residual else None, f64(w)[0], f64(rstd),
                   kind)
