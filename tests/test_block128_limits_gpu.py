"""GPU tests of the block-scaled e4m3 operators where a call can go wrong
without an argument of it being unusual: two host threads at once, long sums,
rows near the ends of fp32, waits that run out."""

import ctypes
import glob
import os
import subprocess
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


# ------------------------------------------------------------- long sums


def long_operand(cuda, rows, k, block, seed, signed):
    """Random finite codes made on the GPU, with scales of 1/4 .. 4; NaN codes and
    scales behind each row."""
    gen = cuda.Generator(device="cuda").manual_seed(seed)
    pitch, groups = up(k, 16), up(k, 128) // 128
    q = cuda.randint(0, 127, (rows, pitch), dtype=cuda.uint8, device="cuda", generator=gen)
    if signed:
        q |= cuda.randint(0, 2, (rows, pitch), dtype=cuda.uint8, device="cuda", generator=gen) << 7
    q[:, k:] = 0x7F
    s = cuda.full((-(-rows // block), groups + 3), 255, dtype=cuda.uint8, device="cuda")
    s[:, :groups] = cuda.randint(125, 130, (s.shape[0], groups), dtype=cuda.uint8, device="cuda",
                                 generator=gen)
    return q, s


def long_values(q, s, rows, k, block):
    """What those rows stand for, in 64 bits."""
    groups = up(k, 128) // 128
    codes = q[rows][:, :k].cpu().numpy()
    scales = s[rows // block][:, :groups].cpu().numpy()
    return ref.VALUES[codes] * ref.spread(scales, len(rows), k, 1)


def long_product(cuda, cmb, m, n, k, block_b, out, signed):
    """Of the product the rows and columns that are compared (the ends and a few), the
    same in 64 bits, the same of magnitudes; and all of it as it is."""
    a, b = long_operand(cuda, m, k, 1, 1, signed), long_operand(cuda, n, k, block_b, 2, signed)
    c = cuda.full((m, n), float("nan"), dtype=cuda.bfloat16 if out == "bf16" else cuda.float32,
                  device="cuda")
    status = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    cmb.check("cmb_gemm_e4m3_block128", addr(a[0]), a[0].shape[1], addr(a[1]), a[1].shape[1],
              addr(b[0]), b[0].shape[1], addr(b[1]), b[1].shape[1], block_b, addr(c), n, CODE[out],
              m, n, k, addr(status), stream_handle(cuda))
    assert int(status.item()) == 0 and bool(cuda.isfinite(c).all())
    rng = np.random.default_rng(k)
    pick = lambda size, some: np.unique(np.concatenate([[0, size - 1], rng.integers(0, size, some)]))
    rows, cols = pick(m, 24), pick(n, 40)
    got = f64(c[cuda.from_numpy(rows).cuda()][:, cuda.from_numpy(cols).cuda()])
    x = long_values(*a, rows, k, 1)
    y = long_values(*b, cols, k, block_b)
    return got, x @ y.T, np.abs(x) @ np.abs(y).T, c


# few tokens and many, one CTA a tile and up to eight, whole and odd sizes
LONG = [(128, 18944, 16384), (160, 8192, 28672), (128, 9472, 53248), (2048, 2048, 131072),
        (512, 1000, 100003), (97, 700, 70001), (3, 1030, 2 ** 21 - 77), (16, 256, 2 ** 21),
        (300, 5000, 30000)]


@pytest.mark.parametrize("m,n,k", LONG)
@pytest.mark.parametrize("signed", [False, True])
def test_gemm_fp32_sums_of_any_length(cuda, cmb, m, n, k, signed):
    """An fp32 C adds accumulators of 2048 of K.  An accumulator's 64 MMAs are off
    by at most 4 u32 of the sum so far each, as in gemm_bound; then come the
    ceil(K / 2048) parts, and at most 8 of a cluster, with a rounding each."""
    got, want, mags, _ = long_product(cuda, cmb, m, n, k, 128, "f32", signed)
    parts = -(-k // 2048) + 8
    err = np.abs(got - want)
    assert (err <= (4 * 64 + parts + 1) * ref.U32 * mags).all()
    if not signed:
        # the sums so far of terms that are positive and alike average half the
        # last one, in an accumulator and over the parts
        room = (4 * 64 + parts + 1) / 2 * ref.U32 * np.linalg.norm(want)
        assert np.linalg.norm(err) <= room, np.linalg.norm(err) / np.linalg.norm(want) / ref.U32


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 131072), (128, 9472, 100003), (3000, 3000, 40000),
                                   (16, 256, 2 ** 22), (5, 8192, 2 ** 18), (300, 600, 32768)])
@pytest.mark.parametrize("signed", [False, True])
def test_gemm_bf16_sums_of_any_length(cuda, cmb, m, n, k, signed):
    """A bf16 C is off by its own rounding and little else: it adds accumulators of at
    most 32768 of K, each off by at most 4 u32 of the sum so far for each 32, and at
    most 8 of a cluster."""
    got, want, mags, _ = long_product(cuda, cmb, m, n, k, 128, "bf16", signed)
    steps = 4 * 1024 + -(-k // 32768) + 8
    room = steps * ref.U32 * mags + ref.U16 * np.abs(want) * (1 + 1e-3)
    assert (np.abs(got - want) <= room).all()


@pytest.mark.parametrize("m,n,k", [(1024, 1024, 2 ** 19), (2000, 2100, 300001), (128, 4800, 2 ** 19),
                                   (16, 4096, 2 ** 20), (48, 8000, 2 ** 19 - 77)])
def test_gemm_bf16_sums_do_not_drift(cuda, cmb, m, n, k):
    """Positive terms and K past 8 x 32768, so that every CTA of a cluster has more
    than one accumulator of a bf16 C.  Against the fp32 C of the same operands the
    mean difference is that of the sums, (4096 + parts) / 2 and (256 + parts) / 2 u32
    of C by the same count as in the fp32 test, and what is left of the roundings to
    bf16: each is uniform within half a step, at most 2^-8 of C, a third of its
    square on average, and six deviations of the mean of all of them are allowed
    for."""
    sums = {}
    for out in ("bf16", "f32"):
        sums[out] = long_product(cuda, cmb, m, n, k, 128, out, False)[3].double()
    drift = float((sums["bf16"] / sums["f32"] - 1).mean())
    room = (4 * 1024 + 4 * 64 + -(-k // 32768) + -(-k // 2048) + 16) / 2 * ref.U32
    room += 6 * ref.U16 / np.sqrt(3 * m * n)
    assert abs(drift) <= room, (drift / ref.U32, room / ref.U32)


# --------------------------------------------------- a wait that runs out


class Lost:
    """The norms of tests/lost_copy.cu, called as the library's."""

    def __init__(self, lib, signatures):
        self.lib = lib
        for name in ("cmb_rmsnorm_e4m3_block128", "cmb_rmsnorm_backward",
                     "cmb_rmsnorm_backward_workspace_bytes"):
            f = getattr(lib, name)
            f.restype, f.argtypes = signatures[name]

    def check(self, name, *args):
        assert getattr(self.lib, name)(*args) == 0

    def lose(self, address):
        assert self.lib.lose_row(ctypes.c_uint64(address)) == 0


@pytest.fixture(scope="module")
def lost(cuda, cmb, tmp_path_factory):
    from cuda_micro_bench_b200 import capi

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    home = os.path.join(root, "cuda_micro_bench_b200")
    out = str(tmp_path_factory.mktemp("lost") / "liblost.so")
    objects = [o for o in glob.glob(home + "/_obj/**/*.o", recursive=True)
               if os.path.basename(o) != "rmsnorm.cu.o"]
    subprocess.run(["/usr/local/cuda/bin/nvcc", "-O3", "-std=c++17", "-gencode",
                    "arch=compute_100a,code=sm_100a", "-Xcompiler", "-fPIC", "-shared", "-Xlinker",
                    "-Bsymbolic", "-I", home + "/csrc", "-I", root + "/include",
                    os.path.join(root, "tests", "lost_copy.cu"), *objects, "-lpthread", "-ldl",
                    "-o", out], check=True, timeout=600)
    return Lost(ctypes.CDLL(out), capi.SIGNATURES)


@pytest.mark.parametrize("rows,cols,row", [(1500, 8192, 777), (1500, 8192, 0), (1500, 1032, 1499)])
def test_norm_whose_wait_runs_out(cuda, cmb, lost, rows, cols, row):
    """A row's copy never comes (a wait ends after 2 s): the row and what its CTA
    has left hold NaN in every output, all other rows are right, and the next
    call works."""
    rng = np.random.default_rng(rows)
    x, r = (on_gpu(cuda, rng.normal(size=(rows, cols)), "bf16")[1] for _ in range(2))
    w = on_gpu(cuda, np.ones((1, cols)), "bf16")[1]
    call = lambda: run_norm(cuda, lost, x, r, w, "bf16", "bf16", 1e-5)
    want = run_norm(cuda, cmb, x, r, w, "bf16", "bf16", 1e-5)
    lost.lose(r.data_ptr() + 2 * cols * row)
    got = call()
    lost.lose(0)
    again = call()
    spoilt = cuda.isnan(got["rstd"])
    assert bool(spoilt[row]) and int(spoilt[:row].sum()) <= 1  # rows are taken in order, two at a time
    assert int(spoilt.sum()) <= 64  # of one CTA
    for name in ("h", "y"):
        assert cuda.isnan(got[name][spoilt]).all()
    assert (got["q"][spoilt] == 0x7F).all() and (got["s"][spoilt] == 255).all()
    for name in ("h", "y", "q", "s", "rstd"):
        assert cuda.equal(got[name][~spoilt], want[name][~spoilt]), name
        assert cuda.equal(again[name], want[name]), name


@pytest.mark.parametrize("rows,cols,row", [(1500, 8192, 777), (1500, 8192, 0), (1500, 1032, 1499)])
def test_gradient_whose_wait_runs_out(cuda, cmb, lost, rows, cols, row):
    rng = np.random.default_rng(rows)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, rows, cols, "bf16", "bf16")
    call = lambda c: run_backward(cuda, c, dy, h, dh, w, rstd, "bf16", "bf16")
    want = call(cmb)
    lost.lose(h.data_ptr() + 2 * cols * row)
    dx, grad = call(lost)
    lost.lose(0)
    again = call(lost)
    spoilt = cuda.isnan(dx).any(dim=1)
    assert bool(spoilt[row]) and int(spoilt[:row].sum()) <= 1 and int(spoilt.sum()) <= 64
    assert cuda.isnan(dx[spoilt]).all() and cuda.isnan(grad).all()
    assert cuda.equal(dx[~spoilt], want[0][~spoilt])
    assert cuda.equal(again[0], want[0]) and cuda.equal(again[1], want[1])


# ------------------------------------------------------- the largest extents

MOST = 2 ** 31 - 2 ** 16  # rows or columns that a call takes


@pytest.fixture
def space(cuda):
    cuda.cuda.empty_cache()
    if cuda.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    yield
    cuda.cuda.empty_cache()


@pytest.mark.parametrize("side", ["m", "n"])
@pytest.mark.parametrize("k", [1, 16])
def test_gemm_of_the_largest_extent(cuda, cmb, space, side, k):
    """As many rows of one operand as a call takes, one of the other: 2 in the first,
    the last and one between, 1 elsewhere, under scales of 1."""
    long = cuda.full((MOST, 16), 0x38, dtype=cuda.uint8, device="cuda")  # 1.0
    for row in (0, 2 ** 30 + 7, MOST - 1):
        long[row] = 0x40  # 2.0
    scales = cuda.full((MOST,), 127, dtype=cuda.uint8, device="cuda")
    one, s1 = long[1:2].clone(), scales[:1].clone()
    c = cuda.full((MOST,), 7.0, dtype=cuda.bfloat16, device="cuda")
    status = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    m, n = (MOST, 1) if side == "m" else (1, MOST)
    a, sa, b, sb = (long, scales, one, s1) if side == "m" else (one, s1, long, scales)
    cmb.check("cmb_gemm_e4m3_block128", addr(a), 16, addr(sa), 1, addr(b), 16, addr(sb), 1, 1,
              addr(c), n, BF16, m, n, k, addr(status), stream_handle(cuda))
    assert int(status.item()) == 0
    for row in (0, 2 ** 30 + 7, MOST - 1):
        assert float(c[row]) == 2.0 * k
        c[row] = 1.0 * k
    assert float(c.min()) == float(c.max()) == k


def test_norm_and_gradient_of_the_largest_extent(cuda, cmb, space):
    """Rows of one value: y = sign(x) but for eps, whose share is exact here, and a
    gradient that nothing but dh reaches."""
    x = cuda.full((MOST,), 3.0, dtype=cuda.bfloat16, device="cuda")
    x[0] = x[2 ** 30 + 7] = x[-1] = -3.0
    w = cuda.ones(1, dtype=cuda.bfloat16, device="cuda")
    y = cuda.full((MOST,), 7.0, dtype=cuda.bfloat16, device="cuda")
    cmb.check("cmb_rmsnorm_e4m3_block128", addr(x), 1, None, 0, BF16, addr(w), BF16,
              ctypes.c_float(0.0), MOST, 1, None, 0, addr(y), 1, None, 0, None, 0, None,
              stream_handle(cuda))
    for row in (0, 2 ** 30 + 7, MOST - 1):
        assert float(y[row]) == -1.0
        y[row] = 1.0
    assert float(y.min()) == float(y.max()) == 1.0
    # rstd of 1/2 and h of 2: dx = (dy - 2 (1/4) (2 dy)) / 2 = 0, and with dh = dy it is dy
    x.fill_(2.0)
    y[0] = y[2 ** 30 + 7] = y[-1] = 5.0
    rstd = cuda.full((MOST,), 0.5, device="cuda")
    dx = cuda.full((MOST,), 7.0, dtype=cuda.bfloat16, device="cuda")
    cmb.check("cmb_rmsnorm_backward", addr(y), 1, addr(x), 1, addr(y), 1, BF16, addr(w), BF16,
              addr(rstd), MOST, 1, addr(dx), 1, None, None, 0, stream_handle(cuda))
    assert cuda.equal(dx, y)


@pytest.mark.parametrize("rows,cols,block", [(MOST, 1, 1), (1, MOST, 1), (MOST, 1, 128)])
def test_quantize_of_the_largest_extent(cuda, cmb, space, rows, cols, block):
    x = cuda.full((MOST,), 3.0, dtype=cuda.bfloat16, device="cuda")
    x[-1] = 6.0
    q = cuda.full((MOST,), FILL, dtype=cuda.uint8, device="cuda")
    high, wide = -(-rows // block), -(-cols // 128)
    s = cuda.full((high, wide), FILL, dtype=cuda.uint8, device="cuda")
    cmb.check("cmb_quantize_e4m3_block128", addr(x), BF16, rows, cols, cols, block, addr(q), cols,
              addr(s), wide, None, 0, None, 0, stream_handle(cuda))
    wq, ws = ref.quantize(np.array([[3.0]]), 1)
    lq, ls = ref.quantize(np.array([[6.0]]), 1)  # the last block: 6 is its largest
    assert int(s.view(-1)[-1]) == ls[0, 0] and int(q[-1]) == lq[0, 0]
    if high * wide > 1:
        rest = s.view(-1)[:-1]
        assert int(rest.min()) == int(rest.max()) == ws[0, 0]
    head = q[:MOST - 128]
    assert int(head.min()) == int(head.max()) == wq[0, 0]


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n", [(1, 5), (33, 3)])
def test_gemm_of_the_longest_k(cuda, cmb, space, m, n, out):
    """K = 2^28 ones: every sum on the way is a whole number under 2^24 or a multiple
    of 2048 up to 2^28, so C is 2^28 exactly."""
    k = 2 ** 28
    a, b = (cuda.full((rows, k), 0x38, dtype=cuda.uint8, device="cuda") for rows in (m, n))
    sa, sb = (cuda.full((rows, k // 128), 127, dtype=cuda.uint8, device="cuda") for rows in (m, n))
    c = cuda.full((m, n), 7.0, dtype=cuda.bfloat16 if out == "bf16" else cuda.float32, device="cuda")
    status = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    cmb.check("cmb_gemm_e4m3_block128", addr(a), k, addr(sa), k // 128, addr(b), k, addr(sb),
              k // 128, 1, addr(c), n, CODE[out], m, n, k, addr(status), stream_handle(cuda))
    assert int(status.item()) == 0 and bool((c == float(k)).all())
