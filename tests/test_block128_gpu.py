"""GPU parity of the block-scaled e4m3 operators against plain 64-bit
implementations (tests/block128_ref.py), at the sizes, strides and values
where they can go wrong.  Quantisation is bit-exact; the products and norms
are held to bounds derived from the roundings they make."""

import ctypes

import numpy as np
import pytest

from tests import block128_ref as ref
from tests.helpers import dptr, stream_handle

pytestmark = pytest.mark.gpu

BF16, F32 = 0, 1
CODE = {"bf16": BF16, "f32": F32}
FILL = 0xA5  # what the bytes no call may write hold


def up(n, to):
    return -(-n // to) * to


def torch_type(cuda, kind):
    return cuda.bfloat16 if kind == "bf16" else cuda.float32


def on_gpu(cuda, x, kind, pitch=None, offset=0):
    """A float64 array rounded to `kind` on the GPU, with `pitch` elements from
    row to row and `offset` elements before the first; (buffer, view)."""
    rows, cols = x.shape
    pitch = pitch or cols
    buf = cuda.full((offset + rows * pitch,), 77.0, dtype=torch_type(cuda, kind), device="cuda")
    view = buf[offset:].view(rows, pitch)[:, :cols]
    view.copy_(cuda.from_numpy(x))
    return buf, view


def f64(t):
    return t.detach().double().cpu().numpy()


def bytes_buffer(cuda, rows, pitch, offset=0):
    buf = cuda.full((offset + rows * pitch,), FILL, dtype=cuda.uint8, device="cuda")
    return buf, buf[offset:].view(rows, pitch)


def addr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def activations(rng, rows, cols):
    return rng.normal(size=(rows, cols)) * np.exp(rng.normal(size=cols))


# ------------------------------------------------------------------ quantiser


def quantize(cuda, cmb, view, kind, block, which="both", pad=0, offset=0):
    rows, cols = view.shape
    tall, tall_t = -(-rows // block), -(-cols // block)
    g, gt = up(cols, 128) // 128, up(rows, 128) // 128
    q, s, qt, st = (None,) * 4
    if which in ("both", "rows"):
        q = bytes_buffer(cuda, rows, cols + pad, offset)[1]
        s = bytes_buffer(cuda, tall, g + pad)[1]
    if which in ("both", "columns"):
        qt = bytes_buffer(cuda, cols, rows + pad, offset)[1]
        st = bytes_buffer(cuda, tall_t, gt + pad)[1]
    pitch = lambda t: t.shape[1] if t is not None else 0
    cmb.check("cmb_quantize_e4m3_block128", addr(view), CODE[kind], rows, cols, view.stride(0),
              block, addr(q), pitch(q), addr(s), pitch(s), addr(qt), pitch(qt), addr(st), pitch(st),
              stream_handle(cuda))
    cuda.cuda.synchronize()
    out = []
    for t, width in ((q, cols), (s, g), (qt, rows), (st, gt)):
        if t is None:
            out.append(None)
            continue
        a = t.cpu().numpy()
        assert (a[:, width:] == FILL).all(), "wrote between the rows"
        out.append(a[:, :width])
    return out


def same_quantized(got, x, block):
    q, s, qt, st = got
    if q is not None:
        wq, ws = ref.quantize(x, block)
        assert np.array_equal(s, ws) and np.array_equal(q, wq)
    if qt is not None:
        wq, ws = ref.quantize(x.T, block)
        assert np.array_equal(st, ws) and np.array_equal(qt, wq)


@pytest.mark.parametrize("which", ["rows", "columns", "both"])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (128, 128), (130, 333),
                                       (257, 1000), (1, 8192), (300, 16)])
def test_quantize(cuda, cmb, rows, cols, kind, block, which):
    rng = np.random.default_rng(rows * 1000 + cols)
    _, view = on_gpu(cuda, activations(rng, rows, cols), kind)
    same_quantized(quantize(cuda, cmb, view, kind, block, which), f64(view), block)


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("pitch,pad,offset", [(333, 3, 1), (336, 8, 0), (335, 0, 3), (344, 7, 8),
                                              (331, 6, 0)])
def test_quantize_strides_and_alignment(cuda, cmb, kind, block, pitch, pad, offset):
    rng = np.random.default_rng(pitch)
    _, view = on_gpu(cuda, activations(rng, 131, 330), kind, pitch, offset)
    same_quantized(quantize(cuda, cmb, view, kind, block, "both", pad, offset), f64(view), block)


@pytest.mark.parametrize("which", ["rows", "both"])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("cols,pad,offset", [(1304, 0, 0), (1304, 8, 0), (1304, 1, 0), (1301, 0, 3)])
def test_quantize_many_tiles(cuda, cmb, kind, cols, pad, offset, which):
    """More tiles than SMs, whose edges and odd rows are read ahead of one
    another, with values that are not finite in some."""
    rng = np.random.default_rng(cols + pad)
    x = activations(rng, 2500, cols)
    x[rng.integers(0, 2500, 9), rng.integers(0, cols, 9)] = [np.inf, -np.inf, np.nan] * 3
    x[0, 0] = x[-1, -1] = np.inf
    _, view = on_gpu(cuda, x, kind, offset=offset)
    same_quantized(quantize(cuda, cmb, view, kind, 1, which, pad), f64(view), 1)


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_quantize_borders(cuda, cmb, kind, block):
    """Blocks that end exactly at 448 * 2^n or just above, blocks of zeros, of
    the type's smallest and largest values, ties between two codes, negative
    zero, NaN and infinities among finite values and alone."""
    rng = np.random.default_rng(5)
    x = rng.normal(size=(12 * 128, 256))
    first = x[::128] if block == 128 else x[:12]
    x[:] = np.clip(x, -3, 3)
    for i, top in enumerate([448.0, 450.0, 446.0, 3.5, 7.0, 7.0625]):
        first[i] = np.clip(first[i], -top, top)
        first[i, 5] = -top
    first[6] = 0.0
    first[7] = rng.integers(-3, 4, 256) * 2.0 ** -133
    first[8] = rng.choice([1, -1], 256) * 3.0e38
    first[9] = np.tile([17.0, 19.0, 21.0, 23.0, -17.0, -19.0, 448.0, 2.0 ** -10], 32)  # ties
    first[10, :4] = [np.nan, np.inf, -np.inf, -0.0]
    first[11] = np.inf
    if block == 128:
        for i in (6, 7, 8, 11):
            x[i * 128:(i + 1) * 128] = first[i]
    _, view = on_gpu(cuda, x, kind)
    got = quantize(cuda, cmb, view, kind, block)
    same_quantized(got, f64(view), block)
    assert (got[0][first_rows(block, 6)] == 0).all() and (got[1][6] == 127).all()
    assert (got[0][first_rows(block, 11)] == 0x7F).all()


def first_rows(block, i):
    return i * 128 if block == 128 else i


def test_quantize_many_tile_rows(cuda, cmb):
    """More rows of tiles than a grid's second dimension counts."""
    rows = 65536 * 128 + 5
    x = cuda.zeros(rows, 4, dtype=cuda.bfloat16, device="cuda")
    x[-5:] = 3.0
    q = cuda.full((rows, 4), FILL, dtype=cuda.uint8, device="cuda")
    s = cuda.full((65537, 1), FILL, dtype=cuda.uint8, device="cuda")
    cmb.check("cmb_quantize_e4m3_block128", addr(x), BF16, rows, 4, 4, 128, addr(q), 4, addr(s), 1,
              None, 0, None, 0, stream_handle(cuda))
    assert int(s[:-1].min()) == int(s[:-1].max()) == 127
    want_q, want_s = ref.quantize(np.full((5, 4), 3.0), 128)
    assert np.array_equal(q[-5:].cpu().numpy(), want_q) and int(s[-1]) == want_s[0, 0]
    assert int(q[:-5].max()) == 0


# ----------------------------------------------------------------- the product


def operand(cuda, rng, rows, cols, block, pitch=None, wide=10, fill=0x7F):
    """Random finite e4m3 codes and scales (2^+-wide); the bytes behind each
    row hold NaN codes and NaN scales, which no product may read into C."""
    pitch = pitch or up(cols, 16)
    q = np.full((rows, pitch), fill, np.uint8)
    q[:, :cols] = rng.integers(0, 127, (rows, cols)) | (rng.integers(0, 2, (rows, cols)) << 7)
    groups = up(cols, 128) // 128
    s = np.full((-(-rows // block), groups + 3), 255, np.uint8)
    s[:, :groups] = 127 + rng.integers(-wide, wide + 1, (s.shape[0], groups))
    return (cuda.from_numpy(q).cuda(), cuda.from_numpy(s).cuda(), q[:, :cols], s[:, :groups])


def product(cuda, cmb, a, b, block_b, m, n, k, out, pad=0, offset=0, stream=None, status=None):
    buf = cuda.full((offset + m * (n + pad),), 55.0, dtype=torch_type(cuda, out), device="cuda")
    c = buf[offset:].view(m, n + pad)
    st = status if status is not None else cuda.zeros(1, dtype=cuda.int32, device="cuda")
    cmb.check("cmb_gemm_e4m3_block128", addr(a[0]), a[0].shape[1], addr(a[1]), a[1].shape[1],
              addr(b[0]), b[0].shape[1], addr(b[1]), b[1].shape[1], block_b, addr(c), c.shape[1],
              CODE[out], m, n, k, addr(st), stream or stream_handle(cuda))
    cuda.cuda.synchronize()
    assert int(st.item()) == 0, "a device-side wait timed out"
    assert (buf[:offset] == 55.0).all() and (c[:, n:] == 55.0).all(), "wrote outside of C"
    return c[:, :n]


def check_product(cuda, cmb, m, n, k, block_b, out, pad=0, offset=0, seed=0, rows=None):
    rng = np.random.default_rng(seed + m * 7 + n * 11 + k)
    a, b = operand(cuda, rng, m, k, 1), operand(cuda, rng, n, k, block_b)
    c = f64(product(cuda, cmb, a, b, block_b, m, n, k, out, pad, offset))
    want, mags = ref.gemm(a[2], a[3], b[2], b[3], block_b)
    err, room = np.abs(c - want), ref.gemm_bound(want, mags, k, out)
    assert (err <= room).all(), (np.argwhere(~(err <= room))[:4], (err / room).max())


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("block_b", [1, 128])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 128, 128), (1, 1000, 2064), (1, 8, 16), (2, 129, 300), (5, 200, 333),
    (7, 640, 1024), (8, 130, 129), (9, 512, 500), (16, 384, 4096), (17, 300, 257), (31, 256, 1000),
    (33, 700, 640), (48, 1024, 2048), (64, 512, 1040), (65, 333, 512), (100, 513, 777),
    (127, 256, 2064)])
def test_gemm_few_rows(cuda, cmb, m, n, k, block_b, out):
    check_product(cuda, cmb, m, n, k, block_b, out)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("block_b", [1, 128])
@pytest.mark.parametrize("m,n,k", [
    (128, 128, 128), (129, 127, 300), (200, 136, 72), (256, 512, 1024), (257, 1, 500),
    (300, 7, 130), (512, 640, 2048), (1000, 700, 520), (1000, 1100, 2064), (2048, 1500, 129),
    (4096, 250, 1), (1500, 2000, 16)])
def test_gemm_many_rows(cuda, cmb, m, n, k, block_b, out):
    check_product(cuda, cmb, m, n, k, block_b, out)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("n,pad,offset", [(200, 1, 0), (200, 8, 1), (203, 5, 4), (256, 0, 2), (96, 3, 3)])
def test_gemm_rows_of_c(cuda, cmb, m, n, pad, offset, out):
    """C with gaps between its rows and off every alignment: exact places, and
    nothing between them."""
    check_product(cuda, cmb, m, n, 260, 128, out, pad, offset)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_gemm_not_a_number(cuda, cmb, m):
    """A NaN code or a NaN scale reaches its row or column of C and no other."""
    rng = np.random.default_rng(m)
    n, k = 260, 400
    a, b = operand(cuda, rng, m, k, 1), operand(cuda, rng, n, k, 1)
    row = m // 2
    a[0][row, 333] = 0x7F
    b[0][17, 3] = 0xFF
    b[1][200, 2] = 255
    c = product(cuda, cmb, a, b, 1, m, n, k, "f32")
    bad = np.isnan(f64(c))
    want = np.zeros((m, n), bool)
    want[row] = want[:, 17] = want[:, 200] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("m", [2, 300])
def test_gemm_no_terms(cuda, cmb, m):
    """K = 0: zeros, between gaps that stay."""
    c = cuda.full((m, 50), 5.0, device="cuda")
    cmb.check("cmb_gemm_e4m3_block128", None, 0, None, 0, None, 0, None, 0, 128, addr(c), 50, F32, m,
              40, 0, None, stream_handle(cuda))
    assert (c[:, :40] == 0).all() and (c[:, 40:] == 5).all()


@pytest.mark.parametrize("m", [3, 200])
def test_gemm_far_scales(cuda, cmb, m):
    """Scales over the whole range of products that fp32 holds: 2^-60 .. 2^60
    each, so one group rules each sum."""
    rng = np.random.default_rng(m)
    a, b = operand(cuda, rng, m, 520, 1, wide=50), operand(cuda, rng, 300, 520, 1, wide=50)
    c = f64(product(cuda, cmb, a, b, 1, m, 300, 520, "f32"))
    want, mags = ref.gemm(a[2], a[3], b[2], b[3], 1)
    assert (np.abs(c - want) <= ref.gemm_bound(want, mags, 520, "f32")).all()


@pytest.mark.parametrize("m,n,k,block_b,out", [
    (8192, 8192, 8192, 128, "bf16"), (8192, 8192, 8192, 1, "f32"), (6000, 8200, 1040, 128, "bf16"),
    (5000, 4600, 300, 1, "f32"), (48, 8192, 8192, 128, "bf16"), (1, 8192, 8192, 128, "f32"),
    (40000, 520, 264, 128, "bf16")])
def test_gemm_large_sampled(cuda, cmb, m, n, k, block_b, out):
    """Every output is finite; sampled rows (first and last among them) against
    the 64-bit product of those rows with all of B."""
    rng = np.random.default_rng(m + n + k)
    a, b = operand(cuda, rng, m, k, 1), operand(cuda, rng, n, k, block_b)
    c = product(cuda, cmb, a, b, block_b, m, n, k, out)
    assert cuda.isfinite(c).all()
    pick = np.unique(np.concatenate([[0, m - 1], rng.integers(0, m, 60)]))
    want, mags = ref.gemm(a[2][pick], a[3][pick], b[2], b[3], block_b)
    err = np.abs(f64(c[cuda.from_numpy(pick).cuda()]) - want)
    assert (err <= ref.gemm_bound(want, mags, k, out)).all()


@pytest.mark.parametrize("m,n,k", [(1, 300, 8192), (100, 512, 6000), (128, 18000, 8192),
                                   (40, 20000, 4200), (250, 4096, 8192), (2000, 1500, 2049),
                                   (2100, 2100, 8192), (1500, 4096, 4096), (3000, 3000, 2300)])
def test_gemm_long_sums_in_fp32(cuda, cmb, m, n, k):
    """An fp32 C adds accumulators of at most 2048 (2816) of K: all products
    positive, where truncation would drift one way."""
    rng = np.random.default_rng(k)
    a, b = operand(cuda, rng, m, k, 1, wide=0), operand(cuda, rng, n, k, 128, wide=0)
    for q in (a, b):
        q[0][:, :k] &= 0x7F
    qa, qb = a[2] & 0x7F, b[2] & 0x7F
    c = product(cuda, cmb, a, b, 128, m, n, k, "f32")
    pick = np.unique(np.concatenate([[0, m - 1], rng.integers(0, m, 40)]))
    want, mags = ref.gemm(qa[pick], a[3][pick], qb, b[3], 128)
    err = np.abs(f64(c[cuda.from_numpy(pick).cuda()]) - want)
    assert (err <= ref.gemm_bound(want, mags, k, "f32")).all()
    # each of an accumulator's 64 (88) MMAs is off by at most 4 u32 of the sum so
    # far, as in gemm_bound (2 for the addition and 2 for the alignment of the
    # products, both downwards, so they do not average out), and the sums so far
    # of terms that are all positive and alike average half the last one: 88 * 4 *
    # 1/2.  One accumulator for 8192 would drift by up to 256 * 4 * 1/2.
    assert np.linalg.norm(err) <= 176 * ref.U32 * np.linalg.norm(want)


@pytest.mark.parametrize("m,n,k", [(1, 1000, 2064), (48, 4096, 4096), (200, 1000, 3000),
                                   (3000, 4096, 1024), (3000, 4096, 4500)])
def test_gemm_same_bits_again(cuda, cmb, m, n, k):
    """No atomics, no order that changes: the same bits from every call, on
    two streams at once too."""
    rng = np.random.default_rng(m)
    a, b = operand(cuda, rng, m, k, 1), operand(cuda, rng, n, k, 128)
    first = product(cuda, cmb, a, b, 128, m, n, k, "f32").clone()
    outs, streams = [], [cuda.cuda.Stream() for _ in range(2)]
    for i in range(12):
        c = cuda.full((m, n), float("nan"), device="cuda")
        outs.append(c)
    cuda.cuda.synchronize()
    for i, c in enumerate(outs):
        s = ctypes.c_void_p(streams[i % 2].cuda_stream)
        cmb.check("cmb_gemm_e4m3_block128", addr(a[0]), a[0].shape[1], addr(a[1]), a[1].shape[1],
                  addr(b[0]), b[0].shape[1], addr(b[1]), b[1].shape[1], 128, addr(c), n, F32, m, n,
                  k, None, s)
    cuda.cuda.synchronize()
    assert all(cuda.equal(first, c) for c in outs)


def test_gemm_status_keeps_what_the_caller_left(cuda, cmb):
    """The status word is the caller's to clear: a call without a timeout
    leaves it as it was."""
    rng = np.random.default_rng(1)
    a, b = operand(cuda, rng, 4, 128, 1), operand(cuda, rng, 64, 128, 1)
    st = cuda.full((1,), 3, dtype=cuda.int32, device="cuda")
    c = cuda.empty(4, 64, device="cuda")
    cmb.check("cmb_gemm_e4m3_block128", addr(a[0]), 128, addr(a[1]), 4, addr(b[0]), 128, addr(b[1]),
              4, 1, addr(c), 64, F32, 4, 64, 128, addr(st), stream_handle(cuda))
    assert int(st.item()) == 3


# ------------------------------------------------------------------- the norm


def run_norm(cuda, cmb, x, r, w, kind, wkind, eps, want=("y", "q", "rstd"), pad=0, in_place=None):
    rows, cols = x.shape
    t = torch_type(cuda, kind)
    out = {}
    if r is not None:
        out["h"] = {"x": x, "r": r}.get(in_place)
        if out["h"] is None:
            out["h"] = cuda.full((rows, cols + pad), 9.0, dtype=t, device="cuda")
    if "y" in want:
        out["y"] = cuda.full((rows, cols + pad), 9.0, dtype=t, device="cuda")
    if "q" in want:
        out["q"] = bytes_buffer(cuda, rows, cols + pad)[1]
        out["s"] = bytes_buffer(cuda, rows, up(cols, 128) // 128 + pad)[1]
    if "rstd" in want:
        out["rstd"] = cuda.full((rows,), 9.0, device="cuda")
    g = out.get
    pitch = lambda v: v.stride(0) if v is not None else 0
    cmb.check("cmb_rmsnorm_e4m3_block128", addr(x), x.stride(0), addr(r), pitch(r), CODE[kind],
              addr(w), CODE[wkind], ctypes.c_float(eps), rows, cols, addr(g("h")), pitch(g("h")),
              addr(g("y")), pitch(g("y")), addr(g("q")), pitch(g("q")), addr(g("s")),
              pitch(g("s")), addr(g("rstd")), stream_handle(cuda))
    cuda.cuda.synchronize()
    for name, fill in (("h", 9.0), ("y", 9.0), ("q", FILL)):
        if g(name) is not None and in_place is None:
            assert (out[name][:, cols:] == fill).all(), "wrote between the rows"
            out[name] = out[name][:, :cols]
    if g("s") is not None:
        assert (out["s"][:, up(cols, 128) // 128:] == FILL).all()
        out["s"] = out["s"][:, :up(cols, 128) // 128]
    return out


def check_norm(out, x, r, w, kind, eps):
    """`x`, `r`, `w`: 64-bit values of the inputs."""
    h = x
    if r is not None:
        h = f64(out["h"])
        # x + r is exact to one fp32 rounding, then rounded to the type
        assert (np.abs(h - (x + r)) <= (ref.UNIT[kind] + 2 * ref.U32) * np.abs(x + r)).all()
    cols = x.shape[1]
    rstd, y = ref.norm(h, w, eps)
    if "rstd" in out:
        assert (np.abs(f64(out["rstd"]) - rstd) <= ref.rstd_bound(cols) * rstd).all()
    rel = ref.y_bound(cols)
    if "y" in out:
        assert (np.abs(f64(out["y"]) - y) <= (ref.UNIT[kind] * (1 + rel) + rel) * np.abs(y)).all()
    if "q" in out:
        ref.check_quantized(out["q"].cpu().numpy(), out["s"].cpu().numpy(), y, rel)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind,wkind", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16"),
                                        ("f32", "f32")])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 1000), (300, 1024),
                                       (1, 8192), (700, 4600), (3, 8200), (2, 16384), (2, 32768),
                                       (3, 20001)])
def test_norm(cuda, cmb, rows, cols, kind, wkind, residual):
    rng = np.random.default_rng(rows + cols)
    _, x = on_gpu(cuda, activations(rng, rows, cols), kind)
    _, w = on_gpu(cuda, 1 + 0.1 * rng.normal(size=(1, cols)), wkind)
    r = on_gpu(cuda, 3 * rng.normal(size=(rows, cols)), kind)[1] if residual else None
    keep = f64(x), f64(r) if residual else None
    out = run_norm(cuda, cmb, x, r, w, kind, wkind, 1e-5)
    check_norm(out, *keep, f64(w)[0], kind, np.float32(1e-5))
    assert np.array_equal(f64(x), keep[0])  # inputs stay


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1200, 4096), (9000, 64), (5000, 1000), (5000, 1032),
                                       (3000, 255), (2500, 2051), (1, 4601), (700, 8190),
                                       (200, 30001)])
def test_norm_more_rows_than_fit(cuda, cmb, rows, cols, kind, residual):
    """Every width of CTA, several rows each, whole chunks and odd ones."""
    rng = np.random.default_rng(rows + cols)
    _, x = on_gpu(cuda, activations(rng, rows, cols), kind)
    _, w = on_gpu(cuda, 1 + 0.1 * rng.normal(size=(1, cols)), "bf16")
    r = on_gpu(cuda, 3 * rng.normal(size=(rows, cols)), kind)[1] if residual else None
    keep = f64(x), f64(r) if residual else None
    out = run_norm(cuda, cmb, x, r, w, kind, "bf16", 1e-5)
    check_norm(out, *keep, f64(w)[0], kind, np.float32(1e-5))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("cols,pitch,offset,pad", [(330, 333, 1, 3), (328, 336, 0, 8), (1000, 1001, 2, 1),
                                                   (9000, 9003, 0, 5), (513, 517, 3, 2), (7, 9, 1, 1)])
def test_norm_strides_and_alignment(cuda, cmb, kind, cols, pitch, offset, pad):
    rng = np.random.default_rng(cols)
    _, x = on_gpu(cuda, activations(rng, 9, cols), kind, pitch, offset)
    _, r = on_gpu(cuda, rng.normal(size=(9, cols)), kind, pitch + 1, offset)
    _, w = on_gpu(cuda, 1 + 0.1 * rng.normal(size=(1, cols)), kind, None, offset)
    keep = f64(x), f64(r)
    out = run_norm(cuda, cmb, x, r, w, kind, kind, 1e-6, pad=pad)
    check_norm(out, *keep, f64(w)[0], kind, np.float32(1e-6))


@pytest.mark.parametrize("where", ["x", "r"])
@pytest.mark.parametrize("rows", [3, 1000])
@pytest.mark.parametrize("cols", [1544, 1547])
def test_norm_residual_in_place(cuda, cmb, where, rows, cols):
    rng = np.random.default_rng(rows)
    _, x = on_gpu(cuda, activations(rng, rows, cols), "bf16")
    _, r = on_gpu(cuda, rng.normal(size=(rows, cols)), "bf16")
    _, w = on_gpu(cuda, np.ones((1, cols)), "bf16")
    keep = f64(x), f64(r)
    out = run_norm(cuda, cmb, x, r, w, "bf16", "bf16", 1e-5, in_place=where)
    check_norm(out, *keep, f64(w)[0], "bf16", np.float32(1e-5))
    assert np.array_equal(f64(r if where == "x" else x), keep[1 if where == "x" else 0])


@pytest.mark.parametrize("want", [("q",), ("y",), ("rstd",), ("q", "rstd"), ()])
def test_norm_only_some_outputs(cuda, cmb, want):
    rng = np.random.default_rng(3)
    _, x = on_gpu(cuda, activations(rng, 20, 500), "bf16")
    _, r = on_gpu(cuda, rng.normal(size=(20, 500)), "bf16")
    _, w = on_gpu(cuda, np.ones((1, 500)), "f32")
    keep = f64(x), f64(r)
    out = run_norm(cuda, cmb, x, r, w, "bf16", "f32", 1e-5, want=want)
    check_norm(out, *keep, f64(w)[0], "bf16", np.float32(1e-5))


def test_norm_rows_of_zeros_and_not_a_number(cuda, cmb):
    """A row of zeros gives zeros and scales of 1 (eps keeps rstd finite); a
    NaN spoils its own row alone; with eps = 0 a row of zeros is NaN, as the
    formula has it."""
    rng = np.random.default_rng(4)
    x = activations(rng, 4, 300)
    x[1] = 0.0
    x[2, 7] = np.nan
    _, xg = on_gpu(cuda, x, "bf16")
    _, w = on_gpu(cuda, np.ones((1, 300)), "bf16")
    out = run_norm(cuda, cmb, xg, None, w, "bf16", "bf16", 1e-5)
    q, s = out["q"].cpu().numpy(), out["s"].cpu().numpy()
    assert (q[1] == 0).all() and (s[1] == 127).all()
    assert (q[2] == 0x7F).all() and (q[[0, 3]] & 0x7F != 0x7F).all()
    out = run_norm(cuda, cmb, xg, None, w, "bf16", "bf16", 0.0)
    assert (out["q"].cpu().numpy()[1] == 0x7F).all() and (out["q"].cpu().numpy()[0] != 0x7F).all()


# ------------------------------------------------------------- its gradients


def run_backward(cuda, cmb, dy, h, dh, w, rstd, kind, wkind, dw=True, pad=0, dx=None, room=None):
    rows, cols = dy.shape
    if dx is None:
        dx = cuda.full((rows, cols + pad), 9.0, dtype=torch_type(cuda, kind), device="cuda")
    grad = cuda.full((cols,), 9.0, device="cuda") if dw else None
    n = cmb.lib.cmb_rmsnorm_backward_workspace_bytes(rows, cols)
    if dw and room is None:
        room = cuda.full((n,), 0xFF, dtype=cuda.uint8, device="cuda")  # NaNs
    cmb.check("cmb_rmsnorm_backward", addr(dy), dy.stride(0), addr(h), h.stride(0), addr(dh),
              dh.stride(0) if dh is not None else 0, CODE[kind], addr(w), CODE[wkind], addr(rstd),
              rows, cols, addr(dx), dx.stride(0), addr(grad), addr(room), n if dw else 0,
              stream_handle(cuda))
    cuda.cuda.synchronize()
    if dx.shape[1] > cols:
        assert (dx[:, cols:] == 9.0).all(), "wrote between the rows"
    return dx[:, :cols], grad


def check_backward(dx, grad, dy, h, dh, w, rstd, kind):
    rows, cols = dy.shape
    past = dh if dh is not None else np.zeros_like(dy)
    want, wdw = ref.norm_backward(dy, h, w, rstd[:, None].repeat(1, 1)[:, 0], past)
    u, g = np.abs(h) * rstd[:, None], np.abs(dy * w)
    r = rstd[:, None]
    # products and differences round a few times each; the row's mean as in sum_steps
    room = ref.U32 * (6 * (r * g + r * u * (g * u).mean(1, keepdims=True) + np.abs(past)) +
                      (ref.sum_steps(cols) + 4) * r * u * (g * u).mean(1, keepdims=True))
    room = room * (1 + 1e-3) + ref.UNIT[kind] * np.abs(want) * (1 + 1e-3)
    err = np.abs(f64(dx) - want)
    assert (err <= room).all(), (err / np.maximum(room, 1e-300)).max()
    if grad is not None:
        room = (rows + 4) * ref.U32 * (np.abs(dy) * u).sum(axis=0)
        err = np.abs(f64(grad) - wdw)
        assert (err <= room).all(), (err / np.maximum(room, 1e-300)).max()


def backward_inputs(cuda, rng, rows, cols, kind, wkind, pitch=None, offset=0):
    _, dy = on_gpu(cuda, rng.normal(size=(rows, cols)), kind, pitch, offset)
    _, h = on_gpu(cuda, activations(rng, rows, cols), kind, pitch, offset)
    _, dh = on_gpu(cuda, rng.normal(size=(rows, cols)), kind, pitch, offset)
    _, w = on_gpu(cuda, 1 + 0.1 * rng.normal(size=(1, cols)), wkind)
    rstd = cuda.rsqrt(h.double().square().mean(dim=1) + 1e-5).float()
    return dy, h, dh, w, rstd


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind,wkind", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16"),
                                        ("f32", "f32")])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8192), (2, 127), (5, 129), (700, 1024),
                                       (333, 4600), (2000, 264), (3, 8200), (400, 16384), (2, 32768),
                                       (3, 20001)])
def test_norm_backward(cuda, cmb, rows, cols, kind, wkind, residual):
    rng = np.random.default_rng(rows + cols)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, rows, cols, kind, wkind)
    dh = dh if residual else None
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, kind, wkind)
    check_backward(dx, grad, f64(dy), f64(h), f64(dh) if residual else None, f64(w)[0], f64(rstd),
                   kind)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1200, 4096), (9000, 64), (5000, 1000), (5000, 1032),
                                       (3000, 255), (2500, 2051), (1, 4601), (700, 8190),
                                       (200, 30001)])
def test_norm_backward_more_rows_than_fit(cuda, cmb, rows, cols, kind, residual):
    rng = np.random.default_rng(rows + cols)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, rows, cols, kind, "bf16")
    dh = dh if residual else None
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, kind, "bf16")
    check_backward(dx, grad, f64(dy), f64(h), f64(dh) if residual else None, f64(w)[0], f64(rstd),
                   kind)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("cols,pitch,offset,pad", [(330, 333, 1, 3), (328, 336, 0, 8), (1000, 1001, 2, 1),
                                                   (513, 517, 3, 2), (7, 9, 1, 1)])
def test_norm_backward_strides_and_alignment(cuda, cmb, kind, cols, pitch, offset, pad):
    rng = np.random.default_rng(cols)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, 40, cols, kind, "f32", pitch, offset)
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, kind, "f32", pad=pad)
    check_backward(dx, grad, f64(dy), f64(h), f64(dh), f64(w)[0], f64(rstd), kind)


@pytest.mark.parametrize("where", ["dy", "dh"])
@pytest.mark.parametrize("cols", [1544, 1547])
def test_norm_backward_in_place(cuda, cmb, where, cols):
    rng = np.random.default_rng(2)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, 900, cols, "bf16", "bf16")
    keep = [f64(t) for t in (dy, h, dh)]
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, "bf16", "bf16",
                            dx={"dy": dy, "dh": dh}[where])
    check_backward(dx, grad, *keep, f64(w)[0], f64(rstd), "bf16")


def test_norm_backward_without_a_weight_gradient(cuda, cmb):
    rng = np.random.default_rng(6)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, 50, 700, "bf16", "bf16")
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, "bf16", "bf16", dw=False)
    check_backward(dx, grad, f64(dy), f64(h), f64(dh), f64(w)[0], f64(rstd), "bf16")


def test_norm_backward_no_rows(cuda, cmb):
    grad = cuda.full((30,), 9.0, device="cuda")
    cmb.check("cmb_rmsnorm_backward", None, 30, None, 30, None, 30, F32, None, F32, None, 0, 30,
              None, 30, addr(grad), None, 0, stream_handle(cuda))
    assert (grad == 0).all()


def test_norm_backward_matches_differences_of_the_forward_kernel(cuda, cmb):
    """Central differences of sum(dy * y) through the forward kernel, fp32.
    The differences are off by the forward's roundings over the step, 2 U32
    |L| sqrt(n) / d for the loss in 64 bits, and by the third derivative."""
    rng = np.random.default_rng(8)
    rows, cols, d = 2, 24, 2.0 ** -6
    h0, w0 = rng.normal(size=(rows, cols)), 1 + 0.1 * rng.normal(size=(1, cols))
    _, dy = on_gpu(cuda, rng.normal(size=(rows, cols)), "f32")
    _, w = on_gpu(cuda, w0, "f32")
    _, h = on_gpu(cuda, h0, "f32")
    out = run_norm(cuda, cmb, h, None, w, "f32", "f32", 1e-5)
    dx, grad = run_backward(cuda, cmb, dy, h, None, w, out["rstd"], "f32", "f32")

    def loss(hv, wv):
        y = run_norm(cuda, cmb, hv, None, wv, "f32", "f32", 1e-5, want=("y",))["y"]
        return float((y.double() * dy.double()).sum())

    size = float((dy.double() * out["y"].double()).abs().sum())
    # sums of 48 terms, each off by y_bound; the third derivative of h * rstd
    # stays under 10 here (|h| ~ 1, 24 columns), and d^2 / 6 of it remains
    room = 2 * ref.y_bound(cols) * size / (2 * d) + 10 * d * d / 6
    for i in range(rows):
        for j in range(cols):
            up_, down = h.clone(), h.clone()
            up_[i, j] += d
            down[i, j] -= d
            step = float(up_[i, j].double() - down[i, j].double())
            assert abs((loss(up_, w) - loss(down, w)) / step - float(dx[i, j])) < room
    for j in range(cols):
        up_, down = w.clone(), w.clone()
        up_[0, j] += d
        down[0, j] -= d
        step = float(up_[0, j].double() - down[0, j].double())
        assert abs((loss(h, up_) - loss(h, down)) / step - float(grad[j])) < room


# ------------------------------------------------------ a layer, all together


class Layer:
    """Norm with residual -> e4m3 projection, forward and backward, as a
    training step calls it: every product in e4m3, buffers kept."""

    def __init__(self, cuda, cmb, tokens, width, out, seed=0):
        self.cuda, self.cmb = cuda, cmb
        self.m, self.k, self.n = tokens, width, out
        rng = np.random.default_rng(seed)
        t = lambda a: cuda.from_numpy(a).cuda().bfloat16()
        self.x, self.r = t(activations(rng, tokens, width)), t(rng.normal(size=(tokens, width)))
        self.g = t(1 + 0.1 * rng.normal(size=(1, width)))
        self.w = t(rng.normal(size=(out, width)) * width ** -0.5)
        self.dc, self.dres = t(rng.normal(size=(tokens, out))), t(rng.normal(size=(tokens, width)))
        byte = lambda r, c: cuda.zeros(r, up(c, 16), dtype=cuda.uint8, device="cuda")
        form = lambda r, c, b=1: (byte(r, c), byte(-(-r // b), -(-c // 128)))
        m, k, n = tokens, width, out
        self.wq, self.wtq = form(n, k, 128), form(k, n, 128)
        self.yq, self.ytq = form(m, k), form(k, m)
        self.dcq, self.dctq = form(m, n), form(n, m)
        z = lambda r, c, d: cuda.zeros(r, c, dtype=d, device="cuda")
        bf, f32 = cuda.bfloat16, cuda.float32
        self.h, self.y, self.c = z(m, k, bf), z(m, k, bf), z(m, n, bf)
        self.dy, self.dx, self.dw = z(m, k, bf), z(m, k, bf), z(n, k, f32)
        self.rstd, self.dg = z(1, m, f32), z(1, k, f32)
        self.room = byte(1, cmb.lib.cmb_rmsnorm_backward_workspace_bytes(m, k))
        self.status = cuda.zeros(1, dtype=cuda.int32, device="cuda")

    def quantize(self, src, block, plain, turned):
        s = stream_handle(self.cuda)
        pair = lambda p: (addr(p[0]), p[0].shape[1], addr(p[1]), p[1].shape[1]) if p else (None, 0, None, 0)
        self.cmb.check("cmb_quantize_e4m3_block128", addr(src), BF16, *src.shape, src.shape[1],
                       block, *pair(plain), *pair(turned), s)

    def gemm(self, a, b, block, c, kind, m, n, k):
        self.cmb.check("cmb_gemm_e4m3_block128", addr(a[0]), a[0].shape[1], addr(a[1]),
                       a[1].shape[1], addr(b[0]), b[0].shape[1], addr(b[1]), b[1].shape[1], block,
                       addr(c), c.shape[1], kind, m, n, k, addr(self.status),
                       stream_handle(self.cuda))

    def forward(self):
        m, k, n = self.m, self.k, self.n
        self.quantize(self.w, 128, self.wq, self.wtq)
        self.cmb.check("cmb_rmsnorm_e4m3_block128", addr(self.x), k, addr(self.r), k, BF16,
                       addr(self.g), BF16, ctypes.c_float(1e-5), m, k, addr(self.h), k,
                       addr(self.y), k, addr(self.yq[0]), self.yq[0].shape[1], addr(self.yq[1]),
                       self.yq[1].shape[1], addr(self.rstd), stream_handle(self.cuda))
        self.gemm(self.yq, self.wq, 128, self.c, BF16, m, n, k)

    def backward(self):
        m, k, n = self.m, self.k, self.n
        self.quantize(self.dc, 1, self.dcq, self.dctq)
        self.quantize(self.y, 1, None, self.ytq)
        self.gemm(self.dcq, self.wtq, 128, self.dy, BF16, m, k, n)
        self.gemm(self.dctq, self.ytq, 1, self.dw, F32, n, k, m)
        self.cmb.check("cmb_rmsnorm_backward", addr(self.dy), k, addr(self.h), k, addr(self.dres),
                       k, BF16, addr(self.g), BF16, addr(self.rstd), m, k, addr(self.dx), k,
                       addr(self.dg), addr(self.room), self.room.numel(), stream_handle(self.cuda))

    def outputs(self):
        return {n: getattr(self, n) for n in ("h", "c", "dy", "dx", "dw", "dg")}


@pytest.mark.parametrize("tokens,width,out", [(1, 640, 500), (17, 1024, 640), (300, 1000, 1400)])
def test_layer_forward_and_backward(cuda, cmb, tokens, width, out):
    """Each step against 64 bits on what the step before it left."""
    L = Layer(cuda, cmb, tokens, width, out)
    L.forward()
    L.backward()
    cuda.cuda.synchronize()
    assert int(L.status.item()) == 0
    v = lambda t: f64(t)
    n8 = lambda t, c: t.cpu().numpy()[:, :c]
    wq, ws = ref.quantize(v(L.w), 128)
    assert np.array_equal(n8(L.wq[0], width), wq) and np.array_equal(n8(L.wtq[0], out), wq.T)
    h = v(L.h)
    rstd, y = ref.norm(h, v(L.g)[0], np.float32(1e-5))
    yq, ys = n8(L.yq[0], width), n8(L.yq[1], -(-width // 128))
    ref.check_quantized(yq, ys, y, ref.y_bound(width))

    def close(got, a, sa, b, sb, block, k, kind):
        want, mags = ref.gemm(a, sa, b, sb, block)
        assert (np.abs(v(got) - want) <= ref.gemm_bound(want, mags, k, kind)).all()

    close(L.c, yq, ys, wq, ws, 128, width, "bf16")
    dq, ds = ref.quantize(v(L.dc), 1)
    dtq, dts = ref.quantize(v(L.dc).T, 1)
    ytq, yts = ref.quantize(v(L.y).T, 1)
    close(L.dy, dq, ds, wq.T, ws.T, 128, out, "bf16")
    close(L.dw, dtq, dts, ytq, yts, 1, tokens, "f32")
    check_backward(L.dx, L.dg[0], v(L.dy), h, v(L.dres), v(L.g)[0], v(L.rstd)[0], "bf16")
    # and as a whole: the e4m3 layer's gradients are near the exact layer's.  Two operands, each
    # rounded by at most 2^-4 of a value: their random errors add up to less than that.
    exact_dw = v(L.dc).T @ y
    assert np.linalg.norm(v(L.dw) - exact_dw) <= 2 * ref.U8 * np.linalg.norm(exact_dw)


@pytest.mark.parametrize("tokens", [1, 200])
def test_layer_in_a_graph_and_on_a_stream(cuda, cmb, tokens):
    """Captured on a side stream beside an eager layer with its own buffers,
    and replayed on new inputs: the same bits as direct calls."""
    L, E = Layer(cuda, cmb, tokens, 640, 500, 1), Layer(cuda, cmb, tokens, 640, 500, 1)
    s = cuda.cuda.Stream()
    s.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(s):
        L.forward()
        L.backward()
    s.synchronize()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=s):
        L.forward()
        L.backward()
    for seed in range(3):
        new = Layer(cuda, cmb, tokens, 640, 500, 10 + seed)
        for name in ("x", "r", "g", "w", "dc", "dres"):
            getattr(L, name).copy_(getattr(new, name))
            getattr(E, name).copy_(getattr(new, name))
        for t in L.outputs().values():
            t.fill_(float("nan"))
        cuda.cuda.synchronize()
        graph.replay()
        E.forward()  # eager on the current stream while the graph runs
        E.backward()
        cuda.cuda.synchronize()
        for name, t in L.outputs().items():
            assert cuda.equal(t, E.outputs()[name]), name
    assert int(L.status.item()) == 0


@pytest.mark.parametrize("where", ["x", "r", "both"])
def test_norm_in_place_where_rows_follow_one_another(cuda, cmb, where):
    """More rows than fit at once, so the next row is on its way while h goes
    over the last; x and the residual may be one tensor."""
    rng = np.random.default_rng(4)
    _, x = on_gpu(cuda, activations(rng, 4100, 1544), "bf16")
    r = x if where == "both" else on_gpu(cuda, rng.normal(size=(4100, 1544)), "bf16")[1]
    _, w = on_gpu(cuda, np.ones((1, 1544)), "bf16")
    keep = f64(x), f64(r)
    out = run_norm(cuda, cmb, x, r, w, "bf16", "bf16", 1e-5, in_place="r" if where == "r" else "x")
    check_norm(out, *keep, f64(w)[0], "bf16", np.float32(1e-5))


@pytest.mark.parametrize("where", ["dy", "dh"])
def test_norm_backward_in_place_where_rows_follow_one_another(cuda, cmb, where):
    rng = np.random.default_rng(5)
    dy, h, dh, w, rstd = backward_inputs(cuda, rng, 4100, 1544, "bf16", "bf16")
    keep = [f64(t) for t in (dy, h, dh)]
    dx, grad = run_backward(cuda, cmb, dy, h, dh, w, rstd, "bf16", "bf16",
                            dx={"dy": dy, "dh": dh}[where])
    check_backward(dx, grad, *keep, f64(w)[0], f64(rstd), "bf16")


@pytest.mark.parametrize("m,k", [(20, 400), (700, 1000)])
def test_gemm_of_a_matrix_with_itself(cuda, cmb, m, k):
    rng = np.random.default_rng(m)
    a = operand(cuda, rng, m, k, 1)
    c = f64(product(cuda, cmb, a, a, 1, m, m, k, "f32"))
    want, mags = ref.gemm(a[2], a[3], a[2], a[3], 1)
    assert (np.abs(c - want) <= ref.gemm_bound(want, mags, k, "f32")).all()


def test_products_of_every_kind_on_four_streams(cuda, cmb):
    """Few tokens (clusters that split K), many (pairs), and the per-tensor
    product share the GPU and its tensor memory."""
    rng = np.random.default_rng(6)
    shapes = [(4, 1024, 4096), (700, 2048, 1024), (100, 3000, 2048)]
    sets = [(operand(cuda, rng, m, k, 1), operand(cuda, rng, n, k, 128)) for m, n, k in shapes]
    alone = [product(cuda, cmb, a, b, 128, m, n, k, "bf16").clone()
             for (a, b), (m, n, k) in zip(sets, shapes)]
    streams = [cuda.cuda.Stream() for _ in shapes]
    outs = [cuda.full((6, m, n), 7.0, dtype=cuda.bfloat16, device="cuda") for m, n, _ in shapes]
    size = 1024
    ab = cuda.randint(0, 120, (2, size, size), dtype=cuda.uint8, device="cuda")
    scale = cuda.ones(2, device="cuda")
    per_tensor = cuda.full((6, size, size), 7.0, device="cuda")
    st = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    other = cuda.cuda.Stream()
    cuda.cuda.synchronize()
    for i in range(6):
        for (a, b), (m, n, k), s, out in zip(sets, shapes, streams, outs):
            cmb.check("cmb_gemm_e4m3_block128", addr(a[0]), a[0].shape[1], addr(a[1]),
                      a[1].shape[1], addr(b[0]), b[0].shape[1], addr(b[1]), b[1].shape[1], 128,
                      addr(out[i]), n, BF16, m, n, k, addr(st), ctypes.c_void_p(s.cuda_stream))
        cmb.check("cmb_gemm_e4m3", addr(ab[0]), addr(ab[1]), addr(per_tensor[i]), size, size,
                  size, addr(scale), addr(scale), 2, addr(st), ctypes.c_void_p(other.cuda_stream))
    cuda.cuda.synchronize()
    assert int(st.item()) == 0
    for want, out in zip(alone, outs):
        assert all(cuda.equal(want, c) for c in out)
    assert all(cuda.equal(per_tensor[0], c) for c in per_tensor)


@pytest.mark.parametrize("m,n,k", [(3, 512, 1024), (900, 1024, 1024)])
def test_captured_calls_share_their_buffers(cuda, cmb, m, n, k):
    """One graph in which the same operand buffers and the same workspace are
    filled again for each of eight products and gradients: each kernel may
    start before the last one's end, none may read or write too soon."""
    rng = np.random.default_rng(8)
    xs = [on_gpu(cuda, activations(rng, m, k), "bf16")[1] for _ in range(8)]
    b = operand(cuda, rng, n, k, 128)
    q, s = (cuda.zeros(m, c, dtype=cuda.uint8, device="cuda") for c in (k, up(k // 128, 16)))
    w = on_gpu(cuda, np.ones((1, k)), "bf16")[1]
    rstd = cuda.ones(m, device="cuda")
    bytes_ = cmb.lib.cmb_rmsnorm_backward_workspace_bytes(m, k)
    room = cuda.empty(bytes_ // 4, device="cuda")
    st = cuda.zeros(1, dtype=cuda.int32, device="cuda")

    def steps(wait):
        outs = []
        for x in xs:
            c = cuda.empty(m, n, device="cuda")
            dx = cuda.empty(m, k, dtype=cuda.bfloat16, device="cuda")
            dw = cuda.empty(k, device="cuda")
            room.fill_(float("nan"))
            cmb.check("cmb_quantize_e4m3_block128", addr(x), BF16, m, k, k, 1, addr(q), k, addr(s),
                      s.shape[1], None, 0, None, 0, stream_handle(cuda))
            wait()
            cmb.check("cmb_gemm_e4m3_block128", addr(q), k, addr(s), s.shape[1], addr(b[0]),
                      b[0].shape[1], addr(b[1]), b[1].shape[1], 128, addr(c), n, F32, m, n, k,
                      addr(st), stream_handle(cuda))
            wait()
            cmb.check("cmb_rmsnorm_backward", addr(x), k, addr(x), k, None, 0, BF16, addr(w), BF16,
                      addr(rstd), m, k, addr(dx), k, addr(dw), addr(room), bytes_,
                      stream_handle(cuda))
            wait()
            outs += [c, dx, dw]
        return outs

    want = steps(cuda.cuda.synchronize)
    graph, side = cuda.cuda.CUDAGraph(), cuda.cuda.Stream()
    with cuda.cuda.graph(graph, stream=side):
        got = steps(lambda: None)
    for _ in range(3):
        for t in got:
            t.fill_(5.0)
        graph.replay()
        cuda.cuda.synchronize()
        assert all(cuda.equal(a, c) for a, c in zip(want, got))
    assert int(st.item()) == 0


# --------------------------------------------- offsets that need more than 32 bits


def far_rows(cuda, rows, cols, pitch, dtype, fill):
    """rows x cols with `pitch` elements from row to row, of which only the
    values and the one behind each row are written."""
    assert (rows - 1) * pitch > 2 ** 32
    v = cuda.empty(rows * pitch, dtype=dtype, device="cuda").view(rows, pitch)
    v[:, :cols + 1] = fill
    return v


@pytest.fixture
def room(cuda):
    cuda.cuda.empty_cache()
    if cuda.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    yield
    cuda.cuda.empty_cache()


@pytest.mark.parametrize("m", [7, 300])
def test_gemm_far_offsets(cuda, cmb, room, m):
    n, k, pitch = 200, 300, up(5 * 2 ** 30 // m, 16)
    rng = np.random.default_rng(m)
    a, b = operand(cuda, rng, m, k, 1), operand(cuda, rng, n, k, 128)
    q, s = (far_rows(cuda, m, w, pitch, cuda.uint8, 0x7F) for w in (k, 3))
    q[:, :k], s[:, :3] = a[0][:, :k], a[1][:, :3]
    c = far_rows(cuda, m, n, pitch, cuda.bfloat16, 55.0)
    cmb.check("cmb_gemm_e4m3_block128", addr(q), pitch, addr(s), pitch, addr(b[0]), b[0].shape[1],
              addr(b[1]), b[1].shape[1], 128, addr(c), pitch, BF16, m, n, k, None,
              stream_handle(cuda))
    want, mags = ref.gemm(a[2], a[3], b[2], b[3], 128)
    err, room_ = np.abs(f64(c[:, :n]) - want), ref.gemm_bound(want, mags, k, "bf16")
    assert (err <= room_).all() and (c[:, n] == 55.0).all()


@pytest.mark.parametrize("rows,cols", [(40, 300), (5000, 256)])
def test_norm_and_gradient_far_offsets(cuda, cmb, room, rows, cols):
    pitch = up(9 * 2 ** 29 // rows, 16)
    rng = np.random.default_rng(rows)
    x, dy = (far_rows(cuda, rows, cols, pitch, cuda.bfloat16, 55.0) for _ in range(2))
    q = far_rows(cuda, rows, cols, pitch, cuda.uint8, FILL)
    x[:, :cols] = cuda.from_numpy(activations(rng, rows, cols))
    dy[:, :cols] = cuda.from_numpy(rng.normal(size=(rows, cols)))
    r, w = (on_gpu(cuda, rng.normal(size=(h, cols)), "bf16")[1] for h in (rows, 1))
    s = bytes_buffer(cuda, rows, 3)[1]
    rstd = cuda.empty(rows, device="cuda")
    keep = f64(x[:, :cols]), f64(r), f64(dy[:, :cols])
    cmb.check("cmb_rmsnorm_e4m3_block128", addr(x), pitch, addr(r), cols, BF16, addr(w), BF16,
              ctypes.c_float(1e-5), rows, cols, addr(x), pitch, None, 0, addr(q), pitch, addr(s), 3,
              addr(rstd), stream_handle(cuda))
    out = dict(h=x[:, :cols], q=q[:, :cols], s=s[:, :up(cols, 128) // 128], rstd=rstd)
    check_norm(out, keep[0], keep[1], f64(w)[0], "bf16", np.float32(1e-5))
    assert (x[:, cols] == 55.0).all() and (q[:, cols] == FILL).all()
    h = f64(x[:, :cols])
    grad = cuda.empty(cols, device="cuda")
    n = cmb.lib.cmb_rmsnorm_backward_workspace_bytes(rows, cols)
    space = cuda.empty(n, dtype=cuda.uint8, device="cuda")
    cmb.check("cmb_rmsnorm_backward", addr(dy), pitch, addr(x), pitch, None, 0, BF16, addr(w), BF16,
              addr(rstd), rows, cols, addr(dy), pitch, addr(grad), addr(space), n,
              stream_handle(cuda))
    check_backward(dy[:, :cols], grad, keep[2], h, None, f64(w)[0], f64(rstd), "bf16")
    assert (dy[:, cols] == 55.0).all()


def test_quantize_far_offsets(cuda, cmb, room):
    rows, cols = 1000, 260
    src_pitch, pitch_t = up(9 * 2 ** 29 // rows, 16), up(9 * 2 ** 29 // cols, 16)
    rng = np.random.default_rng(9)
    x = far_rows(cuda, rows, cols, src_pitch, cuda.bfloat16, 55.0)
    x[:, :cols] = cuda.from_numpy(activations(rng, rows, cols))
    q = far_rows(cuda, rows, cols, src_pitch, cuda.uint8, FILL)
    qt = far_rows(cuda, cols, rows, pitch_t, cuda.uint8, FILL)
    s, st = bytes_buffer(cuda, rows, 3)[1], bytes_buffer(cuda, cols, 8)[1]
    cmb.check("cmb_quantize_e4m3_block128", addr(x), BF16, rows, cols, src_pitch, 1, addr(q),
              src_pitch, addr(s), 3, addr(qt), pitch_t, addr(st), 8, stream_handle(cuda))
    got = [t.cpu().numpy() for t in (q[:, :cols], s, qt[:, :rows], st)]
    same_quantized(got, f64(x[:, :cols]), 1)
    assert (q[:, cols] == FILL).all() and (qt[:, rows] == FILL).all()
    q[:, :cols], s[:] = FILL, FILL
    cmb.check("cmb_quantize_e4m3_block128", addr(x), BF16, rows, cols, src_pitch, 1, addr(q),
              src_pitch, addr(s), 3, None, 0, None, 0, stream_handle(cuda))
    same_quantized([q[:, :cols].cpu().numpy(), s.cpu().numpy(), None, None], f64(x[:, :cols]), 1)


FIRST_IN_A_GRAPH = """
import torch
import cuda_micro_bench_b200 as cmb
from tests.test_block128_gpu import Layer
for tokens in (1, 200):
    L = Layer(torch, cmb, tokens, 640, 500, 1)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        L.forward()
        L.backward()
    graph.replay()
    torch.cuda.synchronize()
    got = {n: t.clone() for n, t in L.outputs().items()}
    L.forward()
    L.backward()
    torch.cuda.synchronize()
    assert all(torch.equal(t, got[n]) for n, t in L.outputs().items())
    assert int(L.status.item()) == 0
print("same")
"""


def test_first_call_of_a_process_is_captured(cuda):
    """What the library asks the driver once (addresses, how many clusters fit)
    may be asked while a stream is captured."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH], cwd=root,
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]


def test_command_line_runs_and_checks_the_layer(cuda, tmp_path):
    """`--tensor-ext` times the operators at 8192^3, checks samples of each
    against fp64 and logs what the validator accepts."""
    import json
    import os
    import subprocess

    from cuda_micro_bench_b200 import validate_results

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = tmp_path / "results.json"
    p = subprocess.run([os.path.join(root, "cuda_micro_bench_b200", "bin", "cmb_b200"),
                        "--tensor-ext", f"--out={out}"], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stdout[-2000:] + p.stderr[-2000:]
    doc = json.loads(out.read_text())
    got = doc["results"]["fp8_block128"]
    assert set(got) == {"gemm_8192_tflops", "gemm_8192_max_rel_err", "quantize_8192_gbps",
                        "rmsnorm_8192_gbps", "rmsnorm_backward_8192_gbps", "verified"}
    assert got["verified"]["value"] == 1.0
    assert [m for m in validate_results.check(doc, full=False) if "fp8_block128" in m] == []
