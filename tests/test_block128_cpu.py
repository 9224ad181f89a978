"""CPU tests of the block-scaled e4m3 operators: every refusal comes before
any device call, and the 64-bit implementation that the GPU tests compare
with holds its own definition."""

import ctypes

import numpy as np
import pytest

from tests import block128_ref as ref

P = ctypes.c_void_p(4096)  # never read: the calls below are refused first
Q = ctypes.c_void_p(4096 + 1)
INVALID, UNSUPPORTED = 1, 4
BF16, F32 = 0, 1


def _refused(cmb, fn, args, word):
    rc = getattr(cmb.lib, fn)(*args)
    assert rc == INVALID, (fn, args, rc)
    text = cmb.lib.cmb_last_error().decode()
    assert text.startswith(fn + ":") and word in text, text


def _with(base, **change):
    d = dict(base, **change)
    return list(d.values())


QUANT = dict(src=P, src_type=BF16, rows=4, cols=300, ld_src=300, block_rows=1, dst=P, ld_dst=304,
             scale=P, ld_scale=3, dst_t=P, ld_dst_t=16, scale_t=P, ld_scale_t=1, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(src_type=2), "src_type"), (dict(src_type=-1), "src_type"),
    (dict(block_rows=0), "block_rows"), (dict(block_rows=64), "block_rows"),
    (dict(rows=-1), "values"), (dict(cols=-4), "values"),
    (dict(rows=2**31 - 1), "values"), (dict(cols=2**31 - 1), "values"),
    (dict(scale=None), "together"), (dict(dst=None), "together"), (dict(dst_t=None), "together"),
    (dict(scale_t=None), "together"),
    (dict(dst=None, scale=None, dst_t=None, scale_t=None), "nothing"),
    (dict(src=None), "src"), (dict(src=Q), "src"), (dict(src=ctypes.c_void_p(4098), src_type=F32), "src"),
    (dict(ld_src=299), "overlap"), (dict(ld_dst=299), "overlap"), (dict(ld_scale=2), "overlap"),
    (dict(ld_dst_t=3), "overlap"), (dict(ld_scale_t=0), "overlap")])
def test_quantize_refusals(cmb, change, word):
    _refused(cmb, "cmb_quantize_e4m3_block128", _with(QUANT, **change), word)


GEMM = dict(A=P, lda=304, sa=P, ld_sa=3, B=P, ldb=304, sb=P, ld_sb=3, block_rows_b=128, C=P,
            ldc=200, c_type=BF16, M=5, N=200, K=300, status=None, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(c_type=3), "c_type"), (dict(block_rows_b=2), "block_rows_b"), (dict(M=-1), "M -1"),
    (dict(N=-1), "N -1"), (dict(K=-1), "K -1"), (dict(M=2**31 - 1), "M 2147483647"),
    (dict(N=2**31 - 1), "N 2147483647"), (dict(K=2**28 + 1, lda=2**29, ldb=2**29, ld_sa=2**22, ld_sb=2**22), "K 268435457"), (dict(status=Q), "status"), (dict(C=None), "C is"),
    (dict(C=Q), "C is"), (dict(C=ctypes.c_void_p(4098), c_type=F32), "C is"),
    (dict(ldc=199), "ldc"), (dict(A=None), "null"), (dict(B=None), "null"), (dict(sa=None), "null"),
    (dict(sb=None), "null"), (dict(A=ctypes.c_void_p(4104)), "16-byte"), (dict(lda=312), "16"),
    (dict(ldb=300), "16"), (dict(B=Q), "16-byte"), (dict(lda=288), "overlap"),
    (dict(ldb=288), "overlap"), (dict(ld_sa=2), "overlap"), (dict(ld_sb=2), "overlap")])
def test_gemm_refusals(cmb, change, word):
    _refused(cmb, "cmb_gemm_e4m3_block128", _with(GEMM, **change), word)


NORM = dict(x=P, ld_x=300, residual=P, ld_residual=300, type=BF16, weight=P, weight_type=BF16,
            eps=ctypes.c_float(1e-5), rows=4, cols=300, h=P, ld_h=300, y=P, ld_y=300, q=P,
            ld_q=304, scale=P, ld_scale=3, rstd=P, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(type=2), "types"), (dict(weight_type=7), "types"), (dict(rows=-1), "rows"),
    (dict(rows=2**31 - 1), "rows"),
    (dict(cols=0), "columns"), (dict(cols=32769), "columns"), (dict(eps=ctypes.c_float(-1)), "eps"),
    (dict(eps=ctypes.c_float(float("nan"))), "eps"), (dict(q=None), "together"),
    (dict(scale=None), "together"), (dict(residual=None), "together"), (dict(h=None), "together"),
    (dict(residual=None, h=None, y=None, q=None, scale=None, rstd=None), "nothing"),
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(x=Q), "x is not aligned"),
    (dict(h=Q), "h is not aligned"), (dict(y=Q), "y is not"), (dict(weight=Q), "weight is not"),
    (dict(rstd=Q), "rstd is not"), (dict(ld_x=299), "rows of x"),
    (dict(ld_residual=299), "rows of residual"), (dict(ld_h=299), "rows of h"),
    (dict(ld_y=299), "rows of y"), (dict(ld_q=299), "rows of q"), (dict(ld_scale=2), "scale")])
def test_norm_refusals(cmb, change, word):
    _refused(cmb, "cmb_rmsnorm_e4m3_block128", _with(NORM, **change), word)


BACK = dict(dy=P, ld_dy=300, h=P, ld_h=300, dh=P, ld_dh=300, type=F32, weight=P, weight_type=F32,
            rstd=P, rows=4, cols=300, dx=P, ld_dx=300, dweight=P, workspace=P,
            workspace_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(type=2), "types"), (dict(rows=-1), "rows"), (dict(cols=0), "columns"),
    (dict(dy=None), "null"), (dict(h=None), "null"), (dict(weight=None), "null"),
    (dict(rstd=None), "null"), (dict(dx=None), "null"), (dict(dy=Q), "dy is"), (dict(dx=Q), "dx is"),
    (dict(dh=Q), "dh is"), (dict(dweight=Q), "dweight"), (dict(ld_dy=299), "rows of dy"),
    (dict(ld_h=299), "rows of h"), (dict(ld_dh=299), "rows of dh"), (dict(ld_dx=299), "rows of dx"),
    (dict(workspace=None), "workspace"), (dict(workspace=ctypes.c_void_p(4104)), "workspace"),
    (dict(workspace_bytes=100), "workspace of 100")])
def test_norm_backward_refusals(cmb, change, word):
    _refused(cmb, "cmb_rmsnorm_backward", _with(BACK, **change), word)


def test_empty_calls_touch_nothing(cmb):
    """No rows or columns: done before any device call (there is none here)."""
    for change in (dict(rows=0), dict(cols=0)):
        assert cmb.lib.cmb_quantize_e4m3_block128(*_with(QUANT, **change)) == 0
    for change in (dict(M=0), dict(N=0)):
        assert cmb.lib.cmb_gemm_e4m3_block128(*_with(GEMM, **change)) == 0
    assert cmb.lib.cmb_rmsnorm_e4m3_block128(*_with(NORM, rows=0)) == 0
    assert cmb.lib.cmb_rmsnorm_backward(*_with(BACK, rows=0, dweight=None, workspace=None)) == 0


def test_backward_workspace_bytes(cmb):
    f = cmb.lib.cmb_rmsnorm_backward_workspace_bytes
    assert f(0, 100) == 0 and f(5, 0) == 0
    assert f(1, 1) >= 4 and f(7, 300) >= 4 * 300
    assert f(1 << 30, 8192) <= 1024 * 8192 * 4  # does not grow without end
    assert all(f(r, 300) <= f(r + 1, 300) for r in range(1, 2000, 37))


# ------------------------------------------------- the 64-bit implementation


def test_reference_encoder_matches_torch():
    import torch

    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-448, 448, 20000), ref.E4M3, -ref.E4M3,
                        (ref.E4M3[1:] + ref.E4M3[:-1]) / 2, rng.normal(0, 0.01, 20000)])
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn)
    x = torch.from_numpy(x).float().double().numpy()
    got = torch.from_numpy(ref.encode(x)).view(torch.float8_e4m3fn)
    assert torch.equal(got.float(), want.float())
    assert list(ref.encode(np.array([np.nan, np.inf, -np.inf]))) == [0x7F] * 3


def test_reference_scale_is_the_smallest_power_that_fits():
    tops = np.array([[448.0, 448.0001, 447.0, 1.75, 1.7500001, 0.0, 2.0 ** -140, 3e38, 1e-38]])
    s = ref.scale_bytes(tops)[0].astype(int) - 127
    assert list(s[:6]) == [0, 1, 0, -8, -7, 0] and s[6] == -127
    for t, e in zip(tops[0], s):
        if t:
            assert t / 2.0 ** e <= 448 and (e == -127 or t / 2.0 ** (e - 1) > 448)


def test_reference_gradient_matches_differences():
    """The backward formula against central differences of the forward one."""
    rng = np.random.default_rng(1)
    h, w, dy = rng.normal(size=(3, 20)), 1 + 0.1 * rng.normal(size=20), rng.normal(size=(3, 20))
    rstd, _ = ref.norm(h, w, 1e-5)
    dx, dw = ref.norm_backward(dy, h, w, rstd, np.zeros_like(h))
    loss = lambda h_, w_: (ref.norm(h_, w_, 1e-5)[1] * dy).sum()
    d = 1e-6
    for i in range(3):
        for j in range(20):
            e = np.zeros_like(h)
            e[i, j] = d
            assert abs((loss(h + e, w) - loss(h - e, w)) / (2 * d) - dx[i, j]) < 1e-7
    for j in range(20):
        e = np.zeros_like(w)
        e[j] = d
        assert abs((loss(h, w + e) - loss(h, w - e)) / (2 * d) - dw[j]) < 1e-7


def test_validator_knows_the_layer():
    from cuda_micro_bench_b200 import validate_results

    def problems(**change):
        v = dict(gemm_8192_tflops=2700.0, gemm_8192_max_rel_err=1e-6, quantize_8192_gbps=5000.0,
                 rmsnorm_8192_gbps=5900.0, rmsnorm_backward_8192_gbps=5900.0, verified=1.0)
        v.update(change)
        doc = {"device": "NVIDIA B200", "architecture": "10.0", "sm_count": 148,
               "results": {"fp8_block128": {k: {"value": x, "unit": ""} for k, x in v.items()}}}
        return validate_results.check(doc, full=False)

    assert problems() == []
    for change in (dict(gemm_8192_tflops=5000.0), dict(rmsnorm_8192_gbps=9000.0),
                   dict(verified=0.0), dict(gemm_8192_max_rel_err=0.5)):
        assert len(problems(**change)) == 1, change
