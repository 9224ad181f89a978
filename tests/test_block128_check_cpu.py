"""CPU tests of the checks that the command line's block-scaled e4m3 section makes of
its own outputs: right ones pass, and one wrong byte, scale or sum does not."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

from tests import block128_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "block128_check.h"
using namespace cmb::check;
extern "C" {
int encode(double x) { return e4m3_nearest(x); }
double decode(int code) { return e4m3_value((uint8_t)code); }
int scale(double top) { return scale_byte(top); }
int block(const double *x, const uint8_t *q, int s, int rows, int cols) {
  return block_holds([&](int r, int c) { return x[r * cols + c]; },
                     [&](int r, int c) { return q[r * cols + c]; }, s, rows, cols);
}
int sum(double got, const double *x, int n, int depth) {
  return sum_holds(got, [&](int i) { return x[i]; }, n, depth);
}
}
"""


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    home = tmp_path_factory.mktemp("checks")
    (home / "checks.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "cuda_micro_bench_b200", "csrc", "host"),
                    str(home / "checks.cpp"), "-o", str(home / "checks.so")], check=True)
    lib = ctypes.CDLL(str(home / "checks.so"))
    lib.decode.restype = ctypes.c_double
    lib.encode.argtypes = lib.scale.argtypes = [ctypes.c_double]
    lib.sum.argtypes = [ctypes.c_double, ctypes.c_void_p, ctypes.c_int, ctypes.c_int]
    lib.block.argtypes = [ctypes.c_void_p, ctypes.c_void_p] + [ctypes.c_int] * 3
    return lib


def test_codes_and_scales(checks):
    rng = np.random.default_rng(0)
    assert all(checks.decode(c) == ref.VALUES[c] for c in range(256) if c & 0x7F != 0x7F)
    assert np.isnan(checks.decode(0x7F)) and np.isnan(checks.decode(0xFF))
    ties = (ref.E4M3[1:] + ref.E4M3[:-1]) / 2
    x = np.concatenate([rng.uniform(-448, 448, 2000), rng.normal(0, 0.01, 2000), ties, -ties,
                        [0.0, -0.0, 448.0, -448.0]])
    assert [checks.encode(v) for v in x] == list(ref.encode(x))
    tops = np.array([[448.0, 448.0001, 3.5, 1.75, 1.7500001, 0.0, 2.0 ** -140, 3e38]])
    assert [checks.scale(t) for t in tops[0]] == list(ref.scale_bytes(tops)[0])


def test_block_of_weights(checks):
    rng = np.random.default_rng(1)
    x = rng.normal(size=(128, 128))
    q, s = ref.quantize(x, 128)
    holds = lambda q_, s_: checks.block(x.ctypes.data, q_.ctypes.data, int(s_), 128, 128)
    assert holds(q, s[0, 0]) == 1
    for byte in (s[0, 0] + 1, s[0, 0] - 1):  # the same values under the next scales
        wrong = ref.encode(np.clip(x / 2.0 ** (float(byte) - 127), -448, 448))
        assert holds(q, byte) == 0 and holds(wrong, byte) == 0
    for at in ((0, 0), (127, 127), (64, 3)):
        wrong = q.copy()
        wrong[at] ^= 1
        assert holds(wrong, s[0, 0]) == 0


def test_column_sum(checks):
    rng = np.random.default_rng(2)
    t = rng.normal(size=8192)
    in_order = np.float32(0)
    for part in t.astype(np.float32).reshape(128, 64):  # 64 rows a CTA, then 128 parts
        in_order += np.cumsum(part, dtype=np.float32)[-1]
    holds = lambda got, depth: checks.sum(float(got), t.ctypes.data, 8192, depth)
    assert holds(in_order, 8192 // 128 + 128 + 1) == 1
    assert holds(np.delete(t, 77).sum(), 128) == 0  # a row is missing
    assert holds(0.0, 128) == 0 and holds(float("nan"), 128) == 0 and holds(9.0, 128) == 0


def test_validator_holds_the_product_to_its_sums():
    from cuda_micro_bench_b200 import validate_results

    def problems(err):
        doc = {"device": "NVIDIA B200", "architecture": "10.0", "sm_count": 148,
               "results": {"fp8_block128": {"gemm_8192_max_rel_err": {"value": err, "unit": ""}}}}
        return [p for p in validate_results.check(doc, full=False) if "max_rel_err" in p]

    assert problems(1e-6) == []
    for err in (2e-5, 1e-3, 0.5, float("nan")):
        assert len(problems(err)) == 1, err
