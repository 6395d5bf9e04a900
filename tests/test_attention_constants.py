"""The polynomial exponential of the attention kernels meets the error bound
its comment states. The constants are read from the source; the f32 steps are
evaluated one by one as the kernel does them."""
import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(__file__), "..", "mlk2_b200", "csrc", "tc_common.cuh")


def _coefficients():
    with open(SOURCE) as f:
        src = f.read()
    body = src[src.index("uint64_t ex2_poly(uint64_t x2)"):]
    body = body[:body.index("\n}")]
    first = re.search(r"fma2\(f, pair\(([^,]+), [^)]+\), pair\(([^,]+), [^)]+\)\)", body)
    rest = re.findall(r"fma2\(p, f, pair\(([^,]+), [^)]+\)\)", body)
    values = [np.float32(c.rstrip("f")) for c in (*first.groups(), *rest)]
    assert len(values) == 5
    return values


def _fma(a, b, c):
    # products of two f32 are exact in 64 bits
    return (a.astype(np.float64) * b.astype(np.float64) + np.float64(c)).astype(np.float32)


def ex2_poly(x):
    c = _coefficients()
    v = np.maximum(x.astype(np.float32), np.float32(-126))
    t = v + np.float32(12582912)
    f = v - (t - np.float32(12582912))
    p = _fma(f, c[0], c[1])
    for k in c[2:]:
        p = _fma(p, f, k)
    i = (t.view(np.int32).astype(np.int64) << 23) & 0xffffffff
    return ((p.view(np.int32).astype(np.int64) + i) & 0xffffffff).astype(np.uint32).view(np.float32)


def test_ex2_poly_error():
    """2.7e-6 relative from -126 to 120."""
    x = np.linspace(-126, 120, 4000001).astype(np.float32)
    err = np.abs(ex2_poly(x).astype(np.longdouble) / np.exp2(x.astype(np.longdouble)) - 1)
    assert err.max() < 2.75e-6, err.max()


def test_ex2_poly_far_below():
    """Arguments below -126 give 2^-126, within the same error."""
    x = np.float32([-126, -126.5, -1000, -3e38, -np.inf])
    assert np.all(np.abs(ex2_poly(x) / np.float64(2.0) ** -126 - 1) < 2.75e-6)
