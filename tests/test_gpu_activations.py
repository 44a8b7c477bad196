"""The activations of linear_act by themselves (identity weights) over all values of the 16-bit types and many of fp32: an
error relative to the result, in the tails too, where the result is small beside its argument."""
import numpy as np
import pytest
from scipy.special import expit, ndtr

import rows64 as ref
import sparse_hip as sh

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in DTYPES}
    yield bes
    for b in bes.values():
        b.destroy()


def arguments(dtype):
    """All finite values of a 16-bit type, as float32 (normal numbers of it); of fp32 steps of 2^-13 to 16 and every 2^-6 of a
    power of two."""
    if dtype == sh.F16:
        z = np.arange(1 << 16, dtype=np.uint16).view(np.float16).astype(np.float32)
    elif dtype == sh.BF16:
        z = (np.arange(1 << 16, dtype=np.uint32) << 16).view(np.float32)
    else:
        far = np.exp2(np.arange(-40, 120, 2.0 ** -6))
        near = np.arange(0, 16, 2.0 ** -13)
        z = np.concatenate([near, -near, far, -far]).astype(np.float32)
    return z[np.isfinite(z) & ((np.abs(z) >= 2.0 ** -126) | (z == 0))]


def exact(z, act):
    """(value, bound on the relative error, bound on an absolute one), with no subtraction of nearly equal numbers.

    E is half a step of fp32; the hardware's reciprocal and exponential are within 2 E each.  SiLU: those two, the sum, the
    product, and the exponential's argument, |z| with two roundings: (6 + 2 |z|) E, doubled.  GELU with tanh: the argument
    2 u passes six roundings: (6 + 6 |2 u|) E.  GELU of fp32: t = 1 / (1 + p a) 3 E, times up to 2.4 where the tail's factor
    t Q(t) is steepest, Q's last steps 3 E, three products 3 E, an exponential 2 E: 16 E; its argument a^2 / 2 three roundings.
    Of 16 bits: an exponential 2 E, one minus it and the product 2 E, and the polynomial that is its argument, whose last
    two steps or three are as large as itself, some a^2 / 2 + 3: within the same.  And the fit, 2^-12 in bf16, 2^-14.5 in
    fp16 or 2^-28, 2^-25.2 in fp32.  Exponentials and reciprocals
    below 2^-126 may be zero, which |z| multiplies."""
    a, z = np.abs(z.astype(np.float64)), z.astype(np.float64)
    if act == "silu":
        y, rel = z * expit(z), 2 * (6 + 2 * a) * ref.E
    elif act == "gelu_tanh":
        with np.errstate(over="ignore"):
            u = 2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)
        y, rel = z * expit(u), (6 + 6 * np.minimum(np.abs(u), 200)) * ref.E
    elif act == "gelu":
        y, rel = z * ndtr(z), (16 + 1.5 * np.minimum(a, 20) ** 2) * ref.E
    else:
        y, rel = z, 0 * a
    # Where the factor of z is one, so are the computed exponential's neighbours: nothing but the product's rounding.
    return y, np.where(z > 100, 4 * ref.E, rel), 2.0 ** -126 * a


FIT = {sh.F32: 2.0 ** -25.2, sh.F16: 2.0 ** -14.5, sh.BF16: 2.0 ** -12}


@pytest.mark.parametrize("act", list(sh.ACTS))
@pytest.mark.parametrize("width", [16, 1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_relative_error(backends, dtype, width, act):
    """Through the MFMA kernel (rows of 16) and through the general one (rows of one value)."""
    be, z = backends[dtype], arguments(dtype)
    z = np.concatenate([z, np.zeros(-z.size % width, np.float32)])
    n = z.size // width
    y = be.alloc(z.size)
    be.linear_act(be.upload(z.reshape(n, width)), np.eye(width, dtype=np.float32), None, y, n, width, width, act=act)
    exp, rel, low = exact(z, act)
    err = rel * np.abs(exp) + low
    if act == "gelu":
        err = err + np.maximum(FIT[dtype] * np.abs(exp), 2.0 ** -28 if dtype == sh.F16 else 0.0)
    # The rounding is of the computed value, err beside the exact one.
    ref.check(be.download(y), exp, 1.01 * err + ref.stored(exp, dtype), act)


@pytest.mark.parametrize("act", list(sh.ACTS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_not_finite(backends, dtype, act):
    """An infinity stays one, a NaN a NaN, and -infinity is -infinity times zero (itself without an activation)."""
    be, y = backends[dtype], backends[dtype].alloc(3)
    x = np.array([np.inf, np.nan, -np.inf], np.float32)
    be.linear_act(be.upload(x), np.ones((1, 1), np.float32), None, y, 3, 1, 1, act=act)
    got = be.download(y)
    assert got[0] == np.inf and np.isnan(got[1]) and (got[2] == -np.inf if act == "none" else np.isnan(got[2]))
