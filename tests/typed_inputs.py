"""Inputs in a floating type, their values in float64, and attention of one head in float64 (not collected)."""
import math

import numpy as np

from cinn_amd.common import BFloat16, Float, bfloat16_bits_to_float32, float32_to_bfloat16_bits

# half a step of each type, relative to the value
ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TYPES = sorted(ULP)


def rounded(values, kind):
    """values as the type holds them (bfloat16: bit patterns), and in float64"""
    v = np.asarray(values, np.float32)
    if kind == "bfloat16":
        bits = float32_to_bfloat16_bits(v)
        return bits, bfloat16_bits_to_float32(bits).astype(np.float64)
    v = v.astype(kind)
    return v, v.astype(np.float64)


def normal(rng, shape, kind, scale=1.0):
    return rounded(rng.standard_normal(shape) * scale, kind)


def as_float64(x, kind):
    return (bfloat16_bits_to_float32(x) if kind == "bfloat16" else x).astype(np.float64)


def dtype(kind):
    return BFloat16() if kind == "bfloat16" else Float(32 if kind == "float32" else 16)


def assert_within(got, want, bound, kind):
    """got, in its type, within bound of float64 values, element by element"""
    over = np.abs(as_float64(got, kind) - want) - bound
    over = np.where(np.isnan(over), np.inf, over)
    assert got.shape == want.shape and over.max() <= 0, "%d of %d out of bounds, the worst by %g at %s: %r, wanted %r +- %r" % (
        (over > 0).sum(), over.size, over.max(), np.unravel_index(over.argmax(), over.shape),
        as_float64(got, kind).flat[over.argmax()], want.flat[over.argmax()], np.broadcast_to(bound, want.shape).flat[over.argmax()])


def attend(q, k, v, allowed, scale, kind):
    """float64 result and the bound on its error; what is not allowed is left out.  A score is an fp32 sum of d products (2^-24
    sqrt(d) + 2^-22 of the products' magnitudes); the relative error of a probability is twice that and what exp adds (its
    argument's rounding, 2^-24 of up to 32, and its own 2^-21), together under 2^-18.  16-bit operands of the second product
    are rounded probabilities (half a step, subnormal ones 2^-25), as are their sums' (another half); the result rounds
    once."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    u = ULP[kind]
    for i in range(q.shape[0]):
        kk, vv = k[allowed[i]], v[allowed[i]]
        if not len(kk):
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (kk @ q[i])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i] = p @ vv
            score = (2.0 ** -24 * math.sqrt(q.shape[1]) + 2.0 ** -22) * abs(scale) * (np.abs(kk) @ np.abs(q[i])).max()
            bound[i] = (2 * score + 2.0 ** -18 + 2 * u) * (p @ np.abs(vv)) + u * np.abs(out[i])
            if kind == "float16":
                bound[i] += len(kk) * 2.0 ** -25 * np.abs(vv).max() + 2.0 ** -24
    return out, bound
