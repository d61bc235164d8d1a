"""Inputs in a floating type and their values in float64 (not collected)."""
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
