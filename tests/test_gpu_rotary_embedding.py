"""rotary_embedding and its gradient (rotary.hip) against float64: every width of access, both orders of pairs, heads out of
packed projections, part of a head, far positions, scaled frequencies.

Bounds: the angle's fraction of a turn is rounded once to fp32 (up to half a turn: pi 2^-24 of angle), sine and cosine are
off by less than 2^-23 and rounded again by the magnitude, 2^-24; two products and a sum round three times.  Together less
than 10 * 2^-24 of |u| + |v|, times the magnitude, and the result's own rounding."""
import math

import numpy as np
import pytest

from cinn_amd.common import Int
from cinn_amd.frontend import NetBuilder

from helpers import run
from typed_inputs import TYPES, ULP, assert_within, dtype, normal

pytestmark = pytest.mark.gpu


def frequencies(r, theta=10000.0, factor=1.0, original_length=0, low=1.0, high=4.0):
    f = np.array([theta ** (-2.0 * i / r) for i in range(r // 2)])
    if not original_length:
        return f / factor
    g = np.clip((original_length * f / (2 * math.pi) - low) / (high - low), 0, 1)
    return f * (g + (1 - g) / factor)


def reference(x, positions, heads, r, interleaved, sign, magnitude, kind, **scaling):
    """float64 result and the bound on its error"""
    x = x[..., :heads, :]
    angle = sign * positions.astype(np.float64)[..., None, None] * frequencies(r, **scaling)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
    first = np.arange(0, r, 2) if interleaved else np.arange(r // 2)
    second = first + (1 if interleaved else r // 2)
    y, bound = x.copy(), np.zeros_like(x)
    u, v = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * c - v * s, v * c + u * s
    bound[..., first] = bound[..., second] = (np.abs(u) + np.abs(v)) * 10 * 2.0 ** -24 * abs(magnitude)
    tiny = 2.0 ** -25 if kind == "float16" else 2.0 ** -134
    return y, bound + np.where(bound > 0, ULP[kind] * np.abs(y) + tiny, 0)


def check(kind, lead, total, heads, d, r, interleaved, far, grad=False, wide=False, magnitude=1.0, **scaling):
    rng = np.random.default_rng(d * 131 + total)
    x, xf = normal(rng, (*lead, total, d), kind)
    positions = rng.integers(0, far, lead).astype(np.int64 if wide else np.int32)
    positions.flat[0] = far - 1
    b = NetBuilder("rotary")
    X = b.create_input(dtype(kind), list(x.shape), "x")
    P = b.create_input(Int(64 if wide else 32), list(lead), "positions")
    make = b.rotary_embedding_grad if grad else b.rotary_embedding
    y = make(X, P, heads=heads, rotary_dim=0 if r == d else r, interleaved=interleaved, magnitude=magnitude, **scaling)
    assert y.shape() == [*lead, heads or total, d]
    (got,), _ = run(b, {X: x, P: positions}, [y])
    want, bound = reference(xf, positions, heads or total, r, interleaved, -1 if grad else 1, magnitude, kind, **scaling)
    assert_within(got, want, bound, kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,total,heads,d,r", [
    ((1,), 1, 0, 2, 2), ((3,), 5, 3, 128, 128), ((2, 7), 6, 0, 64, 64), ((33,), 2, 1, 80, 32), ((5,), 3, 2, 24, 12),
    ((65,), 3, 0, 40, 18), ((9,), 2, 2, 7, 6), ((4,), 2, 0, 512, 512), ((257,), 40, 36, 16, 16), ((3, 2, 2), 4, 1, 10, 10)])
def test_shapes(gpu, kind, interleaved, lead, total, heads, d, r):
    check(kind, lead, total, heads, d, r, interleaved, 1000)
    check(kind, lead, total, heads, d, r, interleaved, 1000, grad=True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("far,wide", [(1 << 20, False), ((1 << 31) - 1, False), (1 << 31, True)])
def test_far_positions(gpu, kind, far, wide):
    """the angle itself, a product of a rounded frequency, is only known to a share of its size"""
    rng = np.random.default_rng(1)
    x, xf = normal(rng, (4, 2, 64), kind)
    positions = np.array([far - 1, far // 2, far // 3, 0], np.int64 if wide else np.int32)
    b = NetBuilder("far")
    X = b.create_input(dtype(kind), [4, 2, 64], "x")
    P = b.create_input(Int(64 if wide else 32), [4], "positions")
    (got,), _ = run(b, {X: x, P: positions}, [b.rotary_embedding(X, P)])
    want, bound = reference(xf, positions, 2, 64, False, 1, 1.0, kind)
    # a power on either side (2^-52 each), the product on either side, a division and 2 pi (2^-53 each): 2^-50 of the angle
    angle = positions[:, None, None] * frequencies(64)
    slack = np.concatenate([2.0 ** -50 * angle] * 2, axis=-1) * (np.abs(xf) + np.abs(np.roll(xf, 32, -1)))
    assert_within(got, want, bound + slack, kind)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("scaling", [
    dict(factor=4.0), dict(factor=8.0, original_length=8192, theta=500000.0), dict(factor=2.5, original_length=4096, low=1.0, high=32.0),
    dict(theta=1e6, magnitude=1.25), dict(factor=40.0, original_length=4096, low=1.0, high=32.0, magnitude=0.1 * math.log(40.0) + 1.0)])
def test_scaling(gpu, kind, scaling):
    check(kind, (70,), 4, 3, 64, 64, False, 200000, **scaling)
    check(kind, (70,), 4, 0, 96, 48, True, 200000, grad=True, **scaling)


def test_gradient_is_that_of_differences(gpu):
    """sum(w y) for a small step in one element of x, fp32: the map is linear, so the difference quotient is exact but for
    rounding: 2^-24 of sums of 64 terms of up to 8, over a step of 1"""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 2, 16)).astype(np.float32)
    w = rng.standard_normal((3, 2, 16)).astype(np.float32)
    positions = np.array([1, 50, 999], np.int32)
    options = dict(rotary_dim=12, interleaved=True, theta=100.0, magnitude=1.5)

    def through(method, data):
        b = NetBuilder("rotary")
        X, P = b.create_input(dtype("float32"), [3, 2, 16], "x"), b.create_input(Int(32), [3], "positions")
        return run(b, {X: data, P: positions}, [getattr(b, method)(X, P, **options)])[0][0].astype(np.float64)

    grad = through("rotary_embedding_grad", w)
    base = through("rotary_embedding", x)
    for at in ((0, 0, 0), (1, 1, 5), (2, 0, 11), (2, 1, 14)):
        step = x.copy()
        step[at] += 1.0
        difference = (w * (through("rotary_embedding", step) - base)).sum()
        assert abs(difference - grad[at]) <= 64 * 8 * 2.0 ** -24 * 4


@pytest.mark.parametrize("graph", [False, True])
def test_replayed_with_other_positions(gpu, graph):
    """one compiled program, positions and data changed between its executions"""
    from cinn_amd import runtime
    from cinn_amd.common import DefaultAMDGPUTarget
    from cinn_amd.frontend import Computation
    stream = runtime.Stream()
    b = NetBuilder("steps")
    X, P = b.create_input(dtype("float16"), [5, 3, 32], "x"), b.create_input(Int(32), [5], "positions")
    y = b.rotary_embedding(X, P)
    comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[y], stream=stream)
    for step in range(4):
        rng = np.random.default_rng(step)
        x, xf = normal(rng, (5, 3, 32), "float16")
        positions = rng.integers(-100, 5000, 5).astype(np.int32)
        comp.get_tensor("x").from_numpy(x)
        comp.get_tensor("positions").from_numpy(positions)
        (comp.execute_graph if graph else comp.execute)()
        stream.synchronize()
        want, bound = reference(xf, positions, 3, 32, False, 1, 1.0, "float16")
        assert_within(comp.get_tensor(y.id).numpy(), want, bound, "float16")
