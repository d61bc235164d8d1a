"""packed_attention (packed_attention.hip) against float64 at the edges of its tiles - 32 pairs of query and head per
wavefront, 32 to 256 per block, 32 keys per step - with empty sequences and single rows among the others, heads that share
keys, operands out of packed projections, rows of no sequence, infinities and NaN where nothing attends to them."""
import numpy as np
import pytest

from cinn_amd import runtime
from cinn_amd.common import DefaultAMDGPUTarget, Int
from cinn_amd.frontend import Computation, NetBuilder

from helpers import run
from typed_inputs import TYPES, as_float64, assert_within, attend, dtype, normal, rounded

pytestmark = pytest.mark.gpu


def causal(q, k, v, offsets, scale, kind):
    """[tokens][heads][d] operands of the heads in use"""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    group = q.shape[1] // k.shape[1]
    for first, end in zip(offsets[:-1], offsets[1:]):
        allowed = np.tril(np.ones((end - first, end - first), bool))
        for h in range(q.shape[1]):
            out[first:end, h], bound[first:end, h] = attend(q[first:end, h], k[first:end, h // group], v[first:end, h // group],
                                                            allowed, scale, kind)
    return out, bound


def program(kind, tokens, heads, kv_heads, d, sequences, **options):
    b = NetBuilder("packed")
    Q, K, V = (b.create_input(dtype(kind), [tokens, n, d], name) for name, n in (("q", heads), ("k", kv_heads), ("v", kv_heads)))
    O = b.create_input(Int(32), [sequences + 1], "offsets")
    return b, (Q, K, V, O), b.packed_attention(Q, K, V, O, **options)


def check(kind, lengths, heads, kv_heads, d, lead=0, rest=0, scale=None, seed=0):
    offsets = lead + np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    tokens = int(offsets[-1]) + rest
    rng = np.random.default_rng(seed + tokens * 7 + d)
    (q, qf), (k, kf), (v, vf) = (normal(rng, (tokens, n, d), kind) for n in (heads, kv_heads, kv_heads))
    b, inputs, o = program(kind, tokens, heads, kv_heads, d, len(lengths), **({} if scale is None else dict(scale=scale)))
    (got,), _ = run(b, dict(zip(inputs, (q, k, v, offsets))), [o])
    want, bound = causal(qf, kf, vf, offsets, d ** -0.5 if scale is None else scale, kind)
    assert_within(got, want, bound, kind)
    if lead:
        assert not as_float64(got, kind)[:lead].any()
    if rest:
        assert not as_float64(got, kind)[-rest:].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,d", [
    ([1], 1, 1, 8), ([2], 1, 1, 128), ([31], 2, 2, 64), ([32], 2, 1, 64), ([33], 3, 1, 40), ([63, 64, 65], 2, 2, 32),
    ([1, 0, 5, 0, 0, 1], 4, 2, 16), ([0, 17], 5, 1, 80), ([40, 0], 6, 2, 96), ([7] * 70, 2, 1, 24), ([1] * 130, 3, 3, 8),
    ([127], 8, 8, 120), ([129, 3], 8, 2, 128), ([200], 12, 4, 72), ([97, 300], 10, 5, 104), ([513], 4, 1, 112), ([700], 4, 4, 64),
    ([1025], 2, 2, 48)])
def test_edges(gpu, kind, lengths, heads, kv_heads, d):
    check(kind, lengths, heads, kv_heads, d)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,d", [
    ([300, 1, 0, 450, 77], 32, 8, 128), ([1100], 32, 8, 64), ([900, 40], 24, 12, 80), ([500, 500], 40, 8, 32)])
def test_many_heads(gpu, kind, lengths, heads, kv_heads, d):
    """enough blocks for the wide ones"""
    check(kind, lengths, heads, kv_heads, d, rest=3)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,heads", [([1100, 3, 0, 1040], 4), ([1, 2200, 16], 4), ([30, 17] * 8, 6), ([64, 0, 100, 1] * 4 + [65], 2),
                                           ([0] * 15 + [70], 3), ([5] * 64, 2), ([9] * 65, 1)])
def test_the_order_of_tiles(gpu, kind, lengths, heads):
    """sequences of more than 64 tiles, and as many as share one order of their tiles or do not"""
    check(kind, lengths, heads, 1, 32, lead=2, rest=1)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("lead,rest", [(0, 1), (0, 200), (5, 0), (70, 33)])
def test_rows_of_no_sequence_are_zero(gpu, kind, lead, rest):
    check(kind, [3, 0, 61], 6, 3, 40, lead, rest)
    check(kind, [0], 2, 2, 64, lead, rest + 1)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [1.0, -0.25, 0.0])
def test_scale(gpu, kind, scale):
    check(kind, [50, 90], 4, 2, 64, scale=scale)


@pytest.mark.parametrize("kind", TYPES)
def test_operands_in_packed_projections(gpu, kind):
    """q, k and v as heads of one tensor, and k rotated in another: the same bits as from tensors of their own"""
    rng = np.random.default_rng(2)
    tokens, heads, kv_heads, d = 150, 6, 2, 64
    offsets = np.array([0, 60, 61, 150], np.int32)
    qkv, _ = normal(rng, (tokens, heads + 2 * kv_heads, d), kind)
    spare, _ = normal(rng, (tokens, 1 + heads + kv_heads, d), kind)
    parts = {"q": spare[:, 1:1 + heads], "k": qkv[:, heads:heads + kv_heads], "v": qkv[:, heads + kv_heads:]}
    b = NetBuilder("parts")
    X, S = b.create_input(dtype(kind), list(qkv.shape), "qkv"), b.create_input(dtype(kind), list(spare.shape), "spare")
    O = b.create_input(Int(32), [4], "offsets")
    P = {n: b.create_input(dtype(kind), list(x.shape), n) for n, x in parts.items()}
    apart = b.packed_attention(P["q"], P["k"], P["v"], O)
    inside = b.packed_attention(S, X, X, O, heads=heads, kv_heads=kv_heads, q_head=1, k_head=heads, v_head=heads + kv_heads)
    one = b.packed_attention(X, X, X, O, heads=heads, kv_heads=kv_heads, k_head=heads, v_head=heads + kv_heads)
    feeds = {X: qkv, S: spare, O: offsets, **{P[n]: np.ascontiguousarray(x) for n, x in parts.items()}}
    (a, i, _), _ = run(b, feeds, [apart, inside, one])
    assert np.array_equal(a.view(np.uint8), i.view(np.uint8))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("at,heads", [(0, 1), (37, 4), (69, 4), (99, 1)])
def test_keys_behind_a_row_do_not_count(gpu, kind, at, heads, bad):
    """rows before `at` are as if it were not there, whatever its key and its value hold; other sequences too; from `at` on
    an infinite or NaN value is in the result"""
    rng = np.random.default_rng(4)
    tokens, d = 150, 64
    offsets = np.array([0, 100, 150], np.int32)
    (q, qf), (k, kf), (v, vf) = (normal(rng, (tokens, n, d), kind) for n in (heads, 1, 1))
    for which in (k, v):
        changed = {id(k): k.copy(), id(v): v.copy()}
        changed[id(which)][at, 0, 5] = rounded([bad], kind)[0][0]
        b, inputs, o = program(kind, tokens, heads, 1, d, 2)
        (got,), _ = run(b, dict(zip(inputs, (q, changed[id(k)], changed[id(v)], offsets))), [o])
        want, bound = causal(qf, kf, vf, offsets, d ** -0.5, kind)
        rows = np.r_[0:at, 100:150]
        assert_within(got[rows], want[rows], bound[rows], kind)
        got = as_float64(got, kind)
        if which is v:
            assert not np.isfinite(got[at:100, :, 5]).any()
            others = np.delete(got[at:100], 5, axis=2)
            assert np.isfinite(others).all()
        elif np.isnan(bad):
            assert np.isnan(got[at:100]).all()


@pytest.mark.parametrize("graph", [False, True])
def test_replayed_with_other_offsets(gpu, graph):
    """one compiled program for every division of its rows"""
    kind, tokens, d = "bfloat16", 120, 32
    stream = runtime.Stream()
    b, inputs, o = program(kind, tokens, 4, 2, d, 3)
    comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[o], stream=stream)
    for step, offsets in enumerate(([0, 40, 80, 120], [0, 0, 0, 120], [0, 1, 2, 3], [0, 120, 120, 120], [0, 77, 78, 100])):
        rng = np.random.default_rng(step)
        data = [normal(rng, (tokens, n, d), kind) for n in (4, 2, 2)]
        for name, (x, _) in zip("qkv", data):
            comp.get_tensor(name).from_numpy(x)
        comp.get_tensor("offsets").from_numpy(np.array(offsets, np.int32))
        (comp.execute_graph if graph else comp.execute)()
        stream.synchronize()
        want, bound = causal(*(f for _, f in data), offsets, d ** -0.5, kind)
        assert_within(comp.get_tensor(o.id).numpy(), want, bound, kind)


@pytest.mark.parametrize("offsets", [[0, 50, 20, 64], [-5, 3, 1 << 30, 64], [64, 0, 64, 0], [1 << 30, 1 << 30, 1 << 30, 1 << 30], [-9, -8, -7, -6]])
def test_offsets_out_of_order_or_range_stay_in_bounds(gpu, offsets):
    """the sequences that are as they should be are right; every offset is brought into 0 .. tokens first"""
    kind, tokens, d = "float16", 64, 32
    rng = np.random.default_rng(1)
    data = [normal(rng, (tokens, n, d), kind) for n in (2, 1, 1)]
    b, inputs, o = program(kind, tokens, 2, 1, d, 3)
    (got,), _ = run(b, dict(zip(inputs, [x for x, _ in data] + [np.array(offsets, np.int32)])), [o])
    if offsets[:2] == [0, 50]:
        want, bound = causal(*(f[:20] for _, f in data), [0, 20], d ** -0.5, kind)
        assert_within(got[:20], want, bound, kind)
