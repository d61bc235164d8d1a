"""packed_attention and cached_attention in fp16 where one key takes nearly all of a row and holds nothing, so that what the row
gives is made of many keys whose probabilities fp16 itself cannot hold (2^-24.5 of the largest, half a step of 2^-24 apart).

Bounds: as in typed_inputs.attend, but a probability is rounded as a multiple of 2^-31 of the largest: fp16 ones are held
times 2^7 or more, their last place is 2^-24, so each is off by at most 2^-25 / 2^7 = 2^-32 of the largest one."""
import numpy as np
import pytest

from cinn_amd.common import Int
from cinn_amd.frontend import NetBuilder

from helpers import run
from typed_inputs import ULP, assert_within, dtype, rounded

pytestmark = pytest.mark.gpu

D, TOP = 64, 17.0


def spread(values):
    """out and its bound for rows that see the first key, whose value is zero, and values [others][heads][d]; [rows][heads][d]
    with one more of them a row"""
    total = np.cumsum(values, 0)
    others = np.arange(1, len(values) + 1)[:, None, None]
    p = np.exp(-TOP) / (1 + others * np.exp(-TOP))
    score = (2.0 ** -24 * D ** 0.5 + 2.0 ** -22) * TOP
    u = ULP["float16"]
    out = p * total
    return out, (2 * score + 2.0 ** -18 + 3 * u) * out + (others + 1) * 2.0 ** -32 * values.max() + 2.0 ** -25


def data(rng, rows, heads, kv_heads):
    """queries along the first element, keys across it but for the first, whose score is TOP; values above zero"""
    q, k = np.zeros((rows, heads, D)), rng.standard_normal((rows, kv_heads, D))
    q[..., 0], k[..., 0], k[0] = 8, 0, 0
    k[0, :, 0] = TOP
    v = np.abs(rng.standard_normal((rows, kv_heads, D))) * 30
    v[0] = 0
    return q.astype(np.float16), rounded(k, "float16")[0], rounded(v, "float16")


# blocks of 128 pairs: 1, 25, 176, 544, 576, which four kinds of blocks take
@pytest.mark.parametrize("rows,heads,kv_heads", [(200, 1, 1), (400, 8, 1), (1500, 16, 16), (1100, 64, 16), (1200, 64, 64)])
def test_prompts(gpu, rows, heads, kv_heads):
    q, k, (v, vf) = data(np.random.default_rng(rows), rows, heads, kv_heads)
    b = NetBuilder("packed")
    Q, K, V = (b.create_input(dtype("float16"), list(x.shape), n) for n, x in (("q", q), ("k", k), ("v", v)))
    O = b.create_input(Int(32), [2], "offsets")
    (got,), _ = run(b, {Q: q, K: k, V: v, O: np.array([0, rows], np.int32)}, [b.packed_attention(Q, K, V, O)])
    want, bound = (np.repeat(x, heads // kv_heads, 1) for x in spread(vf[1:]))
    assert not got[0].any()
    assert_within(got[1:], want, bound, "float16")


@pytest.mark.parametrize("first", [0, 300])
@pytest.mark.parametrize("tokens,heads,length", [(1, 2, 1400), (12, 4, 1400), (24, 4, 380), (40, 4, 380), (45, 8, 350), (64, 8, 350), (5, 4, 9000), (64, 8, 3100)])
def test_caches(gpu, tokens, heads, length, first):
    """the key that takes nearly all at the front of the cache and further back; one block a unit and several"""
    kv_heads, page = 2, 32
    q, k, (v, vf) = data(np.random.default_rng(tokens), length + tokens, heads, kv_heads)
    want, bound = (np.repeat(x[-tokens:], heads // kv_heads, 1) for x in spread(vf[1:]))
    for x in (k, v):
        x[[0, first]] = x[[first, 0]]
    table = np.random.default_rng(1).permutation(-(-length // page)).astype(np.int32)

    def pages(x):
        held = np.zeros((len(table), page, kv_heads, D), np.float16)
        held[table] = np.pad(x[:length], ((0, -length % page), (0, 0), (0, 0))).reshape(held.shape)
        return held
    for columns in (len(table), 4 * len(table)):
        feeds = {"q": q[None, length:], "k": k[None, length:], "v": v[None, length:], "k_pages": pages(k), "v_pages": pages(v),
                 "table": np.resize(table, (1, columns)), "lengths": np.array([length], np.int32)}
        b = NetBuilder("cached")
        var = [b.create_input(Int(32) if x.dtype == np.int32 else dtype("float16"), list(x.shape), n) for n, x in feeds.items()]
        (got,), _ = run(b, {n: np.ascontiguousarray(x) for n, x in feeds.items()}, [b.cached_attention(*var)])
        assert_within(got[0], want, bound, "float16")
