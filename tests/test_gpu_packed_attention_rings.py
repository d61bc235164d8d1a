"""packed_attention of 16-bit prompts that are not short: the blocks whose wavefronts share a ring of tiles.  Which kind a call takes
goes by its blocks of 128 pairs of query and head (packed_attention.hip): more than 128, eight wavefronts of which two share 32
queries; more than 512, eight or (fewer than four heads to a key head) four wavefronts with queries of their own.  Every case
says which of them it is.

Every row of every head is held against float64: padding that ends inside a tile, empty sequences, rows of no sequence on either
side, d below the kernel's, tiles that run past the tensor, infinities and NaN far from the diagonal, near it and in rows of no
sequence.  Bounds as in typed_inputs.attend, a whole head at a time."""
import numpy as np
import pytest

from cinn_amd.common import Int
from cinn_amd.frontend import NetBuilder

from helpers import run
from typed_inputs import ULP, as_float64, assert_within, dtype, normal, rounded

pytestmark = pytest.mark.gpu

SHORT, SHARED, FOUR, EIGHT = "no ring", "2 x 4 wavefronts", "4 wavefronts", "8 wavefronts"


def kind_of_blocks(tokens, heads, kv_heads):
    group = heads // kv_heads
    blocks = tokens * group // 128 * kv_heads
    return SHORT if blocks <= 128 else SHARED if blocks <= 512 else EIGHT if group >= 4 else FOUR


def causal(q, k, v, offsets, kind):
    """float64 result and the bound on its error, [tokens][heads][d]; values that a row does not see may be anything"""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    group, d, u = q.shape[1] // k.shape[1], q.shape[2], ULP[kind]
    for first, end in zip(offsets[:-1], offsets[1:]):
        rows = slice(first, end)
        seen = np.tril(np.ones((end - first, end - first), bool))
        for h in range(q.shape[1]) if end > first else []:
            qq, kk, vv = q[rows, h], np.ascontiguousarray(k[rows, h // group].T), v[rows, h // group]
            s = np.where(seen, d ** -0.5 * (qq @ kk), -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[rows, h] = p @ vv
            score = (2.0 ** -24 * d ** 0.5 + 2.0 ** -22) * d ** -0.5 * np.where(seen, np.abs(qq) @ np.abs(kk), 0).max(1, keepdims=True)
            bound[rows, h] = (2 * score + 2.0 ** -18 + 2 * u) * (p @ np.abs(vv)) + u * np.abs(out[rows, h])
            if kind == "float16":
                bound[rows, h] += np.arange(1, end - first + 1)[:, None] * 2.0 ** -25 * np.abs(vv).max() + 2.0 ** -24
    return out, bound


class Prompts(object):
    def __init__(self, kind, lengths, heads, kv_heads, d, lead=0, rest=0):
        self.offsets = lead + np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        self.kind, self.heads, self.tokens = kind, heads, int(self.offsets[-1]) + rest
        rng = np.random.default_rng(self.tokens + d)
        self.data, self.values = {}, {}
        for name, n in (("q", heads), ("k", kv_heads), ("v", kv_heads)):
            self.data[name], self.values[name] = normal(rng, (self.tokens, n, d), kind)

    def run(self, **changed):
        feeds = {**self.data, **changed}
        b = NetBuilder("packed")
        var = [b.create_input(dtype(self.kind), list(feeds[n].shape), n) for n in "qkv"]
        o = b.packed_attention(*var, b.create_input(Int(32), [len(self.offsets)], "offsets"))
        return run(b, {**feeds, "offsets": self.offsets}, [o])[0][0]

    def reference(self):
        return causal(self.values["q"], self.values["k"], self.values["v"], self.offsets, self.kind)


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("blocks,lengths,heads,kv_heads,d,lead,rest", [
    (EIGHT, [1100, 1, 0, 950], 32, 8, 128, 0, 37), (EIGHT, [300, 0, 777], 64, 16, 80, 5, 0), (EIGHT, [65, 800, 64, 130], 64, 16, 64, 0, 1),
    (EIGHT, [515, 1, 1, 1, 60, 600], 80, 16, 32, 129, 3), (EIGHT, [1999], 40, 8, 120, 70, 60), (EIGHT, [31] * 40, 64, 16, 96, 0, 0),
    (FOUR, [950, 0, 250], 64, 64, 64, 3, 40), (FOUR, [2900, 33], 24, 12, 80, 0, 2), (FOUR, [700, 500], 58, 58, 128, 0, 0),
    (FOUR, [31, 1, 900, 0, 255], 60, 60, 24, 64, 1), (FOUR, [1100, 200], 48, 24, 104, 1, 900), (FOUR, [64] * 20, 96, 48, 40, 0, 5),
    (SHARED, [300, 1, 0, 450], 32, 8, 128, 7, 9), (SHARED, [1300], 14, 14, 64, 0, 3), (SHARED, [63, 700], 36, 18, 80, 2, 0),
    (SHARED, [33] * 40, 15, 15, 16, 0, 100), (SHARED, [600, 1, 130], 40, 20, 96, 0, 0)])
def test_every_row(gpu, kind, blocks, lengths, heads, kv_heads, d, lead, rest):
    case = Prompts(kind, lengths, heads, kv_heads, d, lead, rest)
    assert kind_of_blocks(case.tokens, heads, kv_heads) == blocks
    got = case.run()
    want, bound = case.reference()
    assert_within(got, want, bound, kind)
    assert not as_float64(got, kind)[:lead].any() and not as_float64(got, kind)[case.tokens - rest:].any()


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("blocks,heads,kv_heads,d", [(EIGHT, 64, 16, 64), (EIGHT, 64, 16, 88), (FOUR, 60, 60, 32), (FOUR, 96, 48, 72),
                                                     (SHARED, 16, 16, 64), (SHARED, 20, 10, 128)])
def test_what_is_not_attended_may_hold_anything(gpu, kind, bad, blocks, heads, kv_heads, d):
    """Rows before a bad key or value, and rows of other sequences, are as if it were not there; rows from it on have it, in its
    element of d and its key head.  Rows of no sequence are bad throughout."""
    lengths, lead, rest, head = [700, 400], 20, 80, kv_heads - 2
    group = heads // kv_heads
    case = Prompts(kind, lengths, heads, kv_heads, d, lead, rest)
    assert kind_of_blocks(case.tokens, heads, kv_heads) == blocks
    want, bound = case.reference()
    mine = np.zeros((heads, d), bool)
    mine[head * group:(head + 1) * group, 5] = True
    nothing = rounded([bad], kind)[0][0]
    for at in (20, 20 + 37, 20 + 352, 20 + 352 + 31, 719, 720, 720 + 130, 1119):  # the first rows of both, a tile's first and last, the last rows
        end = 720 if at < 720 else 1120
        for name in "kv":
            changed = {n: case.data[n].copy() for n in "kv"}
            for x in changed.values():
                x[:lead], x[-rest:] = nothing, nothing
            changed[name][at, head, 5] = nothing
            got = case.run(**changed)
            hit = np.zeros(want.shape, bool)
            hit[at:end] = mine if name == "v" else mine.any(1)[:, None]
            if name == "v" or np.isnan(bad):
                assert not np.isfinite(as_float64(got, kind)[hit]).any()
            assert_within(np.where(hit, rounded([0], kind)[0][0], got), np.where(hit, 0, want), bound, kind)
