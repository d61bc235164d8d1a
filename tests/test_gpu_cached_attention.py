"""cached_attention (cached_attention.hip) against float64: caches of no row, one row and many, pages that end inside every
tile, trees, chains and single tokens, padding among the tokens, pages that are none, infinities and NaN where nothing
attends to them, and caches whose tiles several blocks share."""
import ctypes

import numpy as np
import pytest

from cinn_amd import _lib, runtime
from cinn_amd.common import DefaultAMDGPUTarget, Int
from cinn_amd.frontend import Computation, NetBuilder

from helpers import run
from test_gpu_gradient_capture import fresh_stream, replays
from typed_inputs import TYPES, as_float64, assert_within, attend, dtype, normal, rounded

pytestmark = pytest.mark.gpu


class Case(object):
    """inputs of one call: their typed arrays by name, and float64 values of the floating ones"""

    def __init__(self, kind, lengths, tokens, heads, kv_heads, d, page, parents=None, layout="row_head", columns=None, seed=0, spare=2):
        rng = np.random.default_rng(seed + sum(lengths) * 3 + tokens + d)
        batch = len(lengths)
        used = [-(-n // page) for n in lengths]
        pages = sum(used) + spare
        order = rng.permutation(pages)
        table = rng.integers(0, pages, (batch, columns or max(1, max(used)))).astype(np.int32)  # behind a sequence's pages: anything
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        shape = (pages, page, kv_heads, d) if layout == "row_head" else (pages, kv_heads, page, d)
        self.kind, self.layout, self.page, self.lengths, self.tokens = kind, layout, page, list(lengths), tokens
        self.data, self.values = {}, {}
        for name, size in (("q", (batch, tokens, heads, d)), ("k", (batch, tokens, kv_heads, d)), ("v", (batch, tokens, kv_heads, d)),
                           ("k_pages", shape), ("v_pages", shape)):
            self.data[name], self.values[name] = normal(rng, size, kind)
        self.data["table"], self.data["lengths"] = table, np.array(lengths, np.int32)
        if parents is not None:
            self.data["parents"] = np.array(parents, np.int32)

    def builder(self, **options):
        b = NetBuilder("cached")
        var = {n: b.create_input(Int(32) if x.dtype == np.int32 else dtype(self.kind), list(x.shape), n) for n, x in self.data.items()}
        o = b.cached_attention(var["q"], var["k"], var["v"], var["k_pages"], var["v_pages"], var["table"], var["lengths"],
                               parents=var.get("parents"), page_layout=self.layout, **options)
        return b, o

    def run(self, **options):
        b, o = self.builder(**options)
        return run(b, self.data, [o], **{})[0][0]

    def seen(self, b):
        """[token][token], and which tokens are none"""
        seen = np.zeros((self.tokens, self.tokens), bool)
        if "parents" not in self.data:
            return np.tril(~seen), np.zeros(self.tokens, bool)
        parents = self.data["parents"][b]
        none = np.array([not -1 <= parent < i for i, parent in enumerate(parents)])
        for i in range(self.tokens):
            j = i
            while j >= 0 and not none[j]:
                seen[i, j] = True
                j = parents[j]
        return seen, none

    def reference(self, scale=None):
        v = self.values
        out, bound = np.zeros(v["q"].shape), np.zeros(v["q"].shape)
        heads, kv_heads, d = v["q"].shape[2], v["k"].shape[2], v["q"].shape[3]
        pages = v["k_pages"].shape[0]
        for b, length in enumerate(self.lengths):
            length = min(max(length, 0), self.data["table"].shape[1] * self.page)
            row = np.arange(length)
            page = self.data["table"][b][row // self.page].astype(np.int64)
            good = (page >= 0) & (page < pages)
            page, slot = page[good], (row % self.page)[good]
            seen, none = self.seen(b)
            allowed = np.concatenate([np.repeat(~none[:, None], len(page), 1), seen], 1)
            for h in range(heads):
                g = h // (heads // kv_heads)
                past = [x[page, slot, g] if self.layout == "row_head" else x[page, g, slot] for x in (v["k_pages"], v["v_pages"])]
                out[b, :, h], bound[b, :, h] = attend(v["q"][b, :, h], np.concatenate([past[0], v["k"][b, :, g]]),
                                                      np.concatenate([past[1], v["v"][b, :, g]]), allowed,
                                                      d ** -0.5 if scale is None else scale, self.kind)
        return out, bound

    def check(self, **options):
        got = self.run(**options)
        want, bound = self.reference(options.get("scale"))
        assert_within(got, want, bound, self.kind)


def tree(rng, batch, tokens, none=0.0):
    return [[-1 if i == 0 else (rng.choice([-2, i, i + 3, 1 << 30]) if rng.random() < none else rng.integers(-1, i)) for i in range(tokens)]
            for _ in range(batch)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,d,page", [
    ([0], 1, 1, 8, 1), ([1], 1, 1, 128, 16), ([31], 4, 2, 64, 3), ([32, 0, 5], 2, 1, 40, 16), ([127, 128, 129], 8, 8, 64, 24),
    ([500, 1, 0, 63, 64, 65, 700], 8, 2, 80, 20), ([1000], 12, 12, 32, 64), ([257] * 9, 6, 1, 96, 7), ([3000, 10], 32, 8, 128, 48),
    ([5, 2049], 16, 2, 120, 1), ([4000], 5, 1, 72, 128), ([90] * 130, 2, 2, 16, 32)])
def test_single_tokens(gpu, kind, lengths, heads, kv_heads, d, page):
    Case(kind, lengths, 1, heads, kv_heads, d, page).check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("layout", ["row_head", "head_row"])
@pytest.mark.parametrize("lengths,tokens,heads,kv_heads,d,page", [
    ([0, 3], 2, 2, 2, 64, 4), ([40, 1000, 0], 3, 12, 4, 48, 20), ([77], 33, 1, 1, 64, 16), ([900, 901], 9, 15, 3, 104, 24),
    ([2000, 31], 64, 8, 1, 128, 32), ([130], 64, 16, 2, 64, 5), ([1500, 0, 64], 17, 32, 8, 80, 48)])
def test_chains_and_trees(gpu, kind, layout, lengths, tokens, heads, kv_heads, d, page):
    Case(kind, lengths, tokens, heads, kv_heads, d, page, layout=layout).check()
    rng = np.random.default_rng(tokens)
    Case(kind, lengths, tokens, heads, kv_heads, d, page, tree(rng, len(lengths), tokens), layout).check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,tokens,heads,kv_heads,d,page", [
    ([900, 3, 0, 4000], 1, 32, 1, 128, 16), ([700, 2500], 5, 4, 1, 96, 32), ([1300], 3, 18, 2, 128, 8), ([600, 33], 8, 8, 2, 64, 32),
    ([2100, 9], 20, 2, 2, 120, 5), ([1800, 100], 16, 4, 1, 128, 16), ([2500, 64], 25, 8, 2, 128, 64), ([2000], 48, 4, 1, 128, 16),
    ([1000, 640], 63, 4, 1, 96, 32), ([3000, 0, 1], 33, 12, 3, 112, 16)])
def test_wide_heads_of_many_pairs(gpu, kind, lengths, tokens, heads, kv_heads, d, page):
    Case(kind, lengths, tokens, heads, kv_heads, d, page).check()
    Case(kind, lengths, tokens, heads, kv_heads, d, page, tree(np.random.default_rng(tokens), len(lengths), tokens, 0.1)).check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,heads,d", [(1, 4, 128), (6, 8, 128), (9, 6, 96), (64, 2, 128)])
def test_infinite_values_past_the_first_tiles(gpu, kind, tokens, heads, d):
    """padding that holds an infinity, behind and among clean tiles: what attends to it is infinite, nothing else changes"""
    parents = [[-1] * tokens, [-2] + [-1] * (tokens - 1)]
    case = Case(kind, [1500, 700], tokens, heads, 2, d, 16, parents)
    want, bound = case.reference()
    case.data["v"][1, 0, :, 1] = rounded([np.inf], kind)[0][0]  # a token that is none
    page = case.data["table"][0, 700 // 16]
    case.data["v_pages"][page, 700 % 16, 1, 2] = rounded([np.inf], kind)[0][0]
    got = case.run()
    hit = np.zeros(want.shape, bool)
    hit[0, :, heads // 2:, 2] = True
    assert (as_float64(got, kind)[hit] == np.inf).all()
    clean = np.where(hit, rounded(np.zeros(1), kind)[0][0], got)
    assert_within(clean, np.where(hit, 0, want), np.where(hit, 1, bound), kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,heads", [(1, 2), (7, 4), (40, 4)])
@pytest.mark.parametrize("length", [0, 50, 1200])
def test_padding_among_the_tokens(gpu, kind, tokens, heads, length):
    """tokens that are none have a result of zero, also where they are all there is, and no descendant sees past them"""
    rng = np.random.default_rng(tokens + length)
    parents = tree(rng, 3, tokens, none=0.4)
    parents[1] = [-2] * tokens
    case = Case(kind, [length, length, 9], tokens, heads, 2, 64, 16, parents)
    got = as_float64(case.run(), kind)
    case.check()
    for b in range(3):
        none = case.seen(b)[1]
        assert not got[b][none].any() and (b != 1 or none.all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens", [1, 20])
def test_pages_that_are_none_hold_no_rows(gpu, kind, tokens):
    case = Case(kind, [100, 1000, 30], tokens, 4, 2, 64, 20)
    pages = case.data["k_pages"].shape[0]
    case.data["table"][0, 2], case.data["table"][1, [0, 7, 40]], case.data["table"][2, :2] = -1, [pages, 1 << 30, -(1 << 31)], pages + 5
    case.check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,heads", [(1, 4), (10, 4), (20, 4), (40, 4), (24, 14), (50, 16)])
@pytest.mark.parametrize("length", [100, 1000, 63, 32])
def test_the_one_page_that_is_none_lies_where_the_cache_ends(gpu, kind, tokens, heads, length):
    """the only rows that are none are in the tile that the cache ends in, in its first 32: none of the units' wavefronts (2, 20,
    40, 80, 168 and 400 pairs of query and head) may count them"""
    case = Case(kind, [length, length + 64], tokens, heads, 2, 64, 16)
    for b, end in enumerate((length, length + 64)):
        case.data["table"][b, end // 64 * 4] = -1
    # keys whose rows are not there score far below the others, where zeros in their place would weigh most
    case.data["q"], case.values["q"] = rounded(np.abs(case.values["q"]), kind)
    for name in ("k", "k_pages"):
        case.data[name], case.values[name] = rounded(-np.abs(case.values[name]), kind)
    case.check()


@pytest.mark.parametrize("length", [-1, -(1 << 31), (1 << 31) - 1, 161])
def test_lengths_beyond_the_table(gpu, length):
    case = Case("float16", [160, 100], 3, 4, 2, 32, 16)
    case.data["lengths"][0] = case.lengths[0] = length
    case.check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
@pytest.mark.parametrize("tokens", [1, 12])
def test_scale(gpu, kind, scale, tokens):
    Case(kind, [70, 900], tokens, 6, 2, 64, 16).check(scale=scale)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("length", [0, 45, 1100])
def test_tokens_that_are_not_attended_do_not_count(gpu, kind, bad, length):
    """an infinite or NaN key or value of one branch does not reach another; rows of the cache behind its length neither"""
    parents = [[-1, 0, 0, 1, 2, 3, 4, -1]]
    clean = Case(kind, [length], 8, 4, 2, 64, 16, parents, columns=length // 16 + 1, spare=5)
    want, bound = clean.reference()
    for name in ("k", "v"):
        case = Case(kind, [length], 8, 4, 2, 64, 16, parents, columns=length // 16 + 1, spare=5)
        case.data[name][0, 2, :, 3] = rounded([bad], kind)[0][0]
        page = case.data["table"][0, length // 16]
        if length % 16:
            for pages in ("k_pages", "v_pages"):
                case.data[pages][page, length % 16:] = rounded([bad], kind)[0][0]
        got = case.run()
        others, hit = [0, 1, 3, 5, 7], [2, 4, 6]
        assert_within(got[:, others], want[:, others], bound[:, others], kind)
        if name == "v" or np.isnan(bad):
            assert not np.isfinite(as_float64(got, kind)[:, hit, :, 3]).any()


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_operands_in_packed_projections(gpu, kind):
    case = Case(kind, [300, 20], 5, 6, 2, 64, 16)
    qkv = np.concatenate([case.data[n] for n in "qkv"], axis=2)
    b = NetBuilder("parts")
    var = {n: b.create_input(Int(32) if x.dtype == np.int32 else dtype(kind), list(x.shape), n) for n, x in case.data.items()}
    X = b.create_input(dtype(kind), list(qkv.shape), "qkv")
    rest = [var[n] for n in ("k_pages", "v_pages", "table", "lengths")]
    apart = b.cached_attention(var["q"], var["k"], var["v"], *rest)
    inside = b.cached_attention(X, X, X, *rest, heads=6, kv_heads=2, k_head=6, v_head=8)
    (a, i), _ = run(b, {**case.data, X: qkv}, [apart, inside])
    assert np.array_equal(a.view(np.uint8), i.view(np.uint8))
    # pages of keys as those of values too
    shared = b.cached_attention(var["q"], var["k"], var["v"], var["k_pages"], var["k_pages"], var["table"], var["lengths"])
    (s,), _ = run(b, {**case.data, X: qkv}, [shared])
    case.values["v_pages"] = case.values["k_pages"]
    want, bound = case.reference()
    assert_within(s, want, bound, kind)


@pytest.mark.parametrize("graph", [False, True])
def test_a_program_serves_every_length(gpu, graph):
    """lengths, table and parents change between executions of one compiled program, also between replays of its graph"""
    stream = runtime.Stream()
    first = Case("bfloat16", [1500, 10, 0, 700], 6, 8, 2, 64, 16, [[-1, 0, 1, 2, 3, 4]] * 4, columns=100)
    b, o = first.builder()
    comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[o], stream=stream)
    pages = first.data["k_pages"].shape[0]
    for step, lengths in enumerate(([1500, 10, 0, 700], [0, 0, 0, 1600], [3, 1599, 2, 600], [1, 1, 1, 1], [2210, 0, 0, 0])):
        rng = np.random.default_rng(step)
        case = Case("bfloat16", lengths, 6, 8, 2, 64, 16, tree(rng, 4, 6, 0.1), columns=100 if max(lengths) <= 1600 else 139, seed=step)
        if case.data["table"].shape[1] != 100:  # more than the table can hold: what it holds
            case.data["table"] = np.ascontiguousarray(case.data["table"][:, :100])
        for name in ("k_pages", "v_pages"):
            padded, values = normal(rng, (pages, 16, 2, 64), "bfloat16")
            case.data[name], case.values[name] = padded, values
        case.data["table"] %= pages
        for name, x in case.data.items():
            comp.get_tensor(name).from_numpy(x)
        (comp.execute_graph if graph else comp.execute)()
        stream.synchronize()
        want, bound = case.reference()
        assert_within(comp.get_tensor(o.id).numpy(), want, bound, "bfloat16")


def test_two_programs_on_two_streams(gpu):
    """programs that overlap have scratch of their own: the bits that each gives alone"""
    cases = [Case("float16", [5000, 3000], 2, 8, 2, 64, 16, seed=s) for s in range(2)]
    alone = [case.run() for case in cases]
    comps = []
    for case in cases:
        b, o = case.builder()
        comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[o], stream=runtime.Stream())
        for name, x in case.data.items():
            comp.get_tensor(name).from_numpy(x)
        comps.append((comp, o))
    for _ in range(20):
        for comp, _ in comps:
            comp.execute()
    runtime.synchronize()
    for (comp, o), want in zip(comps, alone):
        assert np.array_equal(comp.get_tensor(o.id).numpy().view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("kind", ["float16", "float32"])
@pytest.mark.parametrize("tokens,heads", [(1, 4), (12, 4), (64, 4)])
def test_captured_without_an_eager_run(gpu, kind, tokens, heads):
    """called first while its stream is captured, with no scratch to divide a long cache over blocks: one block each"""
    case = Case(kind, [1700, 0, 300], tokens, heads, 2, 64, 16)
    lib = _lib.load()
    lib.cinn_call_hip_cached_attention.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_float] + [ctypes.c_int] * 16 + [ctypes.c_void_p]
    want, bound = case.reference()
    clear = np.full(want.shape, 7, kind)
    out = runtime.DeviceBuffer.from_numpy(clear)
    inputs = [runtime.DeviceBuffer.from_numpy(x) for x in case.data.values()]
    pods = runtime.pod_args(inputs + [out])
    stream = fresh_stream(lib, 0)
    pages, columns = case.data["k_pages"].shape[0], case.data["table"].shape[1]
    args = [64 ** -0.5, 3, tokens, heads, 2, 64, pages, 16, 0, columns, (0x06543210 | 15 << 28) - (1 << 32), heads, 0, 2, 0, 2, 0]
    for got in replays(stream, lambda: lib.cinn_call_hip_cached_attention(pods, 8, *args, stream.handle), out, clear):
        assert_within(got.numpy(), want, bound, kind)
        case.check()
