"""rotary_embedding, packed_attention and cached_attention as a layer uses them: prompts of different lengths through one
product, their rotated keys and values into pages, then steps of new tokens over the pages.  A prompt that is a step longer
holds what the step has to give: both are within their bounds of the same float64 values."""
import numpy as np
import pytest

from cinn_amd import runtime
from cinn_amd.common import DefaultAMDGPUTarget, Int
from cinn_amd.frontend import Computation, NetBuilder

from helpers import run
from typed_inputs import TYPES, as_float64, assert_within, attend, dtype, normal

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, D, WIDTH, PAGE, COLUMNS = 6, 2, 64, 96, 16, 8
TOTAL = HEADS + 2 * KV_HEADS


def layer(kind, lead):
    """x [*lead, WIDTH] -> its projections [*lead, TOTAL, D] and their rotated queries and keys [*lead, HEADS + KV_HEADS, D]"""
    b = NetBuilder("layer")
    X = b.create_input(dtype(kind), [int(np.prod(lead)), WIDTH], "x")
    W = b.create_input(dtype(kind), [WIDTH, TOTAL * D], "w")
    P = b.create_input(Int(32), list(lead), "positions")
    qkv = b.reshape(b.matmul(X, W), [*lead, TOTAL, D])
    return b, qkv, b.rotary_embedding(qkv, P, heads=HEADS + KV_HEADS, theta=5e5)


def prompts(kind, x, w, lengths):
    b, qkv, turned = layer(kind, [len(x)])
    O = b.create_input(Int(32), [len(lengths) + 1], "offsets")
    o = b.packed_attention(turned, turned, qkv, O, heads=HEADS, kv_heads=KV_HEADS, k_head=HEADS, v_head=HEADS + KV_HEADS)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    positions = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
    return run(b, {"x": x, "w": w, "positions": positions, "offsets": offsets}, [qkv, turned, o])[0]


def steps(kind, batch, tokens, pages, graph):
    """a program of one step, and how to run it"""
    b, qkv, turned = layer(kind, [batch, tokens])
    K, V = (b.create_input(dtype(kind), [pages, PAGE, KV_HEADS, D], name) for name in ("k_pages", "v_pages"))
    T, L = b.create_input(Int(32), [batch, COLUMNS], "table"), b.create_input(Int(32), [batch], "lengths")
    o = b.cached_attention(turned, turned, qkv, K, V, T, L, heads=HEADS, kv_heads=KV_HEADS, k_head=HEADS, v_head=HEADS + KV_HEADS)
    stream = runtime.Stream()
    comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[qkv, turned, o], stream=stream)

    def step(**feeds):
        for name, data in feeds.items():
            comp.get_tensor(name).from_numpy(np.ascontiguousarray(data))
        (comp.execute_graph if graph else comp.execute)()
        stream.synchronize()
        return [comp.get_tensor(v.id).numpy() for v in (qkv, turned, o)]
    return step


def attention(q, k, v, kind):
    """the last len(q) rows of len(k) [rows][heads][D] in float64, and their bound"""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    allowed = np.tril(np.ones((len(q), len(k)), bool), len(k) - len(q))
    for h in range(HEADS):
        g = h // (HEADS // KV_HEADS)
        out[:, h], bound[:, h] = attend(q[:, h], k[:, g], v[:, g], allowed, D ** -0.5, kind)
    return out, bound


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("tokens", [1, 4])
def test_steps_continue_their_prompts(gpu, kind, graph, tokens):
    rng = np.random.default_rng(tokens)
    lengths, rounds = np.array([37, 1, 16, 90]), 4
    batch, whole = len(lengths), lengths + rounds * tokens
    w, _ = normal(rng, (WIDTH, TOTAL * D), kind, WIDTH ** -0.5)
    xs = [normal(rng, (n, WIDTH), kind)[0] for n in whole]

    qkv, turned, o = prompts(kind, np.concatenate([x[:n] for x, n in zip(xs, lengths)]), w, lengths)
    table = rng.permutation(batch * COLUMNS).reshape(batch, COLUMNS).astype(np.int32)
    k_pages, v_pages = (np.zeros((batch * COLUMNS, PAGE, KV_HEADS, D), qkv.dtype) for _ in range(2))
    seen = [[], [], [], []]  # what a sequence's rows are, as the device gave them

    def keep(b, row, qkv, turned):
        at = table[b][row // PAGE], row % PAGE
        k_pages[at], v_pages[at] = turned[HEADS:], qkv[HEADS + KV_HEADS:]
        seen[b].append((as_float64(turned, kind), as_float64(qkv, kind)))

    def check(b, first, got):
        turned, qkv = (np.array([row[i] for row in seen[b]]) for i in range(2))
        want, bound = attention(turned[first:, :HEADS], turned[:, HEADS:], qkv[:, HEADS + KV_HEADS:], kind)
        assert_within(got, want, bound, kind)

    first = np.concatenate([[0], np.cumsum(lengths)])
    for b in range(batch):
        for row in range(lengths[b]):
            keep(b, row, qkv[first[b] + row], turned[first[b] + row])
        check(b, 0, o[first[b]:first[b + 1]])

    step = steps(kind, batch, tokens, batch * COLUMNS, graph)
    for r in range(rounds):
        x = np.stack([x[n:n + tokens] for x, n in zip(xs, lengths)])
        positions = (lengths[:, None] + np.arange(tokens)).astype(np.int32)
        qkv, turned, o = step(x=x.reshape(-1, WIDTH), w=w, positions=positions, k_pages=k_pages, v_pages=v_pages, table=table,
                              lengths=lengths.astype(np.int32))
        for b in range(batch):
            for i in range(tokens):
                keep(b, lengths[b] + i, qkv[b, i], turned[b, i])
            check(b, lengths[b], o[b])
        lengths = lengths + tokens
    assert (lengths == whole).all()


@pytest.mark.parametrize("kind", TYPES)
def test_a_step_gives_what_a_longer_prompt_holds(gpu, kind):
    """the same rows of projections both ways: rotated to the same bits, attention within both bounds"""
    rng = np.random.default_rng(9)
    length, tokens = 61, 3
    data, _ = normal(rng, (length + tokens, TOTAL, D), kind)

    def rotate(b, x, positions):
        return b.rotary_embedding(x, positions, heads=HEADS + KV_HEADS)

    parts = dict(heads=HEADS, kv_heads=KV_HEADS, k_head=HEADS, v_head=HEADS + KV_HEADS)
    b = NetBuilder("whole")
    X, P = b.create_input(dtype(kind), list(data.shape), "x"), b.create_input(Int(32), [len(data)], "positions")
    O = b.create_input(Int(32), [2], "offsets")
    t = rotate(b, X, P)
    (turned, whole), _ = run(b, {X: data, P: np.arange(len(data), dtype=np.int32), O: np.array([0, len(data)], np.int32)},
                             [t, b.packed_attention(t, t, X, O, **parts)])

    pages = -(-length // PAGE)
    rows = [np.zeros((pages * PAGE, KV_HEADS, D), data.dtype) for _ in range(2)]
    rows[0][:length], rows[1][:length] = turned[:length, HEADS:], data[:length, HEADS + KV_HEADS:]
    b = NetBuilder("step")
    X, P = b.create_input(dtype(kind), [1, tokens, TOTAL, D], "x"), b.create_input(Int(32), [1, tokens], "positions")
    K, V = (b.create_input(dtype(kind), [pages, PAGE, KV_HEADS, D], name) for name in ("k_pages", "v_pages"))
    T, L = b.create_input(Int(32), [1, pages], "table"), b.create_input(Int(32), [1], "lengths")
    t = rotate(b, X, P)
    feeds = {X: data[None, length:], P: np.arange(length, length + tokens, dtype=np.int32)[None], T: np.arange(pages, dtype=np.int32)[None],
             L: np.array([length], np.int32), K: rows[0].reshape(pages, PAGE, KV_HEADS, D), V: rows[1].reshape(pages, PAGE, KV_HEADS, D)}
    (again, step), _ = run(b, {v: np.ascontiguousarray(x) for v, x in feeds.items()}, [t, b.cached_attention(t, t, X, K, V, T, L, **parts)])
    assert np.array_equal(again[0].view(np.uint8), turned[length:].view(np.uint8))
    turned, data = as_float64(turned, kind), as_float64(data, kind)
    _, bound = attention(turned[length:, :HEADS], turned[:, HEADS:], data[:, HEADS + KV_HEADS:], kind)
    assert_within(step[0], as_float64(whole[length:], kind), 2 * bound, kind)
