"""What a decoder's serving path asks of this framework beside products and norms: rotary positions, attention over whole
prompts packed behind one another, attention of new tokens (single ones or a tree of drafted ones) over a paged cache.

`listed()` are fixed cases, `draw(rng)` gives another one of the same kinds and ranges.  `own` says who computes: programs
built with NetBuilder, or the same formulas in elementary torch operations.  The kinds:

  rotary    rotary positions of the first heads of packed projections, or their gradient
  packed    causal attention with grouped heads over sequences of different lengths
  cached    new tokens of every sequence, which attend to their cache and to the new tokens before them
"""
import math
import random

import torch

own = False

_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "int32": torch.int32}


def listed():
    return [
        # one step of sixteen sequences: a launch, and the latency of a table of angles
        {"name": "rotary_bf16_decode", "kind": "rotary", "tokens": 16, "heads": 40, "total": 48, "d": 128, "rotary": 128,
         "interleaved": False, "theta": 500000.0, "factor": 1.0, "original": 0, "far": 8192, "grad": False,
         "dtype": "bfloat16"},
        # queries and keys of a batch of prompts, read out of the packed projections; memory bound
        {"name": "rotary_bf16_prompts", "kind": "rotary", "tokens": 8191, "heads": 40, "total": 48, "d": 128,
         "rotary": 128, "interleaved": False, "theta": 500000.0, "factor": 1.0, "original": 0, "far": 8192,
         "grad": False, "dtype": "bfloat16"},
        # neighbouring pairs, part of the head, single precision, odd counts
        {"name": "rotary_f32_part", "kind": "rotary", "tokens": 1111, "heads": 12, "total": 12, "d": 80, "rotary": 32,
         "interleaved": True, "theta": 10000.0, "factor": 1.0, "original": 0, "far": 2048, "grad": False,
         "dtype": "float32"},
        # the gradient in a long context whose low frequencies are stretched
        {"name": "rotary_f16_grad_scaled", "kind": "rotary", "tokens": 16384, "heads": 40, "total": 40, "d": 64,
         "rotary": 64, "interleaved": False, "theta": 500000.0, "factor": 8.0, "original": 8192, "far": 131072,
         "grad": True, "dtype": "float16"},
        # eight equal prompts of the benchmark's transformer block, causal
        {"name": "packed_f16_8x512", "kind": "packed", "tokens": 4096, "shortest": 512, "longest": 512, "sequences": 8,
         "heads": 12, "kv_heads": 12, "d": 64, "packed": True, "dtype": "float16"},
        # a batch of prompts of very different lengths, an empty one and one of a token among them, four heads to a key
        {"name": "packed_bf16_ragged", "kind": "packed", "tokens": 8191, "shortest": 0, "longest": 3000, "sequences": 11,
         "heads": 32, "kv_heads": 8, "d": 128, "packed": True, "dtype": "bfloat16"},
        # one long document
        {"name": "packed_bf16_long", "kind": "packed", "tokens": 16384, "shortest": 16384, "longest": 16384,
         "sequences": 1, "heads": 32, "kv_heads": 8, "d": 128, "packed": True, "dtype": "bfloat16"},
        # a few short prompts in single precision, rows between the usual lengths: latency
        {"name": "packed_f32_short", "kind": "packed", "tokens": 233, "shortest": 17, "longest": 100, "sequences": 5,
         "heads": 8, "kv_heads": 2, "d": 80, "packed": False, "dtype": "float32"},
        # the benchmark's decode step: 511 cached tokens and one new
        {"name": "cached_f16_8x511", "kind": "cached", "batch": 8, "new": 1, "shortest": 511, "longest": 511, "page": 16,
         "heads": 12, "kv_heads": 12, "d": 64, "packed": True, "tree": False, "head_pages": False, "dtype": "float16"},
        # a large batch of decode steps over caches of every length: memory bound, unevenly
        {"name": "cached_bf16_ragged", "kind": "cached", "batch": 48, "new": 1, "shortest": 100, "longest": 16000,
         "page": 64, "heads": 32, "kv_heads": 8, "d": 128, "packed": True, "tree": False, "head_pages": False,
         "dtype": "bfloat16"},
        # a tree of drafted tokens for each sequence; pages end inside every tile
        {"name": "cached_bf16_tree", "kind": "cached", "batch": 8, "new": 48, "shortest": 2000, "longest": 5000,
         "page": 24, "heads": 32, "kv_heads": 8, "d": 128, "packed": True, "tree": True, "head_pages": False,
         "dtype": "bfloat16"},
        # three tokens of one sequence behind a very long cache, single precision, pages by head
        {"name": "cached_f32_long", "kind": "cached", "batch": 1, "new": 3, "shortest": 100003, "longest": 100003,
         "page": 20, "heads": 16, "kv_heads": 4, "d": 96, "packed": False, "tree": False, "head_pages": True,
         "dtype": "float32"},
    ]


def _log(rng, low, high):
    """a whole number between low and high, spread over its logarithm"""
    return int(min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _pick_case(rng):
    kind = rng.choice(["rotary", "packed", "cached"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
    heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads < 8 else [1, 2, 4])
    d = rng.choice([32, 40, 64, 64, 80, 96, 120, 128, 128, 128])
    if kind == "rotary":
        rotated = heads + kv_heads
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "heads": rotated,
                "total": rotated + rng.choice([0, kv_heads]), "d": d, "rotary": rng.choice([d, d, d // 2, d // 4 * 2 - 2]),
                "interleaved": rng.random() < 0.4, "theta": rng.choice([10000.0, 500000.0, 1000000.0]),
                "factor": rng.choice([1.0, 4.0, 8.0, 2.5]), "original": rng.choice([0, 4096, 8192]),
                "far": _log(rng, 64, 1000000), "grad": rng.random() < 0.3, "dtype": dtype}
    if kind == "packed":
        longest = _log(rng, 1, 16384)
        sequences = _log(rng, 1, 64)
        return {"kind": kind, "tokens": 0, "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest,
                "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "d": d, "packed": rng.random() < 0.6,
                "dtype": dtype}
    longest = _log(rng, 1, 131072)
    new = rng.choice([1, 1, 1, _log(rng, 2, 64)])
    return {"kind": kind, "batch": _log(rng, 1, 128), "new": new, "shortest": rng.choice([0, longest // 8, longest]),
            "longest": longest, "page": rng.choice([1, 16, 20, 32, 64, 128]), "heads": heads, "kv_heads": kv_heads,
            "d": d, "packed": rng.random() < 0.6, "tree": new > 1 and rng.random() < 0.7,
            "head_pages": rng.random() < 0.3, "dtype": dtype}


def draw(rng):
    while True:
        case = _pick_case(rng)
        if case["kind"] == "packed":
            case["tokens"] = sum(_lengths(case)) + rng.choice([0, 0, 5])  # rows behind the last sequence
            if case["tokens"] == 0:
                continue
        w = work(case)
        # no more than the largest listed cases; single precision has a sixteenth of the matrix rate
        single = 16 if case["dtype"] == "float32" else 1
        if w["bytes"] <= 6e8 and single * w["flops"] <= 2e12:
            return case


# ---- what the cases' sequences and trees look like -----------------------------------------------------------------------
def _lengths(case):
    """of the sequences: what a case says and nothing else; spread over the logarithm"""
    count = case["sequences"] if case["kind"] == "packed" else case["batch"]
    low, high = case["shortest"], case["longest"]
    if low == high:
        return [low] * count
    rng = random.Random(1000003 * high + 1009 * low + count)
    got = [_log(rng, max(1, low), high) if rng.random() < 0.9 else low for _ in range(count)]
    got[0], got[-1] = high, low
    if case.get("tokens"):  # the rows there are, shared out in proportion
        total = sum(got)
        if total > case["tokens"]:
            got = [n * case["tokens"] // total for n in got]
        got[count // 2] = min(1, got[count // 2])
    return got


def _tree(case, seed):
    """parents[b][i] < i of every drafted token, -1 for those that follow the cache"""
    rng = random.Random(seed)
    n = case["new"]
    return [[-1 if i == 0 else rng.choice([i - 1, i - 1, rng.randrange(i), max(-1, i // 3 - 1)]) for i in range(n)]
            for _ in range(case["batch"])]


def _inputs(case, seed):
    """every tensor that a pass reads, made from the seed on the GPU"""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = _TORCH[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    if case["kind"] == "rotary":
        positions = torch.randint(0, case["far"], (case["tokens"],), generator=gen, device="cuda", dtype=torch.int32)
        return {"x": normal(case["tokens"], case["total"], case["d"]), "positions": positions}
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["d"]
    lead = [case["tokens"]] if case["kind"] == "packed" else [case["batch"], case["new"]]
    if case["packed"]:
        data = {"qkv": normal(*lead, heads + 2 * kv_heads, d)}
    else:
        data = {"q": normal(*lead, heads, d), "k": normal(*lead, kv_heads, d), "v": normal(*lead, kv_heads, d)}
    lengths = _lengths(case)
    if case["kind"] == "packed":
        ends = [0]
        for n in lengths:
            ends.append(ends[-1] + n)
        data["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        return data
    page = case["page"]
    used = [(n + page - 1) // page for n in lengths]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32).cpu()
    table = torch.zeros((case["batch"], max(1, max(used))), dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    shape = [pages, kv_heads, page, d] if case["head_pages"] else [pages, page, kv_heads, d]
    data.update(k_pages=normal(*shape), v_pages=normal(*shape), table=table.cuda(),
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if case["tree"]:
        data["parents"] = torch.tensor(_tree(case, seed), dtype=torch.int32, device="cuda")
    return data


# ---- the framework's programs ----------------------------------------------------------------------------------------------
class _DeviceArray(object):
    """device memory of a computation's tensor, as torch takes it"""

    def __init__(self, owner, pointer, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": tuple(shape), "typestr": typestr,
                                         "strides": None, "version": 2}


def _view(comp, name):
    t = comp.get_tensor(name)
    dtype = str(t.type())
    typestr = {"float32": "<f4", "float16": "<f2", "bfloat16": "<i2", "int32": "<i4"}[dtype]
    seen = torch.as_tensor(_DeviceArray(comp, t.device_ptr, t.shape(), typestr), device="cuda")
    return seen.view(_TORCH[dtype]) if dtype == "bfloat16" else seen


_STREAM = []


def _stream():
    """the program's one stream; its computations follow one another on it"""
    if not _STREAM:
        from cinn_amd import runtime
        _STREAM.append(runtime.Stream())
    return _STREAM[0]


def _build(case, b, var):
    if case["kind"] == "rotary":
        scaling = dict(rotary_dim=case["rotary"], interleaved=case["interleaved"], theta=case["theta"],
                       factor=case["factor"], original_length=case["original"])
        if case["grad"]:
            return b.rotary_embedding_grad(var["x"], var["positions"], heads=case["heads"], **scaling)
        return b.rotary_embedding(var["x"], var["positions"], heads=case["heads"], **scaling)
    heads, kv_heads = case["heads"], case["kv_heads"]
    if case["packed"]:
        operands = [var["qkv"]] * 3
        where = dict(heads=heads, kv_heads=kv_heads, q_head=0, k_head=heads, v_head=heads + kv_heads)
    else:
        operands = [var["q"], var["k"], var["v"]]
        where = dict(heads=heads, kv_heads=kv_heads)
    if case["kind"] == "packed":
        return b.packed_attention(*operands, var["offsets"], **where)
    return b.cached_attention(*operands, var["k_pages"], var["v_pages"], var["table"], var["lengths"],
                              parents=var.get("parents"), page_layout="head_row" if case["head_pages"] else "row_head",
                              **where)


def _program(case, data):
    from cinn_amd.common import BFloat16, DefaultAMDGPUTarget, Float, Int
    from cinn_amd.frontend import Computation, NetBuilder
    types = {torch.float32: Float(32), torch.float16: Float(16), torch.bfloat16: BFloat16(), torch.int32: Int(32)}
    b = NetBuilder(case["kind"])
    var = {name: b.create_input(types[t.dtype], list(t.shape), name) for name, t in data.items()}
    out = _build(case, b, var)
    comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[out], stream=_stream())
    for name, t in data.items():
        _view(comp, var[name].id).copy_(t)
    torch.cuda.synchronize()
    return {"comp": comp, "out": _view(comp, out.id)}


def prepare(case, seed):
    data = _inputs(case, seed)
    if own:
        return _program(case, data)
    state = {"case": case, "data": data}
    if case["kind"] != "rotary":
        state["lengths"] = _lengths(case)  # the host made the batch: it knows them
    if case["kind"] == "cached" and case["tree"]:
        state["parents"] = _tree(case, seed)
    return state


def run(state):
    if "comp" in state:
        state["comp"].execute()
        return state["out"]
    return {"rotary": _rotary, "packed": _packed, "cached": _cached}[state["case"]["kind"]](state)


# ---- the plain forms -----------------------------------------------------------------------------------------------------------
def _frequencies(case):
    r = case["rotary"]
    f = case["theta"] ** (-2.0 * torch.arange(r // 2, dtype=torch.float64, device="cuda") / r)
    if case["original"] == 0:
        return f / case["factor"]
    low, high = 1.0, 4.0
    kept = ((case["original"] * f / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
    return f * (kept + (1.0 - kept) / case["factor"])


def _rotary(state):
    case, x = state["case"], state["data"]["x"]
    x = x[:, :case["heads"]].float()
    angle = state["data"]["positions"].double()[:, None, None] * _frequencies(case)
    cos, sin = angle.cos().float(), angle.sin().float()
    if case["grad"]:
        sin = -sin
    r = case["rotary"]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1).to(state["data"]["x"].dtype)


def _operands(state):
    case, data = state["case"], state["data"]
    if case["packed"]:
        return data["qkv"].split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=-2)
    return data["q"], data["k"], data["v"]


def _attend(q, k, v, mask):
    """queries [kv_heads][rows][d], their keys and values [kv_heads][keys][d], what may be attended [rows][keys]; as many
    heads together as keep the scores under a gigabyte"""
    o = torch.empty_like(q)
    step = max(1, (1 << 28) // mask.numel())
    for h in range(0, q.shape[0], step):
        s = torch.matmul(q[h:h + step], k[h:h + step].transpose(1, 2)) * (1.0 / math.sqrt(q.shape[-1]))
        s.masked_fill_(~mask, -math.inf)
        s -= s.amax(-1, keepdim=True)
        p = s.exp_()
        o[h:h + step] = torch.matmul(p, v[h:h + step]) / p.sum(-1, keepdim=True)
    return o


def _grouped(q, kv_heads):
    """[rows][heads][d] -> [kv_heads][group rows][d]"""
    return q.float().transpose(0, 1).reshape(kv_heads, -1, q.shape[-1])


def _ungrouped(o, like):
    return o.reshape(like.shape[1], like.shape[0], like.shape[2]).transpose(0, 1).to(like.dtype)


def _packed(state):
    case = state["case"]
    q, k, v = _operands(state)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=q.dtype, device="cuda")
    first = 0
    for n in state["lengths"]:
        rows = slice(first, first + n)
        first += n
        if n == 0:
            continue
        mask = torch.ones((n, n), dtype=torch.bool, device="cuda").tril_().repeat(group, 1)
        o = _attend(_grouped(q[rows], case["kv_heads"]), _grouped(k[rows], case["kv_heads"]),
                    _grouped(v[rows], case["kv_heads"]), mask)
        out[rows] = _ungrouped(o, q[rows])
    return out


def _cached(state):
    case, data = state["case"], state["data"]
    q, k, v = _operands(state)
    n, kv_heads = case["new"], case["kv_heads"]
    group = case["heads"] // kv_heads
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    for b, length in enumerate(state["lengths"]):
        pages = data["table"][b, :(length + case["page"] - 1) // case["page"]].long()
        past = []
        for cache in (data["k_pages"], data["v_pages"]):
            rows = cache[pages]
            if case["head_pages"]:
                rows = rows.transpose(1, 2)
            past.append(rows.reshape(-1, kv_heads, case["d"])[:length])
        mask = torch.ones((n, length + n), dtype=torch.bool, device="cuda")
        if case["tree"]:
            seen = torch.zeros((n, n), dtype=torch.bool)
            for i, parent in enumerate(state["parents"][b]):
                if parent >= 0:
                    seen[i] = seen[parent]
                seen[i, i] = True
            mask[:, length:] = seen.cuda()
        else:
            mask[:, length:].tril_()
        o = _attend(_grouped(q[b], kv_heads), _grouped(torch.cat([past[0], k[b]]), kv_heads),
                    _grouped(torch.cat([past[1], v[b]]), kv_heads), mask.repeat(group, 1))
        out[b] = _ungrouped(o, q[b])
    return out


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def _softmax_rows(scores, values):
    top = scores.max(dim=1, keepdim=True).values
    weights = torch.exp(scores - top)
    return torch.mm(weights / weights.sum(dim=1, keepdim=True), values)


def _exact_rotary(case, data):
    """each pair as a complex number times exp(i angle)"""
    x = data["x"][:, :case["heads"], :].double()
    r, half = case["rotary"], case["rotary"] // 2
    turns = []
    for i in range(half):
        f = math.exp(-2.0 * i / r * math.log(case["theta"]))
        if case["original"]:
            rounds = case["original"] * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (rounds - 1.0) / 3.0))
            f = keep * f + (1.0 - keep) * f / case["factor"]
        else:
            f /= case["factor"]
        turns.append(f)
    angle = torch.outer(data["positions"].double(), torch.tensor(turns, dtype=torch.float64, device="cuda"))
    factor = torch.polar(torch.ones_like(angle), -angle if case["grad"] else angle).unsqueeze(1)
    even = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    odd = even + (1 if case["interleaved"] else half)
    z = torch.complex(x[..., even], x[..., odd]) * factor
    y = x.clone()
    y[..., even], y[..., odd] = z.real, z.imag
    return y


def _exact_attention(case, data):
    if case["packed"]:
        total = data["qkv"].double()
        q = total[..., :case["heads"], :]
        k = total[..., case["heads"]:case["heads"] + case["kv_heads"], :]
        v = total[..., case["heads"] + case["kv_heads"]:, :]
    else:
        q, k, v = data["q"].double(), data["k"].double(), data["v"].double()
    return q, k, v, case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["d"])


def _exact_packed(case, data):
    q, k, v, group, scale = _exact_attention(case, data)
    y = torch.zeros_like(q)
    start = 0
    for n in _lengths(case):
        for h in range(case["heads"]):
            kh = k[start:start + n, h // group, :].t().contiguous()
            vh = v[start:start + n, h // group, :].contiguous()
            for r0 in range(0, n, 2048):
                r1 = min(n, r0 + 2048)
                s = torch.mm(q[start + r0:start + r1, h, :], kh[:, :r1]) * scale
                row = torch.arange(r0, r1, device="cuda").unsqueeze(1)
                column = torch.arange(r1, device="cuda").unsqueeze(0)
                s = torch.where(column <= row, s, torch.full_like(s, -math.inf))
                y[start + r0:start + r1, h, :] = _softmax_rows(s, vh[:r1])
        start += n
    return y


def _exact_cached(case, data, seed):
    q, k, v, group, scale = _exact_attention(case, data)
    y = torch.empty_like(q)
    trees = _tree(case, seed) if case["tree"] else [[i - 1 for i in range(case["new"])]] * case["batch"]
    for b, length in enumerate(_lengths(case)):
        position = torch.arange(length, device="cuda")
        page = data["table"][b][position // case["page"]].long()
        slot = position % case["page"]
        allowed = torch.ones((case["new"], length + case["new"]), dtype=torch.bool, device="cuda")
        allowed[:, length:] = False
        for i in range(case["new"]):
            j = i
            while j >= 0:
                allowed[i, length + j] = True
                j = trees[b][j]
        for kv in range(case["kv_heads"]):
            if case["head_pages"]:
                pk, pv = data["k_pages"][page, kv, slot], data["v_pages"][page, kv, slot]
            else:
                pk, pv = data["k_pages"][page, slot, kv], data["v_pages"][page, slot, kv]
            kt = torch.cat([pk.double(), k[b, :, kv]]).t().contiguous()
            vt = torch.cat([pv.double(), v[b, :, kv]])
            for h in range(kv * group, (kv + 1) * group):
                s = torch.mm(q[b, :, h], kt) * scale
                s = torch.where(allowed, s, torch.full_like(s, -math.inf))
                y[b, :, h] = _softmax_rows(s, vt)
    return y


def exact(case, seed):
    data = _inputs(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, data)
    if case["kind"] == "packed":
        return _exact_packed(case, data)
    return _exact_cached(case, data, seed)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    """bytes: inputs that count read once, outputs written once; flops: the two products of every query with the keys that
    it attends to, or six operations for every pair"""
    e = _BYTES[case["dtype"]]
    if case["kind"] == "rotary":
        rows = case["tokens"] * case["heads"]
        return {"bytes": 2 * e * rows * case["d"] + 4 * case["tokens"], "flops": 3 * rows * case["rotary"]}
    heads, kv_heads, d, lengths = case["heads"], case["kv_heads"], case["d"], _lengths(case)
    if case["kind"] == "packed":
        rows, pairs = sum(lengths), sum(n * (n + 1) // 2 for n in lengths)
        moved = 2 * (heads + kv_heads) * rows + heads * (case["tokens"] - rows)
        return {"bytes": e * d * moved + 4 * len(lengths), "flops": 4.0 * d * heads * pairs}
    n, batch = case["new"], case["batch"]
    depths = 0
    for parents in _tree(case, 0) if case["tree"] else [[i - 1 for i in range(n)]] * batch:
        depth = []
        for parent in parents:
            depth.append(1 if parent < 0 else depth[parent] + 1)
        depths += sum(depth)
    rows = 2 * kv_heads * sum(lengths) + 2 * (heads + kv_heads) * batch * n
    pages = sum((m + case["page"] - 1) // case["page"] for m in lengths)
    return {"bytes": e * d * rows + 4 * (pages + batch), "flops": 4.0 * d * heads * (n * sum(lengths) + depths)}
