"""What stands between the packed linears of a transformer block when it serves: the norms around a block with its gate, the
paged 8-bit cache of keys and values, the attention that reads it, and the upkeep of its pages.

A case is a dict of plain values; `kind` says which operator it goes through:

  norm    r' = r + residual_scale * gate * post(branch); y = norm(r') * weight * (1 + scale) + shift
  append  new tokens into the cache, then the blocks that changed read back as the values they stand for
  attend  attention of the last tokens of some sequences over all that the cache holds of them
  fork    a beam or guidance step: sequences forked from others, then room reserved for their next tokens
  compact live pages moved together at the front of the pool

Lengths of a ragged batch come from the case (`shape` seeds them), values from the seed.
"""
import math
import random

import torch

own = False  # false: elementary torch operations in 32 bits; true: the framework's entry points

BLOCK = 16  # tokens that share a scale
DTYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the norms between two blocks while one token is generated: the smallest call, latency alone
        {"name": "norm 1", "kind": "norm", "rows": 1, "width": 4096, "groups": 1, "norm": "rms", "post": True, "modulated": False, "residual": "f16", "branch": "f16", "y": "f16"},
        # image tokens of a 1024 x 1024 picture, float32 residual stream, modulated by two conditioning vectors
        {"name": "norm 4096", "kind": "norm", "rows": 4096, "width": 4096, "groups": 2, "norm": "layer", "post": False, "modulated": True, "residual": "f32", "branch": "f16", "y": "f16"},
        # a 2048 x 2048 picture with norms on both sides of the block
        {"name": "norm 16384", "kind": "norm", "rows": 16384, "width": 4096, "groups": 1, "norm": "rms", "post": True, "modulated": True, "residual": "f32", "branch": "f16", "y": "f16"},
        # one generated token of each of 64 requests, somewhere in their 16-token blocks
        {"name": "append 64 x 1", "kind": "append", "batch": 64, "most": 1, "length": 2048, "kv_heads": 8, "head_dim": 128, "page": 64, "x": "f16", "shape": 1},
        # image tokens of a guided pair behind their text prefixes, from the engine's float32
        {"name": "append 2 x 4096", "kind": "append", "batch": 2, "most": 4096, "length": 4173, "kv_heads": 32, "head_dim": 128, "page": 64, "x": "f32", "shape": 2},
        # one token of one short request: launches and latency
        {"name": "attend 1 x 1 of 333", "kind": "attend", "batch": 1, "most": 1, "length": 333, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True, "window": 0, "lse": False, "shape": 3},
        # one token of each of 64 requests of mixed lengths
        {"name": "attend 64 x 1 of 8192", "kind": "attend", "batch": 64, "most": 1, "length": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True, "window": 0, "lse": False, "shape": 4},
        # one token of one very long request: the cache has to be split
        {"name": "attend 1 x 1 of 131071", "kind": "attend", "batch": 1, "most": 1, "length": 131071, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "causal": True, "window": 0, "lse": True, "shape": 5},
        # prompts of mixed lengths, narrow heads
        {"name": "attend 8 x 700", "kind": "attend", "batch": 8, "most": 700, "length": 1111, "heads": 28, "kv_heads": 4, "head_dim": 64, "page": 32, "causal": True, "window": 0, "lse": False, "shape": 6},
        # the image tokens of a guided pair against their text prefixes and themselves, the largest
        {"name": "attend 2 x 4096 of 4173", "kind": "attend", "batch": 2, "most": 4096, "length": 4173, "heads": 32, "kv_heads": 32, "head_dim": 128, "page": 64, "causal": False, "window": 0, "lse": False, "shape": 7},
        # a step of a beam search: 32 sequences replaced by forks of others, pages of all layers
        {"name": "fork 32", "kind": "fork", "sequences": 96, "count": 32, "length": 640, "layers": 16, "pages": 1536, "kv_heads": 8, "head_dim": 128, "page": 32, "shape": 8},
        # a pool with holes after requests of different lengths have ended
        {"name": "compact 1024", "kind": "compact", "sequences": 48, "count": 24, "length": 640, "layers": 16, "pages": 1024, "kv_heads": 8, "head_dim": 128, "page": 32, "shape": 9},
    ]


def _spread(rng, low, high):
    """A whole number of low..high, evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


MOST_SCORES = 2 * 32 * 4096 * 4173   # of the largest listed attention
MOST_CACHED = 64 * 8192 * 8 * 128    # values of K in the largest listed cache


def draw(rng):
    kind = rng.choice(("norm", "norm", "append", "append", "attend", "attend", "attend", "attend", "fork", "compact"))
    if kind == "norm":
        return {"kind": kind, "rows": _spread(rng, 1, 12000), "width": 8 * _spread(rng, 64, 640), "groups": rng.choice((1, 1, 2, 3)), "norm": rng.choice(("rms", "layer")),
                "post": rng.random() < 0.5, "modulated": rng.random() < 0.6, "residual": rng.choice(("f16", "f32")), "branch": rng.choice(("f16", "f32")), "y": rng.choice(("f16", "f32"))}
    shape, head_dim, page = rng.randrange(1 << 20), rng.choice((64, 128, 128)), rng.choice((16, 32, 64, 128))
    if kind == "append":
        most = rng.choice((1, _spread(rng, 1, 4096)))
        batch = _spread(rng, 1, max(1, min(128, 8192 // most)))
        return {"kind": kind, "batch": batch, "most": most, "length": most + _spread(rng, 1, 2000), "kv_heads": rng.choice((1, 2, 4, 8, 8, 24, 32)), "head_dim": head_dim, "page": page,
                "x": rng.choice(("f16", "f32")), "shape": shape}
    if kind == "attend":
        kv_heads = rng.choice((1, 2, 4, 8, 8, 8))
        group = rng.choice((1, 2, 3, 4, 4, 7, 8))
        most = rng.choice((1, 1, rng.randint(2, 8), _spread(rng, 9, 4096)))
        length = most + _spread(rng, 1, 60000 if most <= 8 else 4000)
        room = min(MOST_SCORES // (kv_heads * group * most * length), MOST_CACHED // (kv_heads * 128 * length))
        return {"kind": kind, "batch": _spread(rng, 1, max(1, min(96, room))), "most": most, "length": length, "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": page, "causal": rng.random() < 0.7, "window": rng.choice((0, 0, 0, rng.randint(1, length))), "lse": rng.random() < 0.5, "shape": shape}
    sequences = _spread(rng, 8, 96)
    page = rng.choice((16, 32, 64))
    kv_heads = rng.choice((1, 2, 4, 8))
    length = _spread(rng, page, 640)
    # room for every sequence, for the forks' own pages before the old ones are given back, and for their next tokens
    pages = sequences * (length // page + 1) * 2 + rng.randint(1, 50)
    return {"kind": kind, "sequences": sequences, "count": rng.randint(1, sequences // 2), "length": length, "layers": rng.randint(1, 12), "pages": pages,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "shape": shape}


# ---- inputs ------------------------------------------------------------------------------------------------------


class _Maker:
    def __init__(self, seed):
        self.random = torch.Generator(device="cuda")
        self.random.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.random)

    def uniform(self, low, high, *shape):
        return torch.rand(*shape, device="cuda", generator=self.random) * (high - low) + low

    def activations(self, rows, width, dtype):
        """Normal values, one channel in a hundred eight times as large."""
        channels = torch.where(self.uniform(0.0, 1.0, width) < 0.01, 8.0, 1.0)
        return (self.normal(rows, width) * channels).to(DTYPES[dtype])

    def codes(self, *shape):
        """What normal keys and values quantise to: a bell around 128."""
        out = torch.empty(*shape, dtype=torch.uint8, device="cuda")
        for layer in out:
            layer.copy_((self.normal(*layer.shape) * 40 + 128).round_().clamp_(1, 255))
        return out

    def cache(self, layers, pages, kv_heads, page, head_dim):
        codes, scales = (layers, pages, kv_heads, page, head_dim), (layers, pages, kv_heads, page // BLOCK)
        return {"k_codes": self.codes(*codes), "v_codes": self.codes(*codes),
                "k_scales": self.uniform(0.02, 0.04, *scales), "v_scales": self.uniform(0.01, 0.06, *scales)}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _shape(case):
    """Lengths and numbers of new tokens of a case's batch."""
    rng = random.Random(case["shape"])
    lengths, counts = [], []
    for b in range(case["batch"]):
        most = case["most"]
        count = most if b == 0 or most == 1 else rng.randint(max(1, most // 3), most)
        lengths.append(case["length"] if b == 0 else rng.randint(max(count, case["length"] // 4), case["length"]))
        counts.append(count)
    return lengths, counts


def _offsets(counts):
    return [sum(counts[:b]) for b in range(len(counts) + 1)]


def _table(rng, lengths, page, width, pages):
    """Pages of sequences, scattered over the pool; and how often each is held."""
    order = list(range(pages))
    rng.shuffle(order)
    table, references = [], [0] * pages
    for length in lengths:
        mine = [order.pop() for _ in range(-(-length // page))]
        for p in mine:
            references[p] = 1
        table.append(mine + [-1] * (width - len(mine)))
    return table, references


def _framework():
    import importlib

    return importlib.import_module("qwen-image-cplus_b200")  # the folder's name has a hyphen


def _sequences(state, make, case, lengths, layers):
    """Cache, tables and lengths of a batch, and the structures of the framework that hold them."""
    rng, page = random.Random(case["shape"] + 1), case["page"]
    width = -(-max(lengths) // page)
    pages = sum(-(-n // page) for n in lengths) + 5
    table, references = _table(rng, lengths, page, width, pages)
    state["cache"] = make.cache(layers, pages, case["kv_heads"], page, case["head_dim"])
    state["table"], state["lengths"], state["references"] = _ints(table), _ints(lengths), _ints(references)


def _handles(state):
    """The framework's descriptions of the buffers; made at the first pass of a state, as a program makes them once."""
    if "handles" not in state:
        qi = _framework()
        state["handles"] = (qi, qi.KvCache(**state["cache"]), qi.KvPages(state["table"], state["lengths"], state["references"]))
    return state["handles"]


def prepare(case, seed):
    make, kind = _Maker(seed), case["kind"]
    state = {"case": case}
    if kind == "norm":
        rows, width = case["rows"], case["width"]
        state["residual"] = (make.normal(rows, width) * 4).to(DTYPES[case["residual"]])
        state["branch"] = make.activations(rows, width, case["branch"])
        state["post"] = make.uniform(0.5, 1.5, width) if case["post"] else None
        state["weight"] = make.uniform(0.5, 1.5, width) if case["norm"] == "rms" else None
        # one row of six vectors for each conditioning vector, as the modulation linear of a block gives them
        vectors = (make.normal(case["groups"], 6 * width) * 0.3).half() if case["modulated"] else None
        state["vectors"] = [vectors[:, i * width:(i + 1) * width] if case["modulated"] else None for i in (2, 4, 3)]  # gate, scale, shift
        state["residual_out"] = torch.empty(rows, width, dtype=DTYPES[case["residual"]], device="cuda")
        state["y"] = torch.empty(rows, width, dtype=DTYPES[case["y"]], device="cuda")
    elif kind == "append":
        lengths, counts = _shape(case)
        heads, dim = case["kv_heads"], case["head_dim"]
        _sequences(state, make, case, lengths, 1)
        tokens = sum(counts)
        state["kv"] = make.activations(tokens, 2 * heads * dim, case["x"])  # keys and values side by side, as one linear writes them
        back = [n + (length - n) % BLOCK for n, length in zip(counts, lengths)]  # from the start of the first block that changes
        state["slots"], state["counts"], state["back"] = _ints(list(range(len(counts)))), counts, back
        state["offsets"], state["back_offsets"] = _ints(_offsets(counts)), _ints(_offsets(back))
        state["k"], state["v"] = (torch.empty(sum(back), heads, dim, device="cuda") for _ in range(2))
    elif kind == "attend":
        lengths, counts = _shape(case)
        _sequences(state, make, case, lengths, 2)
        heads, dim, tokens = case["heads"], case["head_dim"], sum(counts)
        state["q"] = (make.normal(tokens, heads, dim) * 1.5).half()
        state["slots"], state["offsets"], state["counts"] = _ints(list(range(len(counts)))), _ints(_offsets(counts)), counts
        state["y"] = torch.empty(tokens, heads, dim, dtype=torch.float16, device="cuda")
        state["lse"] = torch.empty(tokens, heads, device="cuda") if case["lse"] else None
    else:
        rng, page, count = random.Random(case["shape"]), case["page"], case["count"]
        lengths = [rng.randint(1, case["length"]) for _ in range(case["sequences"])]
        width = -(-(case["length"] + 1) // page) + 1
        table, references = _table(rng, lengths, page, width, case["pages"])
        chosen = rng.sample(range(case["sequences"]), count)
        state["cache"] = make.cache(case["layers"], case["pages"], case["kv_heads"], page, case["head_dim"])
        if kind == "compact":  # the chosen sequences have ended
            for s in chosen:
                for p in table[s]:
                    if p >= 0:
                        references[p] = 0
                table[s], lengths[s] = [-1] * width, 0
        # table, lengths and references in one buffer, so that a snapshot of them is one copy
        parts = [[p for row in table for p in row], lengths, references]
        state["book"] = _ints(sum(parts, []))
        state["table"], state["lengths"], state["references"] = torch.split(state["book"], [len(p) for p in parts])
        state["table"] = state["table"].view(case["sequences"], width)
        state["snapshot"] = state["book"].clone()
        state["children"], state["ones"] = _ints(chosen), _ints([1] * count)
        state["parents"] = _ints([rng.randrange(case["sequences"]) for _ in range(count)])
        state["told"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _norm(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)


def _plain_norm(s):
    case = s["case"]
    branch = s["branch"].float()
    if s["post"] is not None:
        branch = _norm(branch, case["norm"]) * s["post"]
    owner = torch.arange(case["rows"], device="cuda") // -(-case["rows"] // case["groups"])
    gate, scale, shift = (None if v is None else v.float()[owner] for v in s["vectors"])
    residual = s["residual"].float() + 0.5 * (branch if gate is None else gate * branch)
    y = _norm(residual, case["norm"])
    if s["weight"] is not None:
        y = y * s["weight"]
    if scale is not None:
        y = y * (1 + scale) + shift
    return residual.to(DTYPES[case["residual"]]), y.to(DTYPES[case["y"]])


def _positions(lengths, counts, most):
    """Positions of the last counts[b] tokens of each sequence, padded to `most` columns; which columns are tokens."""
    column = torch.arange(most, device="cuda")
    return (lengths - counts)[:, None] + column, column < counts[:, None]


def _places(s, positions, inside):
    """Page and place within it of each position (page 0 outside)."""
    page = s["case"]["page"]
    at = torch.where(inside, positions, 0)
    return torch.where(inside, torch.gather(s["table"], 1, at // page), 0).long(), at % page


def _values(s, layer, which, pages, places):
    """Cached values in 32 bits: [sequences, tokens, heads, head_dim]."""
    codes = s["cache"][which + "_codes"][layer][pages, :, places]
    return (codes.float() - 128) * s["cache"][which + "_scales"][layer][pages, :, places // BLOCK][..., None]


def _plain_append(s):
    case, cache, lengths = s["case"], s["cache"], s["lengths"].long()
    counts = s["offsets"].long().diff()
    blocks = (case["most"] + 2 * BLOCK - 2) // BLOCK
    # whole blocks, from the one that the first new token falls into
    first = (lengths - counts) // BLOCK * BLOCK
    positions = first[:, None] + torch.arange(blocks * BLOCK, device="cuda")
    held = positions < lengths[:, None]
    new = held & (positions >= (lengths - counts)[:, None])
    pages, places = _places(s, positions, held)
    token = torch.where(new, positions - (lengths - counts)[:, None] + s["offsets"].long()[:-1, None], 0)
    heads, dim = case["kv_heads"], case["head_dim"]
    for which, x in (("k", s["kv"][:, :heads * dim]), ("v", s["kv"][:, heads * dim:])):
        x = torch.where(new[..., None, None], x.float().view(-1, heads, dim)[token], 0.0)
        codes, scales = cache[which + "_codes"][0], cache[which + "_scales"][0]
        split = (len(counts), blocks, BLOCK, heads)
        largest = x.abs().amax(-1).view(split).amax(2) / 127
        at, block = pages.view(split[:3])[:, :, 0], places.view(split[:3])[:, :, 0] // BLOCK
        before = (held & ~new).view(split[:3]).any(2)
        old = torch.where(before[..., None], scales[at, :, block], 0.0)
        scale = torch.maximum(old, largest)
        each = scale.repeat_interleave(BLOCK, 1)[..., None]
        fresh = torch.where(each > 0, x / each, 0.0).round().clamp(-127, 127)
        factor = torch.where(scale > 0, old / scale, 1.0).repeat_interleave(BLOCK, 1)[..., None]
        kept = ((codes[pages, :, places].float() - 128) * factor).round()
        out = (torch.where(new[..., None, None], fresh, kept) + 128).to(torch.uint8)
        codes[pages[held], :, places[held]] = out[held]
        touched = new.view(split[:3]).any(2)
        scales[at[touched], :, block[touched]] = scale[touched]
    back = s["back_offsets"].long().diff()
    positions, inside = _positions(lengths, back, case["most"] + BLOCK - 1)
    pages, places = _places(s, positions, inside)
    return [_values(s, 0, which, pages, places)[inside] for which in "kv"]


def _plain_attend(s):
    case, lengths = s["case"], s["lengths"].long()
    heads, kv_heads, dim, most, batch = case["heads"], case["kv_heads"], case["head_dim"], case["most"], case["batch"]
    counts = s["offsets"].long().diff()
    positions = torch.arange(case["length"], device="cuda").expand(batch, -1)
    held = positions < lengths[:, None]
    pages, places = _places(s, positions, held)
    k, v = (_values(s, 1, which, pages, places).masked_fill(~held[..., None, None], 0.0).transpose(1, 2) for which in "kv")
    mine, inside = _positions(lengths, counts, most)
    token = torch.where(inside, mine - (lengths - counts)[:, None] + s["offsets"].long()[:-1, None], 0)
    q = s["q"].float()[token].view(batch, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(batch, kv_heads, -1, dim) @ k.transpose(2, 3)).mul_(dim ** -0.5)
    seen = held[:, None, :].expand(-1, most, -1)
    if case["causal"]:
        seen = seen & (positions[:, None, :] <= mine[:, :, None])
    if case["window"]:
        seen = seen & (positions[:, None, :] > mine[:, :, None] - case["window"])
    scores.view(batch, kv_heads, -1, most, case["length"]).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    y = torch.where(total > 0, (scores @ v) / total, 0.0).view(batch, kv_heads, -1, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    outputs = [y[inside].half()]
    if s["lse"] is not None:
        outputs.append((top + total.log()).view(batch, heads, most).transpose(1, 2)[inside])
    return outputs


def _copy_pages(cache, sources, targets):
    for pool in cache.values():
        pool[:, targets] = pool[:, sources]


def _plain_fork(s):
    page, table, lengths, references = s["case"]["page"], s["table"], s["lengths"], s["references"]
    parents, children = s["parents"].long(), s["children"].long()
    other = parents != children
    parents, children = parents[other], children[other]
    rows, have = table[parents], lengths[parents]
    column = torch.arange(table.shape[1], device="cuda")
    whole, part = have // page, have % page > 0
    free = (references == 0).nonzero()[:, 0]
    missing = (part.sum() - len(free)).clamp(min=0)
    s["told"][0] = missing
    if missing > 0:
        return
    new = free[torch.cumsum(part, 0) - 1].int()
    shared = torch.where(column < whole[:, None], rows, -1)
    last = (column == whole[:, None]) & part[:, None]
    result = torch.where(last, new[:, None], shared)
    references.index_add_(0, result[result >= 0].long(), torch.ones_like(result[result >= 0]))
    gone = table[children]
    references.index_add_(0, gone[gone >= 0].long(), -torch.ones_like(gone[gone >= 0]))
    table[children], lengths[children] = result, have
    _copy_pages(s["cache"], rows[last].long(), result[last].long())


def _plain_reserve(s):
    page, table, lengths, references = s["case"]["page"], s["table"], s["lengths"], s["references"]
    slots = s["children"].long()
    have, want = (lengths[slots] + page - 1) // page, (lengths[slots] + s["ones"] + page - 1) // page
    need = want - have
    free = (references == 0).nonzero()[:, 0]
    missing = (need.sum() - len(free)).clamp(min=0)
    s["told"][1] = missing
    if missing > 0:
        return
    column = torch.arange(table.shape[1], device="cuda")
    rank = (torch.cumsum(need, 0) - need - have)[:, None] + column
    fresh = (column >= have[:, None]) & (column < want[:, None])
    table[slots] = torch.where(fresh, free[rank.clamp(0, len(free) - 1)].int(), table[slots])
    references[free[: need.sum()]] = 1
    lengths[slots] += s["ones"]


def _plain_compact(s):
    table, references = s["table"], s["references"]
    live = references > 0
    used = live.sum()
    index = torch.arange(len(references), device="cuda")
    sources, targets = (live & (index >= used)).nonzero()[:, 0], (~live & (index < used)).nonzero()[:, 0]
    where = index.clone()
    where[sources] = targets
    table.copy_(torch.where(table >= 0, where[table.clamp(min=0).long()].int(), -1))
    references[targets] = references[sources]
    references[sources] = 0
    s["told"][0] = used
    _copy_pages(s["cache"], sources, targets)


# ---- one pass ----------------------------------------------------------------------------------------------------


def _ok(status):
    if status != 0:
        raise RuntimeError(f"status {status}")


def _pool(s):
    """The pool's bytes as words: pages are moved as they are, whatever their codes stand for."""
    cache = s["cache"]
    return [s["table"], s["lengths"], s["references"], s["told"], cache["k_codes"].view(torch.int32), cache["v_codes"].view(torch.int32), cache["k_scales"], cache["v_scales"]]


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind in ("fork", "compact"):
        s["book"].copy_(s["snapshot"])  # the tables as they were; the pages behind them are not cleared
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "append":
            return _plain_append(s)
        if kind == "attend":
            return _plain_attend(s)
        if kind == "fork":
            _plain_fork(s)
            _plain_reserve(s)
        else:
            _plain_compact(s)
        return _pool(s)
    if kind == "norm":
        qi = _framework()
        if "norm" not in s:
            code = {"f16": qi.DTYPE_F16, "f32": qi.DTYPE_F32}
            gate, scale, shift = s["vectors"]
            s["norm"] = qi.GatedNorm(case["rows"], case["width"], kind=qi.NORM_RMS if case["norm"] == "rms" else qi.NORM_LAYER, epsilon=1e-6, residual=s["residual"],
                                     residual_dtype=code[case["residual"]], branch=s["branch"], branch_dtype=code[case["branch"]], branch_norm=case["post"], branch_weight=s["post"],
                                     residual_scale=0.5, gate=gate, scale=scale, shift=shift, vector_dtype=qi.DTYPE_F16, ld_vector=6 * case["width"],
                                     rows_per_vector=-(-case["rows"] // case["groups"]), weight=s["weight"], residual_out=s["residual_out"], y=s["y"], y_dtype=code[case["y"]])
        _ok(qi.gated_norm_ex(s["norm"]))
        return s["residual_out"], s["y"]
    qi, cache, pages = _handles(s)
    if kind == "append":
        heads, dim, tokens = case["kv_heads"], case["head_dim"], sum(s["counts"])
        if "batch" not in s:
            s["batch"] = qi.KvBatch(s["slots"], s["offsets"], tokens, max(s["counts"]))
            s["back_batch"] = qi.KvBatch(s["slots"], s["back_offsets"], sum(s["back"]), max(s["back"]))
        dtype = qi.DTYPE_F16 if case["x"] == "f16" else qi.DTYPE_F32
        width = 2 * heads * dim
        _ok(qi.kv_append_ex(cache, pages, s["batch"], 0, s["kv"], s["kv"][:, heads * dim:], dtype, width, width))
        _ok(qi.kv_read_ex(cache, pages, s["back_batch"], 0, s["k"], s["v"], qi.DTYPE_F32, heads * dim, heads * dim))
        return s["k"], s["v"]
    if kind == "attend":
        heads, dim = case["heads"], case["head_dim"]
        if "batch" not in s:
            s["batch"] = qi.KvBatch(s["slots"], s["offsets"], sum(s["counts"]), max(s["counts"]))
            s["workspace"] = torch.zeros(qi.kv_attention_workspace(cache, s["batch"], heads, case["length"]), dtype=torch.uint8, device="cuda")
        _ok(qi.kv_attention_ex(cache, pages, s["batch"], 1, s["q"], heads * dim, s["y"], heads * dim, heads, dim ** -0.5, case["length"], causal=case["causal"], window=case["window"],
                               lse=s["lse"], workspace=s["workspace"]))
        return [s["y"]] if s["lse"] is None else [s["y"], s["lse"]]
    if "workspace" not in s:
        s["workspace"] = torch.zeros(qi.kv_pages_workspace(cache, pages), dtype=torch.uint8, device="cuda")
    if kind == "fork":
        _ok(qi.kv_pages_fork_ex(cache, pages, s["parents"], s["children"], case["count"], s["told"], s["workspace"]))
        _ok(qi.kv_pages_reserve_ex(cache, pages, s["children"], s["ones"], case["count"], s["told"][1:], s["workspace"]))
    else:
        _ok(qi.kv_pages_compact_ex(cache, pages, s["told"], s["workspace"]))
    return _pool(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def _pairs(case):
    """Scores that the masks leave: for each sequence, over its queries."""
    total = 0
    for length, count in zip(*_shape(case)):
        for p in range(length - count, length):
            total += (p + 1 if case["causal"] else length) - (max(0, p + 1 - case["window"]) if case["window"] else 0)
    return total


def _moved(case):
    """Pages that a fork or a compaction copies."""
    rng, page = random.Random(case["shape"]), case["page"]
    lengths = [rng.randint(1, case["length"]) for _ in range(case["sequences"])]
    table, references = _table(rng, lengths, page, 1 << 10, case["pages"])
    chosen = rng.sample(range(case["sequences"]), case["count"])
    if case["kind"] == "fork":
        parents = [rng.randrange(case["sequences"]) for _ in range(case["count"])]
        return sum(p != c and lengths[p] % page > 0 for p, c in zip(parents, chosen))
    for s in chosen:
        for p in table[s]:
            if p >= 0:
                references[p] = 0
    used = sum(references)
    return sum(references[used:])


def work(case):
    kind, size = case["kind"], {"f16": 2, "f32": 4}
    if kind == "norm":
        each = 2 * size[case["residual"]] + size[case["branch"]] + size[case["y"]]
        vectors = case["width"] * (4 * case["post"] + 4 * (case["norm"] == "rms") + 6 * case["groups"] * case["modulated"])
        return {"bytes": case["rows"] * case["width"] * each + vectors, "flops": 12.0 * case["rows"] * case["width"]}
    token = 2 * case["kv_heads"] * case["head_dim"]  # codes of a token's keys and values
    scales = 2 * case["kv_heads"] * 4 / BLOCK
    if kind == "append":
        lengths, counts = _shape(case)
        back = sum(n + (length - n) % BLOCK for n, length in zip(counts, lengths))
        return {"bytes": sum(counts) * (token * (size[case["x"]] + 1) + scales) + back * (token * 5 + scales), "flops": 4.0 * back * token}
    if kind == "attend":
        lengths, counts = _shape(case)
        ends = sum(min(length, count + case["window"] - 1) if case["window"] else length for length, count in zip(lengths, counts))
        return {"bytes": ends * (token + scales) + sum(counts) * case["heads"] * (4 * case["head_dim"] + 4 * case["lse"]), "flops": 4.0 * case["head_dim"] * case["heads"] * _pairs(case)}
    page = case["layers"] * case["page"] * (token + scales)
    width = -(-(case["length"] + 1) // case["page"]) + 1
    return {"bytes": 2 * _moved(case) * page + 4.0 * (2 * case["pages"] + 2 * case["sequences"] * width), "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def _exact_norm(case, s):
    def normed(x):
        if case["norm"] == "layer":
            x = x - x.mean(1, keepdim=True)
        return x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt()

    branch = s["branch"].double()
    if case["post"]:
        branch = normed(branch) * s["post"].double()
    each = -(-case["rows"] // case["groups"])
    if case["modulated"]:
        gate, scale, shift = (v.double().repeat_interleave(each, 0)[:case["rows"]] for v in s["vectors"])
        branch = branch * gate
    residual = s["residual"].double() + branch / 2
    y = normed(residual)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    return [residual, y * (1 + scale) + shift if case["modulated"] else y]


def _exact_cached(case, s, b, layer, which):
    """Codes less 128 and scales of sequence b, one row a token."""
    page, length = case["page"], int(s["lengths"][b])
    mine = s["table"][b, : -(-length // page)].long()
    codes = s["cache"][which + "_codes"][layer, mine].transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"])[:length].double() - 128
    scales = s["cache"][which + "_scales"][layer, mine].transpose(1, 2).reshape(-1, case["kv_heads"])
    return codes, scales


def _exact_append(case, s):
    lengths, counts = _shape(case)
    heads, dim = case["kv_heads"], case["head_dim"]
    out = {"k": [], "v": []}
    for b, (length, count) in enumerate(zip(lengths, counts)):
        begin = sum(counts[:b])
        first = (length - count) // BLOCK * BLOCK
        early = length - count - first
        for i, which in enumerate("kv"):
            x = s["kv"][begin:begin + count, i * heads * dim:(i + 1) * heads * dim].view(count, heads, dim).double()
            codes, scales = _exact_cached(case, s, b, 0, which)
            padded = torch.cat([torch.zeros(early, heads, dim, device="cuda", dtype=torch.float64), x])
            padded = torch.cat([padded, padded.new_zeros(-len(padded) % BLOCK, heads, dim)]).view(-1, BLOCK, heads, dim)
            scale = (padded.abs().amax((1, 3)).float() / 127).double()  # stored in 32 bits
            old = scales[first // BLOCK].double()
            if early:
                scale[0] = torch.maximum(scale[0], old)
            q = torch.nan_to_num(padded / scale[:, None, :, None]).round()
            if early:
                q[0, :early] = (codes[first:first + early] * torch.nan_to_num(old / scale[0])[:, None]).round()
            out[which].append((q * scale[:, None, :, None]).view(-1, heads, dim)[: early + count])
    return [torch.cat(out["k"]), torch.cat(out["v"])]


def _exact_attend(case, s):
    lengths, counts = _shape(case)
    group, dim = case["heads"] // case["kv_heads"], case["head_dim"]
    ys, lses = [], []
    for b, (length, count) in enumerate(zip(lengths, counts)):
        begin = sum(counts[:b])
        q = s["q"][begin:begin + count].double()
        k, v = ((codes * scales.double().repeat_interleave(BLOCK, 0)[:length, :, None]) for codes, scales in (_exact_cached(case, s, b, 1, which) for which in "kv"))
        p, j = torch.arange(length - count, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
        hidden = torch.zeros(count, length, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= j > p
        if case["window"]:
            hidden |= j <= p - case["window"]
        y, lse = torch.zeros(count, case["heads"], dim, dtype=torch.float64, device="cuda"), torch.empty(count, case["heads"], dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            scores = (q[:, h] @ k[:, h // group].T / math.sqrt(dim)).masked_fill_(hidden, -math.inf)
            lse[:, h] = scores.logsumexp(1)
            y[:, h] = torch.nan_to_num(torch.exp(scores - lse[:, h, None])) @ v[:, h // group]
        ys.append(y)
        lses.append(lse)
    return [torch.cat(ys)] + ([torch.cat(lses)] if case["lse"] else [])


def exact(case, seed):
    """Pages are only moved, and tables are whole numbers: those cases have no such values."""
    if case["kind"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend}[case["kind"]](case, s)
