"""The operators of serving over a paged key/value cache: what is measured, in plain form and through the library.

A serving loop over the paged cache (``xpu_playground_b200.kv_cache.KvCache``) uses five operators: causal attention
over the packed prompts that arrive together, attention of a tree of drafted tokens over the cache (a tree of one node
is the ordinary decode step), appending the keys and values of prompts or accepted drafts to the cache's pages,
forking sequences, and compacting the pool.

``own = False`` runs each operator as elementary torch operations in 32 bits, ``own = True`` as a program that uses the
library calls it. ``exact`` computes the same outputs in 64 bits from the definitions.

Layouts: packed tokens [tokens, heads, head_dim]; the pool [layers, pages, kv_heads, page_size, head_dim] for keys and
for values; tables [sequences, width] of page ids (-1: none); lens [sequences]; refs [pages] counts each page's users.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # one short chat turn: latency of a single prompt
        {"name": "prompt one short", "op": "prompt", "type": "bf16", "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "sequences": 1, "shortest": 37, "longest": 37, "mix": 1},
        # sixteen users' prompts of very different lengths, packed
        {"name": "prompt packed ragged", "op": "prompt", "type": "fp16", "q_heads": 16, "kv_heads": 8, "head_dim": 128,
         "sequences": 16, "shortest": 1, "longest": 2047, "mix": 2},
        # one long document
        {"name": "prompt long", "op": "prompt", "type": "bf16", "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "sequences": 1, "shortest": 8192, "longest": 8192, "mix": 3},
        # ordinary decode of one sequence: a tree of one node
        {"name": "tree single token", "op": "tree", "type": "bf16", "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 16, "sequences": 1, "shortest": 2048, "longest": 2048, "fewest": 1, "nodes": 1, "mix": 4},
        # sixteen sequences with small trees of different sizes at different lengths
        {"name": "tree batch ragged", "op": "tree", "type": "fp16", "q_heads": 16, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "sequences": 16, "shortest": 1, "longest": 2051, "fewest": 1, "nodes": 23, "mix": 5},
        # sixteen long sequences with the largest trees
        {"name": "tree long", "op": "tree", "type": "bf16", "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "page_size": 16, "sequences": 16, "shortest": 8192, "longest": 16384, "fewest": 64, "nodes": 64, "mix": 6},
        # the accepted tokens of sixteen trees, all layers
        {"name": "append accepted", "op": "append", "type": "bf16", "kv_heads": 8, "head_dim": 128, "layers": 36,
         "page_size": 16, "sequences": 16, "shortest": 100, "longest": 500, "fewest": 1, "tokens": 6, "spread": True,
         "mix": 7},
        # four prompts entering the cache, all layers
        {"name": "append prompts", "op": "append", "type": "bf16", "kv_heads": 8, "head_dim": 128, "layers": 36,
         "page_size": 16, "sequences": 4, "shortest": 0, "longest": 0, "fewest": 301, "tokens": 2048, "spread": False,
         "mix": 8},
        # four samples of one prompt
        {"name": "fork samples", "op": "fork", "type": "bf16", "kv_heads": 8, "head_dim": 128, "layers": 28,
         "page_size": 16, "sequences": 1, "children": 4, "shortest": 137, "longest": 137, "mix": 9},
        # eight prompts with eight beams each, large pages
        {"name": "fork beams", "op": "fork", "type": "fp16", "kv_heads": 8, "head_dim": 128, "layers": 36,
         "page_size": 128, "sequences": 8, "children": 64, "shortest": 500, "longest": 4000, "mix": 10},
        # a small pool after a few sequences left
        {"name": "compact small", "op": "compact", "type": "bf16", "kv_heads": 8, "head_dim": 128, "layers": 28,
         "page_size": 16, "sequences": 4, "shortest": 30, "longest": 200, "filled": 80, "mix": 11},
        # a large pool, half empty
        {"name": "compact large", "op": "compact", "type": "bf16", "kv_heads": 8, "head_dim": 128, "layers": 36,
         "page_size": 64, "sequences": 24, "shortest": 200, "longest": 2000, "filled": 50, "mix": 12},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "append", "fork", "compact"])
    q_heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (16, 8, 128), (8, 8, 128), (28, 4, 128), (24, 8, 128),
                                              (4, 2, 128), (32, 8, 64), (14, 2, 64), (16, 1, 64)])
    case = {"op": op, "type": rng.choice(["bf16", "fp16"]), "kv_heads": kv_heads, "head_dim": head_dim,
            "mix": rng.randrange(1 << 30)}
    if op == "prompt":
        longest = _log(rng, 1, 8192)
        most = max(1, min(64, 32 * 8192 * 8192 // (q_heads * longest * longest), 32768 // longest))
        return case | {"q_heads": q_heads, "sequences": _log(rng, 1, most), "longest": longest,
                       "shortest": _log(rng, 1, longest)}
    case["page_size"] = rng.choice([16, 32, 64, 128])
    if op == "tree":
        longest, nodes = _log(rng, 1, 16384), _log(rng, 1, 64)
        rows = 32 * 64 * 16 * 12288 // (q_heads * nodes * longest)
        keys = 16 * 12288 * 8 * 128 // (longest * kv_heads * head_dim)
        return case | {"q_heads": q_heads, "sequences": _log(rng, 1, max(1, min(32, rows, keys))), "longest": longest,
                       "shortest": _log(rng, 1, longest), "nodes": nodes, "fewest": _log(rng, 1, nodes)}
    case["layers"] = _log(rng, 1, 36)
    room = 36 * 8 * 128 * 4000 // (case["layers"] * kv_heads * head_dim)  # rows that cost what the largest case's do
    if op == "append":
        tokens = _log(rng, 1, 2048)
        return case | {"tokens": tokens, "fewest": _log(rng, 1, tokens), "sequences": _log(rng, 1, max(1, min(64, room // tokens))),
                       "shortest": 0, "longest": _log(rng, 1, 600), "spread": rng.random() < 0.5}
    if op == "fork":
        longest = _log(rng, 1, 2000)
        return case | {"sequences": _log(rng, 1, 8), "children": _log(rng, 1, 64), "longest": longest,
                       "shortest": _log(rng, 1, longest)}
    longest = _log(rng, 1, 2000)
    return case | {"sequences": _log(rng, 1, 16), "longest": longest, "shortest": _log(rng, 1, longest),
                   "filled": rng.randrange(30, 96)}


def _spread(case, low, high, salt):
    """One whole number of [low, high] per sequence, `high` among them: part of the case, not of the seed."""
    r = random.Random(case["mix"] * 7 + salt)
    many = [high] + [r.randint(low, high) for _ in range(case["sequences"] - 1)]
    r.shuffle(many)
    return many


def _lengths(case):
    return _spread(case, case["shortest"], case["longest"], 1)


def _counts(case):
    """Nodes of each tree, or tokens that each sequence appends."""
    return _spread(case, case["fewest"], case["nodes"] if case["op"] == "tree" else case["tokens"], 2)


def _pages(positions, size):
    return -(-positions // size)


def _pool(case, lens):
    """Pages of the pool, and entries of a sequence's table."""
    size, used = case["page_size"], [_pages(n, case["page_size"]) for n in lens]
    if case["op"] == "compact":
        return max(sum(used), sum(used) * 100 // case["filled"]), max(used)
    if case["op"] == "fork":
        return sum(used) + case["children"] + 5, max(used) + 1
    if case["op"] == "append":
        after = [_pages(n + c, size) for n, c in zip(lens, _counts(case))]
        return sum(after) + 5, max(after) + 1
    return sum(used) + 5, max(used) + 1


def work(case):
    lens, d, kv = _lengths(case), case["head_dim"], case["kv_heads"]
    row = 2 * kv * d  # bytes of one position's keys, or values, in one layer
    if case["op"] == "prompt":
        tokens, q = sum(lens), case["q_heads"]
        return {"bytes": tokens * (4 * q * d + 2 * row + 4 * q), "flops": 4 * d * q * sum(n * (n + 1) // 2 for n in lens)}
    if case["op"] == "tree":
        counts, q = _counts(case), case["q_heads"]
        entries = sum(_pages(n, case["page_size"]) for n in lens)
        return {"bytes": 2 * row * (sum(lens) + sum(counts)) + sum(counts) * (4 * q * d + 4 * q + 8) + 4 * entries,
                "flops": 4 * d * q * sum(c * (n + 1) for n, c in zip(lens, counts))}
    if case["op"] == "append":
        return {"bytes": case["layers"] * 4 * row * sum(_counts(case)) + 4 * _pool(case, lens)[0], "flops": 0}
    if case["op"] == "fork":
        size, shared = case["page_size"], [lens[i % len(lens)] for i in range(case["children"])]
        return {"bytes": case["layers"] * 4 * row * sum(n % size for n in shared) +
                8 * sum(_pages(n, size) for n in shared) + 4 * _pool(case, lens)[0], "flops": 0}
    pages, width = _pool(case, lens)
    live = sum(_pages(n, case["page_size"]) for n in lens)
    moved = live * (pages - live) / pages  # expected: live pages behind the first `live` ones
    return {"bytes": case["layers"] * 4 * row * case["page_size"] * moved + 4 * pages + 8 * width * len(lens), "flops": 0}


# ----------------------------------------------------------------- inputs ----

def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _starts(counts):
    return [0] + list(np.cumsum(counts))


def _values(g, case, *shape):
    return torch.randn(*shape, device="cuda", dtype=TYPES[case["type"]], generator=g)


def _queries(g, case, tokens):
    """Normalised and rotated queries, flat in some heads and peaked in others."""
    heat = torch.linspace(0.5, 2.0, case["q_heads"], device="cuda")[:, None]
    return (torch.randn(tokens, case["q_heads"], case["head_dim"], device="cuda", generator=g) * heat).to(TYPES[case["type"]])


def _cache(g, r, case, lens, layers, spare_sequences=0):
    """A pool in use: sequences at `lens`, their pages anywhere in it."""
    pages, width = _pool(case, lens)
    at, order = 0, r.permutation(pages)
    tables = np.full((len(lens) + spare_sequences, width), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    for i, n in enumerate(lens):
        used = _pages(n, case["page_size"])
        tables[i, :used] = order[at:at + used]
        refs[order[at:at + used]] = 1
        at += used
    shape = (layers, pages, case["kv_heads"], case["page_size"], case["head_dim"])
    return {"k": _values(g, case, *shape), "v": _values(g, case, *shape), "tables": _ints(tables), "refs": _ints(refs),
            "lens": _ints(list(lens) + [0] * spare_sequences)}


def _trees(seed, counts):
    """Each node's set of attended nodes of its own tree (bit j: node j), for random trees grown from the context."""
    r, sets = random.Random(seed), []
    for n in counts:
        tree = []
        for i in range(n):
            parent = r.randint(max(-1, i - 8), i - 1)
            tree.append((tree[parent] if parent >= 0 else 0) | 1 << i)
        sets += tree
    return torch.tensor(np.array(sets, np.uint64).view(np.int64), device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 32))
    lens, d, kv = _lengths(case), case["head_dim"], case["kv_heads"]
    s = {"case": case, "op": case["op"]}
    if case["op"] == "prompt":
        tokens = sum(lens)
        s |= {"q": _queries(g, case, tokens), "k": _values(g, case, tokens, kv, d), "v": _values(g, case, tokens, kv, d),
              "lens": _ints(lens), "longest": max(lens)}
        if own:
            from xpu_playground_b200 import kernels
            s["plan"] = kernels.PromptPlan(lens, case["q_heads"], kv, d)  # one batch's, for every layer
        return s
    if case["op"] == "tree":
        counts = _counts(case)
        nodes = sum(counts)
        s |= _cache(g, r, case, lens, 2)
        s |= {"q": _queries(g, case, nodes), "new_k": _values(g, case, nodes, kv, d), "new_v": _values(g, case, nodes, kv, d),
              "sequences": _ints(r.permutation(len(lens))), "nodes": nodes, "most": max(counts), "longest": max(lens)}
        placed = [counts[i] for i in s["sequences"].tolist()]  # a tree goes with its sequence
        s |= {"starts": _ints(_starts(placed)), "sets": _trees(seed, placed)}
    elif case["op"] == "append":
        counts = _counts(case)
        tokens = sum(counts)
        held = 2 * tokens if case["spread"] else tokens  # accepted rows stand among rejected ones
        s |= _cache(g, r, case, lens, case["layers"])
        s |= {"new_k": _values(g, case, case["layers"], held, kv, d), "new_v": _values(g, case, case["layers"], held, kv, d),
              "sequences": _ints(range(len(lens))), "before": _ints(lens), "starts": _ints(_starts(counts)), "tokens": tokens,
              "rows": _ints(np.sort(r.permutation(held)[:tokens])) if case["spread"] else None}
    elif case["op"] == "fork":
        many = case["children"]
        s |= _cache(g, r, case, lens, case["layers"], many)
        s |= {"parents": _ints([i % len(lens) for i in range(many)]), "children": _ints(len(lens) + r.permutation(many)),
              "none": _ints([0] * many)}
    else:
        s |= _cache(g, r, case, lens, case["layers"])
        s |= {"tables_then": s["tables"].clone(), "refs_then": s["refs"].clone()}
    if own:
        from xpu_playground_b200 import kernels
        from xpu_playground_b200.kv_cache import KvCache
        s["cache"] = KvCache.wrap(s["k"], s["v"], s["tables"], s["lens"], s["refs"])
        if case["op"] == "tree":
            s["workspace"] = kernels.tree_attention_workspace(len(lens), s["nodes"], case["q_heads"], kv, d)
    return s


# ------------------------------------------------------------- plain forms ----

def _attend(q, k, v, allowed):
    """softmax(q k^T / sqrt(d)) v over the allowed keys in 32 bits, and the logarithm of each row's sum; a row that is
    allowed no key gives zeros and -inf. q [.., rows, d], k and v [.., keys, d]."""
    scores = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(q.shape[-1])).masked_fill_(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out, (top + total.log())[..., 0]


def _prompt(s):
    case, lens, longest, tokens = s["case"], s["lens"].long(), s["longest"], s["q"].shape[0]
    many, kv, d = case["sequences"], case["kv_heads"], case["head_dim"]
    starts, at = lens.cumsum(0) - lens, torch.arange(longest, device="cuda")
    place = (starts[:, None] + at).clamp(max=tokens - 1)
    q = s["q"][place].float().view(many, longest, kv, -1, d).permute(0, 2, 3, 1, 4)
    k, v = (s[x][place].float().permute(0, 2, 1, 3)[:, :, None] for x in ("k", "v"))
    allowed = (at[None, :] <= at[:, None]) & (at < lens[:, None])[:, None, :]
    out, lse = _attend(q, k, v, allowed[:, None, None])
    owner = torch.repeat_interleave(torch.arange(many, device="cuda"), lens, output_size=tokens)
    inside = torch.arange(tokens, device="cuda") - starts[owner]
    out = out.permute(0, 3, 1, 2, 4)[owner, inside].reshape(tokens, -1, d)
    return out.to(s["q"].dtype), lse.permute(0, 3, 1, 2)[owner, inside].reshape(tokens, -1)


def _tree(s):
    case, longest, most, nodes = s["case"], s["longest"], s["most"], s["nodes"]
    kv, d, size = case["kv_heads"], case["head_dim"], case["page_size"]
    sequences, starts = s["sequences"].long(), s["starts"].long()
    many, counts, lens = len(sequences), starts.diff(), s["lens"].long()[s["sequences"].long()]
    held = s["tables"].long()[sequences][:, :_pages(longest, size)].clamp(min=0)
    old_k, old_v = (s[x][1, held].float().transpose(1, 2).reshape(many, kv, -1, d) for x in ("k", "v"))
    at, bits = torch.arange(old_k.shape[2], device="cuda"), torch.arange(most, device="cuda")
    place = (starts[:-1, None] + bits).clamp(max=nodes - 1)
    q = s["q"][place].float().view(many, most, kv, -1, d).permute(0, 2, 3, 1, 4)
    k, v = (torch.cat([old, s[x][place].float().transpose(1, 2)], 2)[:, :, None]
            for old, x in ((old_k, "new_k"), (old_v, "new_v")))
    drafted = ((s["sets"][place][..., None] >> bits) & 1).bool() & (bits < counts[:, None])[:, None, :]
    context = (at < lens[:, None])[:, None, :].expand(-1, most, -1)
    out, lse = _attend(q, k, v, torch.cat([context, drafted], 2)[:, None, None])
    owner = torch.repeat_interleave(torch.arange(many, device="cuda"), counts, output_size=nodes)
    inside = torch.arange(nodes, device="cuda") - starts[owner]
    out = out.permute(0, 3, 1, 2, 4)[owner, inside].reshape(nodes, -1, d)
    return out.to(s["q"].dtype), lse.permute(0, 3, 1, 2)[owner, inside].reshape(nodes, -1)


def _trim(s, sequences, lens):
    """Shortens sequences to `lens`; pages wholly behind the new length lose a user."""
    sequences, size = sequences.long(), s["case"]["page_size"]
    old = s["lens"][sequences].long()
    new = torch.minimum(old, lens.long())
    at, held = torch.arange(s["tables"].shape[1], device="cuda"), s["tables"][sequences]
    drop = (at >= ((new + size - 1) // size)[:, None]) & (at < ((old + size - 1) // size)[:, None])
    s["refs"].scatter_add_(0, held.long().clamp(min=0).flatten(), -drop.int().flatten())
    s["tables"][sequences] = torch.where(drop, -1, held)
    s["lens"][sequences] = new.int()


def _free(s):
    """Page ids, the free ones first in ascending order."""
    return torch.argsort((s["refs"] != 0).int(), stable=True)


def _append(s):
    """Takes the lowest free pages in the sequences' order, then writes every layer's rows."""
    case, size, tokens = s["case"], s["case"]["page_size"], s["tokens"]
    _trim(s, s["sequences"], s["before"])
    sequences, starts = s["sequences"].long(), s["starts"].long()
    old, counts = s["lens"][sequences].long(), starts.diff()
    first, last = (old + size - 1) // size, (old + counts + size - 1) // size
    rank = (last - first).cumsum(0) - (last - first)
    at, free = torch.arange(s["tables"].shape[1], device="cuda"), _free(s)
    fresh = (at >= first[:, None]) & (at < last[:, None])
    ids = free[(rank[:, None] + at - first[:, None]).clamp(0, len(free) - 1)]
    s["refs"].scatter_add_(0, ids.flatten(), fresh.int().flatten())
    s["tables"][sequences] = torch.where(fresh, ids.int(), s["tables"][sequences])
    s["lens"][sequences] = (old + counts).int()
    owner = torch.repeat_interleave(torch.arange(case["sequences"], device="cuda"), counts, output_size=tokens)
    place = old[owner] + torch.arange(tokens, device="cuda") - starts[owner]
    page, slot = s["tables"][sequences[owner], place // size].long(), place % size
    for_rows = slice(None) if s["rows"] is None else s["rows"].long()
    s["k"][:, page, :, slot] = s["new_k"][:, for_rows].transpose(0, 1)
    s["v"][:, page, :, slot] = s["new_v"][:, for_rows].transpose(0, 1)
    return s["k"], s["v"], s["tables"], s["lens"], s["refs"]


def _fork(s):
    """Children share their parents' full pages; a last page that is not full is copied, as far as it is in use, to the
    lowest free page in the children's order."""
    size = s["case"]["page_size"]
    _trim(s, s["children"], s["none"])
    parents, children = s["parents"].long(), s["children"].long()
    lens, rows = s["lens"][parents].long(), s["tables"][parents].long()
    full, part = lens // size, lens % size
    own_page = part > 0
    new = _free(s)[own_page.long().cumsum(0) - own_page.long()]
    at = torch.arange(rows.shape[1], device="cuda")
    shared, fresh = at < full[:, None], (at == full[:, None]) & own_page[:, None]
    s["refs"].scatter_add_(0, rows.clamp(min=0).flatten(), shared.int().flatten())
    s["refs"].scatter_add_(0, new, own_page.int())
    s["tables"][children] = torch.where(shared, rows, torch.where(fresh, new[:, None], -1)).int()
    s["lens"][children] = lens.int()
    which = own_page.nonzero()[:, 0]
    old, new = rows[which, full[which]], new[which]
    used = (torch.arange(size, device="cuda") < part[which][:, None])[None, :, None, :, None]
    s["k"][:, new] = torch.where(used, s["k"][:, old], s["k"][:, new])
    s["v"][:, new] = torch.where(used, s["v"][:, old], s["v"][:, new])
    return s["k"], s["v"], s["tables"], s["lens"], s["refs"]


def _compact(s):
    """With n pages in use, those whose id is n or more move to the free pages below n, both in ascending order."""
    refs, ids = s["refs"], torch.arange(len(s["refs"]), device="cuda")
    live = refs > 0
    many = live.sum()
    moved, holes = (live & (ids >= many)).nonzero()[:, 0], (~live & (ids < many)).nonzero()[:, 0]
    to = ids.scatter(0, moved, holes)
    s["k"][:, holes], s["v"][:, holes] = s["k"][:, moved], s["v"][:, moved]
    s["tables"].copy_(torch.where(s["tables"] >= 0, to[s["tables"].long().clamp(min=0)].int(), -1))
    refs[holes], refs[moved] = refs[moved], 0
    return s["k"], s["v"], s["tables"], s["lens"], s["refs"]


def run(s):
    """One pass. The page operators begin from the state that `prepare` left: appending first takes back what the last
    pass appended, forking first frees the children, compacting first puts the scattered tables back."""
    if s["op"] == "compact":
        s["tables"].copy_(s["tables_then"])
        s["refs"].copy_(s["refs_then"])
    if not own:
        return {"prompt": _prompt, "tree": _tree, "append": _append, "fork": _fork, "compact": _compact}[s["op"]](s)
    if s["op"] in ("prompt", "tree"):
        from xpu_playground_b200 import kernels
        if s["op"] == "prompt":
            return kernels.prompt_attention(s["plan"], s["q"], s["k"], s["v"])
        return kernels.tree_attention(s["cache"], 1, s["sequences"], s["starts"], s["sets"], s["q"], s["new_k"], s["new_v"],
                                      s["workspace"])
    cache = s["cache"]
    if s["op"] == "append":
        cache.trim(s["sequences"], s["before"])
        cache.append(s["sequences"], s["starts"], s["new_k"], s["new_v"], s["rows"])
    elif s["op"] == "fork":
        cache.trim(s["children"], s["none"])
        cache.fork(s["parents"], s["children"])
    else:
        cache.compact()
    return cache.k, cache.v, cache.tables, cache.lens, cache.refs


# ---------------------------------------------------------------- in 64 bits ----

def _rows64(q, k, v, allowed):
    """Outputs and logarithms of sums of one head's rows, as a softmax is defined."""
    z = torch.einsum("rd,kd->rk", q.double(), k.double()) / float(q.shape[-1]) ** 0.5
    z = torch.where(allowed, z, torch.full_like(z, -math.inf))
    lse = torch.logsumexp(z, -1)
    w = torch.where(allowed, torch.exp(z - lse[:, None]), torch.zeros_like(z))
    return w @ v.double(), lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("prompt", "tree"):
        q, group = s["q"], case["q_heads"] // case["kv_heads"]
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
        begin = 0
        for i in range(case["sequences"]):
            if case["op"] == "prompt":
                n = int(s["lens"][i])
                keys, values = s["k"][begin:begin + n], s["v"][begin:begin + n]
                allowed = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            else:
                begin, n = int(s["starts"][i]), int(s["starts"][i + 1] - s["starts"][i])
                sequence = int(s["sequences"][i])
                context = int(s["lens"][sequence])
                keys, values = ([], [])
                for p in range(_pages(context, case["page_size"])):
                    fill = min(case["page_size"], context - p * case["page_size"])
                    page = int(s["tables"][sequence, p])
                    keys.append(s["k"][1, page, :, :fill].transpose(0, 1))
                    values.append(s["v"][1, page, :, :fill].transpose(0, 1))
                keys = torch.cat(keys + [s["new_k"][begin:begin + n]])
                values = torch.cat(values + [s["new_v"][begin:begin + n]])
                sets = [[b >> j & 1 for j in range(n)] for b in s["sets"][begin:begin + n].tolist()]
                allowed = torch.cat([torch.ones(n, context, dtype=torch.bool, device="cuda"),
                                     torch.tensor(sets, dtype=torch.bool, device="cuda")], 1)
            for h in range(case["q_heads"]):
                out[begin:begin + n, h], lse[begin:begin + n, h] = _rows64(
                    q[begin:begin + n, h], keys[:, h // group], values[:, h // group], allowed)
            begin += n if case["op"] == "prompt" else 0
        return out, lse
    size, k, v = case["page_size"], s["k"], s["v"]
    tables, lens, refs = (s[x].tolist() for x in ("tables", "lens", "refs"))
    if case["op"] == "append":
        starts = s["starts"].tolist()
        rows = list(range(s["tokens"])) if s["rows"] is None else s["rows"].tolist()
        spots = []
        for i, sequence in enumerate(s["sequences"].tolist()):
            for _ in range(starts[i], starts[i + 1]):
                n = lens[sequence]
                if n % size == 0:
                    tables[sequence][n // size] = refs.index(0)
                    refs[tables[sequence][n // size]] = 1
                spots.append(tables[sequence][n // size] * size + n % size)
                lens[sequence] = n + 1
        spots, rows = torch.tensor(spots, device="cuda"), torch.tensor(rows, device="cuda")
        for layer in range(case["layers"]):
            for pool, new in ((k, s["new_k"]), (v, s["new_v"])):
                flat = pool[layer].transpose(1, 2).clone().reshape(-1, case["kv_heads"], case["head_dim"])  # by position
                flat[spots] = new[layer, rows]
                pool[layer] = flat.view(-1, size, case["kv_heads"], case["head_dim"]).transpose(1, 2)
    elif case["op"] == "fork":
        for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
            n = lens[child] = lens[parent]
            for p in range(_pages(n, size)):
                page = tables[parent][p]
                if n < (p + 1) * size:
                    new = refs.index(0)
                    k[:, new, :, :n - p * size] = k[:, page, :, :n - p * size]
                    v[:, new, :, :n - p * size] = v[:, page, :, :n - p * size]
                    page = new
                tables[child][p] = page
                refs[page] += 1
    else:
        live = [p for p, n in enumerate(refs) if n > 0]
        holes = [p for p, n in enumerate(refs) if n == 0 and p < len(live)]
        moves = dict(zip([p for p in live if p >= len(live)], holes))
        for old, new in moves.items():
            k[:, new], v[:, new] = k[:, old], v[:, old]
            refs[new], refs[old] = refs[old], 0
        tables = [[moves.get(p, p) for p in row] for row in tables]
    return k, v, _ints(tables), _ints(lens), _ints(refs)
