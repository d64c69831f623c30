"""The timed operators of speculative decoding: attention of drafted token trees over a K/V cache, the walk that accepts drafted tokens,
the move that keeps the accepted rows of a cache, and copies of cache rows.

A sequence `s` of a batch has `prefix[s]` cached rows and a tree of drafted tokens, rows row_start[s] .. row_start[s + 1] - 1 of the batch.  Node i of a
tree is written at cache row prefix[s] + i and names an earlier node of the same tree (or -1) as its parent.  A node sees the cached rows before the tree and,
of the tree, its ancestors and itself.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one conversation, a small tree behind a short prompt: the smallest verification step, where latency counts
        dict(name="attn 1 x 8, 500 rows", op="attn", n_seq=1, tree=8, ctx=500, ragged=False, heads=32, kv_heads=8, hd=128, q="bf16", cache="bf16", page=0, window=0, sinks=False),
        # a single token (a tree that is its root) behind a long paged context
        dict(name="attn 1 x 1, 4095 rows, pages", op="attn", n_seq=1, tree=1, ctx=4095, ragged=False, heads=32, kv_heads=8, hd=128, q="bf16", cache="bf16", page=64, window=0, sinks=False),
        # a serving batch: 32 conversations of different lengths, trees of 8 to 16 nodes, a paged pool
        dict(name="attn 32 x 16, 2048 rows, pages", op="attn", n_seq=32, tree=16, ctx=2048, ragged=True, heads=32, kv_heads=8, hd=128, q="bf16", cache="bf16", page=64, window=0, sinks=False),
        # f32 queries (this runtime's own activations) with 64 heads of 64 over 8 K/V heads, a sliding window and sinks; odd sizes
        dict(name="attn 5 x 13, window 128, f32", op="attn", n_seq=5, tree=13, ctx=1001, ragged=True, heads=64, kv_heads=8, hd=64, q="f32", cache="bf16", page=64, window=128, sinks=True),
        # wide trees and eight query heads per K/V head: bound by the products
        dict(name="attn 8 x 64, 4096 rows, 8 per head", op="attn", n_seq=8, tree=64, ctx=4096, ragged=False, heads=64, kv_heads=8, hd=64, q="bf16", cache="bf16", page=0, window=0, sinks=False),
        # long contexts: 16 sequences of up to 32768 rows in small pages
        dict(name="attn 16 x 32, 32768 rows, pages", op="attn", n_seq=16, tree=32, ctx=32768, ragged=True, heads=32, kv_heads=8, hd=128, q="bf16", cache="bf16", page=16, window=0, sinks=False),
        # one conversation's step: which of 8 drafted tokens stand, over a vocabulary of 128256
        dict(name="accept 1 x 8", op="accept", n_seq=1, tree=8, accepted=4, ragged=False, vocab=128256),
        # a serving batch with wide trees
        dict(name="accept 32 x 64", op="accept", n_seq=32, tree=64, accepted=5, ragged=True, vocab=128256),
        # the accepted rows of one conversation close up, all 32 layers
        dict(name="compact 1 x 8, 32 layers", op="compact", n_seq=1, tree=8, accepted=4, ctx=500, ragged=False, layers=32, row=1024, page=0),
        # the same for a serving batch with a paged pool, odd lengths
        dict(name="compact 32 x 64, 32 layers, pages", op="compact", n_seq=32, tree=64, accepted=7, ctx=333, ragged=True, layers=32, row=1024, page=64),
        # eight sequences fork in the middle of a page: the rows of that page are copied in every layer
        dict(name="copy 8 x 37 rows, 32 layers", op="copy", spans=8, rows=37, ragged=True, layers=32, row=1024),
        # a prompt's rows given to two other contiguous slots
        dict(name="copy 2 x 4001 rows, 32 layers", op="copy", spans=2, rows=4001, ragged=False, layers=32, row=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "accept", "compact", "copy"])
    if op == "attn":
        while True:
            kv, g, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 128])
            n, t, ctx = _log(rng, 1, 48), _log(rng, 1, 100), _log(rng, 1, 32768)
            q = rng.choice(["bf16", "bf16", "f32"])
            c = dict(op=op, n_seq=n, tree=t, ctx=ctx, ragged=rng.random() < 0.6, heads=kv * g, kv_heads=kv, hd=hd, q=q, cache="f32" if q == "f32" and rng.random() < 0.4 else "bf16",
                     page=rng.choice([0, 0, 16, 64, 128]), window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]), sinks=rng.random() < 0.25)
            # at most the largest listed case's keys and products, a third of them in 32 bits
            part = 1 if q == "bf16" else 3
            if n * (ctx + t) * kv * hd * part <= 16 * 32800 * 8 * 128 and n * t * (ctx + t) * kv * g * hd * part <= 16 * 32 * 32800 * 32 * 128:
                return c
    if op == "accept":
        while True:
            n, t, v = _log(rng, 1, 48), _log(rng, 1, 128), _log(rng, 1000, 201088)
            if n * t * v <= 32 * 64 * 128256:
                return dict(op=op, n_seq=n, tree=t, accepted=rng.randint(1, min(t, 8)), ragged=rng.random() < 0.5, vocab=v)
    if op == "compact":
        while True:
            n, t, ctx, layers, row = _log(rng, 1, 48), _log(rng, 1, 128), _log(rng, 1, 1000), rng.randint(1, 36), 16 * _log(rng, 1, 128)
            if n * (ctx + t) * layers * row <= 32 * 400 * 32 * 1024:
                return dict(op=op, n_seq=n, tree=t, accepted=rng.randint(1, min(t, 8)), ctx=ctx, ragged=rng.random() < 0.5, layers=layers, row=row, page=rng.choice([0, 16, 64]))
    while True:
        n, rows, layers, row = _log(rng, 1, 64), _log(rng, 1, 4000), rng.randint(1, 36), 8 * _log(rng, 1, 256)
        if n * rows * layers * row <= 2 * 4001 * 32 * 1024:
            return dict(op="copy", spans=n, rows=rows, ragged=rng.random() < 0.5, layers=layers, row=row)


def _sizes(case):
    """Nodes and cached rows of every sequence."""
    n, t = case["n_seq"], case["tree"]
    ctx = case.get("ctx", 0)
    if not case["ragged"]:
        return [t] * n, [ctx] * n
    return [t - s * 5 % ((t + 1) // 2) for s in range(n)], [ctx - s * 7919 % (ctx * 3 // 4 + 1) for s in range(n)]


def _accepted(case):
    return [min(t, 1 + (case["accepted"] - 1 + s) % case["accepted"]) if case["ragged"] else min(t, case["accepted"]) for s, t in enumerate(_sizes(case)[0])]


def _spans(case):
    n, r = case["spans"], case["rows"]
    return [r - s * 3 % ((r + 1) // 2) if case["ragged"] else r for s in range(n)]


def _tree_state(case, g):
    """The trees: row_start, prefix, parent, and the same facts spread over a [n_seq, tree] grid for the plain forms."""
    nodes, ctx = _sizes(case)
    n, t = case["n_seq"], case["tree"]
    row_start = torch.zeros(n + 1, dtype=torch.int64)
    row_start[1:] = torch.tensor(nodes).cumsum(0)
    dev = dict(device="cuda")
    nodes_d, row_start_d = torch.tensor(nodes, **dev), row_start.to(device="cuda", dtype=torch.int32)
    i = torch.arange(t, **dev)
    # half of the nodes continue the node before, the others hang below any earlier one: deep paths and wide levels
    u = torch.rand(n, t, generator=g, **dev)
    back = torch.rand(n, t, generator=g, **dev)
    parent = torch.where(u < 0.5, i - 1, (back * i).long().clamp(max=t - 1)).minimum((i - 1).expand(n, t))
    live = i < nodes_d[:, None]
    return dict(n_seq=n, max_rows=t, max_prefix=max(ctx), row_start=row_start_d, prefix=torch.tensor(ctx, dtype=torch.int32, **dev), parent=parent[live].to(torch.int32),
                n_rows=int(row_start[-1]))


def _pages(case, g):
    """Where the rows of the sequences are: (rows of the pool, page table or None, rows of a slot)."""
    nodes, ctx = _sizes(case)
    page, most = case["page"], max(a + b for a, b in zip(nodes, ctx))
    if not page:
        return case["n_seq"] * most, None, most
    per = -(-most // page)
    need = torch.tensor([-(-(a + b) // page) for a, b in zip(nodes, ctx)], device="cuda")
    total = int(need.sum()) + 3
    order = torch.randperm(total, generator=g, device="cuda")[: total - 3].to(torch.int32)
    table = torch.full((case["n_seq"], per), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(per, device="cuda") < need[:, None]] = order
    return total * page, table, most


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = dict(device="cuda")
    state = dict(case=case)
    if case["op"] == "copy":
        lens = _spans(case)
        n, r = len(lens), case["rows"]
        rows = 2 * n * r + 5
        kv = torch.randn(2 * case["layers"], rows, case["row"], generator=g, dtype=torch.bfloat16, **dev)
        first = torch.randperm(2 * n, generator=g, **dev) * r + 2
        spans = torch.stack([first[:n], first[n:], torch.tensor(lens, **dev)], 1).to(torch.int32)
        return dict(state, kv=kv, spans=spans, max_rows=max(lens), planes=_planes(kv))
    state.update(_tree_state(case, g))
    if case["op"] == "attn":
        t = _TYPES[case["cache"]]
        rows, table, most = _pages(case, g)
        width = case["kv_heads"] * case["hd"]
        k = torch.randn(rows, width, generator=g, dtype=t, **dev)
        v = torch.randn(rows, width, generator=g, dtype=t, **dev)
        q = (torch.randn(state["n_rows"], case["heads"] * case["hd"], generator=g, **dev) * 1.5).to(_TYPES[case["q"]])
        sinks = torch.randn(case["heads"], generator=g, **dev) if case["sinks"] else None
        return dict(state, k=k, v=v, q=q, sinks=sinks, out=torch.zeros_like(q), rows=rows, table=table, max_seq=most)
    path = _planted_path(case, state, g)
    if case["op"] == "accept":
        logits = torch.randn(state["n_rows"], case["vocab"], generator=g, **dev)
        tokens = torch.randint(case["vocab"], (state["n_rows"],), generator=g, dtype=torch.int32, **dev)
        # the model agrees with the drafts along the path: the next node's token stands out
        a, b, s = path[:, :-1], path[:, 1:], state["row_start"][:-1, None].long()
        at, child = (a + s)[b >= 0], (b + s)[b >= 0]
        logits[at, tokens[child].long()] = 9.0
        return dict(state, logits=logits, tokens=tokens, path_len=case["tree"])
    rows, table, most = _pages(case, g)
    kv = torch.randn(2 * case["layers"], rows, case["row"], generator=g, dtype=torch.bfloat16, **dev)
    return dict(state, kv=kv, rows=rows, table=table, max_seq=most, path=path.to(torch.int32).contiguous(), n_accepted=(path >= 0).sum(1).to(torch.int32), planes=_planes(kv))


def _planes(kv):
    """Address and bytes of a row of every plane, as the operators on cache rows take them."""
    step = kv.stride(0) * kv.element_size()
    return torch.tensor([[kv.data_ptr() + i * step, kv.stride(1) * kv.element_size()] for i in range(kv.shape[0])], dtype=torch.int64, device="cuda")


def _planted_path(case, state, g):
    """[n_seq, tree]: node 0 and then accepted - 1 more nodes, each the child of the one before, -1 behind them.  The trees are changed so that the path exists."""
    n, t = case["n_seq"], case["tree"]
    dev = dict(device="cuda")
    nodes = (state["row_start"][1:] - state["row_start"][:-1]).long()
    want = torch.tensor(_accepted(case), **dev)
    order = torch.rand(n, t, generator=g, **dev)
    order = torch.where(torch.arange(t, **dev) < nodes[:, None], order, 2.0)
    order[:, 0] = -1.0
    chosen = order.argsort(1).argsort(1) < want[:, None]                     # node 0 and want - 1 others
    at = torch.where(chosen, torch.arange(t, **dev), t).sort(1).values
    path = torch.where(at < t, at, -1)
    a, b, s = path[:, :-1], path[:, 1:], state["row_start"][:-1, None].long()
    state["parent"][(b + s)[b >= 0]] = a[b >= 0].to(torch.int32)
    return path


# ------------------------------------------------------------------------------------------------------------ the plain forms


def _grid(state):
    """(rows of the batch on the grid, -1 behind a tree's last node; parents on the grid)."""
    i = torch.arange(state["max_rows"], device="cuda")
    row = state["row_start"][:-1, None].long() + i
    row = torch.where(row < state["row_start"][1:, None], row, -1)
    parent = torch.where(row >= 0, state["parent"].long()[row.clamp(min=0)], -1)
    return row, parent


def _ancestors(parent):
    """[n_seq, tree, tree]: whether node j is an ancestor of node i, or i itself.  The sum of the powers of the parent matrix P is the inverse of I - P."""
    n, t = parent.shape
    eye = torch.eye(t, device="cuda").expand(n, t, t)
    p = (parent[:, :, None] == torch.arange(t, device="cuda")).float()
    return torch.linalg.solve_triangular(eye - p, eye, upper=False, unitriangular=True) > 0.5


def _cache_rows(state, page, count):
    """[n_seq, count]: cache rows 0 .. count - 1 of every sequence."""
    j = torch.arange(count, device="cuda")
    if state["table"] is None:
        return torch.arange(state["n_seq"], device="cuda")[:, None] * state["max_seq"] + j
    return state["table"].long()[:, j // page].clamp(min=0) * page + j % page


def _plain_attn(state):
    c = state["case"]
    n, t, h, kvh, hd = state["n_seq"], state["max_rows"], c["heads"], c["kv_heads"], c["hd"]
    row, parent = _grid(state)
    anc = _ancestors(parent)
    keys = state["max_prefix"] + t
    where = _cache_rows(state, c["page"], keys).clamp(max=state["rows"] - 1)
    k = state["k"][where].float().view(n, keys, kvh, hd).permute(0, 2, 3, 1)
    q = state["q"].float()[row.clamp(min=0)].view(n, t, kvh, h // kvh, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, hd)
    x = (q @ k).view(n, kvh, h // kvh, t, keys) * (1.0 / math.sqrt(hd))
    del k
    j, prefix = torch.arange(keys, device="cuda"), state["prefix"].long()[:, None, None]
    node = j - prefix                                                        # [n, 1, keys]: which node of the tree a key is
    depth = anc.sum(2) - 1
    in_tree = (node >= 0) & (node < t) & anc.gather(2, node.clamp(0, t - 1).expand(n, t, keys))
    sees = (node < 0) | in_tree
    if c["window"]:
        place = torch.where(node < 0, j, prefix + depth[:, None, :].gather(2, node.clamp(0, t - 1)))
        sees &= prefix + depth[:, :, None] - place < c["window"]
    x = x.masked_fill(~sees[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(1, kvh, h // kvh, 1, 1)
        top = torch.maximum(top, sink)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sink - top)
    del x
    v = state["v"][where].float().view(n, keys, kvh, hd).permute(0, 2, 1, 3)
    o = (w.view(n, kvh, -1, keys) @ v).view(n, kvh, h // kvh, t, hd) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, t, h * hd)
    out = state["out"]
    out[row[row >= 0]] = o[row >= 0].to(out.dtype)
    return out


def _plain_accept(state):
    n, t = state["n_seq"], state["max_rows"]
    row, parent = _grid(state)
    pick = state["logits"].argmax(1)
    token = torch.where(row >= 0, state["tokens"].long()[row.clamp(min=0)], -1)
    i = torch.arange(t, device="cuda")
    # a node stands if its token is what its parent's row picks, no earlier child of that parent has it too, and all its ancestors stand
    wanted = torch.where(parent >= 0, pick[(state["row_start"][:-1, None].long() + parent).clamp(min=0)], -2)
    same = (parent[:, :, None] == parent[:, None, :]) & (token[:, :, None] == token[:, None, :]) & (i[None, :, None] > i)
    match = ((token == wanted) & ~same.any(2)) | (i == 0)
    stands = (_ancestors(parent).float() @ (~match).float()[:, :, None])[:, :, 0] == 0
    stands &= (row >= 0)
    reached = _ancestors(parent)[:, :, 0] & stands
    count = reached.sum(1)
    path = torch.where(reached, i, t).sort(1).values
    path = torch.where(path < t, path, -1)
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])[:, 0]
    after = torch.where(count > 0, pick[(state["row_start"][:-1].long() + last).clamp(min=0)], -1)
    return path.to(torch.int32), count.to(torch.int32), after.to(torch.int32)


def _plain_compact(state):
    c = state["case"]
    t = state["max_rows"]
    where = _cache_rows(state, c["page"], state["max_prefix"] + t)
    path, prefix = state["path"].long(), state["prefix"].long()[:, None]
    live = path >= 0
    src = where.gather(1, prefix + path.clamp(min=0))[live]
    dst = where.gather(1, (prefix + torch.arange(t, device="cuda")).expand_as(path))[live]
    state["kv"][:, dst] = state["kv"][:, src]
    return state["kv"]


def _plain_copy(state):
    i = torch.arange(state["max_rows"], device="cuda")
    src, dst, n = state["spans"].long().unbind(1)
    live = i < n[:, None]
    state["kv"][:, (dst[:, None] + i)[live]] = state["kv"][:, (src[:, None] + i)[live]]
    return state["kv"]


# ------------------------------------------------------------------------------------------------------------ one pass


def run(state):
    c = state["case"]
    if not own:
        return {"attn": _plain_attn, "accept": _plain_accept, "compact": _plain_compact, "copy": _plain_copy}[c["op"]](state)
    from __graft_entry__ import load_package

    drafts = load_package().drafts
    if c["op"] == "copy":
        drafts.kv_copy(state["planes"], state["kv"].shape[1], state["spans"], max_rows=state["max_rows"])
        return state["kv"]
    tree = drafts.DraftTree(state["row_start"], state["prefix"], state["parent"], max_rows=state["max_rows"], max_prefix=state["max_prefix"])
    if c["op"] == "accept":
        return drafts.tree_accept(tree, state["tokens"], logits=state["logits"], path_len=state["path_len"])
    kv_map = drafts.KvMap(state["rows"], page_table=state["table"], page_rows=c["page"], max_seq=state["max_seq"])
    if c["op"] == "attn":
        return drafts.attn_tree(state["q"], state["k"], state["v"], tree, kv_map, n_kv_heads=c["kv_heads"], head_dim=c["hd"], window=c["window"], sinks=state["sinks"], out=state["out"])
    drafts.kv_compact(state["planes"], kv_map, tree, state["path"], state["n_accepted"])
    return state["kv"]


def work(case):
    op = case["op"]
    if op == "copy":
        return {"bytes": 2 * sum(_spans(case)) * 2 * case["layers"] * case["row"] * 2, "flops": 0}
    nodes, ctx = _sizes(case)
    if op == "accept":
        # the rows of the nodes that stand, each picked from once
        return {"bytes": sum(_accepted(case)) * case["vocab"] * 4 + 12 * sum(nodes), "flops": 0}
    if op == "compact":
        # node 0 stays where it is
        return {"bytes": 2 * sum(a - 1 for a in _accepted(case)) * 2 * case["layers"] * case["row"] * 2 + 8 * sum(nodes), "flops": 0}
    q, e = (2 if case["q"] == "bf16" else 4), (2 if case["cache"] == "bf16" else 4)
    seen = [min(p, case["window"]) if case["window"] else p for p in ctx]
    keys = sum(p + t for p, t in zip(seen, nodes))
    pairs = sum(t * (p + (t + 1) / 2) for p, t in zip(seen, nodes))
    return {"bytes": keys * case["kv_heads"] * case["hd"] * 2 * e + 2 * sum(nodes) * case["heads"] * case["hd"] * q, "flops": 4 * pairs * case["heads"] * case["hd"]}


# ------------------------------------------------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    """Sequence by sequence and node by node, from the definition.  Copies and whole numbers have no rounding to speak of: None."""
    if case["op"] != "attn":
        return None
    st = prepare(case, seed)
    starts, prefix, parent = st["row_start"].tolist(), st["prefix"].tolist(), st["parent"].tolist()
    kvh, hd, group = case["kv_heads"], case["hd"], case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s in range(case["n_seq"]):
        first, count, p = starts[s], starts[s + 1] - starts[s], prefix[s]
        if count == 0:
            continue
        total = p + count
        if st["table"] is None:
            at = torch.arange(total, device="cuda") + s * st["max_seq"]
        else:
            pages = st["table"][s].tolist()
            at = torch.cat([torch.arange(case["page"], device="cuda") + e * case["page"] for e in pages if e >= 0])[:total]
        place = [0] * count
        sees = torch.zeros(count, total, dtype=torch.bool)
        sees[:, :p] = True
        for i in range(count):
            up = parent[first + i]
            if up >= 0:
                sees[i, p:] = sees[up, p:]
                place[i] = place[up] + 1
            sees[i, p + i] = True
        if case["window"]:
            where = torch.cat([torch.arange(p), p + torch.tensor(place)])
            sees &= (p + torch.tensor(place))[:, None] - where[None, :] < case["window"]
        sees = sees.cuda()
        k, v = st["k"][at].double().view(total, kvh, hd), st["v"][at].double().view(total, kvh, hd)
        q = st["q"][first:first + count].double().view(count, kvh, group, hd)
        for h in range(kvh):
            x = torch.einsum("tgd,kd->gtk", q[:, h], k[:, h]) / math.sqrt(hd)
            x = torch.where(sees, x, -torch.inf)
            if st["sinks"] is not None:
                sink = st["sinks"][h * group:(h + 1) * group].double()[:, None, None].expand(group, count, 1)
                w = torch.softmax(torch.cat([x, sink], 2), 2)[:, :, :total]
            else:
                w = torch.softmax(x, 2)
            out[first:first + count].view(count, kvh, group, hd)[:, h] = torch.einsum("gtk,kd->tgd", w, v[:, h])
    return out
