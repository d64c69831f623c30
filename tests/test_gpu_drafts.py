"""The operators of speculative decoding (include/lum_tree.h, oneiron_luminal_b200.drafts) against float64 statements of them."""
import numpy as np
import pytest

import drafts_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "GPU tests need a CUDA device"
    t.cuda.set_device(0)
    return t


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.drafts


class Batch:
    """Sequences with their trees, a cache that holds nothing but NaN where no sequence has a row, and the same facts as numpy arrays."""

    def __init__(self, torch, ops, nodes, prefix, *, n_kv=2, group=2, dim=64, q="bf16", cache=None, page=0, seed=0, kind="mixed", slots=None, gap=0, head=0, q_pad=0, kv_pad=0, sinks=False,
                 hint=0):
        rng = np.random.default_rng(seed)
        self.torch, self.ops, self.nodes, self.prefix, self.n_kv, self.dim, self.heads = torch, ops, nodes, prefix, n_kv, dim, n_kv * group
        cache = cache or "bf16"
        types = {"bf16": torch.bfloat16, "f32": torch.float32}
        n = len(nodes)
        self.parents = [plain.random_parents(rng, t, kind) for t in nodes]
        self.start = np.concatenate([[0], np.cumsum(nodes)]) + head
        self.rows = int(self.start[-1]) + gap
        i32 = dict(dtype=torch.int32, device="cuda")
        flat = [-7] * head + sum(self.parents, []) + [-7] * gap
        most = max(t + p for t, p in zip(nodes, prefix))
        self.slot = slots if slots is not None else list(range(n))
        n_slots = max(self.slot) + 2
        width = n_kv * dim
        if page:
            per = -(-most // page) + 1
            need = [-(-(t + p) // page) for t, p in zip(nodes, prefix)]
            order = rng.permutation(sum(need) + 5)
            table = np.full((n_slots, per), -1, np.int32)
            at = 0
            for s, m in zip(self.slot, need):
                table[s, :m] = order[at:at + m]
                at += m
            total = (sum(need) + 5) * page
            self.where = [(table[s, np.arange(t + p) // page].astype(np.int64) * page + np.arange(t + p) % page) for s, t, p in zip(self.slot, nodes, prefix)]
            self.map = ops.KvMap(total, max_seq=per * page, page_table=torch.tensor(table, **i32), page_rows=page)
        else:
            total = n_slots * most
            self.where = [s * most + np.arange(t + p) for s, t, p in zip(self.slot, nodes, prefix)]
            self.map = ops.KvMap(total, max_seq=most, slots=n_slots)

        def cache_rows():
            full = torch.full((total, width + kv_pad), float("nan"), dtype=types[cache])
            x = torch.tensor(rng.standard_normal((total, width)), dtype=types[cache])
            for w in self.where:
                full[w, :width] = x[w]
            return full.cuda()[:, :width]

        self.k, self.v = cache_rows(), cache_rows()
        qw = self.heads * dim
        self.q = torch.tensor(rng.standard_normal((self.rows, qw + q_pad)) * 1.5, dtype=types[q]).cuda()[:, :qw]
        self.sinks = torch.tensor(rng.standard_normal(self.heads), dtype=torch.float32).cuda() if sinks else None
        self.tree = ops.DraftTree(torch.tensor(self.start, **i32), torch.tensor(prefix, **i32), torch.tensor(flat, **i32), max_rows=max(max(nodes), 1), max_prefix=max(prefix) + hint,
                                  slot=None if slots is None else torch.tensor(slots, **i32))

    def run(self, **kw):
        return self.ops.attn_tree(self.q, self.k, self.v, self.tree, self.map, n_kv_heads=self.n_kv, head_dim=self.dim, sinks=self.sinks, **kw)

    def want(self, window=0, scale=None):
        """(result, bound) as [rows, heads * dim], NaN where the rows belong to no sequence."""
        out = np.full((self.rows, self.heads, self.dim), np.nan)
        off = np.zeros_like(out)
        k, v, q = (x.double().cpu().numpy() for x in (self.k, self.v, self.q))
        sinks = None if self.sinks is None else self.sinks.double().cpu().numpy()
        for s, w in enumerate(self.where):
            a, b = self.start[s], self.start[s + 1]
            if a < b:
                shape = (len(w), self.n_kv, self.dim)
                out[a:b], off[a:b] = plain.attention(q[a:b].reshape(-1, self.heads, self.dim), k[w].reshape(shape), v[w].reshape(shape), self.parents[s], self.prefix[s], self.n_kv, window, sinks,
                                                     scale)
        return out.reshape(self.rows, -1), off.reshape(self.rows, -1)

    def check(self, got, window=0, scale=None):
        want, off = self.want(window, scale)
        live = ~np.isnan(want[:, 0])
        g = got.double().cpu().numpy()[live]
        want, off = want[live], off[live]
        if got.dtype == self.torch.bfloat16:
            off = off + 2.0 ** -8 * (np.abs(want) + off) + 2.0 ** -16 * np.abs(self.v[np.concatenate(self.where)].double().cpu().numpy()).max()
        bad = ~(np.abs(g - want) <= off)
        assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(g - want) / off)} of the bound, NaN {np.isnan(g).sum()}"


TYPES = [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")]


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes, prefix", [([1], [0]), ([1], [1]), ([2], [63]), ([5], [64]), ([8], [500]), ([64], [130]), ([33], [31]), ([3, 1, 17, 9], [0, 200, 77, 129])])
def test_attention(torch, ops, q, cache, dim, nodes, prefix):
    b = Batch(torch, ops, nodes, prefix, dim=dim, q=q, cache=cache, seed=len(nodes) + prefix[0])
    b.check(b.run())
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_attention_pages_and_slots(torch, ops, q, cache, page):
    b = Batch(torch, ops, [7, 20, 1], [150, 15, 64], q=q, cache=cache, page=page, slots=[4, 0, 2], seed=page)
    b.check(b.run())
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("group, n_kv, nodes", [(1, 3, 40), (3, 2, 43), (8, 1, 33), (7, 2, 19), (16, 1, 9), (1, 1, 200), (5, 1, 26), (64, 1, 3)])
def test_attention_heads(torch, ops, q, cache, group, n_kv, nodes):
    b = Batch(torch, ops, [nodes], [90], n_kv=n_kv, group=group, q=q, cache=cache, seed=group)
    b.check(b.run())


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("kind", ["chain", "star", "forest"])
def test_attention_of_tree_shapes(torch, ops, q, cache, kind):
    b = Batch(torch, ops, [256, 100], [70, 3], n_kv=1, group=2, q=q, cache=cache, kind=kind)
    b.check(b.run())


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000])
@pytest.mark.parametrize("page", [0, 16])
def test_attention_window_and_sinks(torch, ops, q, cache, window, page):
    b = Batch(torch, ops, [30, 6], [333, 0], q=q, cache=cache, kind="mixed", page=page, sinks=True, seed=window)
    b.check(b.run(window=window), window=window)
    b = Batch(torch, ops, [30, 6], [333, 0], q=q, cache=cache, kind="chain", page=page, seed=window)
    b.check(b.run(window=window), window=window)


@pytest.mark.parametrize("q, cache", TYPES)
def test_attention_strides_scale_and_rows_of_nobody(torch, ops, q, cache):
    b = Batch(torch, ops, [4, 0, 9], [100, 5, 31], q=q, cache=cache, head=2, gap=3, q_pad=16, kv_pad=32)
    out = torch.full((b.rows, b.q.shape[1] + 8), 5.0, dtype=b.q.dtype, device="cuda")
    got = b.run(out=out[:, :-8], scale=0.37)
    b.check(got, scale=0.37)
    assert (out[:2] == 5.0).all() and (out[-3:] == 5.0).all() and (out[:, -8:] == 5.0).all()
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
def test_attention_of_long_and_uneven_batches(torch, ops, q, cache):
    """Chunks of keys that are joined, sequences of very different lengths, a bound on the lengths that is far above them."""
    for hint in (0, 20000):
        b = Batch(torch, ops, [3, 12, 1], [5000, 64, 1], n_kv=1, group=4, dim=128, q=q, cache=cache, page=64, hint=hint)
        b.check(b.run())
        ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("short, n_kv", [(34, 8), (17, 8), (140, 2), (20, 8)])
def test_attention_of_one_long_sequence_among_many_short_ones(torch, ops, q, cache, page, short, n_kv):
    """About as many short units as CTAs that run at once, and a long unit that is cut as well: every piece has to be computed by some CTA."""
    b = Batch(torch, ops, [1] * (short // 2) + [2] + [1] * (short - short // 2), [5] * (short // 2) + [6000] + [7] * (short - short // 2), n_kv=n_kv, group=1, dim=64, q=q,
              cache=cache, page=page)
    b.check(b.run())
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 3.0e38])
def test_attention_leaves_out_what_is_masked_whatever_it_holds(torch, ops, q, cache, value):
    """A node that the others do not see, a row of the cache outside the window, and keys of the next sequence hold infinities: only who sees them is touched."""
    b = Batch(torch, ops, [6, 4], [70, 66], q=q, cache=cache, kind="star", seed=3)
    want, _ = b.want(window=40)
    rows = [int(b.where[0][70 + 3]), int(b.where[0][2]), int(b.where[1][66 + 2])]      # node 3, a far row, node 2 of the other
    for r in rows:
        b.k[r], b.v[r] = value, value
    got = b.run(window=40).double().cpu().numpy()
    sees = {3, 6 + 2}
    for i in range(10):
        if i in sees:
            if not abs(value) < 1e39:
                assert not np.isfinite(got[i]).all()
        else:
            assert np.abs(got[i] - want[i]).max() < 0.05, i
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
def test_attention_large_scores(torch, ops, q, cache):
    """One key takes everything, scores of some hundred: no overflow, and -inf keys weigh nothing."""
    b = Batch(torch, ops, [5], [100], q=q, cache=cache, kind="chain")
    b.k[int(b.where[0][17])] *= 200.0
    b.check(b.run())
    b = Batch(torch, ops, [2], [40], q=q, cache=cache)
    b.q[:] = b.q.abs()
    b.k[int(b.where[0][7])] = float("-inf")
    got = b.run().double().cpu().numpy()
    b.k[int(b.where[0][7])] = -1e4
    want, off = b.want()
    assert np.abs(got - want).max() < 0.05


def rounded(b, want, off):
    """The bound of bf16 results: the rounding of the result, and weights in two bf16 terms against the largest value of the cache that is finite."""
    if b.q.dtype != b.torch.bfloat16:
        return off
    v = b.v[np.concatenate(b.where)].double().cpu().numpy()
    return off + 2.0 ** -8 * (np.abs(want) + off) + 2.0 ** -16 * np.abs(v[np.abs(v) < 1e30]).max()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [70, 1000])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 3.0e38])
def test_attention_beside_masked_values_keeps_its_bound(torch, ops, q, cache, dim, prefix, value):
    """What nobody sees changes nothing, down to the bound of f32 arithmetic: one key more or less, of some 40, would be far outside it."""
    b = Batch(torch, ops, [6, 4], [prefix, 66], dim=dim, q=q, cache=cache, kind="star", seed=3)
    want, off = b.want(window=40)
    bound = rounded(b, want, off)
    for r in (b.where[0][prefix + 3], b.where[0][2], b.where[1][66 + 2]):                # node 3, a far row, node 2 of the other
        b.k[int(r)], b.v[int(r)] = value, value
    got = b.run(window=40).double().cpu().numpy()
    keep = [i for i in range(10) if i not in (3, 6 + 2)]
    assert (np.abs(got[keep] - want[keep]) <= bound[keep]).all()
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix", [40, 1000])
def test_attention_without_a_key_of_minus_infinity_keeps_its_bound(torch, ops, q, cache, dim, prefix):
    """A visible key whose score is -inf weighs nothing: the result is that of the sequence without it."""
    b = Batch(torch, ops, [2], [prefix], dim=dim, q=q, cache=cache)
    b.q[:] = b.q.abs() + 2.0 ** -10
    b.k[int(b.where[0][7])] = float("-inf")
    got = b.run().double().cpu().numpy()
    ops.status()
    k, v, x = (t.double().cpu().numpy() for t in (b.k, b.v, b.q))
    rows = np.delete(b.where[0], 7)
    shape = (len(rows), b.n_kv, dim)
    want, off = plain.attention(x.reshape(2, b.heads, dim), k[rows].reshape(shape), v[rows].reshape(shape), b.parents[0], prefix - 1, b.n_kv)
    want, off = want.reshape(2, -1), off.reshape(2, -1)
    assert (np.abs(got - want) <= rounded(b, want, off)).all()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("hint", [0, 30000])
@pytest.mark.parametrize("prefix", [40, 1000])
@pytest.mark.parametrize("dim, sinks", [(64, False), (128, False), (64, True)])
def test_attention_of_rows_whose_scores_are_all_minus_infinity(torch, ops, q, cache, hint, prefix, dim, sinks):
    """The definition's 0 / 0: undefined, unless a sink is in the denominator (then nothing).  A node that sees one finite score takes that key alone."""
    b = Batch(torch, ops, [3, 2], [prefix, 50], dim=dim, q=q, cache=cache, kind="star", hint=hint, sinks=sinks, seed=prefix)
    b.q[:] = b.q.abs() + 2.0 ** -10
    want, off = b.want()
    at = b.where[0]
    b.k[[int(r) for r in at[:prefix + 2]]] = float("-inf")   # all but node 2's
    got = b.run().double().cpu().numpy()
    assert np.isnan(got[:2]).all() if not sinks else (got[:2] == 0.0).all()
    k, v, x = (t.double().cpu().numpy() for t in (b.k[int(at[prefix + 2])], b.v[int(at[prefix + 2])], b.q[2]))
    sink = None if b.sinks is None else b.sinks.double().cpu().numpy()
    one, one_off = plain.attention(x.reshape(1, b.heads, dim), k.reshape(1, b.n_kv, dim), v.reshape(1, b.n_kv, dim), [-1], 0, b.n_kv, 0, sink)
    want[2], off[2] = one.reshape(-1), one_off.reshape(-1)
    bound = off[2:] + (2.0 ** -8 * (np.abs(want[2:]) + off[2:]) + 2.0 ** -16 * np.abs(v).max() if q == "bf16" else 0.0)
    bound[1:] += 2.0 ** -14 if q == "bf16" else 0.0          # (weights in two terms, of values up to 4)
    assert (np.abs(got[2:] - want[2:]) <= bound).all()
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("hint", [0, 30000])
@pytest.mark.parametrize("prefix", [40, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_with_infinite_sinks(torch, ops, q, cache, hint, prefix, dim):
    """-inf is no sink, +inf leaves nothing to the keys, whatever way the work is shared out; an undefined one stays undefined."""
    b = Batch(torch, ops, [3, 2], [prefix, 50], group=4, n_kv=1, dim=dim, q=q, cache=cache, hint=hint, sinks=True, seed=prefix)
    b.sinks.copy_(torch.tensor([float("-inf"), 0.7, float("inf"), float("nan")]))
    got = b.run().unflatten(1, (4, dim))
    ops.status()
    assert (got[:, 2] == 0.0).all() and torch.isnan(got[:, 3]).all()
    b.sinks.copy_(torch.tensor([-1e30, 0.7, 0.0, 0.0]))      # (-inf in the float64 statement's exponentials)
    want, off = (x.reshape(5, 4, dim)[:, :2] for x in b.want())
    bound = off + (2.0 ** -8 * (np.abs(want) + off) + 2.0 ** -16 * np.abs(b.v[np.concatenate(b.where)].double().cpu().numpy()).max() if q == "bf16" else 0.0)
    assert (np.abs(got[:, :2].double().cpu().numpy() - want) <= bound).all()


def test_attention_under_capture_on_another_stream_and_twice_at_once(torch, ops):
    b = Batch(torch, ops, [9, 30], [700, 90], dim=128, group=4, page=64)
    c = Batch(torch, ops, [3], [2000], dim=64, group=8, q="f32", seed=5)
    first, second = b.run().clone(), c.run().clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            x = b.run()
        with torch.cuda.stream(s2):
            y = c.run()
        outs.append((x, y))
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, first) and torch.equal(y, second)
    out = torch.zeros_like(b.q.contiguous())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(out=out)
        y = c.run()
    out.zero_()
    b.q.mul_(0.5)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    b.check(out)
    assert torch.equal(y, second)
    ops.status()


def test_attention_bad_numbers_on_the_device_are_left_out_and_reported(torch, ops, pkg):
    def refused():
        with pytest.raises(pkg.LumError) as e:
            ops.status()
        assert e.value.code == -4
        ops.status()

    b = Batch(torch, ops, [4, 5], [100, 40], page=16)
    good = b.run().clone()
    b.map.tensors[0][1, 1] = 10 ** 6                         # a page outside the pool: the other sequence is untouched
    got = b.run()
    assert torch.equal(got[:4], good[:4])
    refused()
    b = Batch(torch, ops, [4, 5], [100, 40])
    good = b.run().clone()
    b.tree.tensors[1][1] = 10 ** 6                           # more cached rows than the call named
    out = torch.full_like(b.q, 3.0)
    b.run(out=out)
    assert torch.equal(out[:4], good[:4]) and (out[4:] == 3.0).all()
    refused()
    b.tree.tensors[1][1] = 40
    b.tree.tensors[2][6] = 3                                 # a parent that is a later node
    assert torch.equal(b.run()[:4], good[:4])
    refused()
    b.tree.tensors[2][6] = 0
    b.tree.tensors[0][2] = 10 ** 6                           # rows outside the batch
    assert torch.equal(b.run()[:4], good[:4])
    refused()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("hint", [1000, 30000])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes, prefix, group", [([1, 0, 3], [0, 9, 300], 1), ([12, 2], [70, 1], 4), ([40, 33], [700, 2], 4), ([3], [63], 3), ([200], [500], 2)])
def test_attention_of_few_keys_in_the_room_of_many(torch, ops, q, cache, hint, dim, nodes, prefix, group):
    """The call's bounds ask for many CTAs per unit, the lengths leave some of them without a key."""
    for window, sinks in ((0, False), (90, True)):
        b = Batch(torch, ops, nodes, prefix, group=group, dim=dim, q=q, cache=cache, hint=hint, page=16, sinks=sinks)
        b.check(b.run(window=window), window=window)
    ops.status()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("hint", [0, 30000])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_attention_leaves_out_infinities_where_a_unit_is_shared(torch, ops, q, cache, hint, group):
    """As above, where several CTAs share a unit: their rows that are not finite are computed once more."""
    b = Batch(torch, ops, [16], [1000], group=group, dim=128, q=q, cache=cache, kind="star", hint=hint)
    at = [int(b.where[0][1000 + 5]), int(b.where[0][3])]     # a node, and a row that no node sees with this window
    for r in at:
        b.v[r] = float("inf")
    got = b.run(window=990).clone()
    ops.status()
    for r in at:
        b.v[r] = 0.0
    want, off = b.want(window=990)
    keep = [i for i in range(16) if i != 5]
    bound = off[keep] + (2.0 ** -8 * (np.abs(want[keep]) + off[keep]) + 2.0 ** -14 if q == "bf16" else 0.0)
    assert (np.abs(got.double().cpu().numpy()[keep] - want[keep]) <= bound).all()
    assert not np.isfinite(got[5].float().cpu().numpy()).all()


@pytest.mark.parametrize("q, cache", TYPES)
@pytest.mark.parametrize("masked", [0.0, float("inf")])
def test_attention_takes_the_rows_of_an_unknown_page_as_zeros(torch, ops, pkg, q, cache, masked):
    """Also where a row is computed key by key, because a value that it does not see is infinite."""
    b = Batch(torch, ops, [6], [100], page=16, q=q, cache=cache, kind="star")
    node = int(b.where[0][100 + 5])                          # the others do not see it
    b.v[node] = masked
    b.map.tensors[0][0, 2] = 10 ** 6
    got = b.run()[:5].clone()
    with pytest.raises(pkg.LumError):
        ops.status()
    gone = b.where[0][32:48]
    b.k[gone], b.v[gone], b.v[node] = 0.0, 0.0, 0.0
    want, off = b.want()
    bound = off[:5] + (2.0 ** -8 * (np.abs(want[:5]) + off[:5]) + 2.0 ** -14 if q == "bf16" else 0.0)
    assert (np.abs(got.double().cpu().numpy() - want[:5]) <= bound).all()


def test_tensors_expanded_along_their_rows_are_refused(torch, ops, pkg):
    """Their rows are all one: nothing is launched, out and what lies behind stay as they are."""
    b = Batch(torch, ops, [4, 3], [30, 9], q="f32", cache="f32")
    out = torch.full_like(b.q, 2.0)
    one = lambda t: t[:1].clone().expand(t.shape)  # noqa: E731
    call = lambda q=b.q, k=b.k, v=b.v, out=out: ops.attn_tree(q, k, v, b.tree, b.map, n_kv_heads=b.n_kv, head_dim=b.dim, out=out)  # noqa: E731
    for kw in (dict(q=one(b.q)), dict(k=one(b.k)), dict(v=one(b.v)), dict(k=one(b.k), v=one(b.v)), dict(out=one(out)), dict(q=one(b.q).unflatten(1, (b.heads, b.dim)))):
        with pytest.raises(pkg.LumError) as e:
            call(**kw)
        assert e.value.code == -1
    tokens = torch.zeros(b.rows, dtype=torch.int32, device="cuda")
    with pytest.raises(pkg.LumError) as e:
        ops.tree_accept(b.tree, tokens, logits=torch.randn(1, 50, device="cuda").expand(b.rows, 50))
    assert e.value.code == -1
    torch.cuda.synchronize()
    assert (out == 2.0).all()
    b.check(call(k=b.k, v=b.v))
    ops.status()


# ---------------------------------------------------------------------------------------------------- accepted nodes


def accept_case(torch, ops, nodes, vocab, seed, agree=0.7, spread=0):
    rng = np.random.default_rng(seed)
    parents = [plain.random_parents(rng, t) for t in nodes]
    start = np.concatenate([[0], np.cumsum(nodes)])
    rows = int(start[-1])
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    logits = rng.standard_normal((rows, vocab)).astype(np.float32)
    for s, ps in enumerate(parents):
        for i, p in enumerate(ps):
            if p >= 0 and rng.random() < agree:
                logits[start[s] + p, tokens[start[s] + i]] = 20.0 + i
    i32 = dict(dtype=torch.int32, device="cuda")
    tree = ops.DraftTree(torch.tensor(start, **i32), torch.zeros(len(nodes), **i32), torch.tensor(sum(parents, []), **i32), max_rows=max(nodes), max_prefix=0)
    return parents, start, tokens, logits, tree, torch.tensor(tokens, **i32)


def check_accept(got, parents, start, tokens, picks):
    path, count, after = (x.cpu().numpy() for x in got)
    for s, ps in enumerate(parents):
        a, b = start[s], start[s + 1]
        want, nxt = plain.accept(tokens[a:b], ps, picks[a:b])
        assert count[s] == len(want) and after[s] == nxt, (s, want, path[s], count[s], after[s], nxt)
        assert list(path[s][:len(want)]) == want and (path[s][len(want):] == -1).all()


@pytest.mark.parametrize("nodes, vocab", [([1], 5), ([8], 1000), ([64, 1, 30], 4097), ([256], 300), ([5] * 40, 50), ([16] * 8, 32064), ([3, 0, 2], 1), ([2], 128256), ([64], 128256)])
def test_accept(torch, ops, nodes, vocab):
    for seed in range(3):
        parents, start, tokens, logits, tree, t = accept_case(torch, ops, nodes, vocab, seed)
        picks = [plain.pick(r) for r in logits]
        check_accept(ops.tree_accept(tree, t, logits=torch.tensor(logits).cuda()), parents, start, tokens, picks)
        check_accept(ops.tree_accept(tree, t, picks=torch.tensor(picks, dtype=torch.int32, device="cuda"), path_len=max(nodes) + 3), parents, start, tokens, picks)
        wide = torch.full((len(tokens), vocab + 3), 1e30).cuda()
        wide[:, :vocab] = torch.tensor(logits).cuda()
        check_accept(ops.tree_accept(tree, t, logits=wide[:, :vocab]), parents, start, tokens, picks)
    ops.status()


@pytest.mark.parametrize("vocab", [7, 33, 4096, 130000])
def test_accept_ties_and_undefined_logits(torch, ops, vocab):
    """The last maximum wins, NaN counts as -inf, -0 equals 0; the same token twice under one node: the first of them."""
    i32 = dict(dtype=torch.int32, device="cuda")
    tree = ops.DraftTree(torch.tensor([0, 5], **i32), torch.zeros(1, **i32), torch.tensor([-1, 0, 0, 2, 1], **i32), max_rows=5, max_prefix=0)
    last = vocab - 1
    tokens = np.array([0, last, last, 2, 3], np.int32)
    rows = np.zeros((5, vocab), np.float32)
    rows[0, 1] = -0.0
    rows[1] = np.nan
    rows[1, 3] = -5.0
    rows[4] = np.nan
    picks = [plain.pick(r) for r in rows]
    assert picks[0] == last and picks[1] == 3 and picks[4] == last
    got = ops.tree_accept(tree, torch.tensor(tokens, **i32), logits=torch.tensor(rows).cuda())
    check_accept(got, [[-1, 0, 0, 2, 1]], [0, 5], tokens, picks)
    rows[0] = -np.inf
    rows[0, 2] = np.inf
    rows[0, 4] = np.inf
    check_accept(ops.tree_accept(tree, torch.tensor(tokens, **i32), logits=torch.tensor(rows).cuda()), [[-1, 0, 0, 2, 1]], [0, 5], tokens, [plain.pick(r) for r in rows])


def test_accept_bad_trees_are_reported(torch, ops, pkg):
    parents, start, tokens, logits, tree, t = accept_case(torch, ops, [6, 6], 50, 1)
    tree.tensors[2][2] = 4
    ops.tree_accept(tree, t, logits=torch.tensor(logits).cuda())
    with pytest.raises(pkg.LumError):
        ops.status()
    tree.tensors[0][1] = -3
    ops.tree_accept(tree, t, logits=torch.tensor(logits).cuda())
    with pytest.raises(pkg.LumError):
        ops.status()


# ---------------------------------------------------------------------------------------------------- cache rows


@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("row_bytes", [16, 48, 1024, 2080])
def test_compact(torch, ops, page, row_bytes):
    rng = np.random.default_rng(page + row_bytes)
    b = Batch(torch, ops, [40, 1, 256, 9], [10, 3, 130, 0], page=page, slots=[2, 0, 5, 1])
    planes = [torch.randint(-30000, 30000, (b.map.rows, n), dtype=torch.int16, device="cuda") for n in (row_bytes // 2, 8)]
    want = [p.clone() for p in planes]
    path, count = np.full((4, 256), -1, np.int32), []
    for s, t in enumerate(b.nodes):
        n = [17, 1, 256, 0][s]
        pick = np.sort(rng.choice(t, n, replace=False)) if n else np.zeros(0, int)
        path[s, :n] = pick
        count.append(n)
        w, p = b.where[s], b.prefix[s]
        for x, y in zip(want, planes):
            x[torch.tensor(w[p:p + n])] = y[torch.tensor(w[p + pick])]
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.kv_compact(ops.kv_planes(planes), b.map, b.tree, torch.tensor(path, **i32), torch.tensor(count, **i32))
    for x, y in zip(planes, want):
        assert torch.equal(x, y)
    ops.status()


def test_compact_refuses_what_is_no_path(torch, ops, pkg):
    b = Batch(torch, ops, [6, 6], [4, 5])
    planes = [torch.randn(b.map.rows, 16, device="cuda")]
    before = planes[0].clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    table = ops.kv_planes(planes)
    for path, count in (([[0, 3, 2], [0, 1, 2]], [3, 3]), ([[0, 6, 7], [0, 1, 2]], [3, 3]), ([[0, 1, 2], [0, 1, 2]], [7, 3]), ([[0, 1, 2], [0, 1, 2]], [-1, 3]), ([[-1, 1, 2], [0, 1, 2]], [2, 3])):
        ops.kv_compact(table, b.map, b.tree, torch.tensor(path, **i32), torch.tensor(count, **i32))
        with pytest.raises(pkg.LumError):
            ops.status()
        assert torch.equal(planes[0], before)


@pytest.mark.parametrize("row_elems", [8, 40, 512])
@pytest.mark.parametrize("lens", [[1], [3, 0, 5], [700, 1, 64], [37] * 50])
def test_copy(torch, ops, row_elems, lens):
    rng = np.random.default_rng(len(lens))
    most = max(lens)
    rows = 2 * len(lens) * most + 3
    kv = torch.randn(5, rows, row_elems, device="cuda").to(torch.bfloat16)
    first = rng.permutation(2 * len(lens)) * most + 3
    spans = [[first[i], first[len(lens) + i], n] for i, n in enumerate(lens)]
    want = kv.clone()
    for a, b, n in spans:
        want[:, b:b + n] = kv[:, a:a + n]
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.kv_copy(ops.kv_planes([kv]), rows, torch.tensor(np.array(spans), **i32), max_rows=most)
    assert torch.equal(kv, want)
    ops.status()


def test_copy_of_spans_outside_the_cache_is_left_out(torch, ops, pkg):
    kv = torch.randn(2, 100, 64, device="cuda")
    want = kv.clone()
    want[:, 50:60] = kv[:, 0:10]
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.kv_copy(ops.kv_planes([kv]), 100, torch.tensor([[0, 50, 10], [95, 20, 6], [10, 96, 5], [-1, 30, 2], [0, 70, 11]], **i32), max_rows=10)
    with pytest.raises(pkg.LumError):
        ops.status()
    assert torch.equal(kv, want)


def test_planes_whose_rows_are_no_multiple_of_16_bytes_are_left_out(torch, ops, pkg):
    kv = torch.randn(2, 40, 16, device="cuda")
    want = kv.clone()
    want[0, 20:24] = kv[0, 3:7]
    planes = ops.kv_planes([kv])
    planes[1, 1] = 60
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.kv_copy(planes, 40, torch.tensor([[3, 20, 4]], **i32), max_rows=4)
    with pytest.raises(pkg.LumError):
        ops.status()
    assert torch.equal(kv, want)
    with pytest.raises(pkg.LumError):
        ops.kv_planes([kv[:, :, :3]])


@pytest.mark.parametrize("q, cache", TYPES)
def test_attention_with_a_window_that_reaches_over_everything(torch, ops, q, cache):
    b = Batch(torch, ops, [200, 3], [70, 500], n_kv=1, group=1, q=q, cache=cache, kind="chain")
    for window in (2 ** 31 - 1, 756, 700, 270):
        b.check(b.run(window=window), window=window)
    ops.status()


def test_attention_with_a_workspace_of_the_caller(torch, ops, pkg):
    b = Batch(torch, ops, [9, 30], [3000, 90], dim=128, group=4, hint=30000)     # (a shorter bound needs none)
    want = b.run().clone()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    assert torch.equal(b.run(workspace=ws), want)
    with pytest.raises(pkg.LumError):
        b.run(workspace=ws[:16])
    with pytest.raises(pkg.LumError):
        b.run(workspace=ws.view(-1, 64)[:, :32])
    with pytest.raises(pkg.LumError):
        b.run(out=b.q)


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing is allocated or synchronised: even the first calls can be captured (the kernels are loaded then)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch, drafts_plain, test_gpu_drafts as t
from __graft_entry__ import load_package
ops = load_package().drafts
b = t.Batch(torch, ops, [9, 30], [700, 90], dim=128, group=4, page=64)
out = torch.zeros_like(b.q.contiguous())
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b.run(out=out)
g.replay()
torch.cuda.synchronize()
b.check(out)
""" % (root, os.path.join(root, "tests"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_a_step_of_speculative_decoding(torch, ops):
    """Attention over drafts, acceptance, compaction: the kept rows are those of the path, and attending again from a chain over them gives what the tree gave."""
    b = Batch(torch, ops, [12, 7], [100, 33], page=16, q="f32", dim=64)
    out = b.run().clone()
    rng = np.random.default_rng(9)
    tokens = rng.integers(0, 90, b.rows).astype(np.int32)
    logits = rng.standard_normal((b.rows, 90)).astype(np.float32)
    for s, ps in enumerate(b.parents):
        at = 0
        for i, p in enumerate(ps):
            if p == at and len(set(tokens[b.start[s]:b.start[s + 1]])) > 0:
                logits[b.start[s] + at, tokens[b.start[s] + i]] = 30.0
                at = i
    i32 = dict(dtype=torch.int32, device="cuda")
    path, count, after = ops.tree_accept(b.tree, torch.tensor(tokens, **i32), logits=torch.tensor(logits).cuda())
    check_accept((path, count, after), b.parents, b.start, tokens, [plain.pick(r) for r in logits])
    kept = [path[s, :int(count[s])].cpu().numpy() for s in range(2)]
    assert all(len(p) > 1 for p in kept)
    ops.kv_compact(ops.kv_planes([b.k, b.v]), b.map, b.tree, path, count)
    chain = [list(range(-1, len(p) - 1)) for p in kept]
    start = np.concatenate([[0], np.cumsum([len(p) for p in kept])])
    tree = ops.DraftTree(torch.tensor(start, **i32), b.tree.tensors[1], torch.tensor(sum(chain, []), **i32), max_rows=12, max_prefix=100)
    rows = np.concatenate([b.start[s] + p for s, p in enumerate(kept)])
    again = ops.attn_tree(b.q[torch.tensor(rows)], b.k, b.v, tree, b.map, n_kv_heads=b.n_kv, head_dim=b.dim)
    # other tiles, another order of sums: two f32 results, each within the bound of the same exact one
    assert (again - out[torch.tensor(rows)]).abs().max().item() < 2e-5
    ops.status()
