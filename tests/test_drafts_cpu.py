"""Host side of speculative decoding: refusals that need no GPU, the ctypes and Rust mirrors of include/lum_tree.h, the drafter and the serving loop against a
stand-in runtime."""
import ctypes as C
import os
import re
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def strip_comments(text):
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


HEADER = strip_comments(open(os.path.join(ROOT, "include", "lum_tree.h")).read())
RUST = strip_comments(open(os.path.join(ROOT, "oneiron-luminal_b200", "host", "rust", "luminal_b200", "src", "tree.rs")).read())
STRUCTS = {"lum_draft_tree": "DraftTreeDesc", "lum_kv_map": "KvMapDesc", "lum_tree_attn": "TreeAttnDesc", "lum_kv_plane": "KvPlaneDesc"}
SCALARS = {"int32_t": "i32", "uint32_t": "u32", "int64_t": "i64", "uint64_t": "u64", "size_t": "usize", "float": "f32", "void": "c_void", **{n: n for n in STRUCTS}}


def rust_type(c):
    toks = re.findall(r"\w+|\*", c)
    const = toks[0] == "const"
    toks = toks[1:] if const else toks
    return ("*const " if const else "*mut ") * toks.count("*") + SCALARS[toks[0]]


def fields(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, flags=re.S).group(1)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        ty, names = re.match(r"((?:const )?\w+\s*\**)\s*(.*)", decl, flags=re.S).groups()
        out += [(n.strip(), rust_type(ty)) for n in names.split(",")]
    return out


@pytest.mark.parametrize("name", list(STRUCTS))
def test_structs_have_the_same_fields_everywhere(pkg, name):
    body = re.search(r"pub struct %s \{(.*?)\}" % name, RUST, flags=re.S).group(1)
    assert [(m.group(1), m.group(2).strip()) for m in re.finditer(r"pub (\w+): ([^,]+),", body)] == fields(name)
    ct = {C.c_int32: "i32", C.c_uint32: "u32", C.c_float: "f32", C.c_uint64: "u64", C.c_int64: "i64"}
    mirror = getattr(pkg.runtime, STRUCTS[name])._fields_
    assert [n for n, _ in mirror] == [n for n, _ in fields(name)]
    assert all(ct.get(t) == want if t is not C.c_void_p else want.startswith("*") for (_, t), (_, want) in zip(mirror, fields(name)))


def test_functions_are_declared_in_rust_as_in_the_header_and_exported(pkg):
    want = []
    for m in re.finditer(r"^(size_t|int32_t) (lum_\w+)\(([^;{}]*?)\);", HEADER, flags=re.M | re.S):
        args = [re.match(r"(.*?)(\w+)$", " ".join(a.split())).groups() for a in m.group(3).split(",")]
        want.append((m.group(2), [(n, rust_type(t)) for t, n in args], SCALARS[m.group(1)]))
    got = []
    for m in re.finditer(r"pub fn (\w+)\((.*?)\) -> (\w+);", RUST, flags=re.S):
        got.append((m.group(1), [tuple(x.strip() for x in a.split(":", 1)) for a in filter(None, (p.strip() for p in m.group(2).split(",")))], m.group(3)))
    assert len(want) == 6 and got == want
    lib = pkg.load_library()
    for name, _, _ in want:
        assert getattr(lib, name).argtypes is not None


# ---- refusals: numbers that the host can see are wrong never reach a device (there is none here)

TREE = dict(row_start=4096, prefix=4096, parent=4096, slot=None, n_seq=2, n_rows=10, max_rows=8, max_prefix=100)
MAP = dict(page_table=None, rows=1000, slots=2, max_seq=200, page_rows=0, pages_per_seq=0)
ATTN = dict(q_dtype=2, kv_dtype=2, n_q_heads=8, n_kv_heads=2, head_dim=64, window=0, scale=0.0, reserved=0, q_stride=0, kv_stride=0, out_stride=0)


def attn(pkg, ptr=(4096,) * 4, **kw):
    t, m, a = ({k: kw.get(k, v) for k, v in d.items()} for d in (TREE, MAP, ATTN))
    args = pkg.runtime.TreeAttnDesc(**a), pkg.runtime.DraftTreeDesc(**t), pkg.runtime.KvMapDesc(**m)
    q, k, v, o = ptr
    return pkg.load_library().lum_op_attn_tree(*args, q, k, v, None, o, None, 0, None)


@pytest.mark.parametrize("kw, code", [
    (dict(n_seq=-1), -1), (dict(n_seq=70000), -1), (dict(n_rows=-1), -1), (dict(max_rows=0), -1), (dict(max_rows=257), -1), (dict(max_prefix=-1), -1), (dict(max_prefix=2 ** 31 - 1), -1),
    (dict(row_start=None), -1), (dict(parent=None), -1), (dict(prefix=None), -1),
    (dict(rows=0), -1), (dict(rows=2 ** 31), -1), (dict(slots=0), -1), (dict(max_seq=0), -1), (dict(rows=300), -1), (dict(page_rows=8), -1), (dict(page_rows=48, page_table=4096, pages_per_seq=3), -1),
    (dict(page_rows=64), -1), (dict(page_rows=64, page_table=4096), -1),
    (dict(head_dim=96), -3), (dict(n_q_heads=7), -1), (dict(n_kv_heads=0), -1), (dict(n_q_heads=2048), -1), (dict(q_dtype=1), -3), (dict(kv_dtype=7), -3), (dict(kv_dtype=0), -3),
    (dict(window=-1), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(q_stride=100), -1), (dict(kv_stride=64), -1), (dict(out_stride=513), -1),
    (dict(q_stride=516), -1), (dict(n_q_heads=512, n_kv_heads=2), -3), (dict(n_seq=65535, max_prefix=2 ** 30), -3), (dict(n_rows=2 ** 31 - 1, n_q_heads=64, n_kv_heads=64), -3),
    (dict(ptr=(None, 4096, 4096, 4096)), -1), (dict(ptr=(4096, 4096, 4096, None)), -1), (dict(ptr=(4104, 4096, 4096, 4096)), -1),
])
def test_attention_refuses(pkg, kw, code):
    assert attn(pkg, **kw) == code
    assert len(pkg.load_library().lum_last_error(None)) > 10


def test_empty_batches_need_nothing(pkg):
    assert attn(pkg, n_seq=0) == 0 and attn(pkg, n_rows=0) == 0
    lib = pkg.load_library()
    tree = pkg.runtime.DraftTreeDesc(**dict(TREE, n_seq=0))
    assert lib.lum_op_tree_accept(tree, None, None, 0, 0, None, None, 0, None, None, None, 0, None) == 0
    assert lib.lum_op_kv_copy(4096, 2, 100, None, 0, 5, None) == 0
    assert lib.lum_op_kv_compact(4096, 2, pkg.runtime.KvMapDesc(**MAP), tree, None, 1, None, None) == 0


def test_accept_compact_and_copy_refuse(pkg):
    lib, tree, cache = pkg.load_library(), pkg.runtime.DraftTreeDesc(**TREE), pkg.runtime.KvMapDesc(**MAP)
    p = 4096
    accept = lambda tokens=p, logits=p, vocab=50, ld=0, picks=None, path=p, length=8, n=p, nxt=p: lib.lum_op_tree_accept(tree, tokens, logits, vocab, ld, picks, path, length, n, nxt, None, 0, None)  # noqa: E731
    for kw in (dict(tokens=None), dict(logits=None), dict(picks=p), dict(vocab=0), dict(vocab=2 ** 30 + 1), dict(logits=p + 2), dict(ld=49), dict(path=None), dict(length=7), dict(n=None), dict(nxt=None)):
        assert accept(**kw) == -1, kw
    assert lib.lum_op_kv_compact(None, 2, cache, tree, p, 8, p, None) == -1
    assert lib.lum_op_kv_compact(p, 0, cache, tree, p, 8, p, None) == -1
    assert lib.lum_op_kv_compact(p, 2, cache, tree, None, 8, p, None) == -1
    assert lib.lum_op_kv_compact(p, 2, cache, tree, p, 0, p, None) == -1
    assert lib.lum_op_kv_copy(p, 2, 0, p, 1, 5, None) == -1
    assert lib.lum_op_kv_copy(p, 2, 100, None, 1, 5, None) == -1
    assert lib.lum_op_kv_copy(p, 2, 100, p, -1, 5, None) == -1
    assert lib.lum_op_kv_copy(p, 65535, 100, p, 65535, 5, None) == -1
    assert lib.lum_op_attn_tree_workspace(None, tree, cache) == C.c_size_t(-1).value
    assert lib.lum_op_tree_accept_workspace(tree, 0) == C.c_size_t(-1).value


def test_the_workspace_of_a_walk_says_why_it_refuses(pkg):
    lib, tree = pkg.load_library(), pkg.runtime.DraftTreeDesc(**TREE)
    for vocab in (0, -3, 2 ** 30 + 1):
        assert lib.lum_op_attn_tree_workspace(None, tree, None) == C.c_size_t(-1).value              # another operator's message is the last one
        assert lib.lum_op_tree_accept_workspace(tree, vocab) == C.c_size_t(-1).value
        assert b"vocabulary" in lib.lum_last_error(None) and str(vocab).encode() in lib.lum_last_error(None)


def test_python_calls_refuse_tensors_of_the_wrong_kind(pkg):
    import torch
    d = pkg.drafts
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(pkg.LumError):
        d.DraftTree(i, i[:2], i, max_rows=1, max_prefix=0)           # not on a GPU
    with pytest.raises(pkg.LumError):
        d.KvMap(100, max_seq=10, page_rows=16)
    with pytest.raises(pkg.LumError):
        d.KvMap(100, max_seq=10, page_table=torch.zeros(1, 2, dtype=torch.int32), page_rows=16)
    with pytest.raises(pkg.LumError):
        d.kv_planes([])


@pytest.mark.parametrize("rows, ok", [(1, True), (2, False), (7, False)])
def test_rows_that_share_memory_are_refused(pkg, rows, ok):
    """A row stride of 0 (or less than a row) must not reach a call, where 0 means rows without gaps."""
    import torch
    d = pkg.drafts
    d._use_torch()
    cpu = torch.device("cpu")
    dense = torch.zeros(rows, 16)
    assert d._rows_of("x", dense, cpu, 16, rows) == (dense.data_ptr(), 16)
    padded = torch.zeros(rows, 24)[:, :16]
    assert d._rows_of("x", padded, cpu, 16, rows) == (padded.data_ptr(), 24 if rows > 1 else 16)
    room = torch.zeros(16 * rows + 16)
    for t in (torch.zeros(1, 16).expand(rows, 16), torch.zeros(1, 2, 8).expand(rows, 2, 8), room.as_strided((rows, 16), (15, 1)), room.as_strided((rows, 2, 8), (8, 8, 1))):
        if ok:
            assert d._rows_of("x", t, cpu, 16, rows)[1] == 16
        else:
            with pytest.raises(pkg.LumError) as e:
                d._rows_of("x", t, cpu, 16, rows)
            assert e.value.code == -1


def test_gradients_are_refused_where_they_are_recorded(pkg):
    import torch
    d = pkg.drafts
    x, y = torch.zeros(2, 64), torch.zeros(2, 64, requires_grad=True)
    for tensors in ((y, x, x, None), (x, y, x, None), (x, x, y, None), (x, x, x, y)):
        with pytest.raises(pkg.LumError) as e:
            d._no_gradient(*tensors)
        assert e.value.code == -1 and "gradient" in str(e.value)
        with torch.no_grad():
            d._no_gradient(*tensors)
    d._no_gradient(x, x, x, None)
    with pytest.raises(pkg.LumError) as e:
        d.attn_tree(y, x, x, None, None, n_kv_heads=1, head_dim=64)
    assert "gradient" in str(e.value)


# ---- the drafter and the loop


def test_prompt_lookup(pkg):
    look = pkg.serving.PromptLookup(length=3, match=2, places=2)
    assert look([1, 2, 3, 4, 1, 2], 10) == ([3, 4, 1], [0, 1, 2])
    assert look([1, 2, 3, 9, 1, 2, 4, 8, 1, 2], 10) == ([4, 8, 1, 3, 9, 1], [0, 1, 2, 0, 4, 5])     # the later place first, two branches
    assert look([1, 2, 3, 9, 1, 2, 3, 8, 1, 2], 10) == ([3, 8, 1, 9, 1], [0, 1, 2, 1, 4])           # what they share is one path
    assert look([1, 2, 3, 9, 1, 2, 3, 8, 1, 2], 2) == ([3, 8], [0, 1])
    assert look([5, 6, 7], 10) == ([], []) and look([5], 10) == ([], []) and look([], 10) == ([], [])
    assert look([7, 1, 7], 10) == ([1, 7], [0, 1])                                                   # one token matches
    for bad in (dict(length=0), dict(match=0), dict(places=0)):
        with pytest.raises(ValueError):
            pkg.serving.PromptLookup(**bad)


class Stand:
    """A 'model' whose next token depends on every cached token; verification as lum_draft_verify documents it."""

    def __init__(self, max_batch=3, max_seq=64):
        self.desc = types.SimpleNamespace(max_batch=max_batch, max_seq=max_seq, max_new_tokens=16)
        self.cache = [[None] * max_seq for _ in range(max_batch)]
        self.cur, self.passes, self.rows = 0, 0, 0

    @staticmethod
    def next(rows):
        return (sum(rows) * 31 + len(rows) * 7 + 3) % 5

    def seq_select(self, s):
        self.cur = s

    def set_data(self, toks):
        self.data = list(toks)

    def execute(self, dims):
        p = dims["p"]
        self.cache[self.cur][p:p + len(self.data)] = self.data
        self.tok = self.next(self.cache[self.cur][:p + len(self.data)])

    def get_token(self):
        return self.tok

    def draft_verify(self, trees, positions, slots):
        self.passes += 1
        out = []
        for (tokens, parents), p, s in zip(trees, positions, slots):
            assert len(tokens) == len(parents) and parents[0] == -1 and all(0 <= q < i for i, q in enumerate(parents) if i)
            assert p + len(tokens) <= self.desc.max_seq and None not in self.cache[s][:p]
            self.rows += len(tokens)
            at, kept, new = 0, [tokens[0]], []
            while True:
                new.append(self.next(self.cache[s][:p] + kept))
                child = [i for i in range(len(tokens)) if parents[i] == at and tokens[i] == new[-1]]
                if not child:
                    break
                at = child[0]
                kept.append(tokens[at])
            self.cache[s][p:p + len(tokens)] = kept + [None] * (len(tokens) - len(kept))
            out.append(new)
        return out


def generate(prompt, n, eos=()):
    rows, out = list(prompt), []
    while len(out) < n:
        out.append(Stand.next(rows))
        rows.append(out[-1])
        if out[-1] in eos:
            break
    return out


@pytest.mark.parametrize("steps", [1, 4])
def test_the_loop_with_a_drafter_gives_plain_decoding(pkg, steps):
    rt = Stand()
    b = pkg.serving.ContinuousBatcher(rt, steps_per_round=steps, drafter=pkg.serving.PromptLookup(4, 2, 2))
    prompts = [[1, 2, 3], [4], [2, 2, 2, 2, 2, 2], [0, 1, 2, 3, 4, 0, 1, 2, 3], [3, 1]]
    ids = [b.submit(p, max_new=1 + 9 * i, eos=[] if i % 2 else [0]) for i, p in enumerate(prompts)]
    got = b.run()
    for i, (rid, p) in enumerate(zip(ids, prompts)):
        assert got[rid] == generate(p, 1 + 9 * i, [] if i % 2 else [0]), i
    st = b.stats()
    assert st["stood"] > 0 and st["drafted"] >= st["stood"] and st["live"] == 0
    assert rt.passes < sum(len(t) for t in got.values())


def test_a_drafter_that_breaks_its_promise_is_refused(pkg):
    for bad in (lambda text, room: ([1] * (room + 1), [0] * (room + 1)), lambda text, room: ([1], [1]), lambda text, room: ([1, 2], [0])):
        b = pkg.serving.ContinuousBatcher(Stand(), drafter=bad)
        b.submit([1, 2], max_new=6)
        with pytest.raises(ValueError):
            b.run()


class Narrow(Stand):
    """A stand-in whose passes take a limited number of nodes, as those of lum_draft_verify."""

    def __init__(self, capacity, **kw):
        super().__init__(**kw)
        self.capacity, self.widest = capacity, 0

    def draft_capacity(self):
        return self.capacity

    def draft_verify(self, trees, positions, slots):
        n = sum(len(t) for t, _ in trees)
        assert n <= self.capacity, f"{n} nodes in all, a pass takes {self.capacity}"
        self.widest = max(self.widest, n)
        return super().draft_verify(trees, positions, slots)


@pytest.mark.parametrize("sequences, capacity, max_seq", [(32, 256, 256), (8, 128, 128), (5, 5, 64), (7, 9, 64), (3, 1000, 64)])
def test_the_loop_keeps_to_the_nodes_that_a_pass_takes(pkg, sequences, capacity, max_seq):
    rt = Narrow(capacity, max_batch=sequences, max_seq=max_seq)
    b = pkg.serving.ContinuousBatcher(rt, drafter=pkg.serving.PromptLookup())
    prompts = [[(i + j) % 5 for j in range(5)] * 4 + [i % 5] for i in range(sequences + 3)]
    ids = [b.submit(p, max_new=30) for p in prompts]
    got = b.run()
    assert [got[i] for i in ids] == [generate(p, 30) for p in prompts]
    assert b.stats()["drafted"] > 0 or capacity == sequences


def test_room_that_one_sequence_does_not_use_goes_to_the_next_ones(pkg):
    rt, rooms = Narrow(11, max_batch=3), []

    def drafter(text, room):
        rooms.append(room)
        return ([], []) if len(rooms) % 3 == 1 else ([4] * room, list(range(room)))

    b = pkg.serving.ContinuousBatcher(rt, steps_per_round=1, drafter=drafter)
    for i in range(3):
        b.submit([i, 1, 2], max_new=20)
    b.round()
    assert rooms == [2, 4, 4] and rt.widest == 11
