"""Speculative steps of whole models (lum_draft_verify, the serving loop's drafter): whatever is guessed, the tokens are those of plain decoding."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 1000, 3, 3, 8, 44], [9] * 40 + [7, 2], [(31 * i + 7) % 1900 for i in range(70)]]


def runtime(pkg, name="small_q8", **kw):
    rt = pkg.B200Runtime.initialize(device=0)
    rt.load_model(pkg.CONFIGS[name].copy(**kw))
    rt.synth(77)
    return rt


def prompts_in(rt, prompts):
    first = []
    for s, p in enumerate(prompts):
        rt.seq_select(s)
        rt.set_data(p)
        rt.execute({"s": len(p), "p": 0})
        first.append(rt.get_token())
    return first


def plain_tokens(pkg, n, sampling=None, **kw):
    """What plain batched steps give: [sequence][n] and the caches' rows of the first and last layer."""
    rt = runtime(pkg, max_batch=3, **kw)
    try:
        if sampling:
            rt.set_sampling(**sampling)
        first = prompts_in(rt, PROMPTS)
        rt.batch_begin(first, [len(p) for p in PROMPTS])
        rt.batch_decode(n - 1)
        log = np.asarray(rt.batch_get_decoded(n - 1))
        rows = []
        for s, p in enumerate(PROMPTS):
            rt.seq_select(s)
            rows.append([rt.kv_read(layer, kind, len(p) + n - 1) for layer in (0, rt.desc.n_layers - 1) for kind in ("k", "v")])
        return [[first[s]] + [int(t) for t in log[:, s]] for s in range(3)], rows
    finally:
        rt.close()


def guesses(kind, ahead, rng):
    """(tokens, parents) of guesses behind node 0, whose true continuation is `ahead`."""
    wrong = lambda: int(rng.integers(0, 2048))  # noqa: E731
    if kind == "none":
        return [], []
    if kind == "right":
        t = list(ahead[:5])
        return t, list(range(len(t)))
    if kind == "wrong":
        return [wrong() for _ in range(6)], [0, 1, 1, 0, 4, 5]
    # the right path among wrong branches, its nodes in between
    tokens, parents, at = [], [], 0
    for t in ahead[:4]:
        for _ in range(int(rng.integers(0, 3))):
            tokens.append(wrong())
            parents.append(int(rng.integers(0, len(tokens))))
        tokens.append(t)
        parents.append(at)
        at = len(tokens)
    return tokens + [wrong()], parents + [at]


@pytest.mark.parametrize("page, kv", [(0, "bf16"), (64, "bf16"), (64, "f32")])
@pytest.mark.parametrize("kind", ["none", "right", "wrong", "tree"])
def test_verified_drafts_are_plain_decoding(pkg, kind, page, kv):
    n = 24
    cfg = dict(kv_page_rows=page, kv_dtype=pkg.DTYPE[kv])
    want, want_rows = plain_tokens(pkg, n, **cfg)
    rt = runtime(pkg, max_batch=3, **cfg)
    rng = np.random.default_rng(4)
    try:
        got = [[t] for t in prompts_in(rt, PROMPTS)]
        pos = [len(p) for p in PROMPTS]
        steps = 0
        while min(len(g) for g in got) < n:
            order = [int(s) for s in rng.permutation(3) if len(got[s]) < n]        # sequences in any order, those that are done left out
            trees = []
            for s in order:
                tokens, parents = guesses(kind, want[s][len(got[s]):n - 1], rng)
                trees.append(([got[s][-1]] + tokens, [-1] + parents))
            for s, new in zip(order, rt.draft_verify(trees, [pos[s] for s in order], order)):
                got[s] += new
                pos[s] += len(new)
            steps += 1
        for s in range(3):
            assert got[s][:n] == want[s], s
            rt.seq_select(s)
            rows = [rt.kv_read(layer, k, len(PROMPTS[s]) + n - 1) for layer in (0, rt.desc.n_layers - 1) for k in ("k", "v")]
            for a, b in zip(rows, want_rows[s]):
                # the same values but for the order of sums: a step of the cache's type here and there
                assert np.abs(a - b).max() <= (2.0 ** -6 if kv == "bf16" else 1e-3) * np.abs(b).max()
        assert steps == (n - 1 if kind in ("none",) else steps)
        if kind in ("right", "tree"):
            assert steps <= (n + 3) // 4 + 3, steps
    finally:
        rt.close()


def test_verified_drafts_of_a_sampler(pkg):
    """The draw at a node is that of plain decoding at its position, so guesses stand exactly where plain sampling would have drawn them."""
    n, sampling = 16, dict(temperature=0.9, top_k=40, top_p=0.95, seed=11)
    want, _ = plain_tokens(pkg, n, sampling)
    rt = runtime(pkg, max_batch=3)
    rng = np.random.default_rng(5)
    try:
        rt.set_sampling(**sampling)
        got = [[t] for t in prompts_in(rt, PROMPTS)]
        pos = [len(p) for p in PROMPTS]
        while min(len(g) for g in got) < n:
            order = [s for s in range(3) if len(got[s]) < n]
            trees = []
            for s in order:
                tokens, parents = guesses("tree", want[s][len(got[s]):n - 1], rng)
                trees.append(([got[s][-1]] + tokens, [-1] + parents))
            for s, new in zip(order, rt.draft_verify(trees, [pos[s] for s in order], order)):
                got[s] += new
                pos[s] += len(new)
        assert [g[:n] for g in got] == want
    finally:
        rt.close()


def test_single_token_steps_go_on_behind_a_verified_draft(pkg):
    """max_batch 1: a verified step between steps of the device-resident loop."""
    solo = runtime(pkg, max_seq=128)
    want = solo.generate(PROMPTS[0], 12)
    solo.close()
    rt = runtime(pkg, max_seq=128, kv_page_rows=64)
    try:
        first = prompts_in(rt, PROMPTS[:1])[0]
        new = rt.draft_verify([([first, want[1], want[2], 1], [-1, 0, 1, 1])], [len(PROMPTS[0])])[0]
        assert [first] + new == want[:1 + len(new)] and len(new) == 3
        assert rt.get_token() == new[-1]
        rt.decode_reset()
        rt.decode_greedy(8)
        assert [first] + new + list(rt.get_decoded(8)) == want
        assert rt.kv_pool()[1] == 1                      # one page of two holds the 18 rows
    finally:
        rt.close()


def test_pages_of_what_did_not_stand_go_back_and_shared_pages_are_left_alone(pkg):
    rt = runtime(pkg, max_batch=3, kv_page_rows=64, max_seq=128)
    try:
        prompt = [(3 * i + 1) % 2000 for i in range(60)]
        rt.seq_select(0); rt.set_data(prompt); rt.execute({"s": 60, "p": 0})
        first = rt.get_token()
        rt.kv_copy(0, 1, 60)                             # a fork
        before = np.asarray(rt.kv_save(0, "k", 60)).copy()
        free = rt.kv_pool()[1]
        tree = ([first] + [1] * 20, [-1] + list(range(20)))
        new = rt.draft_verify([tree], [60], [1])[0]
        assert rt.kv_pool()[1] == free                   # rows 60 .. 80 reached a second page, which went back
        rt.seq_select(0)
        assert np.array_equal(np.asarray(rt.kv_save(0, "k", 60)), before)
        rt.batch_begin_slots([0], [first], [60]); rt.batch_decode(2)
        assert rt.batch_get_decoded(2)[0][0] == new[0]
    finally:
        rt.close()


def test_refusals(pkg):
    rt = runtime(pkg, max_batch=2, max_seq=64)
    try:
        ok = ([3, 4, 5], [-1, 0, 0])
        for trees, positions, slots in ((  # noqa: E741
                [([3], [0])], [5], None), ([([3, 4], [-1, 1])], [5], None), ([([3, 4], [-1, -1])], [5], None), ([([3, 5000], [-1, 0])], [5], None),
                ([ok], [62], None), ([ok], [-1], None), ([ok], [5], [2]), ([ok, ok], [5, 5], [1, 1]), ([ok, ok, ok], [5, 5, 5], None),
                ([([], [])], [5], None), ([([1] * 257, [-1] + [0] * 256)], [0], None), ([([3, 4], [-1])], [5], None), ([ok], [5, 6], None)):
            with pytest.raises(pkg.LumError) as e:
                rt.draft_verify(trees, positions, slots)
            assert e.value.code == -1
        rt.set_data([1, 2, 3, 4]); rt.execute({"s": 4, "p": 0})
        assert len(rt.draft_verify([([rt.get_token()], [-1])], [4])[0]) == 1       # and goes on
    finally:
        rt.close()
    rt = runtime(pkg, "tiny_f32")
    try:
        with pytest.raises(pkg.LumError) as e:
            rt.draft_verify([([1], [-1])], [0])
        assert e.value.code == -3
    finally:
        rt.close()


@pytest.mark.parametrize("page", [0, 64])
def test_serving_with_a_drafter(pkg, page):
    """The loop with prompt lookup gives every request the tokens it gets without, in fewer passes where the text repeats."""
    out = []
    for drafter in (None, pkg.serving.PromptLookup(length=6, match=2, places=2)):
        rt = runtime(pkg, max_batch=3, kv_page_rows=page)
        try:
            b = pkg.serving.ContinuousBatcher(rt, steps_per_round=4, drafter=drafter)
            ids = [b.submit(p, max_new=20, eos=[77]) for p in PROMPTS + [[6, 5, 4, 6, 5, 4, 6, 5], [2] * 12]]
            res = b.run()
            out.append([res[i] for i in ids])
            if drafter:
                st = b.stats()
                assert st["drafted"] > 0 and 0 <= st["stood"] <= st["drafted"]
        finally:
            rt.close()
    assert out[0] == out[1]


def test_serving_with_more_guesses_than_a_pass_takes(pkg, monkeypatch):
    """Passes of 32 rows, and a drafter that would fill 41 for each of three sequences: the loop shares the rows out."""
    monkeypatch.setenv("LUM_ROWS_CAP", "32")
    out = []

    def look(text, room):
        tokens, parents = pkg.serving.PromptLookup(length=20, match=1, places=2)(text, room)
        return tokens + [3] * (room - len(tokens)), parents + [0] * (room - len(tokens))

    for drafter in (None, look):
        rt = runtime(pkg, max_batch=3, max_seq=256)
        try:
            b = pkg.serving.ContinuousBatcher(rt, steps_per_round=4, drafter=drafter)
            ids = [b.submit(p, max_new=20) for p in PROMPTS + [[6, 5, 4, 6, 5, 4, 6, 5], [2] * 12]]
            res = b.run()
            out.append([res[i] for i in ids])
            if drafter:
                assert rt.draft_capacity() == 32
                with pytest.raises(pkg.LumError) as e:   # the runtime itself still refuses what does not fit
                    rt.draft_verify([([1] * 33, [-1] + [0] * 32)], [5], [0])
                assert e.value.code == -1
        finally:
            rt.close()
    assert out[0] == out[1]


def test_capacity_of_a_model_that_cannot_verify(pkg):
    rt = runtime(pkg, "tiny_f32")
    try:
        with pytest.raises(pkg.LumError) as e:
            rt.draft_capacity()
        assert e.value.code == -3
    finally:
        rt.close()
    rt = runtime(pkg, max_seq=64)
    try:
        assert rt.draft_capacity() == 64
        rt.set_data([1, 2, 3]); rt.execute({"s": 3, "p": 0})
        assert len(rt.draft_verify([([rt.get_token()] + [1] * 60, [-1] + [0] * 60)], [3])[0]) >= 1
    finally:
        rt.close()


@pytest.mark.parametrize("bits, words", [(1 << 8, "no tree"), (1 << 9, "cache row or page"), (1 << 8 | 1 << 9, "no path through one; cache row or page")])
def test_the_runtime_says_what_was_wrong_with_a_tree_or_a_page(pkg, bits, words):
    rt = runtime(pkg, max_seq=64)
    try:
        rt.set_data([1, 2, 3]); rt.execute({"s": 3, "p": 0})
        cur = rt.get_token()
        rt.debug_set_status(bits)
        with pytest.raises(pkg.LumError) as e:
            rt.draft_verify([([cur, 1], [-1, 0])], [3])
        assert e.value.code == -4 and words in str(e.value) and hex(bits) in str(e.value)
        assert len(rt.draft_verify([([cur, 1], [-1, 0])], [3])[0]) >= 1                  # and goes on
    finally:
        rt.close()


def test_steps_that_grow_keep_no_more_memory_than_the_largest_one(pkg):
    """The buffers of a step that was outgrown go back: what is left is what a runtime holds that ran the largest step first."""
    import torch
    used = []
    for sizes in ([256], [256], [8, 30, 60, 100, 150, 200, 256]):                        # (the first time loads the kernels)
        before = torch.cuda.mem_get_info()[0]
        rt = runtime(pkg, max_batch=8, max_seq=2048)
        try:
            for n in sizes:
                rt.draft_verify([([1] * n, [-1] + [0] * (n - 1))] * 8, [0] * 8)
            used.append(before - torch.cuda.mem_get_info()[0])
        finally:
            rt.close()
    # a block of the allocator (2 MB) for each of the step's four buffers.  Without giving back, the logits alone (2048 values of f32) leave 1.5 x 8 x
    # (8 + 30 + 60 + 100 + 200) rows of 8 KB: 39 MB, where the largest step needs 17
    assert used[2] <= used[1] + 8 * 2 ** 20, used


def test_a_step_that_the_pool_cannot_hold_takes_no_page(pkg):
    """Three sequences that share a prompt's pages; the pool runs out at the third.  One page more and the same step goes through."""
    prompt = [(3 * i + 1) % 2000 for i in range(160)]
    for pages, ok in ((5, False), (6, True)):
        rt = runtime(pkg, max_batch=4, kv_page_rows=64, max_seq=256, kv_pool_pages=pages)
        try:
            rt.set_data(prompt); rt.execute({"s": 160, "p": 0})                          # 3 pages, the last one half full
            cur = rt.get_token()
            rt.kv_copy(0, 1, 128); rt.kv_copy(0, 2, 128)                                 # two of them shared
            assert rt.kv_pool()[1] == pages - 3
            tree = ([cur, 1], [-1, 0])
            # a page each for sequences 1 and 2 behind row 128, and a copy of the second page, whose last row sequence 1 writes
            trees, positions, slots = [tree, tree, ([cur], [-1])], [127, 128, 160], [1, 2, 0]
            if ok:
                assert [len(x) >= 1 for x in rt.draft_verify(trees, positions, slots)] == [True] * 3
            else:
                with pytest.raises(pkg.LumError) as e:
                    rt.draft_verify(trees, positions, slots)
                assert e.value.code == -5 and "pool" in str(e.value) and rt.kv_pool()[1] == pages - 3
            assert len(rt.draft_verify([([cur, 1, 2], [-1, 0, 1])], [160], [0])[0]) >= 1   # and goes on
        finally:
            rt.close()


def test_pages_of_a_step_that_a_kernel_gave_up_go_back(pkg):
    rt = runtime(pkg, max_batch=2, kv_page_rows=64, max_seq=256)
    try:
        prompt = [(3 * i + 1) % 2000 for i in range(64)]
        first = prompts_in(rt, [prompt, prompt])
        free = rt.kv_pool()[1]
        trees = [([t] + [1] * 100, [-1] + list(range(100))) for t in first]              # two pages each behind the prompt's
        rt.debug_set_status(1 << 9)
        with pytest.raises(pkg.LumError) as e:
            rt.draft_verify(trees, [64, 64])
        assert e.value.code == -4 and rt.kv_pool()[1] == free
        again = rt.draft_verify(trees, [64, 64])                                         # and the step can be made again
        assert [len(x) >= 1 for x in again] == [True, True]
    finally:
        rt.close()


def test_results_outlive_a_refused_step(pkg):
    import ctypes as C
    ints = lambda *v: (C.c_int32 * len(v))(*v)  # noqa: E731
    rt = runtime(pkg, max_batch=2, max_seq=64)
    try:
        first = prompts_in(rt, PROMPTS[:1])[0]
        want = rt.draft_verify([([first], [-1])], [len(PROMPTS[0])])[0]
        verify = lambda p, *t: rt._lib.lum_draft_verify(rt._h, 1, None, ints(p), ints(0, len(t)), ints(*t), ints(*range(-1, len(t) - 1)))  # noqa: E731
        counts, out = (C.c_int32 * 1)(), (C.c_int32 * 1)()
        assert verify(len(PROMPTS[0]), first) == 0
        assert verify(64, first) == -1 and verify(3, 10 ** 6) == -1 and verify(3, *[1] * 65) == -1
        assert rt._lib.lum_draft_get(rt._h, counts, out, 1) == 0 and [counts[0], out[0]] == [1] + want
        assert rt._lib.lum_draft_get(rt._h, counts, out, 1) == -1                        # read once
    finally:
        rt.close()
