"""A continuous-batching decode loop over the runtime's cache slots.

The reference's example loop serves one sequence: prompt, then one ``execute`` per token with the sample taken on the host
(examples/llama/src/main.rs:82-148).  This is the step after it for a server: requests arrive in a queue, each one takes a
free cache slot (its prompt runs as rows on the tensor cores), all live slots then advance together — one row per sequence
and step, samples fed back on the device — and a request that ends (token budget or an end-of-sequence id) frees its slot for
the next one in the queue between two groups of steps.  Prompt prefixes computed once can be parked in a slot and copied into
a new request's slot on the device instead of being recomputed.  With a paged cache the loop admits a request only when
the pool can hold its whole life (prompt and every token it may generate) next to what is already promised, and gives a
finished request's pages back.

With a ``drafter`` the steps are speculative: every live sequence brings a tree of guesses of what follows its last token, one pass of
the model verifies them all (``draft_verify``), and a sequence moves on by as many tokens as it guessed right, plus one — the tokens are
those of plain decoding.  :class:`PromptLookup` is a drafter that needs no second model.  What one pass takes (``draft_capacity``, where the runtime
has it) is shared out evenly among the sequences' guesses.

Everything here is host-side bookkeeping over four calls of the runtime: ``seq_select`` + ``execute`` (admission),
``kv_copy`` (prefix reuse), ``batch_begin_slots`` + ``batch_decode`` (the steps).  The runtime object only needs those methods
plus ``set_data``, ``get_token``, ``batch_get_decoded`` and ``desc.max_batch`` / ``desc.max_seq`` / ``desc.max_new_tokens``.
"""
from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field
from typing import Deque, Dict, Iterable, List, Optional, Sequence, Set, Tuple


@dataclass
class Request:
    """One generation request and its progress."""

    rid: int
    prompt: List[int]
    max_new: int
    eos: Set[int] = field(default_factory=set)
    tokens: List[int] = field(default_factory=list)   # generated so far (the end-of-sequence id, if met, is the last one)
    slot: int = -1
    pos: int = 0                                      # rows of this sequence in its cache slot
    done: bool = False
    reused_rows: int = 0                              # prompt rows taken from a parked prefix instead of being computed
    pages: int = 0                                    # paged cache: pages set aside for this request's whole life

    @property
    def cur(self) -> int:
        return self.tokens[-1]


class PromptLookup:
    """Guesses that the text goes on as it did before: where the last ``match`` tokens (or fewer, down to one) occurred earlier in a sequence, what
    followed them there, up to ``length`` tokens.  The ``places`` most recent such places are branches of the tree; what they have in common is one
    path of it."""

    def __init__(self, length: int = 8, match: int = 3, places: int = 2):
        if length < 1 or match < 1 or places < 1:
            raise ValueError("length, match and places must be at least 1")
        self.length, self.match, self.places = length, match, places

    def __call__(self, text: Sequence[int], room: int) -> Tuple[List[int], List[int]]:
        text, room = list(text), min(room, self.length * self.places)
        tokens: List[int] = []
        parents: List[int] = []
        for n in range(min(self.match, len(text) - 1), 0, -1):
            tail, found = text[-n:], 0
            for i in range(len(text) - n - 1, -1, -1):
                if text[i:i + n] != tail:
                    continue
                at = 0                                   # node 0 is the last token of the text
                for t in text[i + n:i + n + self.length]:
                    known = [j + 1 for j in range(len(tokens)) if parents[j] == at and tokens[j] == t]
                    if known:
                        at = known[0]
                    elif len(tokens) < room:
                        tokens.append(t)
                        parents.append(at)
                        at = len(tokens)
                    else:
                        break
                found += 1
                if found == self.places:
                    break
            if tokens:
                break
        return tokens, parents


class ContinuousBatcher:
    """Keeps up to ``max_batch`` (minus parked prefixes) sequences decoding together and refills slots as requests end."""

    def __init__(self, rt, steps_per_round: int = 8, drafter=None):
        """``drafter(text, room)``: at most ``room`` guesses of what follows the tokens ``text``, as (tokens, parents) with parent 0 = the last
        token of the text and parent k = the k-th guess, which comes before its children (None: plain steps)."""
        if steps_per_round < 1:
            raise ValueError("steps_per_round must be at least 1")
        self.rt = rt
        self.drafter = drafter
        self.steps_per_round = steps_per_round
        self.free: List[int] = list(range(rt.desc.max_batch))[::-1]      # pop() hands out slot 0 first
        self.queue: Deque[Request] = deque()
        self.live: Dict[int, Request] = {}                               # slot -> request
        self.finished: Dict[int, Request] = {}
        self.prefixes: List[Tuple[Tuple[int, ...], int]] = []            # (tokens, slot), longest first
        self._next_id = 0
        # Paged cache: a request is admitted only when the pool can hold its prompt AND every token it may still generate, next to
        # what the live requests and the parked prefixes were promised — so no step ever finds the pool empty.  (Pages a request
        # shares with a parked prefix are counted for the request too: it may write into them, which gives it copies of its own.)
        pool = getattr(rt, "kv_pool", None)
        self.page_rows = 0
        self.pool_pages = 0
        if pool is not None:
            total, _free, rows = pool()
            self.page_rows, self.pool_pages = rows, total
        self.promised = 0           # pages promised to live requests and parked prefixes
        self.rounds = 0
        self.steps_run = 0          # batched steps issued
        self.rows_run = 0           # rows those steps carried (sum of live sequences per step; with a drafter, of nodes)
        self.drafted = 0            # guesses made, and those that stood
        self.stood = 0
        self.pass_nodes: Optional[int] = None        # nodes that a pass takes, of all trees (asked for by the first speculative step)

    # ---- requests ------------------------------------------------------------------------------------------------
    def submit(self, prompt: Sequence[int], max_new: int, eos: Optional[Iterable[int]] = None) -> int:
        prompt = [int(t) for t in prompt]
        if not prompt:
            raise ValueError("empty prompt")
        if max_new < 1:
            raise ValueError("max_new must be at least 1")
        if len(prompt) + max_new > self.rt.desc.max_seq:
            raise ValueError(f"prompt of {len(prompt)} tokens + {max_new} new ones pass the cache capacity {self.rt.desc.max_seq}")
        if self.page_rows and self._pages_for(len(prompt) + max_new) > self.pool_pages:
            raise ValueError(f"{len(prompt) + max_new} rows need more pages than the pool has ({self.pool_pages} of {self.page_rows} rows)")
        r = Request(self._next_id, prompt, max_new, set(int(e) for e in (eos or ())))
        self._next_id += 1
        self.queue.append(r)
        return r.rid

    def _pages_for(self, rows: int) -> int:
        return -(-rows // self.page_rows) if self.page_rows else 0

    def park_prefix(self, tokens: Sequence[int]) -> int:
        """Compute a prompt prefix once into a slot of its own; later requests that start with it copy its rows on the device.
        Returns the slot (it no longer serves requests)."""
        tokens = tuple(int(t) for t in tokens)
        if not tokens:
            raise ValueError("empty prefix")
        if len(self.free) < 2:
            raise RuntimeError("parking a prefix would leave no slot for requests")
        if self.page_rows and self.promised + self._pages_for(len(tokens)) > self.pool_pages:
            raise RuntimeError("the page pool cannot hold this prefix next to what is already promised")
        self.promised += self._pages_for(len(tokens))
        slot = self.free.pop()
        self.rt.seq_select(slot)
        self.rt.set_data(list(tokens))
        self.rt.execute({"s": len(tokens), "p": 0})
        self.prefixes.append((tokens, slot))
        self.prefixes.sort(key=lambda e: -len(e[0]))
        return slot

    # ---- the loop ------------------------------------------------------------------------------------------------
    def _admit(self, r: Request, slot: int) -> None:
        rt = self.rt
        start = 0
        for toks, pslot in self.prefixes:
            # leave at least one prompt token to run: its row produces the first sample
            if len(toks) < len(r.prompt) and tuple(r.prompt[:len(toks)]) == toks:
                rt.kv_copy(pslot, slot, len(toks))
                start = len(toks)
                break
        rt.seq_select(slot)
        rt.set_data(r.prompt[start:])
        rt.execute({"s": len(r.prompt) - start, "p": start})
        r.tokens = [int(rt.get_token())]
        r.slot, r.pos, r.reused_rows = slot, len(r.prompt), start
        r.pages = self._pages_for(len(r.prompt) + r.max_new)
        self.promised += r.pages
        self.live[slot] = r
        self._check_done(r)

    def _check_done(self, r: Request) -> None:
        if r.done:
            return
        if len(r.tokens) >= r.max_new or (r.tokens and r.tokens[-1] in r.eos):
            r.done = True
            self.promised -= r.pages
            del self.live[r.slot]
            release = getattr(self.rt, "kv_release", None)
            if release is not None:
                release(r.slot)                          # a paged cache gets the sequence's pages back
            self.free.append(r.slot)
            self.finished[r.rid] = r

    def round(self) -> List[Request]:
        """Admit what fits, run one group of steps for every live sequence, retire what ended.  Returns the requests that ended."""
        before = set(self.finished)
        while self.queue and self.free:
            nxt = self.queue[0]
            if self.page_rows and self.promised + self._pages_for(len(nxt.prompt) + nxt.max_new) > self.pool_pages:
                break                                    # first come, first served: it waits for pages, nobody overtakes it
            self._admit(self.queue.popleft(), self.free.pop())
        if self.live and self.drafter is not None:
            for _ in range(self.steps_per_round):
                if self.live and not self._speculate():
                    break
        elif self.live:
            slots = sorted(self.live)
            reqs = [self.live[s] for s in slots]
            n = min(self.steps_per_round, self.rt.desc.max_new_tokens, min(r.max_new - len(r.tokens) for r in reqs))
            self.rt.batch_begin_slots(slots, [r.cur for r in reqs], [r.pos for r in reqs])
            self.rt.batch_decode(n)
            log = self.rt.batch_get_decoded(n)          # [n][rows]
            self.steps_run += n
            self.rows_run += n * len(reqs)
            for j, r in enumerate(reqs):
                for s in range(n):
                    r.tokens.append(int(log[s][j]))
                    r.pos += 1
                    if r.tokens[-1] in r.eos:
                        break                            # what the row decoded after its end is dropped
                self._check_done(r)
        self.rounds += 1
        return [self.finished[i] for i in sorted(set(self.finished) - before)]

    def _speculate(self) -> bool:
        """One speculative step of every live sequence.  False: a request has ended, its slot can be filled."""
        slots = sorted(self.live)
        reqs = [self.live[s] for s in slots]
        if self.pass_nodes is None:
            capacity = getattr(self.rt, "draft_capacity", None)
            self.pass_nodes = 1 << 30 if capacity is None else capacity()
        trees = []
        left = self.pass_nodes - len(reqs)               # guesses that the pass has room for, next to a node of every sequence
        for i, r in enumerate(reqs):
            # guesses that could all stand without passing what the request may still generate (the sample behind them is one more), and no more than an
            # even share of what the sequences before have left
            room = min(r.max_new - len(r.tokens) - 1, self.max_nodes - 1, left // (len(reqs) - i))
            tokens, parents = self.drafter(r.prompt + r.tokens, room) if room > 0 else ([], [])
            if len(tokens) > room or len(tokens) != len(parents) or any(not 0 <= p <= i for i, p in enumerate(parents)):
                raise ValueError(f"the drafter returned {len(tokens)} tokens and {len(parents)} parents for room {room}, or a parent that is no earlier guess")
            left -= len(tokens)
            trees.append(([r.cur] + [int(t) for t in tokens], [-1] + [int(p) for p in parents]))
        self.steps_run += 1
        ended = False
        for r, (tokens, _), new in zip(reqs, trees, self.rt.draft_verify(trees, [r.pos for r in reqs], slots)):
            self.rows_run += len(tokens)
            self.drafted += len(tokens) - 1
            self.stood += len(new) - 1
            r.pos += len(new)
            for t in new:
                r.tokens.append(int(t))
                if r.tokens[-1] in r.eos:
                    break                                # what was decoded after its end is dropped
            self._check_done(r)
            ended = ended or r.done
        return not ended

    max_nodes = 64                  # nodes of a tree

    def stats(self) -> Dict[str, float]:
        """Counters of the loop so far: how full the batched steps were is what decides the tokens/s of a server."""
        return {"rounds": self.rounds, "steps": self.steps_run, "rows": self.rows_run,
                "rows_per_step": self.rows_run / self.steps_run if self.steps_run else 0.0,
                "drafted": self.drafted, "stood": self.stood, "live": len(self.live), "queued": len(self.queue), "finished": len(self.finished),
                "pages_promised": self.promised, "pages_in_pool": self.pool_pages}

    def run(self) -> Dict[int, List[int]]:
        """Until the queue and the live set are empty.  Returns request id -> generated tokens."""
        while self.queue or self.live:
            self.round()
        return {rid: r.tokens for rid, r in sorted(self.finished.items())}
