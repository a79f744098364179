"""Forked sequences on the host: pages held by several slots, the page a sequence ends in and its state copied, nothing lost or
freed early, errors that change nothing; several answers to a prompt and log probabilities in the generation loop."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from test_cache import FULL, STATE, WIN, make
from zinfer_b200.cache import CacheError, CallCacheSpec, NoFreeSlot, OutOfPages
from zinfer_b200.engine.generate import GenerationLoop, TokenScores
from zinfer_b200.parts.base import KVRequest, StateRequest


def cache(calls=None, **kw):
    """A cache whose copies are written down instead of launched."""
    c = make(calls, **kw)
    c.copies = []
    c._copy_pages = lambda g, src, dst, tokens: c.copies.append((c.groups.index(g), list(src), list(dst), list(tokens)))
    c._copy_states = lambda src, dst: c.copies.append(("state", list(src), list(dst)))
    return c


def grow(c, slot, n):
    c.reserve([slot], [n])
    c.advance([slot], [n])


def test_a_fork_holds_the_whole_pages_and_a_copy_of_the_last():
    c = cache(max_slots=4, max_tokens=256)
    s, = c.alloc_slots(1)
    grow(c, s, 37)                                           # pages of 16: two whole ones and 5 tokens of a third
    new = c.fork(s, 2)
    assert len(new) == 2 and all(c.lengths[f] == 37 and c.active[f] for f in new)
    g = c.groups[0]
    tables = g.table_host[[s, *new], :3]
    assert (tables[:, :2] == tables[0, :2]).all() and len(set(tables[:, 2].tolist())) == 3
    assert c.copies == [(0, [tables[0, 2]] * 2, tables[1:, 2].tolist(), [5, 5]), ("state", [s, s], new)]
    assert c.free_page_count() == [16 - 5] and g.shared_pages == 2
    c.check_consistency()
    grow(c, new[0], 20)                                      # a fork's own growth touches nobody else's pages
    assert (g.table_host[s, :3] == tables[0]).all() and g.table_host[s, 3] == -1
    c.check_consistency()
    assert c.shared_prefixes([new[1], s, new[0]]) == [([0, 1, 2], 32)]
    assert c.shared_prefixes([s]) == [] and c.shared_prefixes([new[0], s]) == [([0, 1], 32)]


def test_a_sequence_of_whole_pages_copies_no_page():
    c = cache([CallCacheSpec(kv=FULL)])
    s, = c.alloc_slots(1)
    grow(c, s, 32)
    new = c.fork(s, 1)
    assert c.copies == [] and c.free_page_count() == [14]
    grow(c, s, 1)
    grow(c, new[0], 1)
    assert c.groups[0].table_host[s, 2] != c.groups[0].table_host[new[0], 2]
    c.check_consistency()


def test_pages_go_back_with_their_last_holder_in_any_order():
    for order in ([0, 1, 2], [2, 0, 1], [1, 2, 0]):
        c = cache([CallCacheSpec(kv=FULL)], max_slots=3)
        s, = c.alloc_slots(1)
        grow(c, s, 40)
        slots = [s, *c.fork(s, 2)]
        for i, x in enumerate(order):
            c.free_slots([slots[x]])
            c.check_consistency()
            assert c.free_page_count() == [16 - (2 + 2 - i) if i < 2 else 16]
        assert c.groups[0].shared_pages == 0 and not c.groups[0].holders.any()


def test_forks_of_forks():
    c = cache([CallCacheSpec(kv=FULL)], max_slots=8, max_tokens=512, max_seq_len=200)
    a, = c.alloc_slots(1)
    grow(c, a, 33)
    b, = c.fork(a, 1)
    grow(c, b, 40)                                           # 73 tokens: four whole pages
    d, e = c.fork(b, 2)
    c.check_consistency()
    assert c.shared_prefixes([a, b, d, e]) == [([0, 1, 2, 3], 32)] and c.shared_prefixes([d, e, b]) == [([0, 1, 2], 64)]
    other, = c.alloc_slots(1)
    grow(c, other, 20)
    assert c.shared_prefixes([other, d, a, e]) == [([1, 2, 3], 32)]
    c.free_slots([a, b])
    c.check_consistency()
    assert c.shared_prefixes([d, e]) == [([0, 1], 64)]
    c.free_slots([d])
    assert c.shared_prefixes([e, other]) == [] and c.groups[0].shared_pages == 0
    c.free_slots([e, other])
    assert c.free_page_count() == [32]
    c.check_consistency()


def test_windows_and_stretches_give_shared_pages_back_once_each():
    keep = KVRequest(2, 16, 40, keep_first=5)
    chunk = KVRequest(2, 16, chunk=32)
    c = cache([CallCacheSpec(kv=WIN), CallCacheSpec(kv=FULL), CallCacheSpec(kv=keep), CallCacheSpec(kv=chunk)], max_tokens=512, max_seq_len=300)
    s, = c.alloc_slots(1)
    grow(c, s, 75)
    new = c.fork(s, 2)
    c.check_consistency()
    assert [len(x[1]) for x in c.copies] == [2, 2, 2, 2]
    for x, n in ((new[0], 100), (s, 1), (new[1], 30), (s, 60)):
        grow(c, x, n)
        c.check_consistency()
    assert c.shared_prefixes([s, *new]) == [([0, 1, 2], 64)]
    c.free_slots([s, *new])
    assert c.free_page_count() == [32] * 4
    c.check_consistency()


def test_a_cache_without_an_unwindowed_group_shares_no_prefix():
    c = cache([CallCacheSpec(kv=WIN), CallCacheSpec(state=STATE)])
    s, = c.alloc_slots(1)
    grow(c, s, 70)
    new = c.fork(s, 1)
    assert c.shared_prefixes([s, *new]) == []
    c = cache([CallCacheSpec(state=STATE), CallCacheSpec(state=StateRequest((3,)))])
    s, = c.alloc_slots(1)
    new = c.fork(s, 2)
    assert c.copies == [("state", [s, s], new)] and c.shared_prefixes([s, *new]) == []


def test_an_empty_sequence_and_no_forks():
    c = cache()
    s, = c.alloc_slots(1)
    new = c.fork(s, 1)
    assert c.lengths[new[0]] == 0 and c.copies == [("state", [s], new)] and c.shared_prefixes([s, *new]) == []
    assert c.fork(s, 0) == []
    c.check_consistency()


def test_fork_errors_change_nothing():
    c = cache([CallCacheSpec(kv=FULL)], max_slots=4, max_tokens=64)
    s, = c.alloc_slots(1)
    grow(c, s, 50)                                           # four pages: none is left
    for bad, error in ((lambda: c.fork(s, 1), OutOfPages), (lambda: c.fork(s, 4), NoFreeSlot), (lambda: c.fork(3, 1), CacheError),
                       (lambda: c.fork(-1, 1), CacheError), (lambda: c.fork(9, 1), CacheError), (lambda: c.fork(s, -1), CacheError)):
        with pytest.raises(error):
            bad()
    assert c.copies == [] and c.free_slot_count() == 3 and c.groups[0].shared_pages == 0
    c.check_consistency()
    grow(c, s, 14)                                           # whole pages: nothing to copy, nothing needed
    assert len(c.fork(s, 3)) == 3
    c.check_consistency()


def test_a_copy_that_fails_gives_everything_back():
    for broken in ("_copy_pages", "_copy_states"):
        c = cache(max_slots=4)
        s, = c.alloc_slots(1)
        grow(c, s, 37)

        def fail(*args):
            raise RuntimeError("no copy")
        setattr(c, broken, fail)
        with pytest.raises(RuntimeError, match="no copy"):
            c.fork(s, 2)
        assert c.free_slot_count() == 3 and c.free_page_count() == [13] and c.lengths[s] == 37
        c.check_consistency()


def test_random_histories_lose_no_page():
    rng = np.random.default_rng(5)
    for trial in range(20):
        c = cache([CallCacheSpec(kv=FULL), CallCacheSpec(kv=WIN), CallCacheSpec(state=STATE)], max_slots=6, max_tokens=640, max_seq_len=120)
        live = []
        for _ in range(60):
            what = rng.integers(0, 4)
            try:
                if what == 0:
                    live += c.alloc_slots(1)
                elif what == 1 and live:
                    live += c.fork(live[rng.integers(len(live))], int(rng.integers(1, 3)))
                elif what == 2 and live:
                    grow(c, live[rng.integers(len(live))], int(rng.integers(1, 40)))
                elif live:
                    c.free_slots([live.pop(rng.integers(len(live)))])
            except CacheError:
                pass
            c.check_consistency()
            for rows, tokens in c.shared_prefixes(live):
                pages = c.groups[0].table_host[[live[r] for r in rows], :tokens // 16]
                assert (pages == pages[0]).all() and (pages >= 0).all() and all(c.lengths[live[r]] >= tokens for r in rows)
        c.free_slots(live)
        assert c.free_page_count() == [40, 40]


# ------------------------------------------------------------------------------- the loop

class Backend:
    """Request r's k-th new token is 1000 * r + k; a slot learns its request from the sampler's rows."""

    def __init__(self, slots):
        self.free, self.log, self.fed = list(range(slots)), [], {}

    def start(self, n):
        return [self.free.pop(0) for _ in range(n)]

    def fork(self, slot, n):
        new = [self.free.pop(0) for _ in range(n)]
        for s in new:
            self.fed[s] = list(self.fed[slot])
        self.log.append(("fork", slot, tuple(new)))
        return new

    def finish(self, slots):
        self.free += slots

    def prefill(self, slots, prompts):
        self.log.append(("prefill", tuple(slots), tuple(map(len, prompts))))
        for s, p in zip(slots, prompts):
            self.fed[s] = list(p)
        return torch.tensor([float(p[0]) for p in prompts])

    def decode(self, slots, tokens):
        for s, t in zip(slots, tokens):
            self.fed[s].append(t)
        return torch.zeros(len(slots))

    def read_tokens(self, toks):
        return list(toks)

    def token_logprobs(self, logits, tokens, top):
        n = len(tokens)
        return SimpleNamespace(logprob=torch.tensor([-0.5 * t for t in tokens]), rank=torch.arange(n) + 1, entropy=torch.ones(n),
                               top_ids=torch.arange(n * top).reshape(n, top), top_logprobs=torch.zeros((n, top)))


class Sampler:
    def __init__(self, n):
        self.step, self.rows, self.history = [0] * n, [], {}

    def accept(self, r, toks):
        self.history.setdefault(r, []).extend(toks)

    def sample(self, logits, requests):
        self.rows.append((list(requests), logits.tolist()))
        out = []
        for r in requests:
            out.append(1000 * r + self.step[r])
            self.step[r] += 1
        return out


PROMPTS = [[7, 1, 2], [8], [9, 9, 9, 9]]


@pytest.mark.parametrize("slots", [2, 4, 5, 9])
def test_several_answers_to_a_prompt(slots):
    """Whatever the batches: every answer starts from its prompt's logits and is fed its own tokens; a batch runs a prompt once."""
    be, smp = Backend(slots), Sampler(9)
    loop = GenerationLoop(be, slots, 10_000, 1000, 16)
    results = loop.run(PROMPTS, smp, max_new_tokens=4, samples=3)
    assert [r.tokens for r in results] == [[1000 * r + k for k in range(4)] for r in range(9)]
    assert [r.prompt_tokens for r in results] == [len(p) for p in PROMPTS for _ in range(3)]
    assert sorted(be.free) == list(range(slots))
    for rows, logits in smp.rows:
        if smp.history and any(logits):
            assert logits == [float(PROMPTS[r // 3][0]) for r in rows]
    assert all(smp.history[r][:len(PROMPTS[r // 3])] == PROMPTS[r // 3] for r in range(9))
    prompts_run = sum(len(x[1]) for x in be.log if x[0] == "prefill")
    assert prompts_run + sum(len(x[2]) for x in be.log if x[0] == "fork") == 9
    if slots == 9:
        assert prompts_run == 3 and loop.stats.n_prompt == 8


def test_one_answer_forks_nothing():
    be, smp = Backend(4), Sampler(3)
    GenerationLoop(be, 4, 10_000, 1000, 16).run(PROMPTS, smp, max_new_tokens=2)
    assert not any(x[0] == "fork" for x in be.log)


def test_log_probabilities_go_to_their_requests():
    be, smp = Backend(9), Sampler(9)
    stop = [1002, 3000, 8003]
    results = GenerationLoop(be, 9, 10_000, 1000, 16).run(PROMPTS, smp, max_new_tokens=4, stop_ids=stop, samples=3, logprobs=2)
    for r, res in enumerate(results):
        seen = res.tokens + ([res.stop_token] if res.stop_token is not None else [])
        assert res.logprobs.logprobs == [-0.5 * t for t in seen]
        assert len(res.logprobs.ranks) == len(res.logprobs.entropies) == len(res.logprobs.top) == len(seen)
        assert all(len(t) == 2 for t in res.logprobs.top)
    assert results[1].tokens == [1000, 1001] and results[3].tokens == [] and results[8].tokens == [8000, 8001, 8002]
    be, smp = Backend(3), Sampler(3)
    results = GenerationLoop(be, 3, 10_000, 1000, 16).run(PROMPTS, smp, max_new_tokens=3, logprobs=0)
    assert [r.logprobs for r in results] == [TokenScores([-500.0 * r - 0.5 * k for k in range(3)], [r + 1] * 3, [1.0] * 3) for r in range(3)]
    results = GenerationLoop(Backend(3), 3, 10_000, 1000, 16).run(PROMPTS, Sampler(3), max_new_tokens=3)
    assert all(r.logprobs is None for r in results)


class Broken:
    """Numbers on a device that has failed: reading them raises."""

    def tolist(self):
        raise RuntimeError("the reader's error")


@pytest.mark.parametrize("fails", ["decode", "read_tokens", "token_logprobs"])
def test_a_step_that_fails_is_what_is_raised(fails):
    """Log probabilities of the steps before it are not read behind a failure: the step's own error reaches the caller, and the slots
    are given back."""
    be, smp = Backend(3), Sampler(3)
    works, calls = getattr(be, fails), []
    be.token_logprobs = lambda *args: SimpleNamespace(**dict.fromkeys(("logprob", "rank", "entropy", "top_ids", "top_logprobs"), Broken()))

    def step(*args):
        calls.append(args)
        if len(calls) == 2:
            raise RuntimeError("the step's error")
        return (be.__class__.token_logprobs(be, *args) if fails == "token_logprobs" else works(*args))

    setattr(be, fails, step)
    with pytest.raises(RuntimeError, match="the step's error"):
        GenerationLoop(be, 3, 10_000, 1000, 16).run(PROMPTS, smp, max_new_tokens=4, logprobs=1)
    assert sorted(be.free) == [0, 1, 2]


@pytest.mark.parametrize("logprobs", [None, 0, 2])
def test_requests_that_an_interrupt_keeps_from_running_have_no_log_probabilities_but_the_place_for_them(logprobs):
    """Every result of a call that asks for them has an entry per token: none for an answer without tokens."""
    import threading
    stop = threading.Event()
    loop = GenerationLoop(Backend(3), 3, 10_000, 1000, 16, interrupt=stop)
    results = loop.run(PROMPTS, Sampler(6), max_new_tokens=4, samples=2, logprobs=logprobs, on_step=lambda emitted: stop.set())
    assert [len(r.tokens) for r in results] == [1, 1, 1, 0, 0, 0] and {r.finish_reason for r in results} == {"interrupted"}
    if logprobs is None:
        assert all(r.logprobs is None for r in results)
    else:
        assert [len(r.logprobs.logprobs) for r in results] == [1, 1, 1, 0, 0, 0]
