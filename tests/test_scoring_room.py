"""Scored continuations in a cache with little room: which slots and pages are free changes how they are run, not what they are scored with."""
import random
from types import SimpleNamespace

import pytest
import torch

from llmplayer_b200.cache.pages import PAGE_SIZE
from llmplayer_b200.cache.sequence_cache import KVRequest
from llmplayer_b200.engine import scoring
from llmplayer_b200.engine.engine import Engine
from llmplayer_b200.engine.scoring import TokenLogprob
from llmplayer_b200.errors import CacheFull

VOCAB = 50


def told(tokens):
    """A number that says which tokens came before."""
    h = 7
    for t in tokens:
        h = (h * 31 + t + 1) % 1000003
    return float(h)


class Remembering:
    """A model that keeps its tokens in the cache's pages and answers with a number of those that its page table leads to."""
    capture_safe = False

    def __init__(self):
        self.layout = SimpleNamespace(head=SimpleNamespace(vocab_size=VOCAB))
        self.tokens_run = 0

    def cache_requests(self):
        return [KVRequest(1, 16)]

    def groups_sharing_pages(self, cache):
        return [True]

    def forward(self, ctx, cache, rows, logits):
        store = cache.groups[0].storage[0][:, 0, 0, :, 0]                      # [page, place]
        table, ids, positions = ctx.page_tables[0].tolist(), ctx.seq_ids.tolist(), ctx.positions.tolist()
        self.tokens_run += len(ids)
        for b, p, t in zip(ids, positions, ctx.tokens.tolist()):
            store[table[b][p // PAGE_SIZE], p % PAGE_SIZE] = t
        for row, at in zip(logits, rows.tolist()):
            row[0] = told(int(store[table[ids[at]][p // PAGE_SIZE], p % PAGE_SIZE]) for p in range(positions[at] + 1))


def engine_with(max_slots, pages):
    runtime = SimpleNamespace(device=torch.device("cpu"), dtype="float32", kernels="", kv_dtype=torch.float32, fast=False)
    eng = Engine(None, Remembering(), runtime, max_tokens=64 * pages, max_slots=max_slots, context_length=64 * pages,
                 options=SimpleNamespace(profile=False, graphs=False, host_loop=False))
    eng.token_logprobs = lambda logits, tokens, top: [TokenLogprob(t, float(row[0]), 0.0, 0) for t, row in zip(tokens, logits)]
    eng.check = lambda: None
    return eng


@pytest.mark.parametrize("max_slots,pages", [(1, 5), (1, 20), (2, 4), (2, 5), (2, 6), (3, 20), (9, 7), (9, 40)])
@pytest.mark.parametrize("length", [1, 2, 64, 65, 130, 150])
def test_whatever_room_there_is(monkeypatch, max_slots, pages, length):
    rng = random.Random(length)
    prompt = [rng.randrange(VOCAB) for _ in range(length)]
    conts = [[rng.randrange(VOCAB) for _ in range(n)] for n in (4, 1, 0, 90, 17, 33, 2)]
    want = [[told(prompt + c[:i]) for i in range(len(c))] for c in conts]
    for most in (1 << 30, 4 * VOCAB * 30):               # all at once, and in pieces
        with monkeypatch.context() as m:
            m.setattr(scoring, "SCORE_LOGITS_BYTES", most)
            eng = engine_with(max_slots, pages)
            got = eng.score(prompt, conts)
        assert [s.token_ids for s in got] == conts and [[t.logprob for t in s.tokens] for s in got] == want
        assert eng.cache.slots.num_held == 0 and eng.cache.free_pages() == [pages]


def test_the_prompt_runs_once_where_there_is_room():
    eng = engine_with(5, 40)
    eng.score([1] * 150, [[2] * 10] * 6)
    assert eng.model.tokens_run == 149 + 60


def test_one_slot_left_beside_held_ones():
    eng = engine_with(3, 40)
    kept = [eng.acquire(), eng.acquire()]
    eng.step([(s, [5] * 70) for s in kept], [[]] * 2)
    got = eng.score([1, 2, 3], [[4, 5], [6]])
    assert [[t.logprob for t in s.tokens] for s in got] == [[told([1, 2, 3]), told([1, 2, 3, 4])], [told([1, 2, 3])]]
    assert eng.cache.slots.num_held == 2


def test_what_does_not_fit_at_all_is_refused_and_nothing_stays_held():
    eng = engine_with(2, 4)
    kept = eng.acquire()
    eng.step([(kept, [5] * 100)], [[]])
    with pytest.raises(CacheFull):
        eng.score([1] * 120, [[2] * 30, [3] * 30])
    assert eng.cache.slots.num_held == 1 and eng.cache.free_pages() == [2]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_slot_scores_as_several_do(tmp_path, dtype):
    import helpers
    from helpers import make_model, random_tokens, tolerance
    model_dir = make_model(tmp_path, "D", dtype=dtype)
    prompt = random_tokens(140, helpers.TINY_D["vocab_size"], seed=4)
    conts = [random_tokens(n, helpers.TINY_D["vocab_size"], seed=n) for n in (5, 70, 1, 0, 20)]
    scores = []
    for slots in (1, 2, 6):
        eng = Engine.load(model_dir, dtype=dtype, context_length=512, max_batch=2, max_slots=slots)
        scores.append(eng.score(prompt, conts, top=2))
        assert eng.cache.slots.num_held == 0
        eng.close()
    # each engine's logits are within the configuration's bound of the plain implementation's, whose largest are below 20
    slack = 4 * tolerance(dtype, "D") * 20
    for other in scores[1:]:
        for a, b in zip(scores[0], other):
            assert a.token_ids == b.token_ids and all(abs(x.logprob - y.logprob) <= slack for x, y in zip(a.tokens, b.tokens))
