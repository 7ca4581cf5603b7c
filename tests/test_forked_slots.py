"""Slots that are released and forked again between the steps of a decode: a step runs on the pages that its slots hold now."""
import random
from types import SimpleNamespace

import pytest
import torch

import helpers
from helpers import make_model, plain_logits, random_tokens
from llmplayer_b200.cache.pages import PAGE_SIZE
from llmplayer_b200.cache.sequence_cache import KVRequest
from llmplayer_b200.engine.engine import Engine

VOCAB = 50


class Recorder:
    """A model that keeps what each step was told, and computes nothing."""
    capture_safe = False

    def __init__(self, requests):
        self.requests, self.seen, self.shares = requests, [], True
        self.layout = SimpleNamespace(head=SimpleNamespace(vocab_size=VOCAB))

    def cache_requests(self):
        return self.requests

    def groups_sharing_pages(self, cache):
        return [self.shares] * len(cache.groups)

    def forward(self, ctx, cache, rows, logits):
        self.seen.append(([t.tolist() for t in ctx.page_tables], ctx.kv_len.tolist(), ctx.slots.tolist(), ctx.shared_pages))


def engine_on_the_host(max_slots=6, pages=40, requests=(KVRequest(1, 16),)):
    runtime = SimpleNamespace(device=torch.device("cpu"), dtype="float32", kernels="", kv_dtype=torch.float32, fast=False)
    return Engine(None, Recorder(list(requests)), runtime, max_tokens=64 * pages, max_slots=max_slots, context_length=64 * pages,
                  options=SimpleNamespace(profile=False, graphs=False, host_loop=False))


def step(eng, slots, ahead=False):
    """One token for each slot; the step must have been told the cache's own tables and lengths."""
    eng.step([(s, [1]) for s in slots], [[0]] * len(slots))
    tables, lengths, told, shared = eng.model.seen[-1]
    assert told == list(slots) and lengths == [eng.length(s) for s in slots]
    for group, rows in zip(eng.cache.groups, tables):
        for s, row in zip(slots, rows):
            used = group.pages.table(s)[:-(-eng.length(s) // PAGE_SIZE)]
            # pages given back behind a window are read by no one: their entries may be what they were
            assert all(page == mine for page, mine in zip(row, used) if mine >= 0), (s, row, used)
    for n, rows in zip(shared, tables):
        assert all(row[:n] == rows[0][:n] for row in rows)
    if ahead:
        eng._prepare_continue()             # as sampling does while the device is busy


@pytest.mark.parametrize("ahead", [False, True])
@pytest.mark.parametrize("length", [5, 64, 100, 199])
def test_a_slot_released_and_forked_again_between_two_steps(length, ahead):
    eng = engine_on_the_host()
    a = eng.acquire()
    eng.step([(a, [1] * length)], [[]])
    b, = eng.fork(a, 1)
    for _ in range(75):                     # past the end of a page
        step(eng, [a, b], ahead)
    eng.release(b)
    c, = eng.fork(a, 1)
    assert c == b and eng._continue([(a, [1]), (c, [1])], [[0], [0]], advance=False) is None      # the native loop asks this way
    for _ in range(70):
        step(eng, [a, c], ahead)


@pytest.mark.parametrize("ahead", [False, True])
def test_both_slots_from_a_third(ahead):
    eng = engine_on_the_host()
    a = eng.acquire()
    eng.step([(a, [1] * 90)], [[]])
    b, c = eng.fork(a, 2)
    for _ in range(40):
        step(eng, [a, b, c], ahead)
    eng.release(c)
    eng.release(b)
    assert eng.fork(a, 2) == [b, c]
    for _ in range(30):
        step(eng, [a, b, c], ahead)


@pytest.mark.parametrize("seed", range(6))
def test_steps_between_random_forks_and_releases(seed):
    rng = random.Random(seed)
    eng = engine_on_the_host(max_slots=5, pages=60, requests=(KVRequest(1, 16), KVRequest(2, 16, window=100)))
    held = [eng.acquire()]
    eng.step([(held[0], [1] * rng.randint(1, 150))], [[]])
    for _ in range(150):
        for _ in range(rng.randint(0, 3)):
            if len(held) > 1 and rng.random() < 0.5:
                eng.release(held.pop(rng.randrange(len(held))))
            elif len(held) < 5:
                held += eng.fork(rng.choice(held), 1)
        held.sort()
        for _ in range(rng.randint(1, 3)):
            step(eng, held, ahead=rng.random() < 0.5)


def test_a_step_of_the_same_sequences_still_continues():
    eng = engine_on_the_host()
    a = eng.acquire()
    eng.step([(a, [1] * 70)], [[]])
    b, = eng.fork(a, 1)
    step(eng, [a, b])
    ctx = eng._last_ctx
    other, = eng.fork(a, 1)                 # neither slot of the step is another sequence by that
    for _ in range(20):
        step(eng, [a, b])
        assert eng._last_ctx is ctx


def two_on_a_prompt(eng, length):
    """The description of a step of two forks of a prompt, which are released again."""
    a = eng.acquire()
    eng.step([(a, [1] * length)], [[]])
    slots = [a] + eng.fork(a, 1)
    step(eng, slots)
    ctx = eng._last_ctx
    for s in slots:
        eng.release(s)
    return ctx


@pytest.mark.parametrize("shares,single", [(False, 1), (True, 10 ** 9), (True, 1)])
def test_a_graph_depends_on_shared_pages_only_where_they_are_attended_over_once(monkeypatch, shares, single):
    from llmplayer_b200.kernels import ops
    monkeypatch.setattr(ops, "SHARED_PAGES_SINGLE", single)
    eng = engine_on_the_host(requests=(KVRequest(8, 64),))
    eng.model.shares = shares
    shapes = {two_on_a_prompt(eng, length).table_shapes for length in (70, 130, 200, 260)}
    assert shapes == ({((8, n),) for n in (1, 2, 3, 4)} if shares and single == 1 else {((8, 0),)})


@pytest.mark.gpu
@pytest.mark.parametrize("everywhere,graphs", [(False, 1), (True, 3)])
def test_graphs_of_forks_of_prompts_of_several_lengths(tmp_path, monkeypatch, everywhere, graphs):
    from llmplayer_b200.kernels import ops
    if everywhere:
        monkeypatch.setattr(ops, "SHARED_PAGES_SINGLE", 1)
    eng = Engine.load(make_model(tmp_path, "D"), context_length=512, max_batch=4)        # (engines in float32 capture nothing)
    for length in (130, 200, 260, 140):
        a = eng.acquire()
        eng.step([(a, random_tokens(length, eng.vocab_size, seed=length))], [[]])
        slots = [a] + eng.fork(a, 2)
        for _ in range(3):
            eng.step([(s, [3 + s]) for s in slots], [[0]] * 3)
        for s in slots:
            eng.release(s)
    assert len({shapes for _, shapes, _, _ in eng._graphs}) == graphs          # (the buffer of the step's integers moves as it grows, too)
    eng.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("way", ["step", "decode", "drawn"])
def test_the_better_of_two_is_kept_and_forked_again(tmp_path, dtype, way):
    """Two sequences side by side past the end of a page; one is dropped, the other forked in its place, and both go on: against the plain
    implementation. Stepped directly (captured and replayed), with the choice of a token in between, and from the native loop."""
    from llmplayer_b200 import SamplerConfig
    from llmplayer_b200.sampling.sampler import SequenceSampler
    model_dir = make_model(tmp_path, "D", dtype=dtype)
    vocab = helpers.TINY_D["vocab_size"]
    eng = Engine.load(model_dir, dtype=dtype, context_length=512, max_batch=4)
    a = eng.acquire()
    told = {a: random_tokens(150, vocab, seed=2)}
    eng.step([(a, told[a])], [[]])
    b, = eng.fork(a, 1)
    told[b] = list(told[a])
    samplers = [SequenceSampler(SamplerConfig.greedy()) for _ in range(2)]

    def go_on(steps, seed):
        if way == "decode":
            entries = [(s, random_tokens(1, vocab, seed=seed + s)[0]) for s in (a, b)]
            for s, t in entries:
                told[s].append(t)
            done = 0
            while done < steps:
                chosen = eng.decode_steps(entries, samplers, quiet=[100, 100], stops=[(), ()], max_steps=min(16, steps - done))
                done += len(chosen)
                for s, column in zip((a, b), zip(*chosen)):
                    told[s] += list(column)
                entries = [(s, told[s][-1]) for s in (a, b)]
            for s in (a, b):
                told[s].pop()                          # chosen last, fed to nobody yet
        else:
            for i in range(steps):
                pieces = [random_tokens(1, vocab, seed=seed + 7 * i + s) for s in (a, b)]
                logits = eng.step(list(zip((a, b), pieces)), [[0], [0]])
                for s, p in zip((a, b), pieces):
                    told[s] += p
                if way == "drawn":
                    eng.sample(logits, [0, 1], samplers)
        assert [eng.length(s) for s in (a, b)] == [len(told[s]) for s in (a, b)]

    go_on(70, 100)
    eng.release(b)
    assert eng.fork(a, 1) == [b]
    told[b] = list(told[a])
    go_on(60, 900)
    last = [random_tokens(1, vocab, seed=5 + s) for s in (a, b)]
    logits = eng.step([(a, last[0]), (b, last[1])], [[0], [0]]).cpu()
    for s, p, row in zip((a, b), last, logits):
        ref = plain_logits(model_dir, told[s] + p, rows=[len(told[s])])
        helpers.assert_close(row[None], ref, dtype, f"forked again, {way}", "D")
    for s in (a, b):
        eng.release(s)
    eng.check()
    assert eng.cache.free_pages() == [eng.cache.num_pages]


def test_a_fork_whose_copies_fail_leaves_nothing_held(monkeypatch):
    eng = engine_on_the_host(requests=(KVRequest(1, 16), KVRequest(2, 16)))
    a = eng.acquire()
    eng.step([(a, [1] * 100)], [[]])
    before = (eng.cache.free_pages(), eng.cache.slots.num_free, list(eng.cache.groups[0].pages.table(a)))

    class Fails:
        is_cuda = False

        def __getitem__(self, at):
            raise RuntimeError("out of memory")

    for group in eng.cache.groups:                      # in the first group, and in the second when the first has been copied
        with monkeypatch.context() as m:
            m.setattr(group, "storage", Fails())
            with pytest.raises(RuntimeError, match="out of memory"):
                eng.fork(a, 2)
        assert (eng.cache.free_pages(), eng.cache.slots.num_free, eng.cache.groups[0].pages.table(a)) == before
    b, = eng.fork(a, 1)
    eng.release(a)
    eng.release(b)
    assert eng.cache.free_pages() == [40, 40] and eng.cache.slots.num_held == 0


@pytest.mark.parametrize("samples", [0, -3])
def test_the_command_line_refuses_numbers_of_samples_below_one(monkeypatch, samples):
    from llmplayer_b200 import cli, engine
    from llmplayer_b200.errors import RequestError
    monkeypatch.setattr(engine.Engine, "load", classmethod(lambda cls, *args, **kwargs: engine_on_the_host()))
    with pytest.raises(RequestError, match="samples"):
        cli.run(["some_model", "--prompt", "1 2 3", "--samples", str(samples)])


def test_the_command_line_counts_a_prompt_once_and_all_prompts_samples(monkeypatch, capsys):
    from llmplayer_b200 import cli, engine
    from llmplayer_b200.engine.generate import GenerationResponse, GenerationStats

    class Counting:
        def generate_samples(self, prompt, samples, *args, **kwargs):
            # 10 tokens of each sample at 100 or 300 tokens a second
            ms = samples * 10 / (100 if prompt == [1, 2, 3] else 300) * 1e3
            self.last_generation_stats = GenerationStats(generated_tokens=10 * samples, decode_ms=ms)
            return [GenerationResponse([5] * 10, len(prompt), "length") for _ in range(samples)]

        def generate(self, prompts, *args, **kwargs):
            self.last_generation_stats = GenerationStats(generated_tokens=10 * len(prompts), decode_ms=200.0)
            return [GenerationResponse([5] * 10, len(p), "length") for p in prompts]

    monkeypatch.setattr(engine.Engine, "load", classmethod(lambda cls, *args, **kwargs: Counting()))
    cli.run(["some_model", "--prompt", "1 2 3", "--prompt", "4 5", "--samples", "3"])
    out = capsys.readouterr().out
    assert "Tokens: 5 prompt + 60 generated" in out and "(150.0 tok/s)" in out
    cli.run(["some_model", "--prompt", "1 2 3", "--prompt", "4 5"])
    out = capsys.readouterr().out
    assert "Tokens: 5 prompt + 20 generated" in out and "(100.0 tok/s)" in out
