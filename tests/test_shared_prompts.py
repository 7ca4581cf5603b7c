"""One prompt continued many times: forked slots, steps over shared pages, given tokens scored, samples drawn side by side."""
import math
import random

import pytest
import torch

import botuvik_helpers
import dopuvik_helpers
import helpers
import plain_llama as P
import ramupel_helpers
import vomotar_helpers
from helpers import check_error, make_model, plain_logits, random_tokens, relative_error, tolerance
from llmplayer_b200.cache.pages import PAGE_SIZE, PageMap
from llmplayer_b200.cache.sequence_cache import KVRequest, RowsRequest, SequenceCache, StateRequest
from llmplayer_b200.cli import CLIOptions
from llmplayer_b200.engine.generate import GenerationLoop, GenerationRequest
from llmplayer_b200.engine.scoring import TokenLogprob
from llmplayer_b200.errors import CacheError, CacheFull, RequestError
from llmplayer_b200.sampling.params import SamplerConfig


# ------------------------------------------------------------------------------------------------ bookkeeping, on the CPU
def test_a_fork_shares_full_pages_and_copies_the_last():
    pm = PageMap(10)
    pm.open(0)
    pm.extend(0, 3 * PAGE_SIZE + 5)
    a, b = pm.fork(0, 1, 3 * PAGE_SIZE + 5)
    assert pm.table(1) == pm.table(0)[:3] + [b] and a == pm.table(0)[3] and b != a
    assert pm.fork(1, 2, 2 * PAGE_SIZE) is None and pm.table(2) == pm.table(0)[:2]
    assert pm.pool.num_held == 5
    pm.close(0)
    assert pm.pool.num_held == 4                    # its last page was its own
    pm.close(1)
    assert pm.pool.num_held == 2                    # slot 2 still holds two
    with pytest.raises(CacheError, match="already"):
        pm.fork(2, 2, 1)
    pm.close(2)
    assert pm.pool.num_free == 10


def test_pages_behind_a_window_go_back_with_their_last_holder():
    pm = PageMap(12, window=64)
    pm.open(0)
    pm.extend(0, 200)
    pm.fork(0, 1, 200)
    pm.extend(0, 260)
    pm.trim(0, 260)
    held = pm.pool.num_held
    assert pm.table(0)[0] == -1 and pm.table(1)[0] >= 0
    pm.extend(1, 260)
    pm.trim(1, 260)
    assert pm.pool.num_held == held + 1 - 3         # a page more, three shared ones less
    pm.close(0)
    pm.close(1)
    assert pm.pool.num_free == 12


def make_cache(max_tokens=1024, max_slots=8):
    requests = [KVRequest(2, 16), RowsRequest(24), KVRequest(2, 16, window=64), StateRequest((3,)), (StateRequest((2, 2)), StateRequest((5,)))]
    return SequenceCache(requests, max_tokens=max_tokens, max_slots=max_slots, kv_dtype=torch.float32, device="cpu")


@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 200])
def test_forks_hold_what_their_parent_holds(length):
    c = make_cache()
    a = c.acquire()
    if length:
        c.reserve([a], [length])
        c.commit([a], [length])
    g = torch.Generator().manual_seed(length)
    for group in c.groups:
        group.storage.copy_(torch.randn(group.storage.shape, generator=g))
    for rows in (c.view(3).rows, *c.view(4).blocks):
        rows[a] = torch.randn(rows[a].shape, generator=g)
    forks = c.fork(a, 3)
    assert [c.length(s) for s in forks] == [length] * 3
    for s in forks:
        for group in c.groups:
            for block, (mine, theirs) in enumerate(zip(group.pages.table(s), group.pages.table(a))):
                assert (mine == theirs) == (block < length // PAGE_SIZE)
                assert theirs < 0 or torch.equal(group.storage[:, mine], group.storage[:, theirs])
        for rows in (c.view(3).rows, *c.view(4).blocks):
            assert torch.equal(rows[s], rows[a])
    assert c.shared_pages([a] + forks) == [length // PAGE_SIZE, length // PAGE_SIZE, 0] and c.shared_pages([a]) == [0, 0, 0]
    other = c.acquire()
    c.reserve([other], [200])
    c.commit([other], [200])
    assert c.shared_pages([a, other]) == [0, 0, 0]
    for s in [a, other] + forks:
        c.release(s)
    assert c.free_pages() == [16] * 3 and c.slots.num_free == 8


def test_a_fork_that_does_not_fit_changes_nothing():
    c = make_cache(max_tokens=64 * 6, max_slots=4)
    a = c.acquire()
    c.reserve([a], [4 * 64 + 1])
    c.commit([a], [4 * 64 + 1])
    before = c.free_pages()
    with pytest.raises(CacheFull, match="slots"):
        c.fork(a, 4)
    with pytest.raises(CacheFull, match="pages|page"):
        c.fork(a, 2)
    with pytest.raises(CacheError):
        c.fork(a, -1)
    with pytest.raises(CacheError):
        c.fork(3, 1)
    assert c.free_pages() == before and c.slots.num_held == 1 and c.fork(a, 0) == []


def test_no_slot_or_page_is_lost_under_forks():
    rng = random.Random(1)
    c = make_cache(max_tokens=64 * 40, max_slots=12)
    held = set()
    for _ in range(3000):
        op = rng.random()
        try:
            if op < 0.15:
                held.add(c.acquire())
            elif op < 0.35 and held:
                held.update(c.fork(rng.choice(sorted(held)), rng.randint(0, 3)))
            elif op < 0.6 and held:
                s = rng.choice(sorted(held))
                c.release(s)
                held.remove(s)
            elif held:
                s = rng.choice(sorted(held))
                n = rng.randint(1, 90)
                c.reserve([s], [n])
                c.commit([s], [n])
        except CacheFull:
            pass
        for group in c.groups:
            owners = {}
            for s in held:
                table = group.pages.table(s)
                assert len(table) >= -(-c.length(s) // PAGE_SIZE)
                for block, page in enumerate(table):
                    if page >= 0:
                        owners.setdefault(page, []).append((s, block))
            assert group.pages.pool.num_held == len(owners)
            for page, by in owners.items():        # a page that several hold is full for all of them, at the same place
                assert len({block for _, block in by}) == 1
                if len(by) > 1:
                    assert all((block + 1) * PAGE_SIZE <= c.length(s) for s, block in by)
    for s in sorted(held):
        c.release(s)
    assert c.free_pages() == [40] * 3


def test_common_pages_are_found_under_random_forks():
    rng = random.Random(3)
    c = make_cache(max_tokens=64 * 200, max_slots=30)
    held = [c.acquire()]
    for _ in range(1500):
        op, s = rng.random(), rng.choice(held)
        try:
            if op < 0.1:
                held.append(c.acquire())
            elif op < 0.4:
                held += c.fork(s, rng.randint(0, 3))
            elif op < 0.55 and len(held) > 1:
                held.remove(s)
                c.release(s)
            else:
                n = rng.randint(1, 150)
                c.reserve([s], [n])
                c.commit([s], [n])
        except CacheFull:
            for s in held[len(held) // 2:]:
                c.release(s)
            held = held[:len(held) // 2]
        slots = rng.sample(held, rng.randint(1, len(held)))
        shortest = min(c.length(s) for s in slots) // PAGE_SIZE
        for g, found in enumerate(c.shared_pages(slots)):
            tables = [c.groups[g].pages.table(s) for s in slots]
            if len(slots) < 2 or c.groups[g].pages.window is not None:
                assert found == 0
                continue
            want = 0
            while want < shortest and len({t[want] for t in tables}) == 1:
                want += 1
            assert found == want


class ScriptedBackend:
    """Chooses token 10 * slot + step; says so with a log probability."""

    def __init__(self):
        self.free, self.steps, self.forked = list(range(20)), [], []

    def acquire(self):
        return self.free.pop(0)

    def release(self, slot):
        self.free.append(slot)

    def fits(self, counts):
        return True

    def fork(self, slot, count):
        self.forked.append((slot, count))
        return [self.acquire() for _ in range(count)]

    def step(self, entries, want):
        self.steps.append([(s, list(t)) for s, t in entries])
        return torch.arange(float(sum(len(w) for w in want)))[:, None].expand(-1, 4)

    def sample(self, logits, rows, samplers):
        return [100 + len(self.steps) * 10 + i for i in range(len(rows))]

    def token_logprobs(self, logits, tokens, top):
        assert logits.shape[0] == len(tokens)
        return [TokenLogprob(t, -float(t), 0.5, 0, [(k, -1.0) for k in range(top)]) for t in tokens]


def test_the_loop_reports_log_probabilities_of_those_who_ask():
    be = ScriptedBackend()
    loop = GenerationLoop(be, max_batch=4, context_length=100)
    out = loop.run([GenerationRequest([1, 2], max_tokens=3, logprobs=2), GenerationRequest([3], max_tokens=2), GenerationRequest([4], max_tokens=3, logprobs=0,
                                                                                                                         stop_token_ids=[122])])
    assert [r.token_ids for r in out] == [[110, 120, 130], [111, 121], [112]]
    assert [t.token_id for t in out[0].logprobs] == out[0].token_ids and [len(t.top) for t in out[0].logprobs] == [2] * 3
    assert out[1].logprobs is None and [t.logprob for t in out[2].logprobs] == [-112.0] and out[2].logprobs[0].top == []
    assert sorted(be.free) == list(range(20))


def test_the_loop_runs_one_prompt_once():
    be = ScriptedBackend()
    loop = GenerationLoop(be, max_batch=3, context_length=100)
    out = loop.run([GenerationRequest([5, 6, 7], max_tokens=2, logprobs=1) for _ in range(3)], one_prompt=True)
    assert be.steps[0] == [(0, [5, 6, 7])] and be.forked == [(0, 2)] and len(be.steps[1]) == 3
    assert [r.token_ids for r in out] == [[110, 120], [111, 121], [112, 122]] and loop.stats.prompt_tokens == 3
    assert sorted(be.free) == list(range(20))


@pytest.mark.parametrize("logprobs", [-1, 33])
def test_lists_of_a_length_that_is_not_offered_are_refused(logprobs):
    be = ScriptedBackend()
    loop = GenerationLoop(be, max_batch=4, context_length=64)
    out = loop.run([GenerationRequest([1, 2], max_tokens=3, logprobs=logprobs), GenerationRequest([3], max_tokens=2, logprobs=1)])
    assert out[0].finish_reason == "error" and "most likely" in out[0].error and out[0].token_ids == []
    assert len(out[1].logprobs) == 2


@pytest.mark.parametrize("seed", [0, 5, 2 ** 63 - 1, -3, 1234567890123])
def test_first_draws_of_samples_are_spread(seed):
    from llmplayer_b200.sampling.java_random import JavaRandom
    config = SamplerConfig(seed=seed)
    assert config.for_sample(0) == config
    draws = sorted(JavaRandom(config.for_sample(i).seed).next_float() for i in range(400))
    # 400 independent uniform draws: the largest distance to the even spread exceeds 2.2 / sqrt(400) once in 8,000 times
    assert max(max((i + 1) / 400 - x, x - i / 400) for i, x in enumerate(draws)) < 0.11


def test_command_line_options():
    o = CLIOptions.parse(["x", "--samples", "5", "--logprobs", "3"])
    assert o.samples == 5 and o.logprobs == 3
    d = CLIOptions.parse(["x"])
    assert d.samples == 1 and d.logprobs is None


# ------------------------------------------------------------------------------------------------ on the GPU
def everywhere(monkeypatch):
    """Shared pages attended over together however few they are."""
    from llmplayer_b200.kernels import ops
    monkeypatch.setattr(ops, "SHARED_PAGES_SINGLE", 1)
    monkeypatch.setattr(ops, "SHARED_PAGES_SEVERAL", 1)


def spy(monkeypatch):
    from llmplayer_b200.kernels import ops
    calls, real = [], ops.attention_shared

    def counted(*args, **kwargs):
        calls.append(kwargs["shared_pages"])
        return real(*args, **kwargs)

    monkeypatch.setattr(ops, "attention_shared", counted)
    return calls


@pytest.mark.gpu
@pytest.mark.parametrize("prompt_len", [1, 64, 130, 257])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forks_go_on_like_sequences_of_their_own(tmp_path, monkeypatch, dtype, prompt_len):
    """Several tokens at once, then single ones (directly, captured and replayed), against the plain implementation."""
    from llmplayer_b200 import Engine
    everywhere(monkeypatch)
    calls = spy(monkeypatch)
    model_dir = make_model(tmp_path, "D", dtype=dtype)
    vocab = helpers.TINY_D["vocab_size"]
    prompt = random_tokens(prompt_len, vocab, seed=prompt_len)
    eng = Engine.load(model_dir, dtype=dtype, context_length=512, max_batch=8)
    parent = eng.acquire()
    eng.step([(parent, prompt)], [[]])
    slots = [parent] + eng.fork(parent, 4)
    told = [list(prompt) for _ in slots]

    def run(pieces, what):
        logits = eng.step(list(zip(slots, pieces)), [list(range(len(p))) for p in pieces]).cpu()
        at = 0
        for seq, piece in zip(told, pieces):
            seq.extend(piece)
            ref = plain_logits(model_dir, seq, rows=list(range(len(seq) - len(piece), len(seq))))
            helpers.assert_close(logits[at:at + len(piece)], ref, dtype, f"forks of {prompt_len}, {what}", "D")
            at += len(piece)

    run([random_tokens(n, vocab, seed=n + i) for i, n in enumerate((3, 70, 1, 20, 9))], "several tokens")
    for step in range(5):
        run([random_tokens(1, vocab, seed=50 * step + i) for i in range(len(slots))], f"single tokens, step {step}")
    if dtype == "bfloat16" and prompt_len >= 64:
        assert calls and set(calls) == {prompt_len // PAGE_SIZE}
    else:
        assert not calls
    for s in slots:
        eng.release(s)
    eng.check()
    assert eng.cache.free_pages() == [eng.cache.num_pages]


@pytest.mark.gpu
@pytest.mark.parametrize("kit,name,vocab_key", [(ramupel_helpers, "small", "vocab"), (botuvik_helpers, None, None), (dopuvik_helpers, None, None)])
def test_forks_of_designs_with_states_and_windows(tmp_path, monkeypatch, kit, name, vocab_key):
    """A fork of a sequence goes on as the sequence itself does (float32: recurrent states, latent rows, windows)."""
    from llmplayer_b200 import Engine
    everywhere(monkeypatch)
    name = name or sorted(kit.CONFIGS)[0]
    model_dir = kit.make_model(tmp_path, name, "float32")
    eng = Engine.load(model_dir, dtype="float32", max_tokens=2048, max_slots=6)
    prompt = random_tokens(150, eng.vocab_size, seed=3)
    more = [random_tokens(n, eng.vocab_size, seed=n) for n in (5, 1, 1, 1)]
    alone = eng.acquire()
    eng.step([(alone, prompt)], [[]])
    want = [eng.step([(alone, m)], [[len(m) - 1]]).cpu() for m in more]
    eng.release(alone)
    parent = eng.acquire()
    eng.step([(parent, prompt)], [[]])
    forks = eng.fork(parent, 2)
    noise = random_tokens(40, eng.vocab_size, seed=77)
    eng.step([(parent, noise)], [[]])                  # the parent goes elsewhere
    for m, ref in zip(more, want):
        got = eng.step([(s, m) for s in forks], [[len(m) - 1]] * 2).cpu()
        for row in got:
            # the same sums in float32, in another order at most
            check_error("forks against their parent, float32", f"{kit.__name__} {name}", relative_error(row, ref[0]), 2e-5)
    for s in [parent] + forks:
        eng.release(s)
    eng.check()


@pytest.mark.gpu
def test_long_steps_of_a_design_without_pages(tmp_path):
    """Nothing is cached but states: there is no table that a long step could describe on the device."""
    from llmplayer_b200 import Engine
    from llmplayer_b200.engine.step import StepContext
    eng = Engine.load(vomotar_helpers.make_model(tmp_path, "recurrent", "float32"), dtype="float32", max_tokens=4096, max_slots=4)
    assert eng.cache.groups == []
    prompt = random_tokens(StepContext.ON_DEVICE_ENTRIES + 76, eng.vocab_size, seed=8)
    slot, other = eng.acquire(), eng.acquire()
    got = eng.step([(slot, prompt)], [[len(prompt) - 1]]).cpu()
    for a in range(0, len(prompt), 100):
        want = eng.step([(other, prompt[a:a + 100])], [[99]]).cpu()
    # float32 sums over chunks of other lengths: two factors of 1100 terms' rounding, 2 * 1100 * 2^-24
    check_error("a long step without pages", "float32", relative_error(got[0], want[0]), 1.4e-4)
    for fork in eng.fork(slot, 2):
        eng.release(fork)
    eng.release(slot)
    eng.release(other)
    eng.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_against_the_plain_implementation(tmp_path, monkeypatch, dtype):
    from llmplayer_b200 import Engine
    from llmplayer_b200.engine import scoring
    everywhere(monkeypatch)
    model_dir = make_model(tmp_path, "D", dtype=dtype)
    vocab = helpers.TINY_D["vocab_size"]
    eng = Engine.load(model_dir, dtype=dtype, context_length=512, max_batch=6)
    for prompt_len in (1, 2, 65, 200):
        prompt = random_tokens(prompt_len, vocab, seed=prompt_len)
        conts = [random_tokens(n, vocab, seed=9 + n) for n in (4, 1, 0, 90, 17, 33, 2, 8)]
        whole = eng.score(prompt, conts, top=3)
        with monkeypatch.context() as m:               # few rows of logits per step: continuations in pieces, few at a time
            m.setattr(scoring, "SCORE_LOGITS_BYTES", 4 * vocab * 30)
            pieces = eng.score(prompt, conts, top=3)
        assert eng.cache.slots.num_held == 0 and eng.cache.free_pages() == [eng.cache.num_pages]
        for scored in (whole, pieces):
            assert [s.token_ids for s in scored] == conts
            for s, c in zip(scored, conts):
                if not c:
                    assert s.logprob == 0.0
                    continue
                rows = plain_logits(model_dir, prompt + c, rows=list(range(prompt_len - 1, prompt_len - 1 + len(c)))).double()
                slack = 2 * tolerance(dtype, "D") * float(rows.abs().max())       # a logit's bound, and the normaliser's
                lp = torch.log_softmax(rows, dim=1)
                entropy = -(lp.exp() * lp).sum(1)
                for i, t in enumerate(s.tokens):
                    assert abs(t.logprob - float(lp[i, c[i]])) <= slack
                    # |dH| <= sum p |dlp| (1 + |lp|), with |lp| averaging H
                    assert abs(t.entropy - float(entropy[i])) <= slack * (1 + float(entropy[i]))
                    better = int((lp[i] > lp[i, c[i]] + slack).sum()), int((lp[i] > lp[i, c[i]] - slack).sum())
                    assert better[0] <= t.rank <= better[1]
                    assert len(t.top) == 3 and all(abs(v - float(lp[i, k])) <= slack for k, v in t.top)
                    assert t.top[0][1] >= t.top[1][1] >= t.top[2][1] and float(lp[i].max()) - t.top[0][1] <= 2 * slack
                assert s.logprob == pytest.approx(sum(t.logprob for t in s.tokens))
    eng.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_greedy_samples_are_what_generate_gives(tmp_path, monkeypatch, dtype):
    from llmplayer_b200 import Engine, SamplerConfig
    everywhere(monkeypatch)
    model_dir = make_model(tmp_path, "D", dtype=dtype)
    vocab = helpers.TINY_D["vocab_size"]
    eng = Engine.load(model_dir, dtype=dtype, context_length=512, max_batch=6)
    prompt = random_tokens(140, vocab, seed=6)
    one = eng.generate([prompt], SamplerConfig.greedy(), max_tokens=70, stop_token_ids=())[0]
    several = eng.generate_samples(prompt, 5, SamplerConfig.greedy(), max_tokens=70, stop_token_ids=())
    assert len(several) == 5 and all(r.finish_reason == "length" and r.prompt_token_count == 140 for r in several)
    assert all(r.token_ids == several[0].token_ids for r in several)
    cfg, w = P.read_model(model_dir)
    for tokens in (one.token_ids, several[0].token_ids):
        logits = P.forward(cfg, w, prompt + tokens, dtype=torch.float64, rows=list(range(139, 209)))
        for row, tok in zip(logits, tokens):
            assert float(row[tok]) >= float(row.max()) - 2 * tolerance(dtype, "D") * float(row.abs().max())
    if dtype == "float32":
        assert one.token_ids == several[0].token_ids
    with_lp = eng.generate_samples(prompt, 3, SamplerConfig.greedy(), max_tokens=20, stop_token_ids=(), logprobs=2)
    for r in with_lp:
        assert [t.token_id for t in r.logprobs] == r.token_ids and all(t.rank == 0 and t.top[0][0] == t.token_id for t in r.logprobs)
        again = eng.score(prompt, [r.token_ids])[0]
        slack = 4 * tolerance(dtype, "D") * 20
        assert all(abs(a.logprob - b.logprob) <= slack for a, b in zip(again.tokens, r.logprobs))
    assert eng.cache.slots.num_held == 0 and eng.cache.free_pages() == [eng.cache.num_pages]
    eng.check()


@pytest.mark.gpu
def test_drawn_samples_differ_and_repeat(tmp_path, monkeypatch):
    from llmplayer_b200 import Engine, SamplerConfig
    everywhere(monkeypatch)
    calls = spy(monkeypatch)
    model_dir = make_model(tmp_path, "D")
    eng = Engine.load(model_dir, context_length=512, max_batch=9)
    prompt = random_tokens(200, helpers.TINY_D["vocab_size"], seed=8)
    config = SamplerConfig(temperature=1.0, top_k=50, top_p=0.95, seed=5)
    a = eng.generate_samples(prompt, 9, config, max_tokens=40, stop_token_ids=())
    b = eng.generate_samples(prompt, 9, config, max_tokens=40, stop_token_ids=())
    assert [r.token_ids for r in a] == [r.token_ids for r in b]
    assert len({tuple(r.token_ids) for r in a}) == 9
    assert calls and set(calls) == {200 // PAGE_SIZE}
    assert eng.cache.slots.num_held == 0


@pytest.mark.gpu
def test_refusals(tmp_path):
    from llmplayer_b200 import Engine
    model_dir = make_model(tmp_path, "A")
    eng = Engine.load(model_dir, context_length=128, max_batch=2, max_slots=2)
    for prompt, conts, top in (([], [[1]], 0), ([1], [[9999]], 0), ([-1], [[1]], 0), ([1] * 100, [[1] * 30], 0), ([1], [[1]], 33), ([1], [[1]], -1)):
        with pytest.raises(RequestError):
            eng.score(prompt, conts, top=top)
    assert eng.score([1, 2], []) == [] and eng.score([1, 2], [[]])[0].tokens == []
    for n in (0, 5):
        with pytest.raises(RequestError):
            eng.generate_samples([1, 2, 3], n, max_tokens=4)
    assert len(eng.score([1, 2, 3], [[4], [5], [6]])) == 3              # more continuations than slots: one after another
    assert eng.cache.slots.num_held == 0
    logits = torch.zeros(2, eng.vocab_size, device="cuda")
    with pytest.raises(RequestError):
        eng.token_logprobs(logits, [1])
    got = eng.token_logprobs(logits, [1, 3], top=1)
    assert [t.rank for t in got] == [1, 3] and all(abs(t.logprob + math.log(eng.vocab_size)) < 1e-6 for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
def test_a_step_described_on_the_device_is_the_same(tmp_path, seed):
    from llmplayer_b200.engine.step import SequenceStep, StepContext, Workspace
    rng = random.Random(seed)
    c = SequenceCache([KVRequest(1, 8), KVRequest(1, 8, window=70)], max_tokens=64 * 200, max_slots=20, kv_dtype=torch.float32, device="cuda")
    slots = [c.acquire()]
    c.reserve(slots, [300])
    c.commit(slots, [300])
    slots += c.fork(slots[0], rng.randint(0, 9)) + [c.acquire()][:seed % 2]
    counts = [rng.choice([1, 2, 63, 200]) for _ in slots]
    first = [c.length(s) for s in slots]
    shared = c.shared_pages(slots)
    c.reserve(slots, counts)
    steps, at = [], 0
    for s, f, n in zip(slots, first, counts):
        steps.append(SequenceStep(s, at, n, f))
        at += n
    tokens, rows = [rng.randrange(100) for _ in range(at)], [at - 1]
    tables = c.page_tables(slots)
    here = StepContext(Workspace("cuda:0"), steps, tokens, tables, rows, shared_pages=shared)
    there = StepContext(Workspace("cuda:0"), steps, tokens, tables, rows, shared_pages=shared, on_device=True)
    for name in ("tokens", "positions", "kv_len", "seq_ids", "slots", "q_start", "rows"):
        assert torch.equal(getattr(here, name), getattr(there, name)), name
    for a, b in zip(here.page_tables, there.page_tables):
        assert torch.equal(a[:, :b.shape[1]], b) and not bool(a[:, b.shape[1]:].any())
