"""When a step attends over shared pages once for all its sequences: the rule beside what was measured, and steps that outlive the choice."""
import pytest

from llmplayer_b200.cache.sequence_cache import KVRequest
from llmplayer_b200.kernels import ops
from test_forked_slots import engine_on_the_host, step

# Heads of 64 / 128, sequences, shared pages, own pages, new tokens: us per layer without and with the shared form (B200, through the engine, 8 key heads).
MEASURED = [
    (64, 8, 128, 4, 1, 61, 59), (64, 8, 128, 64, 1, 70, 94), (64, 8, 128, 200, 1, 90, 199), (64, 2, 512, 4, 1, 61, 71), (64, 2, 512, 200, 1, 68, 198),
    (64, 64, 8, 0, 1, 60, 61), (64, 64, 16, 0, 1, 68, 63), (64, 64, 16, 200, 1, 329, 313), (64, 32, 128, 64, 1, 158, 114), (64, 16, 512, 64, 1, 211, 143),
    (64, 4, 128, 200, 1, 66, 198), (128, 8, 128, 4, 1, 136, 114), (128, 8, 128, 64, 1, 153, 165), (128, 8, 128, 200, 1, 190, 297), (128, 2, 512, 4, 1, 139, 131),
    (128, 2, 512, 200, 1, 151, 300), (128, 4, 512, 200, 1, 190, 310), (128, 64, 16, 16, 1, 190, 168), (128, 16, 16, 64, 1, 150, 171), (128, 16, 64, 0, 1, 138, 113),
    (64, 2, 16, 0, 24, 76, 61), (64, 8, 4, 0, 24, 103, 107), (128, 8, 4, 0, 24, 209, 212), (64, 60, 1, 0, 24, 242, 209), (128, 20, 64, 100, 24, 1386, 620),
    (64, 4, 8, 100, 1600, 1392, 1925), (128, 4, 16, 100, 96, 401, 584), (128, 2, 64, 100, 96, 341, 493), (128, 60, 8, 0, 96, 2012, 2210), (64, 60, 8, 0, 96, 666, 669),
    (64, 60, 64, 0, 96, 1011, 883), (64, 8, 64, 0, 400, 601, 544), (64, 8, 64, 100, 400, 943, 1071), (64, 8, 256, 100, 400, 1601, 1482), (128, 8, 256, 100, 400, 3378, 2741),
    (128, 2, 256, 16, 1600, 2617, 2016), (64, 20, 256, 0, 96, 873, 584)]


@pytest.mark.parametrize("hd,B,P,own,new,without,with_", MEASURED)
def test_the_choice_is_the_faster_one(hd, B, P, own, new, without, with_):
    """Of two forms that are within 7 % of each other either may be chosen."""
    mean = own + 1 if new == 1 else own + new / 2 / 64              # the longest sequence's last page, or what a token sees in the mean
    chosen = with_ if ops.attention_shared_pays(B, P, new, mean, 8, hd) else without
    assert chosen <= 1.07 * min(without, with_)


def test_a_single_sequence_has_nothing_to_share():
    for new in (1, 5, 500):
        assert not ops.attention_shared_pays(1, 10 ** 6, new, 0, 8, 128)


def forks(eng, count, shared, own):
    """``count`` slots on so many shared pages, each with so many of its own."""
    c = eng.cache
    a = c.acquire()
    c.reserve([a], [shared * 64])
    c.commit([a], [shared * 64])
    slots = [a] + eng.fork(a, count - 1)
    c.reserve(slots, [own * 64] * count)
    c.commit(slots, [own * 64] * count)
    return slots


@pytest.mark.parametrize("own,used", [(0, 128), (4, 128), (64, 0), (250, 0)])
def test_the_engine_weighs_own_pages(own, used):
    eng = engine_on_the_host(max_slots=8, pages=2600, requests=(KVRequest(8, 64),))
    slots = forks(eng, 8, 128, own)
    step(eng, slots)
    assert eng.model.seen[-1][3] == [used]
    eng.step([(s, [1] * 300) for s in slots], [[]] * 8)             # longer runs: their own keys count twice
    assert eng.model.seen[-1][3] == [128 if own < 50 else 0]


def test_a_choice_ends_when_the_own_pages_have_grown():
    """Step by step, and for whoever asks whether the next step continues the last (the native loop)."""
    eng = engine_on_the_host(max_slots=8, pages=2600, requests=(KVRequest(8, 64),))
    reach = int(ops.attention_shared_reach(8, 128, 8, 64))
    slots = forks(eng, 8, 128, reach - 1)
    step(eng, slots)
    ctx = eng._last_ctx
    assert ctx.shared_pages == [128]
    for _ in range(63):
        step(eng, slots)
        assert eng._last_ctx is ctx
    assert eng._continue([(s, [1]) for s in slots], [[0]] * 8, advance=False) is None
    for _ in range(3):
        step(eng, slots)
        assert eng._last_ctx is not ctx and eng._last_ctx.shared_pages == [0]
    ctx = eng._last_ctx
    step(eng, slots)
    assert eng._last_ctx is ctx


def test_a_large_batch_keeps_its_choice():
    eng = engine_on_the_host(max_slots=64, pages=20000, requests=(KVRequest(8, 128),))
    slots = forks(eng, 64, 32, 250)
    step(eng, slots)
    assert eng._last_ctx.shared_pages == [32] and eng._last_ctx.shared_until == float("inf")


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["step", "decode"])
def test_a_decode_goes_on_over_the_end_of_a_choice(tmp_path, monkeypatch, way):
    """Against the plain implementation before and behind the length up to which shared pages are attended over once."""
    import helpers
    from helpers import make_model, plain_logits, random_tokens
    from llmplayer_b200 import Engine, SamplerConfig
    from llmplayer_b200.sampling.sampler import SequenceSampler
    monkeypatch.setattr(ops, "SHARED_PAGES_SINGLE", 1)
    model_dir = make_model(tmp_path, "D")
    eng = Engine.load(model_dir, context_length=512, max_batch=4)
    vocab, B = eng.vocab_size, 4
    until = 64 * (2 + int(ops.attention_shared_reach(B, 2, 2, 64)))
    assert until == 384
    a = eng.acquire()
    prompt = random_tokens(130, vocab, seed=1)
    eng.step([(a, prompt)], [[]])
    slots = [a] + eng.fork(a, B - 1)
    told = [prompt + random_tokens(until - 12 - 130 - i, vocab, seed=i) for i in range(B)]
    eng.step([(s, t[130:]) for s, t in zip(slots, told)], [[]] * B)
    samplers = [SequenceSampler(SamplerConfig.greedy()) for _ in slots]

    def compare(what):
        new = [random_tokens(1, vocab, seed=100 + len(t)) for t in told]
        logits = eng.step(list(zip(slots, new)), [[0]] * B).cpu()
        for t, n, row in zip(told, new, logits):
            t += n
            helpers.assert_close(row[None], plain_logits(model_dir, t, rows=[len(t) - 1]), "bfloat16", what, "D")

    compare("a choice of shared pages, before its end")
    assert eng._last_ctx.shared_pages == [2]
    if way == "step":
        for _ in range(20):
            compare("a choice of shared pages, over its end")
    else:
        done, entries = 0, [(s, 3 + i) for i, s in enumerate(slots)]
        for (_, t), seq in zip(entries, told):
            seq.append(t)
        while done < 24:
            chosen = eng.decode_steps(entries, samplers, quiet=[100] * B, stops=[()] * B, max_steps=4)
            done += len(chosen)
            for seq, column in zip(told, zip(*chosen)):
                seq += list(column)
            entries = [(s, seq[-1]) for s, seq in zip(slots, told)]
        for seq in told:
            seq.pop()
        compare("a choice of shared pages, over its end")
    assert eng._last_ctx.shared_pages == [0] and max(map(len, told)) > until
    eng.check()


@pytest.mark.gpu
def test_which_groups_can_be_attended_over_once(tmp_path):
    """The bfloat16 form of a plain design; not float32, and not what the kernel is not built for (scores with windows, caps or biases; states)."""
    import dopuvik_helpers
    import ramupel_helpers
    from helpers import make_model
    from llmplayer_b200 import Engine

    def groups(eng):
        found = eng.model.groups_sharing_pages(eng.cache)
        assert len(found) == len(eng.cache.groups)
        return found

    assert groups(Engine.load(make_model(tmp_path / "a", "D"), context_length=128, max_batch=2)) == [True]
    assert groups(Engine.load(make_model(tmp_path / "b", "D", dtype="float32"), dtype="float32", context_length=128, max_batch=2)) == [False]
    for kit, name in ((ramupel_helpers, "small"), (dopuvik_helpers, sorted(dopuvik_helpers.CONFIGS)[0])):
        eng = Engine.load(kit.make_model(tmp_path, name, "bfloat16"), max_tokens=512, max_slots=2)
        for found, group in zip(groups(eng), eng.cache.groups):
            assert not found or (group.request.window is None and group.request.head_dim in (64, 128))
