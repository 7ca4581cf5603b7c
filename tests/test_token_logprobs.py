"""Log probabilities of given tokens, entropies, ranks and most likely tokens, against float64."""
import math

import pytest
import torch

from helpers import check_error
from llmplayer_b200.errors import KernelError
from llmplayer_b200.kernels import ops

# A log probability is x[t] - ln(sum): the difference x[t] - m is rounded once (half a step of 2^-24, relative), a term of the sum
# comes from an exponential of a rounded argument d: |d| 2^-24 off from rounding and a few steps of the exponential itself, which
# weighs exp(d): at most 4 steps in all for any d; sums of 512 partial sums of V / 512 terms add fewer than 16 half steps for the sizes
# here (random signs; the bound without that luck is V / 512 + 9). So 2^-24 * (|x - m| + 4 + 16 + the last sum's rounding |ln s| + |log p|).
STEP = 2.0 ** -24


def oracle(x, targets, top):
    x = x.double()
    R, V = x.shape
    lp = torch.log_softmax(x, dim=1)
    best, at = x.max(dim=1, keepdim=True)
    rest = torch.exp(x - best).scatter(1, at, 0.0).sum(dim=1, keepdim=True)
    lp = (x - best) - torch.log1p(rest)
    bad = torch.isnan(x).any(dim=1) | (x == math.inf).any(dim=1) | (x == -math.inf).all(dim=1)
    lp[bad] = math.nan
    p = torch.exp(lp)
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(dim=1)
    key = torch.where(torch.isnan(x), torch.full_like(x, math.inf), -x)
    order = torch.argsort(key, dim=1, stable=True)
    # -inf and no number sort alike by this key: numbers first
    for r in range(R):
        if torch.isnan(x[r]).any() and (x[r] == -math.inf).any():
            nan = torch.isnan(x[r])[order[r]]
            order[r] = torch.cat([order[r][~nan], order[r][nan]])
    place = torch.empty_like(order).scatter_(1, order, torch.arange(V).expand(R, V).contiguous())
    real = (targets >= 0) & (targets < V)
    t = targets.clamp(0, V - 1).long()[:, None]
    logprob = torch.where(real, lp.gather(1, t)[:, 0], torch.full((R,), math.nan, dtype=torch.float64))
    rank = torch.where(real, place.gather(1, t)[:, 0], torch.full((R,), -1))
    ids = order[:, :top]
    return logprob, entropy, rank, ids, lp.gather(1, ids), best[:, 0]


def call(x, targets, top):
    R = x.shape[0]
    outs = [torch.full((R,), 7.0, device="cuda"), torch.full((R,), 7.0, device="cuda"), torch.full((R,), 7, dtype=torch.int32, device="cuda"),
            torch.full((R, top), 7, dtype=torch.int32, device="cuda"), torch.full((R, top), 7.0, device="cuda")]
    ops.token_logprobs(x, targets, outs[0], outs[1], outs[2], top_ids=outs[3] if top else None, top_logprobs=outs[4] if top else None)
    return outs


def same_or_near(got, want, bound, kind, what):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    far = ~torch.isfinite(want)
    assert torch.equal(got[far & ~torch.isnan(want)], want[far & ~torch.isnan(want)]), what
    near = torch.isfinite(want)
    if near.any():
        check_error(kind, what, float(((got - want).abs() / bound)[near].max()), 1.0)


def compare(x, targets, top, what):
    logprob, entropy, rank, ids, lps = call(x, targets, top)
    want = oracle(x.cpu().float(), targets.cpu(), top)
    best = want[5][:, None]
    V = x.shape[1]
    log_s = math.log(V) + 1
    same_or_near(logprob, want[0], STEP * (2 * want[0].abs() + 20 + log_s).nan_to_num(1, 1, 1), "log probabilities", what)
    # the entropy sums p * d, of size |d| <= its largest value with a weight that counts (about 2 ln V + 30)
    same_or_near(entropy, want[1], STEP * 32 * (log_s + 4), "entropies", what)
    assert torch.equal(rank.cpu().long(), want[2]), what
    if top:
        assert torch.equal(ids.cpu().long(), want[3]), what
        same_or_near(lps, want[4], STEP * (2 * want[4].abs() + 20 + log_s).nan_to_num(1, 1, 1), "log probabilities", what)


def rows_of(R, V, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * 3.0
    x[torch.arange(R), torch.randint(0, V, (R,), generator=g)] += torch.rand(R, generator=g) * 20
    return x.to(dtype).cuda(), torch.randint(0, V, (R,), generator=g, dtype=torch.int32).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (1, 2, 2), (3, 31, 31), (2, 33, 32), (5, 1000, 0), (7, 4099, 5), (1, 32000, 20), (19, 50257, 3),
                                     (150, 2051, 1), (300, 777, 8), (2, 128256, 32), (700, 1023, 2)])
def test_sizes(R, V, top, dtype):
    x, t = rows_of(R, V, R * 7 + V, dtype)
    compare(x, t, top, f"{R} x {V}, top {top}, {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("R", [2, 400])
def test_rows_that_lie_apart_and_begin_anywhere(R):
    for V, ld, shift, dtype in ((513, 517, 1, torch.float32), (1001, 1003, 3, torch.bfloat16), (2048, 2056, 0, torch.bfloat16), (640, 641, 2, torch.float32)):
        big, t = rows_of(R + 1, ld, V)
        flat = big.to(dtype).reshape(-1)
        x = torch.as_strided(flat, (R, V), (ld, 1), shift)
        t = (t[:R] % V).to(torch.int32)
        compare(x, t, 4, f"rows {ld} apart from {shift}, {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("R,V", [(6, 1500), (160, 1500), (3, 90001)])
def test_equal_logits_go_by_token(R, V):
    x = torch.zeros(R, V, device="cuda")
    x[:, V // 2] = 1.0
    x[:, V - 1] = 1.0
    x[1] = -4.0
    x[1, ::2] = 2.5
    t = torch.tensor([i * 37 % V for i in range(R)], dtype=torch.int32, device="cuda")
    compare(x, t, 20, "equal logits")
    # only signs of zero
    z = torch.zeros(R, V, device="cuda")
    z[:, ::3] = -0.0
    compare(z, t, 20, "zeros of both signs")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(200, 700), (9, 20011), (450, 20011)])
def test_ranks_among_neighbouring_numbers(R, V, dtype):
    """Zeros of both signs, the numbers next to zero, the largest ones, -inf, and each number's neighbours: the order alone."""
    info = torch.finfo(dtype)
    least = info.tiny * 2.0 ** (-23 if dtype == torch.float32 else -7)                     # the smallest number that is not zero
    one = [1.0, 1.0 + info.eps, 1.0 - info.eps / 2]
    few = torch.tensor([0.0, -0.0, least, -least, 2 * least, info.max, -info.max, info.tiny, -math.inf] + one + [-v for v in one], dtype=torch.float64).to(dtype)
    g = torch.Generator().manual_seed(V)
    x = few[torch.randint(0, len(few), (R, V), generator=g)].cuda()
    targets = torch.randint(0, V, (R,), generator=g, dtype=torch.int32).cuda()
    _, _, rank, ids, _ = call(x, targets, 7)
    want = oracle(x.cpu().float(), targets.cpu(), 7)
    assert torch.equal(rank.cpu().long(), want[2])
    assert torch.equal(ids.cpu().long(), want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1500, 90001])
def test_rising_and_falling_rows(V):
    x = torch.stack([torch.linspace(-9, 9, V), torch.linspace(9, -9, V), torch.arange(V).float() % 64, -(torch.arange(V).float() % 640)]).cuda()
    t = torch.tensor([V - 1, V - 2, 63, 1], dtype=torch.int32, device="cuda")
    compare(x, t, 32, "sorted rows")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [37, 1999, 70003])
def test_infinities_and_what_is_no_number(V, dtype):
    inf, nan = math.inf, math.nan
    x, _ = rows_of(10, V, 5, dtype)
    x[0] = -inf
    x[1] = -inf
    x[1, 17] = -30.0                      # one token is left
    x[2, 3] = inf
    x[3, 30] = nan
    x[4, ::2] = -inf
    x[5] = nan
    x[6] = torch.finfo(dtype).min         # masks of the type's lowest value
    x[7] = torch.finfo(dtype).min
    x[7, 9] = 1.0
    x[8, 5:] = -inf
    x[8, 3] = nan
    x[9] = torch.finfo(dtype).max
    t = torch.tensor([4, 17, 3, 30, 0, 1, 2, 9, 20, 8], dtype=torch.int32, device="cuda")
    compare(x, t, 20, "infinities")
    compare(x, torch.flip(t, [0]), 20, "infinities")


@pytest.mark.gpu
def test_nearly_certain_tokens_keep_their_digits():
    V = 4000
    x = torch.zeros(6, V, device="cuda")
    for r, lead in enumerate((8.0, 16.0, 24.0, 40.0, 80.0, 200.0)):
        x[r, 11] = lead
    t = torch.full((6,), 11, dtype=torch.int32, device="cuda")
    logprob, entropy, rank, _, _ = call(x, t, 0)
    want = oracle(x.cpu(), t.cpu(), 0)
    # ln(1 + r) with r = 3999 exp(-lead): relative to its own size now
    rel = ((logprob.cpu().double() - want[0]).abs() / want[0].abs())[:4].max()
    check_error("log probabilities near zero, relative", "certain tokens", float(rel), STEP * 64)
    rel = ((entropy.cpu().double() - want[1]).abs() / want[1].abs())[:4].max()
    check_error("entropies near zero, relative", "certain tokens", float(rel), STEP * 128)
    assert rank.tolist() == [0] * 6


@pytest.mark.gpu
@pytest.mark.parametrize("R", [3, 200])
def test_targets_outside_the_vocabulary(R):
    x, t = rows_of(R, 300, 3)
    t[0], t[1], t[2] = -1, 300, 2 ** 31 - 1
    compare(x, t, 2, "targets outside")


@pytest.mark.gpu
def test_twice_the_same_and_from_a_graph():
    x, t = rows_of(40, 30011, 8)
    a = call(x, t, 10)
    outs = [torch.empty_like(o) for o in a]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.token_logprobs(x, t, outs[0], outs[1], outs[2], top_ids=outs[3], top_logprobs=outs[4])
        with torch.cuda.graph(graph, stream=side):
            ops.token_logprobs(x, t, outs[0], outs[1], outs[2], top_ids=outs[3], top_logprobs=outs[4])
    torch.cuda.current_stream().wait_stream(side)
    y, u = rows_of(40, 30011, 9)
    b = call(y, u, 10)
    x.copy_(y)
    t.copy_(u)
    graph.replay()
    for got, want in zip(outs, b):
        assert torch.equal(got, want)
    assert not torch.equal(a[0], b[0])


@pytest.mark.gpu
def test_rows_behind_four_gigabytes():
    R, V = 9000, 128256                   # 4.6 GB of float32 (more than 2^32 bytes)
    x = torch.zeros(R, V, device="cuda")
    x[-1, 77], x[-1, 5] = 3.0, 2.0
    t = torch.full((R,), 77, dtype=torch.int32, device="cuda")
    logprob, entropy, rank, ids, lps = call(x, t, 2)
    want = 3.0 - math.log(math.exp(3) + math.exp(2) + V - 2)
    assert abs(float(logprob[-1]) - want) < 4e-6 and ids[-1].tolist() == [77, 5] and int(rank[-1]) == 0
    assert int(rank[0]) == 77 and ids[0].tolist() == [0, 1] and abs(float(logprob[0]) + math.log(V)) < 4e-6


def test_without_a_gpu_it_refuses():
    x = torch.zeros(2, 4)
    with pytest.raises(KernelError, match="CUDA"):
        ops.token_logprobs(x, torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(2), torch.zeros(2, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals():
    x, t = rows_of(4, 50, 1)
    f, i = torch.empty(4, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")

    def refused(match, logits=x, targets=t, logprob=f, entropy=f.clone(), rank=i, **more):
        with pytest.raises(KernelError, match=match):
            ops.token_logprobs(logits, targets, logprob, entropy, rank, **more)

    refused("dtype", logits=x.half())
    refused("rows of consecutive", logits=x.t())
    refused("rows of consecutive", logits=x[0])
    refused("rows of consecutive", logits=x[:1].expand(4, 50))
    refused("dtype", targets=t.long())
    refused("targets", targets=t[:3])
    refused("outputs", logprob=f[:3])
    refused("contiguous", rank=torch.empty(8, dtype=torch.int32, device="cuda")[::2])
    refused("go together", top_ids=torch.empty(4, 2, dtype=torch.int32, device="cuda"))
    for k in (33, 51):
        refused("most likely", top_ids=torch.empty(4, k, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(4, k, device="cuda"))
    refused("most likely", logits=x[:, :0])
    refused("top_ids", top_ids=torch.empty(3, 2, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(4, 2, device="cuda"))
    ops.token_logprobs(x[:0], t[:0], f[:0], f[:0].clone(), i[:0])          # no rows: nothing to do
