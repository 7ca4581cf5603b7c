"""Tables of a step built from lengths, copies of pages, and attention of a batch that shares its first pages."""
import random

import pytest
import torch

from helpers import check_error
from llmplayer_b200.errors import KernelError
from llmplayer_b200.kernels import ops

PAGE = 64
INT = dict(dtype=torch.int32, device="cuda")

# Outputs are weighted means of values of order one. Each is rounded to bfloat16 at the end (half a step, 2^-9 of up to 4: 2^-7 at
# most), and the weights enter the product as bfloat16: every weight is off by at most 2^-9 of itself, so the mean of
# |values| <= 4.5 by at most 4.5 * 2^-9. Together less than 1.7e-2.
BOUND = 1.7e-2


# ------------------------------------------------------------------------------------------------ tables
def tables_oracle(first, count, shared, own, width, page=PAGE):
    starts, positions, ids, rows, at = [0], [], [], [], 0
    for b, (f, n) in enumerate(zip(first, count)):
        starts.append(starts[-1] + n)
        positions += range(f, f + n)
        ids += [b] * n
        blocks = -(-(f + n) // page)
        mine = max(0, blocks - len(shared))
        row = (shared[:blocks] + own[at:at + mine])[:width]
        rows.append(row + [0] * (width - len(row)))
        at += mine
    return starts, [f + n for f, n in zip(first, count)], positions, ids, rows


CASES = [([0], [1], 0), ([64], [1], 1), ([63], [1], 0), ([63], [2], 0), ([128, 128, 128], [1, 70, 3], 2), ([0, 5, 200], [0, 0, 0], 0),
         ([256] * 40, [1] * 40, 4), ([640 + 3 * i for i in range(300)], [1 + i % 7 for i in range(300)], 10), ([64 * 500] * 9, [200] * 9, 500),
         ([0, 10, 300], [0, 3, 9], 4), ([0], [20000], 0), ([70] * 1500, [i % 3 for i in range(1500)], 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("first,count,shared", CASES)
@pytest.mark.parametrize("page", [64, 16])
def test_tables(first, count, shared, page):
    need = [-(-(f + n) // page) for f, n in zip(first, count)]
    rng = random.Random(len(first) + shared)
    own = [rng.randrange(1, 10 ** 6) for _ in range(sum(max(0, n - shared) for n in need))]
    pages = [rng.randrange(1, 10 ** 6) for _ in range(shared)]
    T = sum(count)
    for width in (max(max(need), 1), max(need) + 5):
        want = tables_oracle(first, count, pages, own, width, page)
        out = [torch.full((n,), -7, **INT) for n in (len(first) + 1, len(first), T + 3, T + 3)] + [torch.full((len(first), width), -7, **INT)]
        ops.step_tables(torch.tensor(first, **INT), torch.tensor(count, **INT), torch.tensor(pages, **INT), torch.tensor(own, **INT), *out, page_size=page)
        for got, w in zip(out[:4], want[:4]):
            w = w + [-7] * (got.numel() - len(w))             # behind the last sequence: as it was
            assert got.tolist() == w
        assert out[4].tolist() == want[4]
        alone = torch.full((len(first), width), -7, **INT)
        ops.step_tables(torch.tensor(first, **INT), torch.tensor(count, **INT), torch.tensor(pages, **INT), torch.tensor(own, **INT), None, None, None,
                        None, alone, page_size=page)
        assert torch.equal(alone, out[4])


@pytest.mark.gpu
def test_tables_stay_within_their_tensors():
    """Lengths that say more than the tensors hold: what fits is written, the neighbours stay."""
    room = torch.full((4 + 2 + 5 + 5 + 6 + 8,), -7, **INT)
    q_start, kv_len, positions, seq_ids, table = room[4:7], room[8:10], room[11:14], room[15:18], room[20:24].view(2, 2)
    keep = torch.ones(room.numel(), dtype=torch.bool)
    for a, b in ((4, 7), (8, 10), (11, 14), (15, 18), (20, 24)):
        keep[a:b] = False
    ops.step_tables(torch.tensor([100, 300], **INT), torch.tensor([50, 60], **INT), torch.tensor([3], **INT), torch.tensor([8], **INT), q_start, kv_len,
                    positions, seq_ids, table)
    assert (room.cpu()[keep] == -7).all()
    assert positions.tolist() == [100, 101, 102] and table.tolist() == [[3, 8], [3, 0]] and q_start.tolist() == [0, 50, 110]


@pytest.mark.gpu
def test_tables_of_lengths_that_no_cache_has():
    """Counts below zero count as none; sums that wrap around write nothing outside the tensors and end."""
    most = 2 ** 31 - 1
    for first, count in (([70, 5, 130], [-90, 3, 70]), ([most, most, 3], [1, 1, 2]), ([0, 7, 64], [most, most, 5]), ([-most, -1, 0], [most, 2, most])):
        room = torch.full((200,), -7, **INT)
        q_start, kv_len, positions, seq_ids, table = room[4:8], room[12:15], room[20:60], room[64:104], room[120:150].view(3, 10)
        keep = torch.ones(room.numel(), dtype=torch.bool)
        for a, b in ((4, 8), (12, 15), (20, 60), (64, 104), (120, 150)):
            keep[a:b] = False
        own = torch.arange(1000, 1012, **INT)
        ops.step_tables(torch.tensor(first, **INT), torch.tensor(count, **INT), torch.tensor([3], **INT), own, q_start, kv_len, positions, seq_ids, table)
        torch.cuda.synchronize()
        assert (room.cpu()[keep] == -7).all()
        assert bool(((table == 0) | (table == 3) | ((table >= 1000) & (table < 1012))).all())
        if min(count) == -90:
            assert q_start.tolist() == [0, 0, 3, 73] and kv_len.tolist() == [70, 8, 200]
            assert table[:, :5].tolist() == [[3, 1000, 0, 0, 0], [3, 0, 0, 0, 0], [3, 1001, 1002, 1003, 0]]


@pytest.mark.gpu
def test_tables_refusals():
    def ints(*v):
        return torch.tensor(v, **INT)

    good = dict(first=ints(1, 2), count=ints(1, 1), shared=ints(), own=ints(0, 1), q_start=ints(0, 0, 0), kv_len=ints(0, 0), positions=ints(0, 0),
                seq_ids=ints(0, 0), page_table=torch.zeros(2, 1, **INT))
    ops.step_tables(**good)
    for name, bad in (("first", ints(1)), ("count", ints(1)), ("q_start", ints(0, 0)), ("kv_len", ints(0)), ("seq_ids", ints(0)), ("positions", None),
                      ("page_table", torch.zeros(3, 1, **INT)), ("page_table", torch.zeros(2, 0, **INT)), ("own", ints(0, 1).long()),
                      ("first", torch.zeros(2, dtype=torch.int32)), ("page_size", 0)):
        with pytest.raises(KernelError):
            ops.step_tables(**{**good, name: bad})


# ------------------------------------------------------------------------------------------------ copies
@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype,n", [((3, 9, 2, 2, 64, 16), torch.bfloat16, 1), ((1, 40, 64, 96), torch.bfloat16, 5), ((16, 70, 2, 8, 64, 64), torch.bfloat16, 60),
                                           ((2, 11, 2, 3, 64, 48), torch.float32, 4), ((2, 1000, 64, 8), torch.float32, 900)])
def test_copies(shape, dtype, n):
    g = torch.Generator().manual_seed(n)
    storage = torch.randn(*shape, generator=g).to(dtype).cuda()
    want = storage.clone()
    order = torch.randperm(shape[1], generator=g).tolist()
    targets, rest = order[:n], order[n:]
    sources = [rest[i % len(rest)] for i in range(n)]
    want[:, targets] = want[:, sources]
    ops.copy_pages(storage, sources, targets)
    assert torch.equal(storage, want)
    ops.copy_pages(storage, [], [])
    assert torch.equal(storage, want)


@pytest.mark.gpu
def test_copies_behind_two_gigabytes():
    storage = torch.zeros(2, 70000, 64, 256, dtype=torch.bfloat16, device="cuda")           # 4.6 GB
    storage[1, 69999] = 3.0
    storage[0, 69999] = 2.0
    ops.copy_pages(storage, [69999], [12345])
    assert float(storage[1, 12345].float().min()) == 3.0 and float(storage[0, 12345].float().max()) == 2.0
    assert float(storage[:, 12344].float().abs().max()) == 0.0 and float(storage[:, 12346].float().abs().max()) == 0.0


def test_copies_refusals_before_any_launch():
    storage = torch.zeros(1, 4, 64, 8)
    for sources, targets in (([0], [4]), ([-1], [2]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([1], [1])):
        with pytest.raises(KernelError, match="copy_pages: "):
            ops.copy_pages(storage, sources, targets)
    with pytest.raises(KernelError, match="CUDA"):
        ops.copy_pages(storage, [0], [1])


# ------------------------------------------------------------------------------------------------ attention
class Buffers:
    """A supplier of scratch; it hands the buffers out full of what is no number."""

    def __init__(self):
        self.kept = {}

    def __call__(self, name, shape, dtype):
        key = (name, tuple(shape), dtype)
        if key not in self.kept:
            t = torch.empty(shape, dtype=dtype, device="cuda")
            t.fill_(float("nan") if dtype.is_floating_point else -1)
            self.kept[key] = t
        return self.kept[key]


def batch(shared, lengths, new, H, G, hd, seed=0, junk=float("nan"), extra_rows=0, sharp=1.0):
    """Pages in no order; rows of a page behind its sequence's length hold ``junk``, as do all pages of nobody."""
    g = torch.Generator().manual_seed(seed)
    start = shared * PAGE
    need = [max(0, -(-n // PAGE) - shared) for n in lengths]
    total = shared + sum(need) + 4
    order = torch.randperm(total, generator=g).tolist()
    pages = torch.full((total, 2, G, PAGE, hd), junk, dtype=torch.bfloat16)
    width = shared + max(need + [0]) + 1
    common, rest = order[:shared], order[shared:]
    table = torch.full((len(lengths), width), order[-1], dtype=torch.int32)
    for p in common:
        pages[p] = torch.randn(2, G, PAGE, hd, generator=g).clamp(-4, 4).to(torch.bfloat16)
    at = 0
    for b, n in enumerate(lengths):
        table[b, :shared] = torch.tensor(common, dtype=torch.int32)
        for i in range(need[b]):
            p = rest[at]
            at += 1
            table[b, shared + i] = p
            rows = min(PAGE, n - start - i * PAGE)
            pages[p, :, :, :rows] = torch.randn(2, G, rows, hd, generator=g).clamp(-4, 4).to(torch.bfloat16)
    T = sum(new)
    q = (torch.randn(T + extra_rows, H * hd, generator=g) * sharp).to(torch.bfloat16)
    q[T:] = float("nan")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return q, pages, table, starts, lengths


def attend(case, shared, H, G, hd, max_new=None, scratch=None):
    q, pages, table, starts, lengths = case
    out = torch.full((q.shape[0], H * hd), 5.0, dtype=torch.bfloat16, device="cuda")
    new = [b - a for a, b in zip(starts, starts[1:])]
    ops.attention_shared(q.cuda(), out, pages.cuda(), table.cuda(), torch.tensor(starts, **INT), torch.tensor(lengths, **INT), scratch or Buffers(),
                         shared_pages=shared, max_new=max_new or max(new + [1]), num_heads=H, num_kv_heads=G, head_dim=hd, scale=hd ** -0.5)
    return out


def attention_oracle(case, H, G, hd):
    q, pages, table, starts, lengths = case
    T = starts[-1]
    out = torch.zeros(T, H, hd, dtype=torch.float64, device="cuda")
    pages = pages.cuda().double()
    qd = q.cuda().double().view(-1, G, H // G, hd)
    for b, n in enumerate(lengths):
        a, e = starts[b], starts[b + 1]
        if a == e or n == 0:
            continue
        kv = pages[table[b, :-(-n // PAGE)].long().cuda()]
        k = kv[:, 0].permute(1, 0, 2, 3).reshape(G, -1, hd)[:, :n]
        v = kv[:, 1].permute(1, 0, 2, 3).reshape(G, -1, hd)[:, :n]
        s = torch.einsum("tgrd,gkd->tgrk", qd[a:e], k) * hd ** -0.5
        position = torch.arange(n - (e - a), n, device="cuda")[:, None, None, None]
        s = s.masked_fill(torch.arange(n, device="cuda") > position, float("-inf"))
        out[a:e] = torch.einsum("tgrk,gkd->tgrd", torch.softmax(s, dim=-1), v).reshape(e - a, H, hd)
    return out.view(T, H * hd)


def check(case, shared, H, G, hd, kind, what, **more):
    got = attend(case, shared, H, G, hd, **more)
    T = case[3][-1]
    want = attention_oracle(case, H, G, hd)
    assert torch.isfinite(got[:T].float()).all(), what
    check_error(kind, what, float((got[:T].double() - want).abs().max()) if T else 0.0, BOUND)
    assert (got[T:] == 5.0).all(), "rows behind the last sequence"
    return got


HEADS = [(32, 8, 64), (24, 8, 128), (32, 8, 128), (4, 4, 64), (14, 2, 64), (6, 1, 128), (40, 8, 128), (3, 3, 128), (64, 1, 64), (128, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,hd", HEADS)
@pytest.mark.parametrize("shared,own", [(1, 1), (2, 70), (5, 64), (33, 200)])
def test_single_tokens(H, G, hd, shared, own):
    rng = random.Random(shared * own + H)
    for B in (1, 2, 5, 33, 130):
        lengths = [shared * PAGE + rng.randint(1, own) for _ in range(B)]
        case = batch(shared, lengths, [1] * B, H, G, hd, seed=B)
        check(case, shared, H, G, hd, "shared prefix, single tokens", f"{B} sequences, {H} on {G} of {hd}, {shared} pages, up to {own} own")


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,hd", HEADS)
@pytest.mark.parametrize("shared,new,cached", [(1, 2, 0), (2, 30, 0), (4, 65, 10), (17, 129, 70), (40, 7, 300)])
def test_several_tokens(H, G, hd, shared, new, cached):
    rng = random.Random(shared * new + H)
    for B in (1, 3, 20):
        counts = [rng.randint(1, new) for _ in range(B)]
        lengths = [shared * PAGE + rng.randint(0, cached) + n for n in counts]
        case = batch(shared, lengths, counts, H, G, hd, seed=B + 50)
        check(case, shared, H, G, hd, "shared prefix, several tokens", f"{B} sequences, {H} on {G} of {hd}, {shared} pages, up to {new} new behind {cached}")


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,hd", [(8, 2, 64), (8, 2, 128)])
def test_empty_sequences_and_rows_behind_the_last(H, G, hd):
    """Sequences without new tokens, of length zero, tokens that lie inside the shared pages, a batch filled up with rows."""
    shared = 3
    start = shared * PAGE
    for new, lengths in (([1, 0, 1, 0, 1], [start + 5, start, start + 64, 0, start + 1]), ([4, 0, 0, 9, 1], [start + 4, 0, start + 80, start + 100, start + 1]),
                         ([0, 0, 1], [0, 0, start + 2]), ([1, 1], [start, start - 63]), ([70, 3, 1], [start + 2, 3, 100]), ([0], [start + 7])):
        case = batch(shared, lengths, new, H, G, hd, seed=len(new), extra_rows=37)
        check(case, shared, H, G, hd, "shared prefix, gaps", f"new {new}, lengths {lengths}")


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,hd", [(8, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_shared_pages_that_are_not_full(H, G, hd, junk):
    """Every sequence ends inside the shared pages: what lies there behind the longest is not looked at."""
    for shared, lengths, new in ((1, [5, 3], [1, 1]), (3, [130, 129, 2], [1, 1, 1]), (5, [200, 64, 199], [3, 60, 199]), (9, [64] * 3, [1] * 3), (40, [1000] * 70, [1] * 70),
                                 (21, [900 + i for i in range(12)], [2 + 9 * i for i in range(12)]), (30, [1280, 0], [1, 0]), (1, [64, 64], [64, 1])):
        case = batch(shared, lengths, new, H, G, hd, seed=shared)
        pages, table, reached = case[1], case[2], max(lengths)
        for i in range(shared):
            pages[table[0, i].long(), :, :, max(0, min(PAGE, reached - i * PAGE)):] = junk
        check(case, shared, H, G, hd, "shared prefix, short sequences", f"{shared} pages, lengths up to {reached}, {H} on {G} of {hd}")


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("shared", [0, 2])
def test_nothing_shared_or_a_single_sequence(shared, new):
    for lengths in ([new], [shared * PAGE + 300], [shared * PAGE + 11, shared * PAGE + 200, shared * PAGE + new]):
        counts = [new] * len(lengths)
        lengths = [max(n, shared * PAGE + new) for n in lengths]
        check(batch(shared, lengths, counts, 8, 2, 128, seed=3), shared, 8, 2, 128, "shared prefix, none", f"{lengths}, {shared} shared")


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 20])
def test_sharp_and_large_scores(hd, new):
    """Scores of hundreds (weights of one key), and maxima that keep moving along the pages."""
    shared, B = 12, 6
    lengths = [shared * PAGE + 90 + new] * B
    case = batch(shared, lengths, [new] * B, 8, 2, hd, seed=9, sharp=30.0)
    check(case, shared, 8, 2, hd, "shared prefix, sharp scores", f"heads of {hd}")
    q, pages, table, starts, _ = case
    for i in range(shared):                               # keys grow from page to page, so the running maximum does
        pages[table[0, i].long(), 0] *= 0.25 * (i + 1)
    check((q * 0.2, pages, table, starts, lengths), shared, 8, 2, hd, "shared prefix, sharp scores", f"growing keys, heads of {hd}")


@pytest.mark.gpu
def test_the_same_pages_many_times_over_and_long_ones():
    shared, B, H, G, hd = 600, 70, 8, 2, 128
    lengths = [shared * PAGE + 1 + 13 * i for i in range(B)]
    check(batch(shared, lengths, [1] * B, H, G, hd, seed=2), shared, H, G, hd, "shared prefix, single tokens", "38,400 shared positions")
    counts = [1 + 5 * (i % 9) for i in range(B)]
    lengths = [shared * PAGE + n for n in counts]
    check(batch(shared, lengths, counts, H, G, hd, seed=2), shared, H, G, hd, "shared prefix, several tokens", "38,400 shared positions")


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 9, 32])
@pytest.mark.parametrize("shared", [40, 401, 1100])
def test_one_tile_of_rows_over_many_pages(shared, tokens, hd):
    """The rows fill one tile (or less): a CTA's two halves take alternate pages, tens of them each."""
    check(batch(shared, [shared * PAGE + 1 + i for i in range(tokens)], [1] * tokens, 32, 8, hd, seed=tokens), shared, 32, 8, hd, "shared prefix, single tokens",
          f"{tokens} tokens on {shared} pages")


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 12])
def test_results_repeat_and_graphs_replay(new):
    shared, B, H, G, hd = 20, 9, 32, 8, 64
    lengths = [shared * PAGE + 40 + i + new for i in range(B)]
    case = batch(shared, lengths, [new] * B, H, G, hd, seed=4)
    scratch = Buffers()
    a = attend(case, shared, H, G, hd, scratch=scratch)
    b = attend(case, shared, H, G, hd, scratch=scratch)
    assert torch.equal(a, b)
    q, pages, table, starts, _ = (x.cuda() if isinstance(x, torch.Tensor) else x for x in case)
    out = torch.zeros_like(a)
    q_start, kv_len = torch.tensor(starts, **INT), torch.tensor(lengths, **INT)

    def run():
        ops.attention_shared(q, out, pages, table, q_start, kv_len, scratch, shared_pages=shared, max_new=new, num_heads=H, num_kv_heads=G, head_dim=hd,
                             scale=hd ** -0.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        run()
        with torch.cuda.graph(graph, stream=side):
            run()
    torch.cuda.current_stream().wait_stream(side)
    # the sequences grew meanwhile, their tokens are others
    longer = [n - 7 for n in lengths]
    other = batch(shared, longer, [new] * B, H, G, hd, seed=4)
    kv_len.copy_(torch.tensor(longer, **INT))
    graph.replay()
    want = attention_oracle((case[0], case[1], case[2], starts, longer), H, G, hd)
    check_error("shared prefix, replayed", f"{new} new", float((out.double() - want).abs().max()), BOUND)
    assert other[3] == starts


@pytest.mark.gpu
def test_attention_refusals():
    H, G, hd = 8, 2, 64
    q, pages, table, starts, lengths = (x.cuda() if isinstance(x, torch.Tensor) else torch.tensor(x, **INT) for x in batch(2, [130, 140], [1, 1], H, G, hd, junk=0.0))
    good = dict(q=q, out=torch.empty_like(q), pages=pages, page_table=table, q_start=starts, kv_len=lengths, scratch=Buffers(), shared_pages=2, max_new=1,
                num_heads=H, num_kv_heads=G, head_dim=hd, scale=0.125)
    ops.attention_shared(**good)
    for name, bad in (("q", q.float()), ("q", q[:, :-64]), ("out", torch.empty_like(q)[:1]), ("pages", pages.float()), ("pages", pages[..., :32].contiguous()),
                      ("page_table", table[:1]), ("page_table", table.long()), ("q_start", starts[:2]), ("kv_len", lengths[:1]), ("shared_pages", -1),
                      ("shared_pages", table.shape[1] + 1), ("max_new", 0), ("num_heads", 6), ("head_dim", 32), ("q", q.cpu())):
        with pytest.raises(KernelError):
            ops.attention_shared(**{**good, name: bad})
    ops.attention_shared(**{**good, "q": q[:0], "out": q[:0].clone(), "q_start": torch.zeros_like(starts)})       # no tokens: nothing to do


def test_what_is_served():
    assert ops.attention_shared_serves(32, 8, 64) and ops.attention_shared_serves(128, 1, 128)
    assert not ops.attention_shared_serves(32, 8, 96) and not ops.attention_shared_serves(129, 1, 64) and not ops.attention_shared_serves(6, 4, 64)
    assert not ops.attention_shared_serves(32, 8, 64, 32)
