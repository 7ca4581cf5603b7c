"""What the speed of the operators around a shared prompt is measured on: many continuations of one prompt, drawn or scored.

A prompt is run once, its cached pages are shared by all sequences that continue it (``copy_pages`` gives each its own copy of
the page that is still being filled), a step's tables are built on the device from the sequences' lengths (``step_tables``),
the new tokens attend over the shared pages together (``attention_shared``), and the given tokens are scored
(``token_logprobs``).

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare(case, seed)`` makes what a program
holds before the call, ``run(state)`` is one call (the plain tensor operations, or with ``own`` the library's kernels),
``exact(case, seed)`` the same in 64 bits and ``work(case)`` the bytes and operations that the call cannot do without.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 64           # positions per page of the cache

# (query heads, key/value heads, head size): the Llama shapes of the benchmark (1B, 3B, 8B) and smaller ones
HEADS = {"32x8x64": (32, 8, 64), "24x8x128": (24, 8, 128), "32x8x128": (32, 8, 128), "8x2x128": (8, 2, 128), "16x16x64": (16, 16, 64),
         "14x2x64": (14, 2, 64), "40x8x128": (40, 8, 128)}


def listed():
    return [
        # Greedy decoding of one sequence of a small model that reports each chosen token's log probability: latency.
        {"name": "logprobs_one", "op": "logprobs", "rows": 1, "vocab": 32000, "top": 0, "dtype": "float32", "masked": 0.0},
        # A decode step of a serving batch with five alternatives per token, the benchmark's vocabulary.
        {"name": "logprobs_batch", "op": "logprobs", "rows": 48, "vocab": 128256, "top": 5, "dtype": "float32", "masked": 0.0},
        # Scoring answers token by token: every row of a long step's logits.
        {"name": "logprobs_score", "op": "logprobs", "rows": 2000, "vocab": 128256, "top": 2, "dtype": "float32", "masked": 0.0},
        # Logits kept in 16 bits, an odd vocabulary, a grammar that leaves few tokens, the longest list of alternatives.
        {"name": "logprobs_masked_bf16", "op": "logprobs", "rows": 333, "vocab": 50257, "top": 20, "dtype": "bfloat16", "masked": 0.9},
        # Four samples of one short system prompt (1B shape): a decode step where latency counts.
        {"name": "shared_decode_few", "op": "attention", "heads": "32x8x64", "sequences": 4, "shared": 9, "own": 90, "new": 1},
        # 64 samples of one long document (8B shape): a decode step.
        {"name": "shared_decode_batch", "op": "attention", "heads": "32x8x128", "sequences": 64, "shared": 128, "own": 250, "new": 1},
        # Answers of unequal lengths scored against one prompt (1B shape).
        {"name": "shared_score", "op": "attention", "heads": "32x8x64", "sequences": 24, "shared": 50, "own": 0, "new": 37},
        # Many longer answers to a question about a very long document (8B shape): bound by the products.
        {"name": "shared_score_long", "op": "attention", "heads": "32x8x128", "sequences": 40, "shared": 500, "own": 0, "new": 190},
        # The tables of a decode step of eight samples, and of a scoring step over a long shared document.
        {"name": "tables_decode", "op": "tables", "sequences": 8, "shared": 20, "own": 150, "new": 1},
        {"name": "tables_score", "op": "tables", "sequences": 250, "shared": 500, "own": 0, "new": 130},
        # Eight forks of a sequence in the 16 layers of the 1B shape, 60 forks in the 32 layers of the 8B shape.
        {"name": "fork_few", "op": "fork", "heads": "32x8x64", "layers": 16, "forks": 8},
        {"name": "fork_many", "op": "fork", "heads": "32x8x128", "layers": 32, "forks": 60},
    ]


def _spread(rng, lo, hi):
    """A whole number between the two, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "attention", "attention", "attention", "tables", "fork"])
    if op == "logprobs":
        rows = _spread(rng, 1, 2000)
        vocab = _spread(rng, 1000, min(200000, 2000 * 128256 // rows))
        return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 2, 5, 8, 20]),
                "dtype": rng.choice(["float32", "float32", "bfloat16"]), "masked": rng.choice([0.0, 0.0, 0.5, 0.98])}
    if op == "attention":
        heads = rng.choice(sorted(HEADS))
        if rng.random() < 0.5:
            return {"op": op, "heads": heads, "sequences": _spread(rng, 2, 200), "shared": _spread(rng, 4, 500),
                    "own": _spread(rng, 1, 700), "new": 1}
        new = _spread(rng, 2, 250)
        sequences = _spread(rng, 2, min(200, max(2, 4000 // new)))
        return {"op": op, "heads": heads, "sequences": sequences, "shared": _spread(rng, 4, 400), "own": rng.choice([0, 0, 30, 200]),
                "new": new}
    if op == "tables":
        return {"op": op, "sequences": _spread(rng, 1, 250), "shared": _spread(rng, 1, 500), "own": rng.choice([0, 20, 150, 600]),
                "new": _spread(rng, 1, 130)}
    return {"op": op, "heads": rng.choice(sorted(HEADS)), "layers": rng.randint(2, 32), "forks": _spread(rng, 1, 60)}


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Per sequence: the positions it holds before the step and its new tokens. All lie behind the shared pages. They are the
    case's own (the outputs' shapes go by them), whatever the seed."""
    rng = random.Random(1000003 * case["sequences"] + 7919 * case["shared"] + 31 * case["own"] + case["new"])
    B, new, own_most = case["sequences"], case["new"], case["own"]
    start = case["shared"] * PAGE
    first = [start + (rng.randint(0, own_most) if own_most else 0) for _ in range(B)]
    count = [1 if new == 1 else rng.randint(max(1, new // 4), new) for _ in range(B)]
    count[0] = new
    return first, count


def _page_ids(case, seed, first, count):
    """The shared pages, and each sequence's own ones: the numbers of a cache's pages in no order."""
    need = [-(-(f + n) // PAGE) - case["shared"] for f, n in zip(first, count)]
    total = case["shared"] + sum(need)
    ids = list(range(total))
    random.Random(seed * 7919 + 3).shuffle(ids)
    shared, rest, own_pages = ids[:case["shared"]], ids[case["shared"]:], []
    for n in need:
        own_pages.append(rest[:n])
        rest = rest[n:]
    return total, shared, own_pages


def _logits(case, seed, device):
    gen = torch.Generator(device=device).manual_seed(seed)
    R, V = case["rows"], case["vocab"]
    logits = torch.randn(R, V, generator=gen, device=device, dtype=torch.float32) * 2.5
    # a model prefers a few tokens of every row, in some rows one of them nearly for certain
    liked = torch.randint(0, V, (R, 6), generator=gen, device=device)
    amount = torch.rand(R, 6, generator=gen, device=device) * 14.0 + torch.rand(R, 1, generator=gen, device=device).pow(6) * 25.0
    logits.scatter_add_(1, liked, amount)
    pick = torch.randint(0, 8, (R,), generator=gen, device=device)
    other = torch.randint(0, V, (R,), generator=gen, device=device)
    targets = torch.where(pick < 6, liked.gather(1, pick.clamp(max=5)[:, None])[:, 0], other)
    if case["masked"] > 0:
        logits.masked_fill_(torch.rand(R, V, generator=gen, device=device) < case["masked"], float("-inf"))
        # at least the alternatives of the longest list stay allowed
        logits[:, 7:7 + 40] = torch.randn(R, 40, generator=gen, device=device)
    return logits.to(getattr(torch, case["dtype"])), targets.to(torch.int32)


def _attention_inputs(case, seed, device):
    H, G, hd = HEADS[case["heads"]]
    first, count = _lengths(case)
    total, shared, own_pages = _page_ids(case, seed, first, count)
    gen = torch.Generator(device=device).manual_seed(seed)
    pages = torch.randn(total, 2, G, PAGE, hd, generator=gen, device=device, dtype=torch.float32).to(torch.bfloat16)
    T = sum(count)
    q = (torch.randn(T, H * hd, generator=gen, device=device, dtype=torch.float32) * 1.5).to(torch.bfloat16)
    return H, G, hd, first, count, shared, own_pages, pages, q


def prepare(case, seed):
    if case["op"] == "logprobs":
        logits, targets = _logits(case, seed, DEV)
        R, k = case["rows"], case["top"]
        state = {"op": "logprobs", "logits": logits, "targets": targets, "top": k,
                 "logprob": torch.empty(R, dtype=torch.float32, device=DEV), "entropy": torch.empty(R, dtype=torch.float32, device=DEV),
                 "rank": torch.empty(R, dtype=torch.int32, device=DEV),
                 "top_ids": torch.empty(R, k, dtype=torch.int32, device=DEV) if k else None,
                 "top_logprobs": torch.empty(R, k, dtype=torch.float32, device=DEV) if k else None}
    elif case["op"] == "attention":
        H, G, hd, first, count, shared, own_pages, pages, q = _attention_inputs(case, seed, DEV)
        width = max(len(p) for p in own_pages) + len(shared)
        table = torch.zeros(len(first), width, dtype=torch.int32)
        for i, mine in enumerate(own_pages):
            table[i, :len(shared) + len(mine)] = torch.tensor(shared + mine, dtype=torch.int32)
        starts = [0]
        for n in count:
            starts.append(starts[-1] + n)
        buffers = {}

        def scratch(name, shape, dtype):
            key = (name, tuple(shape), dtype)
            if key not in buffers:
                buffers[key] = torch.empty(shape, dtype=dtype, device=DEV)
            return buffers[key]

        state = {"op": "attention", "heads": (H, G, hd), "q": q, "pages": pages, "page_table": table.to(DEV),
                 "q_start": torch.tensor(starts, dtype=torch.int32, device=DEV),
                 "kv_len": torch.tensor([f + n for f, n in zip(first, count)], dtype=torch.int32, device=DEV),
                 "shared_pages": len(shared), "max_new": max(count), "out": torch.empty_like(q), "scratch": scratch}
    elif case["op"] == "tables":
        first, count = _lengths(case)
        _, shared, own_pages = _page_ids(case, seed, first, count)
        T, B = sum(count), len(first)
        width = len(shared) + max(len(p) for p in own_pages)

        def ints(values):
            return torch.tensor(values, dtype=torch.int32, device=DEV)

        def room(*shape):
            return torch.empty(*shape, dtype=torch.int32, device=DEV)

        state = {"op": "tables", "first": ints(first), "count": ints(count), "shared": ints(shared), "own": ints([p for mine in own_pages for p in mine]),
                 "tokens": T, "width": width, "q_start": room(B + 1), "kv_len": room(B), "positions": room(T), "seq_ids": room(T),
                 "page_table": room(B, width)}
    else:
        H, G, hd = HEADS[case["heads"]]
        n = case["forks"]
        gen = torch.Generator(device=DEV).manual_seed(seed)
        # the page that the forks copy lies among theirs; a few pages beside them belong to others
        ids = list(range(n + 4))
        random.Random(seed).shuffle(ids)
        storage = torch.randn(case["layers"], n + 4, 2, G, PAGE, hd, generator=gen, device=DEV, dtype=torch.float32).to(torch.bfloat16)
        state = {"op": "fork", "storage": storage, "sources": [ids[0]] * n, "targets": ids[1:n + 1]}
    return state


# ------------------------------------------------------------------------------------------------ the calls
def _run_own(state):
    from llmplayer_b200.kernels import ops
    op = state["op"]
    if op == "logprobs":
        ops.token_logprobs(state["logits"], state["targets"], state["logprob"], state["entropy"], state["rank"],
                           top_ids=state["top_ids"], top_logprobs=state["top_logprobs"])
        out = [state["logprob"], state["entropy"], state["rank"]]
        return out + ([state["top_ids"], state["top_logprobs"]] if state["top"] else [])
    if op == "attention":
        H, G, hd = state["heads"]
        return ops.attention_shared(state["q"], state["out"], state["pages"], state["page_table"], state["q_start"], state["kv_len"],
                                    state["scratch"], shared_pages=state["shared_pages"], max_new=state["max_new"], num_heads=H,
                                    num_kv_heads=G, head_dim=hd, scale=hd ** -0.5)
    if op == "tables":
        ops.step_tables(state["first"], state["count"], state["shared"], state["own"], state["q_start"], state["kv_len"],
                        state["positions"], state["seq_ids"], state["page_table"], page_size=PAGE)
        return [state[name] for name in ("q_start", "kv_len", "positions", "seq_ids", "page_table")]
    ops.copy_pages(state["storage"], state["sources"], state["targets"])
    return state["storage"]


def _plain_logprobs(logits, targets, top):
    """Exponentials in 32 bits, their sums and logarithms in 64 (the probability of a token that is nearly certain differs from
    one by less than 32 bits show)."""
    x, t = logits.float(), targets.long()[:, None]
    m = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(dim=1, keepdim=True, dtype=torch.float64)
    log_s = torch.log(s)
    # a token without a probability adds nothing to the entropy
    mean = torch.where(e > 0, e * (x - m), torch.zeros_like(x)).sum(dim=1, keepdim=True, dtype=torch.float64) / s
    at = x.gather(1, t)
    index = torch.arange(x.shape[1], device=x.device)[None, :]
    rank = ((x > at) | ((x == at) & (index < t))).sum(dim=1)
    out = [((at - m).double() - log_s).float()[:, 0], (log_s - mean).float()[:, 0], rank.to(torch.int32)]
    if top:
        values, ids = torch.sort(x, dim=1, descending=True, stable=True)             # equal ones: the lowest index first
        out += [ids[:, :top].to(torch.int32), ((values[:, :top] - m).double() - log_s).float()]
    return out


def _softmax_parts(scores, values):
    """The weighted sum of the values with the weights' sum and the maximum that they are taken against."""
    m = scores.amax(dim=-1, keepdim=True)
    weights = scores.sub_(m).exp_()
    return weights @ values, weights.sum(dim=-1, keepdim=True), m


def _plain_attention(state):
    H, G, hd = state["heads"]
    R, P = H // G, state["shared_pages"]
    pages, table, starts, kv_len = state["pages"], state["page_table"].long(), state["q_start"].long(), state["kv_len"].long()
    T, B, n = state["q"].shape[0], kv_len.numel(), state["max_new"]
    q = state["q"].float().view(T, G, R, hd) * hd ** -0.5
    # over the shared pages: all tokens' queries at once, [G, T R, positions]; every token sees all of them
    kv = pages[table[0, :P]].float()
    k0, v0 = (kv[:, which].permute(1, 0, 2, 3).reshape(G, P * PAGE, hd) for which in (0, 1))
    o0, l0, m0 = _softmax_parts(q.permute(1, 0, 2, 3).reshape(G, T * R, hd) @ k0.transpose(1, 2), v0)
    o0, l0, m0 = (x.view(G, T, R, -1).permute(1, 0, 2, 3) for x in (o0, l0, m0))
    # over each sequence's own pages: the tokens in a batch that is filled up to the longest run, [B, G, n R, positions]
    j = torch.arange(n, device=q.device)[None, :]
    count = (starts[1:] - starts[:-1])[:, None]
    token = (starts[:-1, None] + j).clamp(max=T - 1)
    position = (kv_len[:, None] - count + j)[:, None, :, None, None]                   # [B, 1, n, 1, 1]
    kv = pages[table[:, P:]].float()                                                   # [B, W, 2, G, PAGE, hd]
    k1, v1 = (kv[:, :, which].permute(0, 2, 1, 3, 4).reshape(B, G, -1, hd) for which in (0, 1))
    scores = q[token].permute(0, 2, 1, 3, 4).reshape(B, G, n * R, hd) @ k1.transpose(2, 3)
    key = P * PAGE + torch.arange(k1.shape[2], device=q.device)
    hidden = (key > position).expand(B, G, n, R, -1).reshape(scores.shape)
    o1, l1, m1 = _softmax_parts(scores.masked_fill_(hidden, float("-inf")), v1)
    sequence = torch.repeat_interleave(torch.arange(B, device=q.device), count[:, 0], output_size=T)
    place = torch.arange(T, device=q.device) - starts[sequence]
    o1, l1, m1 = (x.view(B, G, n, R, -1).permute(0, 2, 1, 3, 4)[sequence, place] for x in (o1, l1, m1))
    # the two parts against their common maximum
    m = torch.maximum(m0, m1)
    f0, f1 = torch.exp(m0 - m), torch.exp(m1 - m)
    return ((o0 * f0 + o1 * f1) / (l0 * f0 + l1 * f1)).reshape(T, H * hd).to(torch.bfloat16)


def _plain_tables(state):
    first, count, shared, mine = state["first"], state["count"], state["shared"], state["own"]
    B, P = first.numel(), shared.numel()
    zero = torch.zeros(1, dtype=torch.int32, device=first.device)
    q_start = torch.cat([zero, torch.cumsum(count, 0, dtype=torch.int32)])
    kv_len = first + count
    token = torch.arange(state["tokens"], dtype=torch.int32, device=first.device)
    seq = (token[:, None] >= q_start[None, 1:]).sum(dim=1)
    positions = first[seq] + token - q_start[seq]
    blocks = (kv_len + PAGE - 1) // PAGE
    begin = torch.cat([zero, torch.cumsum(blocks - P, 0, dtype=torch.int32)])[:B]
    column = torch.arange(state["width"], dtype=torch.int32, device=first.device)[None, :]
    at = (begin[:, None] + column - P).clamp(0, mine.numel() - 1)
    ids = torch.where(column < P, shared[column.clamp(max=P - 1)], mine[at])
    table = torch.where(column < blocks[:, None], ids, torch.zeros_like(ids))
    return [q_start, kv_len, positions.to(torch.int32), seq.to(torch.int32), table]


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "logprobs":
        return _plain_logprobs(state["logits"], state["targets"], state["top"])
    if state["op"] == "attention":
        return _plain_attention(state)
    if state["op"] == "tables":
        return _plain_tables(state)
    storage = state["storage"]
    storage[:, state["targets"]] = storage[:, state["sources"]]
    return storage


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] == "logprobs":
        logits, targets = _logits(case, seed, DEV)
        outs = [[] for _ in range(5 if case["top"] else 3)]
        for a in range(0, case["rows"], 64):
            x, t = logits[a:a + 64].double(), targets[a:a + 64].long()
            lp = x - torch.logsumexp(x, dim=1, keepdim=True)
            # near certainty: ln p = -ln(1 + the others' sum against it)
            best, where = x.max(dim=1, keepdim=True)
            rest = torch.exp(x - best).scatter(1, where, 0.0).sum(dim=1, keepdim=True)
            lp = (x - best) - torch.log1p(rest)
            p = torch.exp(lp)
            mine = torch.gather(lp, 1, t[:, None])
            outs[0].append(mine[:, 0])
            outs[1].append(-torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(dim=1))
            better = (x > torch.gather(x, 1, t[:, None])).sum(dim=1)
            same = x == torch.gather(x, 1, t[:, None])
            before = torch.cumsum(same, dim=1).gather(1, t[:, None])[:, 0] - 1
            outs[2].append((better + before).to(torch.int32))
            if case["top"]:
                order = torch.argsort(-x, dim=1, stable=True)[:, :case["top"]]
                outs[3].append(order.to(torch.int32))
                outs[4].append(torch.gather(lp, 1, order))
        return [torch.cat(o) for o in outs]
    if case["op"] == "attention":
        H, G, hd, first, count, shared, own_pages, pages, q = _attention_inputs(case, seed, DEV)
        cost = 4.0 * hd * H * sum(n * (f + n) for f, n in zip(first, count))
        if cost > 1.0e14:
            return None
        out, at = torch.empty(q.shape, dtype=torch.float64, device=DEV), 0
        heads = torch.arange(H, device=DEV) // (H // G)                    # the key/value head of every query head
        for f, n, mine in zip(first, count, own_pages):
            kv = pages[torch.tensor(shared + mine, device=DEV)].double()
            for h in range(H):
                g = int(heads[h])
                keys, values = kv[:, 0, g].reshape(-1, hd)[:f + n], kv[:, 1, g].reshape(-1, hd)[:f + n]
                s = q[at:at + n, h * hd:(h + 1) * hd].double() @ keys.T / math.sqrt(hd)
                seen = torch.ones(n, f + n, dtype=torch.bool, device=DEV).tril(diagonal=f)
                s = s.masked_fill(~seen, float("-inf"))
                out[at:at + n, h * hd:(h + 1) * hd] = torch.softmax(s, dim=1) @ values
            at += n
        return out
    if case["op"] == "tables":
        first, count = _lengths(case)
        _, shared, own_pages = _page_ids(case, seed, first, count)
        width = len(shared) + max(len(p) for p in own_pages)
        starts, positions, ids = [0], [], []
        for i, (f, n) in enumerate(zip(first, count)):
            starts.append(starts[-1] + n)
            positions += range(f, f + n)
            ids += [i] * n
        table = [shared + mine + [0] * (width - len(shared) - len(mine)) for mine in own_pages]
        return [torch.tensor(v, dtype=torch.int32, device=DEV)
                for v in (starts, [f + n for f, n in zip(first, count)], positions, ids, table)]
    state = prepare(case, seed)
    storage = state["storage"]
    for s, d in zip(state["sources"], state["targets"]):
        for layer in range(case["layers"]):
            storage[layer, d].copy_(storage[layer, s])
    return storage


# ------------------------------------------------------------------------------------------------ what a call cannot do without
def work(case):
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "float32" else 2
        # an exponential, two sums and a comparison with the target's logit for every logit
        return {"bytes": R * (V * size + 4 + 12 + 8 * case["top"]), "flops": 6 * R * V}
    if case["op"] == "attention":
        H, G, hd = HEADS[case["heads"]]
        first, count = _lengths(case)
        T, start = sum(count), case["shared"] * PAGE
        cached = start + sum(f + n - start for f, n in zip(first, count))
        pairs = sum(n * f + n * (n + 1) // 2 for f, n in zip(first, count))
        return {"bytes": 2 * (2 * T * H * hd + 2 * cached * G * hd), "flops": 4 * pairs * H * hd}
    if case["op"] == "tables":
        first, count = _lengths(case)
        need = [-(-(f + n) // PAGE) for f, n in zip(first, count)]
        B, T, P = len(first), sum(count), case["shared"]
        return {"bytes": 4 * (2 * B + P + sum(need) - B * P + 2 * B + 1 + 2 * T + B * max(need)), "flops": B + T}
    H, G, hd = HEADS[case["heads"]]
    return {"bytes": case["layers"] * 2 * G * PAGE * hd * 2 * (1 + case["forks"]), "flops": 0}
