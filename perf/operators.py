"""Attention with shaped scores, and over a prefix that a batch shares: cases, plain forms and exact values.

Two operators of the attention handle (``ellm_amd.Attention``), each for chunks of tokens and for single tokens:

  set_scores          x = scale q.k of the query at position p and the key at position j becomes
                          cap tanh(x / cap) - slope[head] |p - j|
                      and the query sees the keys begin <= j < end with p - j < window only (begin, end: one pair for
                      each query position; without them 0 and p + 1).  A row that sees no key is 0, its log-sum-exp -inf.
  set_shared_prefix   one plane of `length` keys and values a K/V head stands ahead of every sequence's own rows:
                      own row p is position length + p, all prefix rows are visible to all queries (inside the window).

Kinds of case: `chunk` (interval > 1 new tokens a sequence, position `start` on), `token` (one new token a sequence), `shared`
(either of them behind a shared prefix).  Head counts are those of the repository's configurations, heads 128 wide.
"""
import math
import random

import torch

own = False

D = 128
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(32, 4), (32, 32), (64, 8)]


def _case(kind, dtype, heads, batch, **more):
    case = dict(kind=kind, dtype=dtype, q_heads=heads[0], kv_heads=heads[1], batch=batch, start=0, interval=1,
                shortest=0, longest=0, len_seed=0, prefix=0, cap=0.0, slopes=False, window=0, mask="causal", lse=True)
    case.update(more)
    return case


def listed():
    return [
        # One conversation of a few hundred tokens, next token of a model that caps its scores: latency.
        dict(_case("token", "f16", (32, 4), 1, start=899, cap=50.0), name="token_capped_1x900"),
        # A serving batch at 8k tokens in a layer that sees the last 4096 of them only.
        dict(_case("token", "f16", (32, 4), 16, start=8191, cap=50.0, window=4096), name="token_window_16x8192"),
        # Continuous batching of conversations of very different lengths, scores falling with distance.
        dict(_case("token", "bf16", (32, 4), 24, shortest=500, longest=30000, len_seed=3, slopes=True, lse=False),
             name="token_slopes_24_of_500_to_30k"),
        # What is left of five prompts after their full chunks, nothing aligned.
        dict(_case("chunk", "bf16", (32, 4), 5, start=777, interval=33, cap=30.0), name="chunk_capped_33x5_on_777"),
        # A chunk appended to a long cache, scores falling with distance, no key older than 4096 positions.
        dict(_case("chunk", "bf16", (32, 32), 1, start=16000, interval=512, slopes=True, window=4096),
             name="chunk_slopes_window_512_on_16k"),
        # Two prompts whose beginning (an instruction, an image) is seen by all of its own positions.
        dict(_case("chunk", "f16", (64, 8), 2, interval=1000, mask="prefix", len_seed=5), name="prompt_prefix_1000x2"),
        # Documents packed into one row of a batch, padding behind the last one.
        dict(_case("chunk", "bf16", (32, 4), 2, interval=6001, mask="documents", len_seed=7, lse=False),
             name="prompt_documents_6001x2"),
        # A whole long prompt with capped scores: the largest call.
        dict(_case("chunk", "f16", (32, 4), 1, interval=8192, cap=50.0, lse=False), name="prompt_capped_8192"),
        # Four samples of one prompt, a few hundred tokens in: latency.
        dict(_case("shared", "f16", (32, 4), 4, prefix=2000, shortest=20, longest=500, len_seed=11),
             name="shared_4_on_2000"),
        # A serving batch behind one long system prompt.
        dict(_case("shared", "f16", (32, 4), 32, prefix=8192, shortest=64, longest=1024, len_seed=13),
             name="shared_32_on_8192"),
        # Many questions about one long document, scores capped.
        dict(_case("shared", "bf16", (64, 8), 128, prefix=32768, shortest=100, longest=2000, len_seed=17, cap=50.0,
                   lse=False), name="shared_capped_128_on_32k"),
        # The questions themselves: 40 tokens of each of 16 sequences behind the prompt they share.
        dict(_case("shared", "f16", (32, 4), 16, prefix=4100, interval=40), name="shared_chunk_40x16_on_4100"),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["token", "token", "chunk", "chunk", "shared", "shared_chunk"])
    heads = rng.choice(SHAPES)
    dtype = rng.choice(["f16", "bf16"])
    cap = rng.choice([0.0, 0.0, round(rng.uniform(10.0, 60.0), 1)])
    slopes = rng.random() < 0.35
    window = _log_int(rng, 100, 8000) if rng.random() < 0.35 else 0
    lse = rng.random() < 0.5
    more = dict(cap=cap, slopes=slopes, window=window, lse=lse, len_seed=rng.randrange(1 << 20))
    if kind == "token":
        batch = _log_int(rng, 1, 64)
        longest = _log_int(rng, 200, min(131072, 2097152 // batch // heads[1]))
        if rng.random() < 0.5:
            return _case(kind, dtype, heads, batch, start=longest - 1, **more)
        return _case(kind, dtype, heads, batch, shortest=_log_int(rng, 1, longest), longest=longest, **more)
    if kind == "chunk":
        batch = _log_int(rng, 1, 8)
        interval = _log_int(rng, 2, 4000 // batch)
        more["mask"] = rng.choice(["causal", "causal", "documents", "prefix"])
        start = _log_int(rng, 64, 16000 // batch) if more["mask"] == "causal" and rng.random() < 0.5 else 0
        if heads[0] * interval * (start + interval) * batch > 600000000:
            start = 0
        return _case(kind, dtype, heads, batch, start=start, interval=interval, **more)
    batch = _log_int(rng, 2, 96)
    prefix = _log_int(rng, 100, 32768)
    if kind == "shared":
        longest = _log_int(rng, 16, 2000)
        return _case(kind, dtype, heads, batch, prefix=prefix, shortest=_log_int(rng, 1, longest), longest=longest, **more)
    interval = _log_int(rng, 2, 1 + 600000000 // (heads[0] * batch * (prefix + 200)))
    return _case("shared", dtype, heads, batch, prefix=prefix, start=rng.choice([0, rng.randint(1, 200)]),
                 interval=min(interval, 600), **more)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _positions(case):
    """Per sequence, the position of its first new token among its own rows."""
    if not case["longest"]:
        return [case["start"]] * case["batch"]
    r = random.Random(case["len_seed"])
    return [r.randint(case["shortest"], case["longest"]) - 1 for _ in range(case["batch"])]


def _bounds(case):
    """Per sequence, (begin, end) of every query position; None without a mask of that kind."""
    if case["mask"] == "causal":
        return None
    r = random.Random(case["len_seed"] + 1)
    n, rows = case["interval"], []
    for _ in range(case["batch"]):
        if case["mask"] == "prefix":
            visible = r.randint(n // 8 + 1, n // 2 + 1)
            rows.append([(0, max(p + 1, visible)) for p in range(n)])
            continue
        row, used = [], n - r.randint(0, n // 8)
        while len(row) < used:
            begin, size = len(row), r.randint(max(1, n // 100), max(1, n // 4))
            row += [(begin, p + 1) for p in range(begin, min(used, begin + size))]
        rows.append(row + [(0, 0)] * (n - used))
    return rows


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, hq, hkv, batch = DTYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["batch"]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=gen)

    where = _positions(case)
    interval = case["interval"]
    last = max(where) + interval - 1
    capacity = (last + 1 + 255) // 256 * 256
    state = dict(case=case, where=where, last=last, q=normal(interval, batch, hq, D, scale=2.0),
                 k=normal(batch, hkv, capacity, D), v=normal(batch, hkv, capacity, D))
    state["positions"] = torch.tensor(where, dtype=torch.int32, device="cuda") if case["longest"] else None
    state["slopes"] = _slopes(hq) if case["slopes"] else None
    state["prefix_k"] = state["prefix_v"] = state["begin"] = state["end"] = None
    if case["prefix"]:
        state["prefix_k"], state["prefix_v"] = normal(hkv, case["prefix"], D), normal(hkv, case["prefix"], D)
    bounds = _bounds(case)
    if bounds:
        both = torch.zeros((2, batch, capacity), dtype=torch.int32)
        both[:, :, :interval] = torch.tensor(bounds, dtype=torch.int32).permute(2, 0, 1)
        state["begin"], state["end"] = both.cuda()
    if own:
        import ellm_amd

        out = torch.zeros_like(state["q"])
        lse = torch.zeros((interval, batch, hq), dtype=torch.float32, device="cuda") if case["lse"] else None
        op = ellm_amd.Attention(state["q"], state["k"], state["v"], out, batch, hq, hkv, D, state["k"].stride(),
                                1.0 / math.sqrt(D), lse=lse)
        op.set_scores(cap=case["cap"], slopes=state["slopes"], window=case["window"], key_begin=state["begin"],
                      key_end=state["end"])
        if case["prefix"]:
            op.set_shared_prefix(state["prefix_k"], state["prefix_v"], case["prefix"])
        state.update(op=op, out=out, lse=lse)
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        case = state["case"]
        if state["positions"] is not None:
            state["op"].run_ragged(state["positions"], state["last"], case["batch"])
        else:
            state["op"].run(case["start"], case["interval"], case["batch"])
        return {"out": state["out"]} if state["lse"] is None else {"out": state["out"], "lse": state["lse"]}
    return _plain(state)


def _visible(state, device):
    """Positions of the queries [batch, interval] and of the keys, and which keys each query sees [batch, interval, keys]
    (the prefix's first, then a sequence's own rows)."""
    case = state["case"]
    first = state["positions"].long() if state["positions"] is not None else torch.full((case["batch"],), case["start"], device=device)
    row = first[:, None] + torch.arange(case["interval"], device=device)
    prefix, keys = case["prefix"], state["last"] + 1
    j = torch.arange(prefix + keys, device=device)
    p = prefix + row
    end = p + 1
    begin = torch.zeros_like(p)
    if state["begin"] is not None:
        begin, end = (torch.gather(t.long(), 1, row) for t in (state["begin"], state["end"]))
    sees = (j >= begin[:, :, None]) & (j < end[:, :, None])
    if case["window"]:
        sees &= p[:, :, None] - j < case["window"]
    return p, j, sees


def _plain(state):
    case = state["case"]
    batch, s, hkv = case["batch"], case["interval"], case["kv_heads"]
    group = case["q_heads"] // hkv
    own_keys, prefix = state["last"] + 1, case["prefix"]
    q = state["q"].float().view(s, batch, hkv, group, D).permute(1, 2, 0, 3, 4).reshape(batch, hkv, s * group, D)
    k, v = state["k"][:, :, :own_keys].float(), state["v"][:, :, :own_keys].float()
    x = q @ k.transpose(-1, -2)
    if prefix:
        rows = q.transpose(0, 1).reshape(hkv, batch * s * group, D)
        ahead = (rows @ state["prefix_k"].float().transpose(-1, -2)).view(hkv, batch, s * group, prefix).transpose(0, 1)
        x = torch.cat([ahead, x], dim=-1)
    x = x.mul_(1.0 / math.sqrt(D)).view(batch, hkv, s, group, prefix + own_keys)
    if case["cap"]:
        x = x.mul_(1.0 / case["cap"]).tanh_().mul_(case["cap"])
    p, j, sees = _visible(state, x.device)
    if case["slopes"]:
        x = x - state["slopes"].view(hkv, 1, group, 1) * (p[:, :, None] - j).abs().float()[:, None, :, None, :]
    x = x.masked_fill_(~sees[:, None, :, None, :], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    weight = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(dim=-1, keepdim=True)
    weight = weight.view(batch, hkv, s * group, prefix + own_keys)
    y = weight[..., prefix:] @ v
    if prefix:
        rows = weight[..., :prefix].transpose(0, 1).reshape(hkv, batch * s * group, prefix)
        y = y + (rows @ state["prefix_v"].float()).view(hkv, batch, s * group, D).transpose(0, 1)
    y = y.view(batch, hkv, s, group, D) / torch.where(total == 0.0, 1.0, total)
    answer = {"out": y.permute(2, 0, 1, 3, 4).reshape(s, batch, hkv * group, D).to(state["q"].dtype)}
    if case["lse"]:
        answer["lse"] = (top + total.log()).squeeze(-1).permute(2, 0, 1, 3).reshape(s, batch, hkv * group)
    return answer


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should return
# ---------------------------------------------------------------------------------------------
def _ranges(case):
    """Per sequence and new token, the half-open range of positions (prefix rows first) that it sees."""
    bounds = _bounds(case)
    found = []
    for b, first in enumerate(_positions(case)):
        row = []
        for t in range(case["interval"]):
            p = case["prefix"] + first + t
            begin, end = bounds[b][t] if bounds else (0, p + 1)
            if case["window"]:
                begin = max(begin, p - case["window"] + 1)
            row.append((begin, max(begin, end)))
        found.append(row)
    return found


def work(case):
    ranges, prefix = _ranges(case), case["prefix"]
    pairs = sum(end - begin for row in ranges for begin, end in row)
    seen = [(begin, end) for row in ranges for begin, end in row if end > begin]
    keys = max([0] + [prefix - begin for begin, _ in seen]) if prefix else 0
    for row in ranges:
        live = [(begin, end) for begin, end in row if end > begin]
        if live:
            keys += max(end for _, end in live) - max(prefix, min(begin for begin, _ in live))
    tokens = case["interval"] * case["batch"]
    nbytes = 2 * keys * case["kv_heads"] * D * 2 + 2 * tokens * case["q_heads"] * D * 2
    nbytes += 4 * case["q_heads"] * (tokens if case["lse"] else 0) + (8 * tokens if case["mask"] != "causal" else 0)
    return {"bytes": nbytes, "flops": 4 * D * case["q_heads"] * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    out = torch.zeros((case["interval"], case["batch"], case["q_heads"], D), dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    for b, row in enumerate(_ranges(case)):
        begin, end = (torch.tensor(side, device="cuda")[:, None] for side in zip(*row))
        first, stop = int(begin.min()), max(int(begin.min()) + 1, int(end.max()))
        j = torch.arange(first, stop, device="cuda")
        p = case["prefix"] + state["where"][b] + torch.arange(case["interval"], device="cuda")[:, None]
        hidden = (j < begin) | (j >= end)
        for h in range(case["q_heads"]):
            kv = h // group
            k, v = state["k"][b, kv], state["v"][b, kv]
            if case["prefix"]:
                k, v = torch.cat([state["prefix_k"][kv], k]), torch.cat([state["prefix_v"][kv], v])
            x = state["q"][:, b, h].double() @ k[first:stop].double().T / math.sqrt(D)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - 2.0 ** (-8.0 * (h + 1) / case["q_heads"]) * (p - j).abs()
            x = x.masked_fill(hidden, -math.inf)
            total = torch.logsumexp(x, dim=-1)
            lse[:, b, h] = total
            weight = torch.exp(x - torch.where(total == -math.inf, 0.0, total)[:, None])
            out[:, b, h] = weight @ v[first:stop].double()
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
