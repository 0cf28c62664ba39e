"""A key/value cache in 8 bits: writing, reading back and attending over it.  Cases, plain forms and exact values.

A cache row (one position of a K/V head, 128 elements) is held as 128 values of the type e4m3 and one scale of the type
e8m0, a power of two.  With a = max |x| over the row:

  scale    the smallest 2^e with a <= 448 2^e, e >= -126
  element  x / 2^e rounded to the nearest e4m3, ties to even (values are first cut to 1.875 times the largest power of two
           of the type they come in, so that what is read back fits that type)

Five operators of the cache (``ellm_amd.KVCache``) and of attention over it (``ellm_amd.Attention``):

  write   new key and value rows to their positions, the keys RMS-normalised and rotated on the way or as they are
  read    rows back in 16 bits
  token   attention of one new token a sequence, sequences of one length or of many
  step    write of a new token's rows and attention over the cache that holds them, as one call
  chunk   causal attention of a chunk of new tokens

Head counts are those of the repository's configurations, heads 128 wide.
"""
import math
import random

import torch

own = False

D = 128
EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LARGEST = {"f16": 1.875 * 2.0 ** 15, "bf16": 1.875 * 2.0 ** 127}
SHAPES = [(32, 4), (32, 32), (64, 8)]


def _case(kind, dtype, heads, batch, **more):
    case = dict(kind=kind, dtype=dtype, q_heads=heads[0], kv_heads=heads[1], batch=batch, start=0, interval=1,
                shortest=0, longest=0, len_seed=0, norm=True, lse=True)
    case.update(more)
    return case


def listed():
    return [
        # The cache write of one layer for a whole long prompt.
        dict(_case("write", "f16", (32, 4), 1, interval=16384), name="write_prompt_16384"),
        # The cache write of a serving batch's next tokens, every sequence at a position of its own: latency.
        dict(_case("write", "bf16", (64, 8), 64, shortest=100, longest=4000, len_seed=3), name="write_token_64_of_100_to_4k"),
        # A conversation that moves to another cache.
        dict(_case("read", "f16", (32, 4), 1, interval=30000, start=101), name="read_30000_at_101"),
        # A few hundred rows of some sequences, as a program takes them for a kernel of its own: latency.
        dict(_case("read", "bf16", (64, 8), 6, interval=333, start=77), name="read_333x6_at_77"),
        # The next token of one conversation of a few hundred tokens: latency.
        dict(_case("token", "f16", (32, 4), 1, start=899), name="token_1x900"),
        # A serving batch in steady state.
        dict(_case("token", "f16", (32, 4), 16, start=8191), name="token_16x8192"),
        # Continuous batching of conversations of very different lengths.
        dict(_case("token", "bf16", (32, 4), 24, shortest=1000, longest=60000, len_seed=5, lse=False),
             name="token_24_of_1k_to_60k"),
        # A layer's cache write and attention for four conversations: latency.
        dict(_case("step", "f16", (32, 4), 4, start=1023), name="step_4x1024"),
        # The same for a serving batch of conversations between some hundred and 16k tokens.
        dict(_case("step", "bf16", (64, 8), 32, shortest=300, longest=16000, len_seed=7, lse=False),
             name="step_32_of_300_to_16k"),
        # What is left of five prompts after their full chunks, nothing aligned.
        dict(_case("chunk", "bf16", (32, 4), 5, start=777, interval=33), name="chunk_33x5_on_777"),
        # A chunk appended to a long cache, no heads in common.
        dict(_case("chunk", "bf16", (32, 32), 1, start=16000, interval=512, lse=False), name="chunk_512_on_16k"),
        # A whole long prompt: the largest call.
        dict(_case("chunk", "f16", (32, 4), 1, interval=8192, lse=False), name="prompt_8192"),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["write", "read", "token", "token", "step", "chunk", "chunk"])
    heads = rng.choice(SHAPES)
    dtype = rng.choice(["f16", "bf16"])
    more = dict(lse=rng.random() < 0.5, norm=rng.random() < 0.6, len_seed=rng.randrange(1 << 20))
    if kind == "chunk":
        batch = _log_int(rng, 1, 8)
        interval = _log_int(rng, 2, 4000 // batch)
        start = _log_int(rng, 1, 20000 // batch) if rng.random() < 0.6 else 0
        if heads[0] * interval * (start + interval) * batch > 600000000:
            start = 0
        return _case(kind, dtype, heads, batch, start=start, interval=interval, **more)
    batch = _log_int(rng, 1, 64)
    if kind == "read" or (kind == "write" and rng.random() < 0.6):
        interval = _log_int(rng, 1, 130000 // batch // heads[1])
        return _case(kind, dtype, heads, batch, start=rng.choice([0, rng.randint(1, 300)]), interval=interval, **more)
    rows = 300000 if kind == "write" else 2000000
    longest = _log_int(rng, 1 if kind != "token" else 100, min(100000, rows // batch // heads[1]))
    if rng.random() < 0.5 or kind == "write":
        more.update(shortest=_log_int(rng, 1, longest), longest=longest)
    return _case(kind, dtype, heads, batch, start=0 if more.get("longest") else longest - 1, **dict(more, norm=True))


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _positions(case):
    """Per sequence, the position of its first new token."""
    if not case["longest"]:
        return [case["start"]] * case["batch"]
    r = random.Random(case["len_seed"])
    return [r.randint(case["shortest"], case["longest"]) - 1 for _ in range(case["batch"])]


def _held(x, largest):
    """Rows of x [..., 128] as (elements, scales): e4m3 and e8m0."""
    x = x.float()
    top = x.abs().amax(dim=-1, keepdim=True)
    part, exponent = torch.frexp(top.double() / 1.75)
    exponent = (exponent - (part == 0.5).int() - 8).clamp_(min=-126)
    elements = torch.ldexp(x.clamp(-largest, largest).double(), -exponent).float().to(torch.float8_e4m3fn)
    return elements, (exponent + 127).to(torch.uint8).squeeze(-1).view(torch.float8_e8m0fnu)


def _rope(positions, dtype):
    """Rotary table [positions, 128], (cos, sin) interleaved."""
    rate = 1.0e6 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device="cuda") / D)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.stack([angle.cos(), angle.sin()], dim=-1).view(positions, D).to(dtype)


def _own_cache(state):
    """A cache of one layer with the state's rows, and its tensors."""
    import ellm_amd

    case = state["case"]
    code = ellm_amd.DTYPE_F16 if case["dtype"] == "f16" else ellm_amd.DTYPE_BF16
    cache = ellm_amd.KVCache(1, case["batch"], case["kv_heads"], state["capacity"], code, e4m3=True)
    tensors = dict(zip(("k", "v", "k_scale", "v_scale"), cache.layer_e4m3_tensors(0)))
    for name, t in tensors.items():
        t.view(torch.uint8).copy_(state[name].view(torch.uint8))
    return cache, tensors


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, hkv, batch = DTYPES[case["dtype"]], case["kv_heads"], case["batch"]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen)

    where = _positions(case)
    interval, kind = case["interval"], case["kind"]
    last = max(where) + interval - 1
    capacity = (last + 1 + 255) // 256 * 256
    state = dict(case=case, where=where, last=last, capacity=capacity)
    state["positions"] = torch.tensor(where, dtype=torch.int32, device="cuda") if case["longest"] else None
    if kind == "write":   # a cache that holds nothing yet
        for name in ("k", "v"):
            state[name] = torch.zeros((batch, hkv, capacity, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
            state[name + "_scale"] = torch.zeros((batch, hkv, capacity), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    else:
        for name, spread in (("k", 0.2), ("v", 0.7)):
            rows = normal(batch, hkv, capacity, D) * normal(batch, hkv, capacity, 1, scale=spread).exp_()
            state[name], state[name + "_scale"] = _held(rows.to(dtype), LARGEST[case["dtype"]])
            del rows
    if kind in ("write", "step"):
        state["k_src"] = normal(interval, batch, hkv, D, scale=3.0).to(dtype)
        state["v_src"] = (normal(interval, batch, hkv, D) * normal(interval, batch, hkv, 1, scale=0.7).exp_()).to(dtype)
        state["rope"] = _rope(last + 1, dtype)
    if kind in ("token", "step", "chunk"):
        state["q"] = normal(interval, batch, case["q_heads"], D, scale=2.0).to(dtype)
    if kind == "read":
        state["k_dst"] = torch.zeros((interval, batch, hkv, D), dtype=dtype, device="cuda")
        state["v_dst"] = torch.zeros_like(state["k_dst"])
    if own:
        import ellm_amd

        if kind in ("write", "read", "step"):
            state["cache"], tensors = _own_cache(state)
            state.update(tensors)
        if kind in ("token", "step", "chunk"):
            state["out"] = torch.zeros_like(state["q"])
            lse = torch.zeros((interval, batch, case["q_heads"]), dtype=torch.float32, device="cuda") if case["lse"] else None
            state["lse"] = lse
            state["op"] = ellm_amd.Attention(state["q"], state["k"], state["v"], state["out"], batch, case["q_heads"], hkv, D,
                                             state["k"].stride(), 1.0 / math.sqrt(D), lse=lse,
                                             kv_scales=(state["k_scale"], state["v_scale"]))
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    case, kind, batch = state["case"], state["case"]["kind"], state["case"]["batch"]
    ragged = dict(positions=state["positions"], max_position=state["last"]) if state["positions"] is not None else {}
    if kind == "write":
        if case["norm"]:
            state["cache"].append_norm_rope(0, case["start"], state["k_src"], state["v_src"], state["rope"], eps=EPS, **ragged)
        else:
            state["cache"].append(0, case["start"], state["k_src"], state["v_src"])
        return _rows_of(state)
    if kind == "read":
        state["cache"].read(0, case["start"], state["k_dst"], state["v_dst"])
        return {"k": state["k_dst"], "v": state["v_dst"]}
    if kind == "step":
        state["cache"].append_norm_rope_with_attention(0, state["op"], case["start"], state["k_src"], state["v_src"],
                                                       state["rope"], eps=EPS, **ragged)
    elif ragged:
        state["op"].run_ragged(state["positions"], state["last"], batch)
    else:
        state["op"].run(case["start"], case["interval"], batch)
    answer = _rows_of(state) if kind == "step" else {}
    answer["out"] = state["out"]
    if case["lse"]:
        answer["lse"] = state["lse"]
    return answer


def _rows_of(state):
    return {name: state[name] for name in ("k", "v", "k_scale", "v_scale")}


def _rows_at(state):
    """Position of every new token [batch, interval]."""
    case, device = state["case"], state["k"].device
    first = state["positions"].long() if state["positions"] is not None else torch.full((case["batch"],), case["start"], device=device)
    return first[:, None] + torch.arange(case["interval"], device=device)


def _write(state):
    case, at = state["case"], _rows_at(state)
    rows = {"k": state["k_src"].float(), "v": state["v_src"].float()}
    if case["norm"]:
        x = rows["k"]
        x = x / (x.square().mean(dim=-1, keepdim=True).sqrt() + EPS)
        turn = state["rope"].float()[at].transpose(0, 1)[:, :, None]   # [interval, batch, 1, 128]
        a, b, c, s = x[..., 0::2], x[..., 1::2], turn[..., 0::2], turn[..., 1::2]
        rows["k"] = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    sequence = torch.arange(case["batch"], device=at.device)[:, None]
    for name, x in rows.items():
        elements, scales = _held(x.transpose(0, 1), LARGEST[case["dtype"]])   # [batch, interval, heads, 128]
        state[name].view(torch.uint8)[sequence, :, at] = elements.view(torch.uint8)
        state[name + "_scale"].view(torch.uint8)[sequence, :, at] = scales.view(torch.uint8)


def _plain(state):
    case = state["case"]
    kind, batch, s, hkv = case["kind"], case["batch"], case["interval"], case["kv_heads"]
    group, keys = case["q_heads"] // hkv, state["last"] + 1
    if kind in ("write", "step"):
        _write(state)
    if kind == "write":
        return _rows_of(state)
    values = {name: state[name][:, :, :keys].float() * state[name + "_scale"][:, :, :keys, None].float() for name in ("k", "v")}
    if kind == "read":
        return {name: x[:, :, case["start"]:].permute(2, 0, 1, 3).to(DTYPES[case["dtype"]], memory_format=torch.contiguous_format)
                for name, x in values.items()}
    q = state["q"].float().view(s, batch, hkv, group, D).permute(1, 2, 0, 3, 4).reshape(batch, hkv, s * group, D)
    x = (q @ values["k"].transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(batch, hkv, s, group, keys)
    later = torch.arange(keys, device=q.device) > _rows_at(state)[:, :, None]
    x = x.masked_fill_(later[:, None, :, None, :], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    weight = x.sub_(top).exp_()
    total = weight.sum(dim=-1, keepdim=True)
    y = (weight.view(batch, hkv, s * group, keys) @ values["v"]).view(batch, hkv, s, group, D) / total
    answer = _rows_of(state) if kind == "step" else {}
    answer["out"] = y.permute(2, 0, 1, 3, 4).reshape(s, batch, hkv * group, D).to(state["q"].dtype)
    if case["lse"]:
        answer["lse"] = (top + total.log()).squeeze(-1).permute(2, 0, 1, 3).reshape(s, batch, hkv * group)
    return answer


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should return
# ---------------------------------------------------------------------------------------------
def work(case):
    where, s, hq, hkv, batch = _positions(case), case["interval"], case["q_heads"], case["kv_heads"], case["batch"]
    held, stored, tokens = D + 1, 2 * D, s * batch   # bytes of a row in the cache, in 16 bits
    nbytes = flops = 0
    if case["kind"] in ("write", "read"):
        nbytes = 2 * tokens * hkv * (held + stored)
        if case["kind"] == "write" and case["norm"]:
            nbytes += stored * (tokens if case["longest"] else s)
            flops = 8 * D * tokens * hkv
        return {"bytes": nbytes, "flops": flops}
    keys = sum(p + s for p in where)
    pairs = sum(s * p + s * (s + 1) // 2 for p in where)
    nbytes = 2 * keys * hkv * held + 2 * tokens * hq * stored + (4 * tokens * hq if case["lse"] else 0)
    if case["kind"] == "step":   # the new rows are written, not read
        nbytes += 2 * tokens * hkv * stored + stored * tokens
    return {"bytes": nbytes, "flops": 4 * D * hq * pairs}


def _exact_rows(case, state):
    """The new rows from their formulas: (values [batch, interval, heads, 128], 2^e) of k and of v, elements not rounded."""
    found = {}
    at = torch.tensor(state["where"], device="cuda")[:, None] + torch.arange(case["interval"], device="cuda")
    for name in ("k", "v"):
        x = state[name + "_src"].double().permute(1, 0, 2, 3)
        if name == "k" and case["norm"]:
            x = x / (torch.sqrt((x * x).sum(-1, keepdim=True) / D) + EPS)
            z = torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous())
            w = torch.view_as_complex(state["rope"].double()[at].view(*at.shape, 1, D // 2, 2))
            x = torch.view_as_real(z * w).flatten(-2)
        a = x.abs().amax(-1)
        e = torch.floor(torch.log2(a.clamp_min(1e-300))) - 9   # at most two below the exponent
        for _ in range(3):
            e = torch.where(a > 448.0 * torch.exp2(e), e + 1, e)
        e = e.clamp_min(-126)
        found[name] = (x.clamp(-LARGEST[case["dtype"]], LARGEST[case["dtype"]]), torch.exp2(e))
    return at, found


def exact(case, seed):
    state = prepare(case, seed)
    kind, batch, hq, hkv, s = case["kind"], case["batch"], case["q_heads"], case["kv_heads"], case["interval"]
    answer = {}
    if kind in ("write", "step"):
        at, rows = _exact_rows(case, state)
        for name, (x, scale) in rows.items():
            whole, scales = state[name].double(), state[name + "_scale"].double()
            for b in range(batch):
                whole[b, :, at[b]] = (x[b] / scale[b][..., None]).transpose(0, 1)
                scales[b, :, at[b]] = scale[b].transpose(0, 1)
            answer[name], answer[name + "_scale"] = whole, scales
        if kind == "write":
            return answer
        for name in ("k", "v"):   # attention is over what the cache then holds
            for b in range(batch):
                rounded = answer[name][b, :, at[b]].float().to(torch.float8_e4m3fn)
                state[name].view(torch.uint8)[b, :, at[b]] = rounded.view(torch.uint8)
                state[name + "_scale"].view(torch.uint8)[b, :, at[b]] = (torch.log2(answer[name + "_scale"][b, :, at[b]]) + 127).to(torch.uint8)
    if kind == "read":
        rows = slice(case["start"], case["start"] + s)
        return {name: (state[name][:, :, rows].double() * state[name + "_scale"][:, :, rows].double()[..., None]).permute(2, 0, 1, 3)
                for name in ("k", "v")}
    out = torch.zeros((s, batch, hq, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((s, batch, hq), dtype=torch.float64, device="cuda")
    for b, first in enumerate(state["where"]):
        n = first + s
        hidden = torch.arange(n, device="cuda") > first + torch.arange(s, device="cuda")[:, None]
        for h in range(hq):
            kv = h * hkv // hq
            k, v = (state[name][b, kv, :n].double() * state[name + "_scale"][b, kv, :n].double()[:, None] for name in ("k", "v"))
            x = (state["q"][:, b, h].double() @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
            lse[:, b, h] = torch.logsumexp(x, dim=-1)
            out[:, b, h] = torch.exp(x - lse[:, b, h, None]) @ v
    answer["out"] = out
    if case["lse"]:
        answer["lse"] = lse
    return answer
