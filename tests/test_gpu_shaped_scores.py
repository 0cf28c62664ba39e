"""Attention with shaped scores and over a shared prefix on the GPU, against the definition in 64 bits: sizes around the
tile edges, masks that leave rows empty, values nobody may see, strides, tables, graphs and streams."""
import math

import pytest
import torch

import ellm_amd
from shaped_util import D, check, rand, reference, slopes_of

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(D)
F16, BF16 = torch.float16, torch.bfloat16


def _u32(rows, cap):
    t = torch.zeros((len(rows), cap), dtype=torch.int32, device="cuda")
    for i, row in enumerate(rows):
        t[i, :len(row)] = torch.tensor([x - (1 << 32) if x >= 1 << 31 else x for x in row], dtype=torch.int32)
    return t


class Setup:
    """Inputs of a call and the operator over them."""

    def __init__(self, seed, dtype, hq, hkv, batch, interval, cap_rows, prefix=0, pitch=None, k_scale=1.0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.batch, self.interval, self.hq, self.hkv = batch, interval, hq, hkv
        pitch = pitch or batch
        self.q = rand(gen, (interval, pitch, hq, D), dtype, 1.5)
        self.k, self.v = rand(gen, (pitch, hkv, cap_rows, D), dtype, k_scale), rand(gen, (pitch, hkv, cap_rows, D), dtype)
        self.prefix = (rand(gen, (hkv, prefix, D), dtype, k_scale), rand(gen, (hkv, prefix, D), dtype)) if prefix else None
        self.out = torch.full_like(self.q, 7.0)
        self.lse = torch.full((interval, pitch, hq), 7.0, dtype=torch.float32, device="cuda")
        self.op = ellm_amd.Attention(self.q, self.k, self.v, self.out, pitch, hq, hkv, D, self.k.stride(), SCALE,
                                     lse=self.lse)

    def want(self, first, **scores):
        b = self.batch
        return reference(self.q[:, :b], self.k, self.v, first, SCALE, prefix=self.prefix, **scores)

    def check(self, want, what):
        torch.cuda.synchronize()
        return check(self.out[:, :self.batch], self.lse[:, :self.batch], want, what)


# ---- chunks ---------------------------------------------------------------------------------

CHUNKS = [  # dtype, query heads, K/V heads, batch, interval, start, scores
    (F16, 8, 1, 1, 2, 0, dict(cap=30.0)),
    (BF16, 8, 2, 2, 33, 77, dict(cap=50.0)),
    (F16, 6, 2, 1, 64, 64, dict(slopes=True)),
    (F16, 4, 4, 2, 129, 0, dict(slopes=True, cap=20.0)),
    (BF16, 16, 1, 1, 65, 300, dict(window=100)),
    (F16, 8, 1, 3, 7, 1000, dict(window=1)),
    (F16, 32, 4, 1, 70, 500, dict(window=64, slopes=True, cap=10.0)),
    (BF16, 5, 1, 1, 300, 13, dict(slopes=True, window=33)),
    (F16, 20, 1, 2, 3, 61, dict(cap=256.0)),
    (F16, 8, 8, 1, 200, 1800, dict(cap=0.5)),
]


@pytest.mark.parametrize("dtype,hq,hkv,batch,interval,start,scores", CHUNKS)
def test_chunk_against_the_definition(dtype, hq, hkv, batch, interval, start, scores):
    t = Setup(1, dtype, hq, hkv, batch, interval, start + interval + 9)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, **scores), "chunk")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("extra", [dict(), dict(cap=30.0, slopes=True), dict(window=40)])
def test_key_ranges_documents_prefixes_padding_and_empty_rows(dtype, extra):
    """Two sequences of 150 tokens: documents of 1, 70, 9 and 50 tokens and 20 padding rows; 40 rows that all see each
    other, then causal ones, with ranges that end ahead of where they begin and past the capacity in between."""
    n, cap = 150, 170
    t = Setup(2, dtype, 8, 2, 2, n, cap)
    docs = []
    for size in (1, 70, 9, 50):
        docs += [(len(docs), p + 1) for p in range(len(docs), len(docs) + size)]
    docs += [(0, 0)] * (n - len(docs))
    pre = [(0, max(p + 1, 40)) for p in range(n)]
    pre[50], pre[51], pre[52] = (60, 20), (0xffffffff, 52), (5, 0xffffffff)
    begin, end = ([[r[side] for r in rows] for rows in (docs, pre)] for side in (0, 1))
    scores = dict(extra, slopes=slopes_of(8) if extra.get("slopes") else None)
    t.op.set_scores(key_begin=_u32(begin, cap), key_end=_u32(end, cap), **scores)
    t.op.run(0, n, 2)
    want = t.want([0, 0], begin=begin, end=end, **scores)
    t.check(want, "ranges")
    assert torch.count_nonzero(t.out[130:, 0]) == 0 and (t.lse[130:, 0] == -math.inf).all()
    assert torch.count_nonzero(t.out[50:52, 1]) == 0
    # one of the two arrays alone
    t.op.set_scores(key_begin=_u32(begin, cap), **scores)
    t.op.run(0, n, 2)
    t.check(t.want([0, 0], begin=begin, **scores), "begin only")


def test_every_row_empty():
    t = Setup(3, F16, 8, 1, 2, 40, 64)
    t.op.set_scores(key_end=torch.zeros((2, 64), dtype=torch.int32, device="cuda"))
    t.op.run(0, 40, 2)
    torch.cuda.synchronize()
    assert torch.count_nonzero(t.out) == 0 and (t.lse == -math.inf).all()
    t.op.run(63, 1, 2)
    torch.cuda.synchronize()
    assert torch.count_nonzero(t.out[0]) == 0 and (t.lse[0] == -math.inf).all()


# ---- single tokens --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,lengths,scores", [
    (8, 1, [1], dict(cap=30.0)),
    (8, 2, [63, 64, 65], dict(slopes=True)),
    (32, 4, [900], dict(cap=50.0)),
    (3, 3, [1, 129, 1000, 2], dict(cap=50.0, slopes=True, window=100)),
    (20, 1, [5000, 17], dict(window=64)),
    (64, 8, [700, 1, 350], dict(window=1, cap=5.0)),
    (40, 2, [257, 2000], dict(slopes=True, window=1999)),
])
def test_single_token_of_uneven_lengths(dtype, hq, hkv, lengths, scores):
    t = Setup(4, dtype, hq, hkv, len(lengths), 1, max(lengths) + 3)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    first = [n - 1 for n in lengths]
    t.op.run_ragged(torch.tensor(first, dtype=torch.int32, device="cuda"), max(first), len(first))
    t.check(t.want(first, **scores), "ragged step")
    t.op.run(lengths[0] - 1, 1, len(lengths))
    t.check(t.want([lengths[0] - 1] * len(lengths), **scores), "even step")


def test_single_token_key_ranges():
    cap, lengths = 700, [600, 600, 1, 333]
    t = Setup(5, F16, 8, 2, 4, 1, cap)
    begin, end = [[0] * cap for _ in lengths], [[0] * cap for _ in lengths]
    for i, r in enumerate([(100, 601), (599, 600), (0, 0), (0, 700)]):   # later keys of the last one are visible too
        begin[i][lengths[i] - 1], end[i][lengths[i] - 1] = r
    t.op.set_scores(cap=20.0, key_begin=_u32(begin, cap), key_end=_u32(end, cap))
    first = [n - 1 for n in lengths]
    t.op.run_ragged(torch.tensor(first, dtype=torch.int32, device="cuda"), max(first), 4)
    t.check(t.want(first, cap=20.0, begin=begin, end=end), "ranges of single tokens")


# ---- shared prefix --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,prefix,lengths,scores", [
    (8, 1, 1, 1, [1], dict()),
    (8, 2, 3, 63, [1, 64, 65], dict(cap=30.0)),
    (32, 4, 4, 1000, [20, 1, 500, 130], dict()),
    (4, 4, 40, 64, None, dict(slopes=True)),
    (16, 2, 33, 257, None, dict(window=300)),
    (5, 1, 27, 65, None, dict(window=20, slopes=True, cap=8.0)),
    (64, 8, 2, 3000, [7, 2], dict(cap=50.0)),
])
def test_shared_prefix_single_token(dtype, hq, hkv, batch, prefix, lengths, scores):
    lengths = lengths or [1 + (37 * i) % 90 for i in range(batch)]
    t = Setup(6, dtype, hq, hkv, batch, 1, max(lengths) + 5, prefix=prefix)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.set_shared_prefix(*t.prefix)
    first = [n - 1 for n in lengths]
    t.op.run_ragged(torch.tensor(first, dtype=torch.int32, device="cuda"), max(first), batch)
    t.check(t.want(first, **scores), "shared prefix, ragged")
    t.op.run(lengths[0] - 1, 1, batch)
    t.check(t.want([lengths[0] - 1] * batch, **scores), "shared prefix, even")


@pytest.mark.parametrize("dtype,hq,hkv,batch,prefix,start,interval,scores", [
    (F16, 8, 1, 3, 100, 0, 2, dict()),
    (BF16, 8, 1, 5, 64, 3, 8, dict(cap=30.0)),
    (F16, 32, 4, 2, 500, 0, 40, dict()),
    (F16, 8, 8, 2, 129, 10, 64, dict(slopes=True)),
    (BF16, 8, 8, 1, 1, 0, 65, dict(window=40)),
    (F16, 4, 1, 2, 333, 20, 200, dict(slopes=True, cap=20.0, window=250)),
    (F16, 12, 2, 9, 70, 5, 10, dict(window=12)),
])
def test_shared_prefix_chunk(dtype, hq, hkv, batch, prefix, start, interval, scores):
    t = Setup(7, dtype, hq, hkv, batch, interval, start + interval + 3, prefix=prefix)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.set_shared_prefix(*t.prefix)
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, **scores), "shared prefix, chunk")


def test_part_of_a_longer_prefix_in_a_cache_layer_and_off_again():
    """The prefix as a slot of a cache layer, of which a part counts; without it and without scores the handle is the
    plain operator again, bit for bit."""
    t = Setup(8, F16, 8, 2, 4, 1, 200)
    plain = t.out.clone()
    t.op.run(150, 1, 4)
    plain.copy_(t.out)
    cache = torch.randn((3, 2, 400, D), device="cuda").to(F16)
    values = torch.randn((3, 2, 400, D), device="cuda").to(F16)
    t.op.set_shared_prefix(cache[1], values[1], 333)
    assert t.op.ragged_path(150, 4) == 2
    t.op.run(150, 1, 4)
    t.prefix = (cache[1, :, :333], values[1, :, :333])
    t.check(t.want([150] * 4), "part of a slot")
    t.op.set_shared_prefix()
    t.op.set_scores(cap=30.0)
    t.op.set_scores()
    assert t.op.ragged_path(150, 4) != 2
    t.op.run(150, 1, 4)
    torch.cuda.synchronize()
    assert torch.equal(t.out, plain)


# ---- what nobody may see or touch -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
def test_keys_and_values_that_are_not_seen_may_hold_anything(dtype, poison):
    """Chunks over documents (unseen rows inside a step that others see), ahead of a window, behind the last token, in
    the tail of the prefix: bit for bit what the same call gives on zeros there."""
    n, cap = 140, 160
    docs = [(0 if p < 50 else 50 if p < 90 else 90, p + 1 if p < 90 else 130) for p in range(n)]
    docs[100:120] = [(0, 0)] * 20
    begin, end = _u32([[r[0] for r in docs]], cap), _u32([[r[1] for r in docs]], cap)

    def run(bad):
        got = []
        t = Setup(9, dtype, 8, 1, 1, n, cap)
        t.k[:, :, 130:], t.v[:, :, 130:] = bad, bad      # behind every range
        t.op.set_scores(key_begin=begin, key_end=end, cap=20.0)
        t.op.run(0, n, 1)
        got += [t.out.clone(), t.lse.clone()]
        if bad == bad and not math.isinf(bad):
            t.check(t.want([0], cap=20.0, begin=[[r[0] for r in docs]], end=[[r[1] for r in docs]]), "documents")
        t = Setup(9, dtype, 8, 1, 1, n, cap)
        t.k[:, :, 20:30], t.v[:, :, 20:30] = bad, bad    # seen by rows 20 .. 49 only
        t.op.set_scores(key_begin=begin, key_end=end)
        t.op.run(0, n, 1)
        rows = list(range(20)) + list(range(50, n))
        got += [t.out[rows].clone(), t.lse[rows].clone()]
        t = Setup(9, dtype, 8, 1, 2, 1, cap, prefix=200)
        t.k[:, :, 41:], t.v[:, :, 41:] = bad, bad
        for x in t.prefix:
            x[:, 150:] = bad
            x[:, :20] = bad
        t.op.set_shared_prefix(*t.prefix, 150)
        t.op.set_scores(window=150)     # at own row 40: positions 41 .. 190
        t.op.run(40, 1, 2)
        got += [t.out.clone(), t.lse.clone()]
        torch.cuda.synchronize()
        return got

    clean, dirty = run(0.0), run(poison)
    for a, b in zip(clean, dirty):
        assert not torch.isnan(b).any()
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_and_nan_among_the_values_a_row_sees(dtype):
    """One value of key 30 an infinity, one of key 31 minus infinity, one of key 32 NaN, one column with both infinities:
    rows from there on show them in their columns, earlier rows and other columns do not."""
    n = 70
    t = Setup(10, dtype, 2, 1, 1, n, 80)
    t.v[0, 0, 30, 3], t.v[0, 0, 31, 40], t.v[0, 0, 32, 90] = math.inf, -math.inf, math.nan
    t.v[0, 0, 33, 127], t.v[0, 0, 34, 127] = math.inf, -math.inf
    t.op.set_scores(cap=20.0)
    t.op.run(0, n, 1)
    torch.cuda.synchronize()
    o = t.out[:, 0].float()
    assert torch.isfinite(o[:30]).all()
    assert (o[30:, :, 3] == math.inf).all() and (o[31:, :, 40] == -math.inf).all()
    assert torch.isnan(o[32:, :, 90]).all() and (o[33, :, 127] == math.inf).all() and torch.isnan(o[34:, :, 127]).all()
    fine = [c for c in range(D) if c not in (3, 40, 90, 127)]
    assert torch.isfinite(o[:, :, fine]).all()


def test_rows_of_sequences_outside_the_call_stay_as_they_were():
    t = Setup(11, F16, 8, 2, 3, 20, 64, pitch=5, prefix=30)
    t.op.set_scores(cap=30.0)
    for prefix in (None, t.prefix):
        if prefix:
            t.op.set_shared_prefix(*prefix)
        for start, interval in ((10, 20), (40, 1)):
            t.out.fill_(7.0)
            t.lse.fill_(7.0)
            t.op.run(start, interval, 3)
            torch.cuda.synchronize()
            assert (t.out[:, 3:] == 7.0).all() and (t.lse[:, 3:] == 7.0).all()
            assert (t.out[interval:] == 7.0).all() and (t.lse[interval:] == 7.0).all()
            assert not (t.out[:interval, :3] == 7.0).all(dim=-1).any()


@pytest.mark.parametrize("batch,interval", [(0, 5), (2, 0), (0, 1)])
def test_empty_calls(batch, interval):
    t = Setup(12, F16, 8, 1, 2, 5, 32, prefix=4)
    t.op.set_scores(cap=30.0)
    t.op.set_shared_prefix(*t.prefix)
    t.op.run(0, interval, batch)
    torch.cuda.synchronize()
    assert (t.out == 7.0).all()


# ---- layouts --------------------------------------------------------------------------------

def test_position_major_state_and_padded_strides():
    """K/V as [position][sequence][kv_head][128] (the state a projection leaves), rows 8 elements further apart; the
    prefix likewise."""
    hq, hkv, batch, n = 8, 2, 3, 100
    t = Setup(13, BF16, hq, hkv, batch, n, 120, prefix=90)
    wide = [torch.zeros((120, batch, hkv, D + 8), dtype=BF16, device="cuda") for _ in range(2)]
    ahead = [torch.zeros((90, hkv, D + 8), dtype=BF16, device="cuda") for _ in range(2)]
    for w, src in zip(wide, (t.k, t.v)):
        w[..., :D] = src.permute(2, 0, 1, 3)
    for w, src in zip(ahead, t.prefix):
        w[..., :D] = src.permute(1, 0, 2)
    k, v = (w[..., :D].permute(1, 2, 0, 3) for w in wide)
    op = ellm_amd.Attention(t.q, k, v, t.out, batch, hq, hkv, D, k.stride(), SCALE, lse=t.lse, sequence_capacity=120)
    for prefix in (False, True):
        if prefix:
            op.set_shared_prefix(*(w[..., :D].permute(1, 0, 2) for w in ahead))
        else:
            op.set_scores(cap=30.0)
        ref = t.prefix if prefix else None
        for start, interval in ((11, n), (99, 1)):
            op.run(start, interval, batch)
            torch.cuda.synchronize()
            want = reference(t.q[:interval], t.k, t.v, [start] * batch, SCALE, cap=30.0, prefix=ref)
            check(t.out[:interval], t.lse[:interval], want, f"strides, prefix {prefix}, {interval}")


def test_cache_with_a_capacity_for_each_sequence():
    caps, lengths, hq, hkv = [40, 300, 129], [40, 250, 1], 8, 2
    cache = ellm_amd.KVCache.ragged(1, caps, hkv, ellm_amd.DTYPE_F16)
    kt, vt = cache.layer_flat_tensors(0, F16)
    kt.normal_()
    vt.normal_()
    view = cache.layer_ragged(0)
    q = torch.randn((1, 3, hq, D), device="cuda").to(F16)
    out, lse = torch.zeros_like(q), torch.zeros((1, 3, hq), device="cuda")
    prefix = [torch.randn((hkv, 77, D), device="cuda").to(F16) for _ in range(2)]
    k, v = (torch.zeros((3, hkv, 300, D), dtype=F16, device="cuda") for _ in range(2))
    at = 0
    for i, c in enumerate(caps):
        k[i, :, :c], v[i, :, :c] = kt[:, at:at + c], vt[:, at:at + c]
        at += c
    op = ellm_amd.Attention(q, kt, vt, out, 3, hq, hkv, D, view.strides,
                            SCALE, lse=lse, seq_table=view, max_position_interval=1)
    first = [n - 1 for n in lengths]
    positions = torch.tensor([first[0] + 50, first[1], first[2]], dtype=torch.int32, device="cuda")   # clamped to its capacity
    op.set_scores(cap=30.0, slopes=slopes_of(hq))
    op.run_ragged(positions, 299, 3)
    torch.cuda.synchronize()
    check(out, lse, reference(q, k, v, first, SCALE, cap=30.0, slopes=slopes_of(hq)), "ragged cache")
    op.set_shared_prefix(*prefix)
    op.run_ragged(positions, 299, 3)
    torch.cuda.synchronize()
    check(out, lse, reference(q, k, v, first, SCALE, cap=30.0, slopes=slopes_of(hq), prefix=prefix), "ragged cache, prefix")


def test_scale_zero_and_negative():
    for scale in (0.0, -0.2):
        for scores in (dict(cap=10.0), dict(window=50), dict(slopes=slopes_of(8))):
            t = Setup(14, F16, 8, 1, 1, 70, 80)
            op = ellm_amd.Attention(t.q, t.k, t.v, t.out, 1, 8, 1, D, t.k.stride(), scale, lse=t.lse)
            op.set_scores(**scores)
            op.run(5, 70, 1)
            torch.cuda.synchronize()
            check(t.out, t.lse, reference(t.q, t.k, t.v, [5], scale, **scores), f"scale {scale}")


def test_scores_that_rise_and_fall_steeply():
    """Keys whose scores rise by hundreds along the walk, then fall: references move, sums stay finite."""
    for dtype in (F16, BF16):
        for step in (0.05, -0.05):
            t = Setup(15, dtype, 8, 1, 1, 64, 1200)
            ramp = torch.arange(1200, device="cuda", dtype=torch.float32) * step
            t.k[0, 0] = (ramp[:, None] * torch.ones(D, device="cuda")).to(dtype)
            t.q.fill_(1.0)
            for scores in (dict(window=1100), dict(cap=200.0)):
                t.op.set_scores(**scores)
                t.op.run(1100, 64, 1)
                t.check(t.want([1100], **scores), f"ramp {step} {dtype}")
                t.op.run(1163, 1, 1)
                torch.cuda.synchronize()
                want = reference(t.q[:1], t.k, t.v, [1163], SCALE, **scores)
                check(t.out[:1], t.lse[:1], want, f"ramp {step} {dtype} token")


# ---- graphs, streams, the calls that contain a run ------------------------------------------

def test_recorded_step_replayed_between_eager_calls():
    batch, prefix, cap = 6, 500, 40
    t = Setup(16, F16, 32, 4, batch, 1, cap, prefix=prefix)
    t.op.set_scores(cap=40.0)
    t.op.set_shared_prefix(*t.prefix)
    positions = torch.arange(batch, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with ellm_amd.StepGraph(stream) as g:
        t.op.run_ragged(positions, cap - 1, batch, stream=stream)
        ellm_amd.positions_advance(positions, stream=stream)
    for step in range(4):
        g.launch()
        stream.synchronize()
        got = t.out.clone(), t.lse.clone()
        t.check(t.want([i + step for i in range(batch)], cap=40.0), f"replay {step}")
        t.out.fill_(0.0)
        t.op.run_ragged(torch.arange(batch, dtype=torch.int32, device="cuda") + step, cap - 1, batch)
        torch.cuda.synchronize()
        assert torch.equal(t.out, got[0]) and torch.equal(t.lse, got[1])


def test_same_bits_every_time_and_on_another_stream():
    t = Setup(17, BF16, 8, 1, 2, 150, 1400, prefix=100)
    t.op.set_scores(cap=40.0, window=700)
    side = torch.cuda.Stream()
    for prefix in (False, True):
        if prefix:
            t.op.set_shared_prefix(*t.prefix)
        for start, interval in ((1200, 150), (1300, 1)):
            t.op.run(start, interval, 2)
            torch.cuda.synchronize()
            first = t.out.clone()
            t.out.zero_()
            side.wait_stream(torch.cuda.current_stream())
            t.op.run(start, interval, 2, stream=side)
            side.synchronize()
            assert torch.equal(t.out[:interval], first[:interval])


def _layer(hidden, hq, hkv, batch, interval, cap, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = rand(gen, (interval, batch, hidden), F16)
    w = [rand(gen, (h * D, hidden), F16, hidden ** -0.5) for h in (hq, hkv, hkv)]
    angle = torch.arange(2048, device="cuda", dtype=torch.float64)[:, None] * (1.0e6 ** (-2.0 * torch.arange(64, device="cuda") / D))
    rope = torch.stack((torch.cos(angle), torch.sin(angle)), dim=-1).reshape(2048, D).to(F16)
    return x, w, rope


@pytest.mark.parametrize("batch", [3, 70])
def test_projection_and_cache_writes_with_shaped_scores(batch):
    """The two combined calls with a handle that has shaped scores and a prefix: what the separate calls leave."""
    hidden, hq, hkv, cap, prefix = 1024, 8, 2, 64, 100
    x, w, rope = _layer(hidden, hq, hkv, batch, 1, cap, 18)
    t = Setup(18, F16, hq, hkv, batch, 1, cap, prefix=prefix)
    t.op.set_scores(cap=30.0)
    t.op.set_shared_prefix(*t.prefix)
    proj = ellm_amd.MatMul3(x, w[0], t.q, w[1], t.k, w[2], t.v, rope[prefix:], D, batch, hq, hkv, t.k.stride(), cap)
    assert proj.attention_path(t.op, batch) == 0
    positions = torch.tensor([i % cap for i in range(batch)], dtype=torch.int32, device="cuda")
    proj.run_ragged(positions, cap - 1, batch)
    t.op.run_ragged(positions, cap - 1, batch)
    torch.cuda.synchronize()
    want = [a.clone() for a in (t.q, t.k, t.v, t.out, t.lse)]
    t.check(t.want([i % cap for i in range(batch)], cap=30.0), "separate calls")
    for a in (t.q, t.out, t.lse):
        a.zero_()
    proj.run_with_attention(t.op, cap - 1, batch, positions=positions)
    torch.cuda.synchronize()
    for a, b in zip((t.q, t.k, t.v, t.out, t.lse), want):
        assert torch.equal(a, b)

    cache = ellm_amd.KVCache(1, batch, hkv, cap, ellm_amd.DTYPE_F16)
    kt, vt = cache.layer_tensors(0, F16)
    kt.copy_(t.k)
    vt.copy_(t.v)
    k, v, strides = cache.layer(0)
    op = ellm_amd.Attention(t.q, kt, vt, t.out, batch, hq, hkv, D, strides, SCALE, lse=t.lse, sequence_capacity=cap)
    op.set_scores(window=80)
    op.set_shared_prefix(*t.prefix)
    src = [torch.randn((1, batch, hkv, D), device="cuda").to(F16) for _ in range(2)]
    cache.append_norm_rope(0, 0, *src, rope[prefix:], positions=positions, max_position=cap - 1)
    op.run_ragged(positions, cap - 1, batch)
    torch.cuda.synchronize()
    want = [a.clone() for a in (kt, vt, t.out, t.lse)]
    kt.copy_(t.k)
    vt.copy_(t.v)
    t.out.zero_()
    cache.append_norm_rope_with_attention(0, op, 0, *src, rope[prefix:], positions=positions, max_position=cap - 1)
    torch.cuda.synchronize()
    for a, b in zip((kt, vt, t.out, t.lse), want):
        assert torch.equal(a, b)


def test_a_prompt_then_a_batch_behind_it():
    """The operators together, as a server uses them: a system prompt once through projection and capped attention into
    its own cache slot, then the questions of four requests and three new tokens of each behind it, against every request
    holding the whole text in its own rows."""
    hidden, hq, hkv, batch, prefix, question, cap = 1024, 16, 2, 4, 130, 21, 64
    x0, w, rope = _layer(hidden, hq, hkv, 1, prefix, cap, 19)
    system = ellm_amd.KVCache(1, 1, hkv, prefix, ellm_amd.DTYPE_F16)
    sk, sv = system.layer_tensors(0, F16)
    q0 = torch.zeros((prefix, 1, hq, D), dtype=F16, device="cuda")
    o0 = torch.zeros_like(q0)
    first = ellm_amd.MatMul3(x0, w[0], q0, w[1], sk, w[2], sv, rope, D, 1, hq, hkv, sk.stride(), prefix)
    att0 = ellm_amd.Attention(q0, sk, sv, o0, 1, hq, hkv, D, sk.stride(), SCALE)
    scores = dict(cap=30.0, slopes=slopes_of(hq), window=140)
    att0.set_scores(**scores)
    first.run(0, prefix, 1)
    att0.run(0, prefix, 1)
    torch.cuda.synchronize()
    check(o0, None, reference(q0, sk, sv, [0], SCALE, **scores), "system prompt")

    x, _, _ = _layer(hidden, hq, hkv, batch, question, cap, 20)
    k, v = (torch.zeros((batch, hkv, cap, D), dtype=F16, device="cuda") for _ in range(2))
    q = torch.zeros((question, batch, hq, D), dtype=F16, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros((question, batch, hq), device="cuda")
    proj = ellm_amd.MatMul3(x, w[0], q, w[1], k, w[2], v, rope[prefix:], D, batch, hq, hkv, k.stride(), cap)
    att = ellm_amd.Attention(q, k, v, out, batch, hq, hkv, D, k.stride(), SCALE, lse=lse)
    att.set_scores(**scores)
    att.set_shared_prefix(sk[0], sv[0])
    for start, interval in ((0, question), (question, 1), (question + 1, 1), (question + 2, 1)):
        if interval == 1:
            proj.run_with_attention(att, start, batch)
        else:
            proj.run(start, interval, batch)
            att.run(start, interval, batch)
        torch.cuda.synchronize()
        whole = [torch.cat([a[0][None].expand(batch, -1, -1, -1), c], dim=2) for a, c in ((sk, k), (sv, v))]
        want = reference(q[:interval], *whole, [prefix + start] * batch, SCALE, **scores)
        check(out[:interval], lse[:interval], want, f"request, {interval} at {start}")


# ---- refusals -------------------------------------------------------------------------------

def test_refusals():
    t = Setup(20, F16, 8, 2, 2, 4, 64, prefix=16)
    pk, pv = t.prefix
    bad = [
        lambda: t.op.set_scores(cap=-1.0), lambda: t.op.set_scores(cap=float("nan")), lambda: t.op.set_scores(cap=1e-5),
        lambda: t.op.set_scores(cap=257.0), lambda: t.op.set_scores(cap=float("inf")),
        lambda: t.op.set_shared_prefix(pk[..., 4:], pv[..., 4:]), lambda: t.op.set_shared_prefix(pk[:1], pv[:1]),
        lambda: t.op.set_shared_prefix(pk, pv, 17), lambda: t.op.set_shared_prefix(pk, pv, -1),
        lambda: t.op.set_shared_prefix(pk.to(BF16), pv.to(BF16)), lambda: t.op.set_shared_prefix(pk.cpu(), pv.cpu()),
        lambda: t.op.set_shared_prefix(pk, None), lambda: t.op.set_shared_prefix(pk, pv[:, ::2]),
        lambda: t.op.set_shared_prefix(pk.transpose(1, 2), pv.transpose(1, 2)),
        lambda: t.op.set_scores(slopes=slopes_of(7)), lambda: t.op.set_scores(slopes=slopes_of(8).double()),
        lambda: t.op.set_scores(slopes=slopes_of(8).cpu()),
        lambda: t.op.set_scores(key_end=torch.zeros((2, 63), dtype=torch.int32, device="cuda")),
        lambda: t.op.set_scores(key_end=torch.zeros((1, 64), dtype=torch.int32, device="cuda")),
        lambda: t.op.set_scores(key_end=torch.zeros((2, 64), dtype=torch.int64, device="cuda")),
        lambda: t.op.set_scores(key_begin=torch.zeros((2, 64), dtype=torch.int32, device="cuda"),
                                key_end=torch.zeros((2, 65), dtype=torch.int32, device="cuda")),
        lambda: t.op.set_scores(window=-1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, ellm_amd.EllmError, OverflowError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert t.op.ragged_path(10, 2) != 2   # nothing of it stuck
    ranges = torch.zeros((2, 64), dtype=torch.int32, device="cuda")
    t.op.set_scores(key_begin=ranges)
    with pytest.raises(ellm_amd.EllmError) as e:
        t.op.set_shared_prefix(pk, pv)
    assert e.value.status == 2
    t.op.set_scores()
    t.op.set_shared_prefix(pk, pv)
    with pytest.raises(ellm_amd.EllmError) as e:
        t.op.set_scores(key_begin=ranges)
    assert e.value.status == 2
    # other head sizes and binary32
    for d, dtype in ((64, F16), (128, torch.float32)):
        q = torch.zeros((1, 1, 2, d), dtype=dtype, device="cuda")
        k = torch.zeros((1, 1, 8, d), dtype=dtype, device="cuda")
        op = ellm_amd.Attention(q, k, k, torch.zeros_like(q), 1, 2, 1, d, k.stride(), 1.0)
        with pytest.raises(ellm_amd.EllmError) as e:
            op.set_scores(cap=30.0)
        assert e.value.status == 2
    # the raw entry point: pitch, alignment, strides
    lib, h = t.op._lib, t.op._handle
    assert lib.ellm_attn_set_scores(h, 0.0, None, 0, ranges.data_ptr(), None, 63) == 1
    assert lib.ellm_attn_set_scores(h, 0.0, ranges.data_ptr() + 2, 0, None, None, 0) == 1
    for k, v, hs, ps, n in ((None, pv.data_ptr(), 2048, 128, 16), (pk.data_ptr() + 2, pv.data_ptr(), 2048, 128, 16),
                            (pk.data_ptr(), pv.data_ptr(), 2048, 120, 16), (pk.data_ptr(), pv.data_ptr(), 2044, 128, 16),
                            (pk.data_ptr(), pv.data_ptr(), 0, 128, 16)):
        assert lib.ellm_attn_set_shared_prefix(h, k, v, hs, ps, n) == 1
    assert lib.ellm_attn_set_shared_prefix(h, pk.data_ptr(), pv.data_ptr(), 2048, (1 << 24) + 8, 16) == 2
    assert lib.ellm_attn_set_shared_prefix(h, pk.data_ptr(), pv.data_ptr(), 2048, 128, 0x7fffffff - 63) == 3
