"""Chunks with shaped scores in every kernel that takes them (short walks on 32 or 64 rows a workgroup, tiles whole or split;
which call takes which is held by the CPU tests): scores, masks, empty rows, values that are not finite."""
import random

import pytest
import torch

import ellm_amd
from shaped_util import D, rand, reference, slopes_of
from test_gpu_shaped_scores import BF16, F16, SCALE, Setup, _u32

pytestmark = pytest.mark.gpu

CHUNKS = {  # query heads, K/V heads, sequences, start, interval
    "short 1": (16, 2, 2, 300, 70),
    "short 1, tails": (8, 2, 3, 30, 150),
    "short 2": (64, 1, 6, 200, 45),
    "short 2, tails": (64, 1, 9, 200, 33),
    "tiles": (64, 1, 12, 0, 70),
    "tiles, split": (8, 1, 2, 2600, 9),
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scores", [dict(cap=30.0), dict(slopes=True), dict(cap=12.0, slopes=True, window=45), dict(window=1),
                                    dict(window=1 << 40)])
@pytest.mark.parametrize("name", CHUNKS)
def test_scores(name, scores, dtype):
    hq, hkv, batch, start, interval = CHUNKS[name]
    t = Setup(51, dtype, hq, hkv, batch, interval, start + interval + 3)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.run(start, interval, batch)
    scores["window"] = min(scores.get("window", 0), 1 << 30)
    t.check(t.want([start] * batch, **scores), name)


def _ranges(seed, batch, start, interval, cap):
    """Key ranges of every kind: causal, documents, later keys too, empty, past the capacity."""
    r = random.Random(seed)
    begin, end = ([[0] * cap for _ in range(batch)] for _ in range(2))
    for i in range(batch):
        doc = 0
        for p in range(start, start + interval):
            if r.random() < 0.1:
                doc = r.randrange(p + 1)
            lo = r.randrange(cap)
            begin[i][p], end[i][p] = r.choice([(doc, p + 1)] * 6 + [(0, p + 1), (0, 0), (lo, lo), (lo, lo + 1), (cap - 1, 5),
                                                                    (lo, 0xffffffff), (0xffffffff, 0xffffffff)])
    return begin, end


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scores", [dict(), dict(cap=20.0, slopes=True, window=60)])
@pytest.mark.parametrize("name", CHUNKS)
def test_key_ranges(name, scores, dtype):
    hq, hkv, batch, start, interval = CHUNKS[name]
    cap = start + interval + 5
    t = Setup(52, dtype, hq, hkv, batch, interval, cap)
    begin, end = _ranges(53, batch, start, interval, cap)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(key_begin=_u32(begin, cap), key_end=_u32(end, cap), **scores)
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, begin=begin, end=end, **scores), name)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ranges", [False, True])
@pytest.mark.parametrize("name", CHUNKS)
def test_values_that_are_not_finite(name, ranges, dtype):
    """Infinities and NaN among the values reach the rows that see them and no others; what no row sees may hold anything."""
    hq, hkv, batch, start, interval = CHUNKS[name]
    cap = start + interval + 5
    t = Setup(54, dtype, hq, hkv, batch, interval, cap)
    begin = end = None
    scores = dict(window=40)
    if ranges:
        begin, end = _ranges(55, batch, start, interval, cap)
        t.op.set_scores(key_begin=_u32(begin, cap), key_end=_u32(end, cap), **scores)
    else:
        t.op.set_scores(**scores)
    sees = torch.zeros((interval, batch, cap), dtype=torch.bool)
    for i in range(batch):
        for n in range(interval):
            p = start + n
            lo = max(p - 39, begin[i][p] if begin else 0, 0)
            sees[n, i, lo:max(lo, min(end[i][p] if end else p + 1, cap))] = True
    clean_k, clean_v = t.k.clone(), t.v.clone()
    unseen = ~sees.any(0).cuda()
    assert unseen.any() or ranges   # (some keys past the last query are seen by a range of their own)
    t.k.transpose(1, 2)[unseen] = float("nan")
    t.v.transpose(1, 2)[unseen] = float("inf")
    odd = []
    for n, value in enumerate((float("inf"), float("-inf"), float("nan"))):
        for j in (start + 1 + 9 * n % interval, max(0, start + interval - 2 - 5 * n)):
            dim = (37 * n + j) % D
            t.v[:, :, j, dim] = value
            clean_v[:, :, j, dim] = 0.0
            odd.append((j, dim, value))
    t.op.run(start, interval, batch)
    torch.cuda.synchronize()
    out, _, tol, _ = reference(t.q, clean_k, clean_v, [start] * batch, SCALE, begin=begin, end=end, **scores)
    touched = torch.zeros((interval, batch, 1, D), dtype=torch.float64)   # what a row's sum comes to: inf - inf is NaN
    for j, dim, value in odd:
        touched[:, :, 0, dim] += torch.where(sees[:, :, j], torch.tensor(value, dtype=torch.float64), 0.0)
    touched = touched.expand(-1, -1, hq, -1).cuda()
    plain = touched == 0
    got = t.out.double()
    assert not plain.all() and plain.any()
    assert torch.isfinite(got[plain]).all()
    assert ((got - out).abs() <= tol)[plain].all()
    assert torch.equal(torch.isnan(got), torch.isnan(touched))
    bad = ~plain & ~torch.isnan(touched)
    assert torch.equal(got[bad], touched[bad])


@pytest.mark.parametrize("name", CHUNKS)
def test_rows_and_columns_around_the_call_stay(name):
    """A batch narrower than the handle's, position-major K and V, a recorded call replayed: the same bits as the eager one."""
    hq, hkv, batch, start, interval = CHUNKS[name]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(56)
    rows, pitch = start + interval + 1, batch + 2
    q = rand(gen, (interval + 1, pitch, hq, D), F16, 1.5)
    k, v = (rand(gen, (rows, pitch, hkv, D), F16).permute(1, 2, 0, 3) for _ in range(2))
    out, lse = torch.full_like(q, 7.0), torch.full((interval + 1, pitch, hq), 7.0, device="cuda")
    op = ellm_amd.Attention(q, k, v, out, pitch, hq, hkv, D, k.stride(), -SCALE, lse=lse)
    op.set_scores(cap=25.0)
    op.run(start, interval, batch)
    torch.cuda.synchronize()
    want = reference(q[:interval, :batch], k, v, [start] * batch, -SCALE, cap=25.0)
    assert ((out[:interval, :batch].double() - want[0]).abs() <= want[2]).all()
    assert ((lse[:interval, :batch].double() - want[1]).abs() <= want[3]).all()
    for x in (out, lse):
        assert (x[interval:] == 7.0).all() and (x[:, batch:] == 7.0).all()
    eager = out.clone(), lse.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with ellm_amd.StepGraph(stream) as g:
        op.run(start, interval, batch, stream=stream)
    for _ in range(3):
        out.fill_(7.0)
        lse.fill_(7.0)
        torch.cuda.synchronize()
        g.launch()
        stream.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


@pytest.mark.parametrize("scores", [dict(window=1100), dict(cap=200.0), dict(slopes=True)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_steep_scores_on_short_walks(dtype, scores):
    """Scores that rise or fall by hundreds over a walk: references move, earlier sums fade to nothing."""
    for step in (0.02, -0.02):
        t = Setup(57, dtype, 8, 1, 1, 64, 600)
        ramp = torch.arange(600, device="cuda", dtype=torch.float32) * step
        t.k[0, 0] = (ramp[:, None] * torch.ones(D, device="cuda")).to(dtype)
        t.q.fill_(2.0)
        more = dict(scores, slopes=slopes_of(8) if scores.get("slopes") else None)
        t.op.set_scores(**more)
        t.op.run(500, 64, 1)
        t.check(t.want([500], **more), f"ramp {step}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scores", [dict(), dict(cap=20.0, slopes=True), dict(window=70), dict(window=9, cap=30.0)])
@pytest.mark.parametrize("hq,hkv,batch,prefix,start,interval", [
    (8, 2, 2, 150, 10, 40), (64, 1, 13, 150, 0, 20), (32, 4, 2, 5000, 0, 9), (8, 2, 1, 1, 0, 33), (16, 1, 2, 32, 5, 64), (4, 4, 3, 65, 31, 2),
])
def test_short_walks_behind_a_prefix(hq, hkv, batch, prefix, start, interval, scores, dtype):
    t = Setup(58, dtype, hq, hkv, batch, interval, start + interval + 2, prefix=prefix)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.set_shared_prefix(*t.prefix)
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, **scores), "behind a prefix")


def test_prefix_rows_that_a_window_leaves_out_may_hold_anything():
    for batch, prefix, interval in ((2, 150, 40), (13, 150, 20)):
        t = Setup(59, F16, 64, 1, batch, interval, 100, prefix=prefix)
        for x in t.prefix:
            x[:, :-20] = float("nan")
        t.op.set_shared_prefix(*t.prefix)
        t.op.set_scores(window=20)
        t.op.run(0, interval, batch)
        for x in t.prefix:
            x[:, :-20] = 0.0
        t.check(t.want([0] * batch, window=20), f"{batch} sequences")
