"""Shaped scores and shared prefixes where planes are many (short walks dealt along a plane's tiles, one XCD to a plane) and
over caches with a capacity for each sequence, in every kernel."""
import random

import pytest
import torch

import ellm_amd
from shaped_util import D, check, rand, reference, slopes_of
from test_gpu_shaped_chunks import _ranges
from test_gpu_shaped_scores import BF16, F16, SCALE, Setup, _u32

pytestmark = pytest.mark.gpu

ALONG = [  # query heads, K/V heads, sequences, start, interval, prefix (tests/test_shaped_walks.py: short walks, along)
    (32, 4, 9, 300, 16, 0),      # 36 planes, 32 rows a workgroup
    (8, 1, 37, 30, 33, 0),       # 37 planes, 64 rows
    (8, 8, 9, 2100, 5, 0),       # 72 planes that overflow the caches
    (8, 1, 33, 30, 45, 50),      # 33 planes behind a prefix, 64 rows
    (36, 9, 5, 300, 5, 50),      # 45 planes behind a prefix, 32 rows
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scores", [dict(cap=30.0), dict(slopes=True, window=45)])
@pytest.mark.parametrize("hq,hkv,batch,start,interval,prefix", ALONG)
def test_short_walks_along_the_tiles_of_many_planes(hq, hkv, batch, start, interval, prefix, scores, dtype):
    t = Setup(91, dtype, hq, hkv, batch, interval, start + interval + 1, prefix=prefix)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    if prefix:
        t.op.set_shared_prefix(*t.prefix)
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, **scores), "along")


@pytest.mark.parametrize("hq,hkv,batch,start,interval,prefix", [c for c in ALONG if not c[-1]])
def test_key_ranges_along_the_tiles_of_many_planes(hq, hkv, batch, start, interval, prefix):
    cap = start + interval + 5
    t = Setup(92, F16, hq, hkv, batch, interval, cap)
    begin, end = _ranges(93, batch, start, interval, cap)
    t.op.set_scores(key_begin=_u32(begin, cap), key_end=_u32(end, cap))
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, begin=begin, end=end), "along, ranges")


class Ragged:
    """A cache whose sequences have capacities of their own, the operator over it, the same rows one plane a sequence."""

    def __init__(self, seed, dtype, hq, hkv, caps, interval, prefix=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.caps, batch = caps, len(caps)
        self.cache = ellm_amd.KVCache.ragged(1, caps, hkv, ellm_amd.DTYPE_F16 if dtype == F16 else ellm_amd.DTYPE_BF16)
        flat = self.cache.layer_flat_tensors(0, dtype)
        for x in flat:
            x.copy_(rand(gen, x.shape, dtype))
        self.k, self.v = (torch.full((batch, hkv, max(caps), D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        at = 0
        for i, c in enumerate(caps):
            self.k[i, :, :c], self.v[i, :, :c] = flat[0][:, at:at + c], flat[1][:, at:at + c]
            at += c
        self.q = rand(gen, (interval, batch, hq, D), dtype, 1.5)
        self.prefix = (rand(gen, (hkv, prefix, D), dtype), rand(gen, (hkv, prefix, D), dtype)) if prefix else None
        self.out, self.lse = torch.full_like(self.q, 7.0), torch.full((interval, batch, hq), 7.0, device="cuda")
        view = self.cache.layer_ragged(0)
        self.op = ellm_amd.Attention(self.q, *flat, self.out, batch, hq, hkv, D, view.strides, SCALE, lse=self.lse,
                                     seq_table=view, max_position_interval=interval)

    def check(self, first, what, **scores):
        torch.cuda.synchronize()
        if "end" in scores:   # a range ends at its sequence's capacity
            scores["end"] = [[min(e, c) for e in row] for row, c in zip(scores["end"], self.caps)]
        check(self.out, self.lse, reference(self.q, self.k, self.v, first, SCALE, prefix=self.prefix, **scores), what)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,start,interval", [
    (16, 2, 2, 300, 70),      # short walks of 32 rows a workgroup
    (64, 1, 6, 200, 45),      # of 64 rows
    (32, 4, 9, 300, 16),      # along
    (64, 1, 12, 0, 70),       # tiles
    (8, 1, 2, 2600, 9),       # tiles, split
])
def test_chunks_over_sequences_of_their_own_capacities(hq, hkv, batch, start, interval, dtype):
    """Ranges that end past a sequence's capacity stop there: the next sequence's rows lie behind it."""
    r = random.Random(94)
    caps = [start + interval + (0 if i == 1 else r.randrange(40)) for i in range(batch)]
    t = Ragged(95, dtype, hq, hkv, caps, interval)
    widest = max(caps)
    begin, end = _ranges(96, batch, start, interval, widest)
    for i, c in enumerate(caps):
        end[i][start + interval // 2] = 0xffffffff
        end[i][start] = c + 1 + r.randrange(30)
        begin[i][start] = 0
    slopes = slopes_of(hq)
    t.op.set_scores(slopes=slopes, key_begin=_u32(begin, widest), key_end=_u32(end, widest))
    t.op.run(start, interval, batch)
    t.check([start] * batch, "ranges", slopes=slopes, begin=begin, end=end)
    t.op.set_scores(cap=30.0)
    t.op.run(start, interval, batch)
    t.check([start] * batch, "capped", cap=30.0)


@pytest.mark.parametrize("hq,hkv,caps,start,interval,prefix", [
    (16, 2, [80, 50, 61], 10, 40, 150),            # short walks
    (32, 4, [40, 9], 0, 8, 5000),                  # prefix tiles and own tiles, joined
    (64, 1, [75] * 5 + [70] * 7, 0, 70, 3000),     # tiles over both
])
def test_chunks_behind_a_prefix_over_sequences_of_their_own_capacities(hq, hkv, caps, start, interval, prefix):
    t = Ragged(97, BF16, hq, hkv, caps, interval, prefix=prefix)
    t.op.set_scores(window=prefix + 20)
    t.op.set_shared_prefix(*t.prefix)
    t.op.run(start, interval, len(caps))
    t.check([start] * len(caps), "behind a prefix", window=prefix + 20)


@pytest.mark.parametrize("hq,hkv,batch,prefix,longest,scores", [
    (32, 4, 2, 2000, 70, dict(cap=30.0)),              # walk
    (32, 4, 12, 5000, 70, dict(slopes=True)),          # mixed
    (8, 4, 70, 801, 300, dict(window=900)),            # apart
    (32, 4, 24, 100, 5000, dict(slopes=True)),         # apart, shares
    (16, 2, 70, 0, 3000, dict(slopes=True, cap=9.0)),  # shares
])
def test_steps_over_sequences_of_their_own_capacities(hq, hkv, batch, prefix, longest, scores):
    """Positions past a sequence's capacity are taken as its last row, in every way of a step."""
    r = random.Random(98)
    caps = [max(1, int(longest * r.random() ** 2)) for _ in range(batch)]
    caps[batch // 2] = longest
    t = Ragged(99, F16, hq, hkv, caps, 1, prefix=prefix)
    positions = [longest - 1 if i % 3 == 0 else r.randrange(c) for i, c in enumerate(caps)]
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    if prefix:
        t.op.set_shared_prefix(*t.prefix)
    t.op.run_ragged(torch.tensor(positions, dtype=torch.int32, device="cuda"), longest - 1, batch)
    t.check([min(p, c - 1) for p, c in zip(positions, caps)], "step", **scores)
