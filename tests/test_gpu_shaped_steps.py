"""Single-token steps with shaped scores or behind a shared prefix on the GPU where their kernels change over: many
sequences of uneven lengths, each way of a step behind a prefix, planes wider than 32-bit offsets, recorded steps."""
import math
import random

import pytest
import torch

import ellm_amd
from shaped_util import D, check, rand, reference, slopes_of
from test_gpu_shaped_scores import BF16, F16, SCALE, Setup, _u32

pytestmark = pytest.mark.gpu


def _positions(first):
    return torch.tensor(first, dtype=torch.int32, device="cuda")


def _lengths(seed, batch, longest):
    r = random.Random(seed)
    out = [max(1, int(longest * r.random() ** 2)) for _ in range(batch)]
    out[r.randrange(batch)], out[r.randrange(batch)] = longest, 1
    return out


# more than 64 sequences: the kernel that deals shares adds the lengths up in LDS
@pytest.mark.parametrize("dtype,hq,hkv,batch,longest,scores", [
    (F16, 8, 2, 100, 2500, dict(cap=30.0)),
    (BF16, 16, 2, 70, 3000, dict(slopes=True, window=700)),
    (F16, 12, 4, 40, 5000, dict(cap=8.0, slopes=True)),
    (BF16, 24, 1, 150, 3000, dict(window=129)),
    (F16, 20, 2, 80, 3000, dict(window=1)),
])
def test_many_sequences(dtype, hq, hkv, batch, longest, scores):
    t = Setup(31, dtype, hq, hkv, batch, 1, longest + 2)
    first = [n - 1 for n in _lengths(32, batch, longest)]
    assert t.op.ragged_path(max(first), batch) == 1
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    assert t.op.ragged_path(max(first), batch) == 2
    t.op.run_ragged(_positions(first), max(first), batch)
    t.check(t.want(first, **scores), "many sequences")


@pytest.mark.parametrize("extra", [dict(), dict(cap=30.0, slopes=True, window=900)])
def test_many_sequences_with_key_ranges(extra):
    batch, cap = 90, 2200
    t = Setup(33, F16, 8, 2, batch, 1, cap)
    r = random.Random(34)
    first = [n - 1 for n in _lengths(35, batch, 2000)]
    begin, end = [[0] * cap for _ in first], [[0] * cap for _ in first]
    for i, p in enumerate(first):
        lo = r.randrange(p + 1)
        begin[i][p], end[i][p] = r.choice([(lo, p + 1), (0, p + 1), (0, 0), (lo, lo), (p + 1, p), (0, lo), (lo, 0xffffffff)])
    scores = dict(extra, slopes=slopes_of(8) if extra.get("slopes") else None)
    t.op.set_scores(key_begin=_u32(begin, cap), key_end=_u32(end, cap), **scores)
    t.op.run_ragged(_positions(first), max(first), batch)
    t.check(t.want(first, begin=begin, end=end, **scores), "key ranges")
    empty = [i for i, p in enumerate(first) if begin[i][p] >= end[i][p]]
    assert empty and torch.count_nonzero(t.out[0, empty]) == 0


def test_many_sequences_at_one_position_with_key_ranges():
    batch, cap, at = 90, 2200, 1999
    t = Setup(61, BF16, 8, 2, batch, 1, cap)
    r = random.Random(62)
    begin, end = [[0] * cap for _ in range(batch)], [[0] * cap for _ in range(batch)]
    for i in range(batch):
        lo = r.randrange(at)
        begin[i][at], end[i][at] = r.choice([(lo, at + 1), (0, at + 1), (lo, lo), (lo, cap), (at, at + 1)])
    t.op.set_scores(key_begin=_u32(begin, cap), key_end=_u32(end, cap), cap=30.0)
    t.op.run(at, 1, batch)
    t.check(t.want([at] * batch, begin=begin, end=end, cap=30.0), "even step")


def test_a_short_prefix_of_more_rows_than_room():
    batch = 2100
    t = Setup(63, F16, 64, 1, batch, 1, 3, prefix=30)
    t.op.set_shared_prefix(*t.prefix)
    t.op.set_scores(slopes=slopes_of(64))
    t.op.run(2, 1, batch)
    t.check(t.want([2] * batch, slopes=slopes_of(64)), "one walk")


# walk: the prefix of all planes together is small.  mixed: few planes.  apart: many planes, or a large group, or much of
# the work behind the prefix; the last two rows have more rows than room for their partial results, and a single K/V row each.
WAYS = [  # query heads, K/V heads, sequences, prefix, longest, scores
    (32, 4, 2, 2000, 70, dict()),
    (8, 8, 64, 300, 130, dict(cap=30.0, window=200)),
    (32, 4, 12, 5000, 70, dict(cap=30.0)),
    (8, 8, 7, 3001, 700, dict(slopes=True, window=2900)),
    (8, 4, 70, 801, 300, dict(cap=50.0)),
    (16, 4, 66, 1000, 129, dict(slopes=True)),
    (80, 1, 8, 21000, 65, dict(cap=30.0)),
    (16, 4, 80, 700, 1500, dict(window=600)),
    (6, 2, 130, 2000, 2000, dict()),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,prefix,longest,scores", WAYS)
def test_ways_of_a_step_behind_a_prefix(dtype, hq, hkv, batch, prefix, longest, scores):
    t = Setup(36, dtype, hq, hkv, batch, 1, longest + 1, prefix=prefix)
    first = [n - 1 for n in _lengths(37, batch, longest)]
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.set_shared_prefix(*t.prefix)
    t.op.run_ragged(_positions(first), max(first), batch)
    t.check(t.want(first, **scores), "ragged step")
    t.op.run(longest - 1, 1, batch)
    t.check(t.want([longest - 1] * batch, **scores), "even step")


def test_more_rows_than_room_for_their_partial_results():
    batch, hq = 2100, 64
    t = Setup(38, F16, hq, 1, batch, 1, 3, prefix=130)
    t.op.set_shared_prefix(*t.prefix)
    first = [i % 3 for i in range(batch)]
    t.op.run_ragged(_positions(first), 2, batch)
    t.check(t.want(first), "walks of their own")


def test_planes_wider_than_32_bits():
    """Rows 2^23 elements apart: the last row of a plane lies 10 GB behind its first, the prefix's rows between them."""
    free, _ = torch.cuda.mem_get_info()
    if free < 16 * 2 ** 30:
        pytest.skip("needs 16 GB of free device memory")
    apart, rows, n_prefix, hq, hkv = 2 ** 23, 600, 500, 8, 2
    gen = torch.Generator(device="cuda")
    gen.manual_seed(39)
    room = torch.empty(apart * (rows - 1) + 4096, dtype=F16, device="cuda")
    k, v = (room.as_strided((1, hkv, rows, D), (8, D, apart, 1), at) for at in (0, hkv * D))
    pk, pv = (room.as_strided((hkv, n_prefix, D), (D, apart, 1), at) for at in (2 * hkv * D, 3 * hkv * D))
    for x in (k, v, pk, pv):
        x.copy_(rand(gen, x.shape, F16))
    q = rand(gen, (70, 1, hq, D), F16, 1.5)
    out, lse = torch.zeros_like(q), torch.zeros((70, 1, hq), device="cuda")
    op = ellm_amd.Attention(q, k, v, out, 1, hq, hkv, D, k.stride(), SCALE, lse=lse)
    for prefix in (None, (pk, pv)):
        for scores in (dict(cap=30.0), dict(slopes=slopes_of(hq))):
            op.set_shared_prefix(*(prefix or (None, None, 0)))
            op.set_scores(**scores)
            for start, interval in ((530, 70), (599, 1), (597, 3)):
                op.run(start, interval, 1)
                torch.cuda.synchronize()
                want = reference(q[:interval], k, v, [start], SCALE, prefix=prefix, **scores)
                check(out[:interval], lse[:interval], want, f"{start} + {interval}")


# walk, mixed, apart, and a step without a prefix that deals shares
@pytest.mark.parametrize("hq,hkv,batch,prefix,longest", [(32, 4, 2, 2000, 70), (32, 4, 12, 5000, 70), (8, 4, 70, 801, 300),
                                                         (8, 2, 100, 0, 2500)])
def test_two_recorded_steps_in_turn(hq, hkv, batch, prefix, longest):
    """Two handles' steps recorded apart and replayed in turn, with eager steps of the same handles between them."""
    steps = 3
    setups, graphs = [], []
    stream = torch.cuda.Stream()
    first = [n - 1 for n in _lengths(41, batch, longest)]
    for i in range(2):
        t = Setup(42 + i, F16, hq, hkv, batch, 1, longest + steps, prefix=prefix)
        t.op.set_scores(cap=20.0 + i)
        if prefix:
            t.op.set_shared_prefix(*t.prefix)
        t.positions = _positions(first)
        setups.append(t)
    stream.wait_stream(torch.cuda.current_stream())
    for t in setups:
        with ellm_amd.StepGraph(stream) as g:
            t.op.run_ragged(t.positions, longest + steps - 1, batch, stream=stream)
            ellm_amd.positions_advance(t.positions, stream=stream)
        graphs.append(g)
    # what a setter changes afterwards, the recorded step does not see
    setups[1].op.set_scores(cap=5.0)
    for step in range(steps):
        for i, (t, g) in enumerate(zip(setups, graphs)):
            g.launch()
            stream.synchronize()
            now = [p + step for p in first]
            t.check(t.want(now, cap=20.0 + i), f"replay {step} of {i}")
            got = t.out.clone()
            t.out.zero_()
            t.op.run_ragged(_positions(now), longest + steps - 1, batch)
            torch.cuda.synchronize()
            assert torch.equal(t.out, got) == (i == 0)


def test_chunk_and_step_recorded_with_key_ranges():
    n, cap, batch = 90, 128, 3
    t = Setup(45, BF16, 8, 2, batch, n, cap)
    begin, end = ([[(p // 40 * 40, p + 1)[side] for p in range(cap)] for _ in range(batch)] for side in (0, 1))
    tb, te = _u32(begin, cap), _u32(end, cap)
    t.op.set_scores(key_begin=tb, key_end=te)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with ellm_amd.StepGraph(stream) as g:
        t.op.run(0, n, batch, stream=stream)
    for step in range(3):   # the arrays are read by every run
        for i in range(batch):
            for p in range(cap):
                begin[i][p] = min(p, 10 * step + i)
        stream.wait_stream(torch.cuda.current_stream())
        tb.copy_(_u32(begin, cap))
        torch.cuda.synchronize()
        g.launch()
        stream.synchronize()
        t.check(t.want([0] * batch, begin=begin, end=end), f"replay {step}")


def test_prefix_alone_is_what_a_window_leaves_out():
    """A window shorter than the own rows: no prefix row is visible, whatever the prefix holds."""
    for batch, prefix in ((2, 500), (12, 5000), (70, 801)):
        t = Setup(46, F16, 8, 4, batch, 1, 200, prefix=prefix)
        t.prefix[0].fill_(float("nan"))
        t.prefix[1].fill_(float("inf"))
        t.op.set_shared_prefix(*t.prefix)
        t.op.set_scores(window=100)
        first = [100 + i % 90 for i in range(batch)]
        t.op.run_ragged(_positions(first), 199, batch)
        kept, t.prefix = t.prefix, None
        t.check(t.want(first, window=100), f"{batch} behind {prefix}")
        t.prefix = kept
        assert math.isfinite(float(t.out.float().abs().sum()))
