"""Calls behind a shared prefix on the GPU where a window hides prefix rows, and where own rows are long and uneven."""
import pytest
import torch

from shaped_util import slopes_of
from test_gpu_shaped_scores import BF16, F16, Setup

pytestmark = pytest.mark.gpu


def _both(seed, dtype, hq, hkv, batch, interval, rows, prefix, scores):
    """The same own rows and scores, behind a prefix and without one."""
    with_prefix = Setup(seed, dtype, hq, hkv, batch, interval, rows, prefix=prefix)
    without = Setup(seed, dtype, hq, hkv, batch, interval, rows)
    for x in with_prefix.prefix:
        x.fill_(float("nan"))
    with_prefix.op.set_shared_prefix(*with_prefix.prefix)
    for t in (with_prefix, without):
        t.op.set_scores(**scores)
    return with_prefix, without


@pytest.mark.parametrize("dtype,hq,hkv,batch,prefix,start,interval,window", [
    (F16, 32, 4, 2, 100000, 1999, 1, 1000),
    (BF16, 32, 4, 12, 5000, 129, 1, 130),
    (F16, 8, 4, 70, 801, 200, 1, 100),
    (F16, 32, 4, 2, 32768, 1023, 64, 1024),
    (BF16, 8, 1, 1, 3000, 500, 300, 64),
    (F16, 32, 4, 2, 500, 0, 40, 1),
])
@pytest.mark.parametrize("slopes", [False, True])
def test_a_window_that_hides_the_whole_prefix_leaves_the_call_as_it_is_without_one(dtype, hq, hkv, batch, prefix, start,
                                                                                    interval, window, slopes):
    scores = dict(window=window, cap=30.0, slopes=slopes_of(hq) if slopes else None)
    a, b = _both(71, dtype, hq, hkv, batch, interval, start + interval + 2, prefix, scores)
    for t in (a, b):
        t.op.run(start, interval, batch)
    torch.cuda.synchronize()
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)
    a.prefix = None
    a.check(a.want([start] * batch, **scores), "hidden prefix")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,prefix,start,interval,window", [
    (32, 4, 2, 7001, 99, 1, 101),       # one prefix row left
    (8, 2, 12, 9000, 20, 1, 1500),
    (8, 4, 70, 5003, 200, 1, 1003),
    (16, 2, 3, 6007, 33, 9, 300),
    (8, 8, 2, 4000, 0, 150, 140),       # later tokens see none of it
])
def test_a_window_that_hides_a_part_of_the_prefix(dtype, hq, hkv, batch, prefix, start, interval, window):
    t = Setup(72, dtype, hq, hkv, batch, interval, start + interval + 2, prefix=prefix)
    hidden = prefix + start + 1 - window
    for x in t.prefix:
        x[:, :hidden] = float("nan")
    scores = dict(window=window, slopes=slopes_of(hq))
    t.op.set_scores(**scores)
    t.op.set_shared_prefix(*t.prefix)
    t.op.run(start, interval, batch)
    t.check(t.want([start] * batch, **scores), "even")
    if interval == 1:   # sequences of their own positions: the first of them sees window - 1 rows at most
        for x in t.prefix:
            x[:, :hidden] = 0.5
        first = [i * start // batch for i in range(batch)]
        t.op.run_ragged(torch.tensor(first, dtype=torch.int32, device="cuda"), start, batch)
        t.check(t.want(first, **scores), "ragged")


@pytest.mark.parametrize("dtype,hq,hkv,batch,prefix,longest,scores", [
    (F16, 32, 4, 24, 100, 5000, dict(cap=30.0)),
    (BF16, 16, 8, 20, 333, 4000, dict(slopes=True)),
    (F16, 8, 1, 200, 65, 3000, dict(window=2900)),
    (F16, 80, 2, 70, 1, 4000, dict()),
])
def test_a_short_prefix_ahead_of_long_uneven_own_rows(dtype, hq, hkv, batch, prefix, longest, scores):
    t = Setup(73, dtype, hq, hkv, batch, 1, longest + 1, prefix=prefix)
    scores = dict(scores, slopes=slopes_of(hq) if scores.get("slopes") else None)
    t.op.set_scores(**scores)
    t.op.set_shared_prefix(*t.prefix)
    first = [(i * i * longest) // (batch * batch) for i in range(batch)]
    first[batch // 2] = longest - 1
    positions = torch.tensor(first, dtype=torch.int32, device="cuda")
    for _ in range(2):
        t.out.fill_(7.0)
        t.op.run_ragged(positions, longest - 1, batch)
        t.check(t.want(first, **scores), "uneven own rows")
