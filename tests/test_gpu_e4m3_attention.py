"""Attention over planes in 8 bits against its definition in 64 bits, and what its handles take and refuse."""
import math

import pytest
import torch

import ellm_amd
from e4m3_util import CODE, D, LARGEST, hold, norm_rope, rope_table, rows, values
from shaped_util import check, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = 1.0 / math.sqrt(D)


class Setup:
    """A handle over random planes: [batch, heads, capacity, 128] contiguous unless `planes` says how to lay them out."""

    def __init__(self, seed, dtype, hq, hkv, batch, interval, capacity, spread=0.7, planes=lambda t: t, q_scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        held = [hold(rows(gen, (batch, hkv, capacity), dtype, spread), LARGEST[dtype]) for _ in range(2)]
        self.values = [values(*h).cuda() for h in held]
        self.codes = [planes(h[0].cuda()).view(torch.float8_e4m3fn) for h in held]
        strides = self.codes[0].stride()
        self.scales = []
        for (_, byte), codes in zip(held, self.codes):   # element x / 128 for the row that begins at x
            flat = torch.full((codes.untyped_storage().nbytes() // D,), 200, dtype=torch.uint8, device="cuda")
            at = flat[codes.storage_offset() // D:].as_strided(byte.shape, [s // D for s in strides[:3]])
            at.copy_(byte.cuda())
            self.scales.append(flat[codes.storage_offset() // D:].view(torch.float8_e8m0fnu))
        self.q = (torch.randn((interval, batch, hq, D), generator=gen) * q_scale).to(dtype).cuda()
        self.out = torch.full_like(self.q, 7.0)
        self.lse = torch.full(self.q.shape[:3], 7.0, dtype=torch.float32, device="cuda")
        self.op = ellm_amd.Attention(self.q, *self.codes, self.out, batch, hq, hkv, D, strides, SCALE, lse=self.lse,
                                     sequence_capacity=capacity, kv_scales=self.scales)

    def want(self, first, interval=None, batch=None):
        n, b = interval or self.q.shape[0], batch or self.q.shape[1]
        k, v = (x[:b].float() for x in self.values)   # (exact)
        return reference(self.q[:n, :b], k, v, first, SCALE)

    def check(self, first, what="", interval=None, batch=None):
        torch.cuda.synchronize()
        n, b = interval or self.q.shape[0], batch or self.q.shape[1]
        check(self.out[:n, :b], self.lse[:n, :b], self.want(first, n, b), what)
        assert (self.out[n:] == 7.0).all() and (self.out[:, b:] == 7.0).all() and (self.lse[:, b:] == 7.0).all()


HEADS = [(1, 1), (8, 4), (8, 1), (5, 1), (16, 1), (17, 1), (40, 2)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("keys", [1, 2, 31, 32, 33, 64, 100, 129, 257, 1000])
def test_single_tokens(dtype, hq, hkv, keys):
    t = Setup(keys + hq, dtype, hq, hkv, 2, 1, keys + 3)
    t.op.run(keys - 1, 1, 2)
    t.check([keys - 1] * 2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("batch,hq,hkv,lengths", [
    (1, 8, 1, [70]), (5, 8, 2, [1, 64, 65, 3, 500]), (70, 8, 4, [1 + 37 * i % 601 for i in range(70)]),
    (6, 16, 4, [9000, 1, 33, 4000, 128, 8999]), (300, 4, 4, [1 + 53 * i % 331 for i in range(300)]),
])
def test_single_tokens_at_positions_of_their_own(dtype, batch, hq, hkv, lengths):
    t = Setup(batch, dtype, hq, hkv, batch, 1, max(lengths) + 5)
    positions = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda")
    t.op.run_ragged(positions, max(lengths) + 4, batch)
    t.check([n - 1 for n in lengths])


def test_both_single_token_kernels_are_reached():
    t = Setup(4, F16, 8, 4, 16, 1, 9000)
    assert t.op.ragged_path(8999, 16) == 1 and t.op.ragged_path(100, 16) == 0
    positions = torch.tensor([8999 - 500 * i for i in range(16)], dtype=torch.int32, device="cuda")
    t.op.run_ragged(positions, 8999, 16)
    t.check(positions.tolist())
    first = t.out.clone()
    t.out.fill_(7.0)
    t.op.run_ragged(positions, 8999, 16)
    torch.cuda.synchronize()
    assert torch.equal(first, t.out)   # equal positions, equal bits


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,start,interval", [
    (1, 1, 1, 0, 2), (8, 1, 1, 0, 65), (8, 2, 3, 63, 2), (5, 1, 2, 0, 130), (40, 2, 1, 31, 33), (17, 1, 1, 100, 40),
    (8, 1, 1, 1500, 3), (8, 8, 2, 200, 129), (32, 4, 1, 0, 70), (16, 1, 5, 640, 9), (3, 3, 1, 5000, 17),
])
def test_chunks(dtype, hq, hkv, batch, start, interval):
    t = Setup(interval, dtype, hq, hkv, batch, interval, start + interval + 2)
    t.op.run(start, interval, batch)
    t.check([start] * batch)


def test_fewer_tokens_and_sequences_than_the_handle_has():
    t = Setup(12, BF16, 8, 2, 4, 50, 300)
    t.op.run(200, 37, 3)
    t.check([200] * 3, interval=37, batch=3)
    t.out.fill_(7.0), t.lse.fill_(7.0)
    t.op.run(290, 1, 2)
    t.check([290] * 2, interval=1, batch=2)
    t.op.run(0, 0, 4), t.op.run(0, 5, 0)   # nothing


def _permuted(t):   # [position][sequence][head][128]
    return t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)


def _apart(t):   # rows three rows apart, in a buffer that begins and ends elsewhere
    b, h, n, d = t.shape
    whole = torch.full((b, h, n, 3 * d), 0x7e, dtype=torch.uint8, device=t.device)
    whole[..., d:2 * d] = t
    return whole.view(-1)[d:].as_strided((b, h, n, d), (h * n * 3 * d, n * 3 * d, 3 * d, 1))


@pytest.mark.parametrize("planes", [_permuted, _apart])
@pytest.mark.parametrize("interval", [1, 40])
def test_any_strides_of_whole_rows(planes, interval):
    t = Setup(13, F16, 8, 2, 3, interval, 333, planes=planes)
    t.op.run(290, interval, 3)
    t.check([290] * 3)
    if interval == 1:
        t.op.run_ragged(torch.tensor([0, 332, 77], dtype=torch.int32, device="cuda"), 332, 3)
        t.check([0, 332, 77])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_and_small_scales(dtype):
    """Rows of one plane whose magnitudes are far apart, scores that are far apart."""
    t = Setup(14, dtype, 8, 2, 2, 20, 400, spread=2.0, q_scale=3.0)
    t.op.run(300, 20, 2)
    t.check([300] * 2)
    out = t.out[1:].clone()
    t.op.run(399, 1, 2)
    torch.cuda.synchronize()
    check(t.out[:1], t.lse[:1], t.want([399] * 2, 1))
    assert torch.equal(t.out[1:], out)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_row_that_is_nan_is_seen_by_those_that_see_its_key(dtype, which):
    """Queries before it are as without it: in a chunk, where the row is in their tile, and as single tokens."""
    t = Setup(15, dtype, 8, 2, 2, 90, 200)
    want = t.want([60, 60])
    bad = 60 + 41
    scales = t.scales[0 if which == "k_scale" else 1].view(torch.uint8).view(2, 2, 200)
    scales[1, 0, bad] = 255   # sequence 1, heads 0..3
    t.op.run(60, 90, 2)
    torch.cuda.synchronize()
    sees = torch.zeros(t.out.shape[:3], dtype=torch.bool, device="cuda")
    sees[41:, 1, :4] = True
    assert torch.isnan(t.out[sees]).all() and torch.isnan(t.lse[sees]).all()
    out, lse = t.out.clone(), t.lse.clone()
    out[sees], lse[sees] = want[0][sees].to(dtype), want[1][sees].float()
    check(out, lse, want, which)
    for first, nan in ((bad - 1, False), (bad, True), (bad + 70, True)):
        t.op.run(first, 1, 2)
        torch.cuda.synchronize()
        assert bool(torch.isnan(t.out[0, 1, :4]).all()) == nan and not torch.isnan(t.out[0, 0]).any() and not torch.isnan(t.out[0, 1, 4:]).any()


def test_rows_past_the_last_key_may_hold_anything():
    for interval in (1, 33):
        t = Setup(16, F16, 8, 2, 2, interval, 300)
        start = 133
        for x in (*t.codes, *t.scales):
            x.view(torch.uint8).view(2, 2, 300, -1)[:, :, start + interval:] = 255   # NaN
        t.op.run(start, interval, 2)
        t.check([start] * 2)


def test_the_result_is_that_over_the_rows_read_back():
    """The 16-bit operator over what the cache reads back, and this one, agree to the rounding of either."""
    t = Setup(17, F16, 8, 2, 2, 64, 500)
    k, v = (x.to(F16) for x in t.values)
    out, lse = torch.zeros_like(t.out), torch.zeros_like(t.lse)
    op = ellm_amd.Attention(t.q, k, v, out, 2, 8, 2, D, k.stride(), SCALE, lse=lse)
    for start, interval in ((400, 64), (499, 1)):
        t.op.run(start, interval, 2), op.run(start, interval, 2)
        torch.cuda.synchronize()
        want = t.want([start] * 2, interval)
        for got, got_lse in ((t.out, t.lse), (out, lse)):
            check(got[:interval], got_lse[:interval], want)


def _step(dtype, ragged, capacities=None, batch=5, hq=16, hkv=4, capacity=700, seed=20):
    gen = torch.Generator().manual_seed(seed)
    if capacities:
        cache = ellm_amd.KVCache.ragged(2, capacities, hkv, CODE[dtype], e4m3=True)
    else:
        cache = ellm_amd.KVCache(2, batch, hkv, capacity, CODE[dtype], e4m3=True)
    caps = capacities or [capacity] * batch
    start = [sum(caps[:i]) for i in range(batch)]
    k, v, ks, vs = cache.layer_e4m3_tensors(1)
    model = []   # the rows that the cache stands for, per sequence [heads, capacity, 128]
    for s in range(batch):
        for codes, byte in ((k, ks), (v, vs)):
            c, b = hold(rows(gen, (hkv, caps[s]), dtype), LARGEST[dtype])
            if capacities:
                codes.view(torch.uint8)[:, start[s]:start[s] + caps[s]] = c.cuda()
                byte.view(torch.uint8)[:, start[s]:start[s] + caps[s]] = b.cuda()
            else:
                codes.view(torch.uint8)[s], byte.view(torch.uint8)[s] = c.cuda(), b.cuda()
            model.append(values(c, b))
    q = torch.randn((1, batch, hq, D), generator=gen).to(dtype).cuda()
    out, lse = torch.full_like(q, 7.0), torch.full((1, batch, hq), 7.0, device="cuda")
    view = cache.layer_e4m3(1)
    op = ellm_amd.Attention(q, k, v, out, batch, hq, hkv, D, view.strides, SCALE, lse=lse, sequence_capacity=capacity,
                            max_position_interval=1, seq_table=view if capacities else None, kv_scales=(ks, vs))
    return cache, op, q, out, lse, model, caps, gen


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ragged,capacities", [(False, None), (True, None), (True, [300, 20, 700, 1, 450])])
def test_a_step_writes_the_rows_and_attends_over_them(dtype, ragged, capacities):
    batch, hq, hkv = 5, 16, 4
    cache, op, q, out, lse, model, caps, gen = _step(dtype, ragged, capacities)
    rope = rope_table(700, dtype)
    for turn in range(3):   # three tokens one after the other
        at = [min(c - 3, 90 + 50 * i) + turn if ragged else 333 + turn for i, c in enumerate(caps)]
        at = [max(0, min(p, c - 1)) for p, c in zip(at, caps)]
        ks, vs = (rows(gen, (1, batch, hkv), dtype) for _ in range(2))
        more = dict(positions=torch.tensor(at, dtype=torch.int32, device="cuda"), max_position=max(at)) if ragged else {}
        cache.append_norm_rope_with_attention(1, op, at[0], ks.cuda(), vs.cuda(), rope.cuda(), **more)
        torch.cuda.synchronize()
        new_k = values(*hold(norm_rope(ks, rope, torch.tensor([at]), 1e-6), LARGEST[dtype]))
        new_v = values(*hold(vs, LARGEST[dtype]))
        for s in range(batch):
            model[2 * s][:, at[s]], model[2 * s + 1][:, at[s]] = new_k[0, s], new_v[0, s]
            want = reference(q[:, s:s + 1], model[2 * s][None].cuda().float(), model[2 * s + 1][None].cuda().float(), [at[s]], SCALE)
            check(out[:, s:s + 1], lse[:, s:s + 1], want, f"sequence {s}, turn {turn}")


def test_a_recorded_step_is_replayed_with_positions_that_move_on():
    """Cache write, attention and the advance of the positions as a graph, each replay against the eager calls."""
    dtype, batch, hkv = BF16, 5, 4
    cache, op, q, out, lse, model, caps, gen = _step(dtype, True)
    other, eager, _, out2, lse2, *_ = _step(dtype, True)   # the same seed: the same rows
    eager_q = eager._keep[0]
    rope = rope_table(700, dtype).cuda()
    ks, vs = (torch.zeros((1, batch, hkv, D), dtype=dtype, device="cuda") for _ in range(2))
    first = torch.tensor([0, 100, 31, 64, 690], dtype=torch.int32, device="cuda")
    positions = first.clone()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        with ellm_amd.StepGraph(stream) as graph:
            cache.append_norm_rope_with_attention(1, op, 0, ks, vs, rope, positions=positions, max_position=699, stream=stream)
            ellm_amd.positions_advance(positions, 1, stream=stream)
    for turn in range(5):
        new = [rows(gen, (1, batch, hkv), dtype).cuda() for _ in range(3)]
        ks.copy_(new[0]), vs.copy_(new[1])
        q.copy_(torch.randn(q.shape, generator=gen).to(dtype)), eager_q.copy_(q)
        torch.cuda.synchronize()
        graph.launch(stream)
        stream.synchronize()
        other.append_norm_rope_with_attention(1, eager, 0, ks, vs, rope, positions=first + turn, max_position=699)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(cache.layer_e4m3_tensors(1), other.layer_e4m3_tensors(1)))
    graph.close()


def test_a_conversation():
    """A prompt in chunks and then single tokens, every call against the rows the cache then stands for."""
    dtype, hq, hkv, batch, capacity = F16, 8, 2, 2, 256
    gen = torch.Generator().manual_seed(30)
    cache = ellm_amd.KVCache(1, batch, hkv, capacity, CODE[dtype], e4m3=True)
    k, v, ks, vs = cache.layer_e4m3_tensors(0)
    rope = rope_table(capacity, dtype)
    q = torch.zeros((64, batch, hq, D), dtype=dtype, device="cuda")
    out = torch.zeros_like(q)
    op = ellm_amd.Attention(q, k, v, out, batch, hq, hkv, D, cache.layer_e4m3(0).strides, SCALE, sequence_capacity=capacity,
                            kv_scales=(ks, vs))
    model = [torch.zeros((batch, hkv, capacity, D), dtype=torch.float64) for _ in range(2)]
    for position, n in ellm_amd.schedule_calls(0, 150, 64, 155):
        new = [rows(gen, (n, batch, hkv), dtype) for _ in range(2)]
        q[:n] = torch.randn((n, batch, hq, D), generator=gen).to(dtype)
        cache.append_norm_rope(0, position, *(x.cuda() for x in new), rope.cuda())
        op.run(position, n, batch)
        torch.cuda.synchronize()
        at = position + torch.arange(n)
        turned = norm_rope(new[0], rope, at[:, None].expand(n, batch), 1e-6)
        for to, x in zip(model, (turned, new[1])):
            to[:, :, at] = values(*hold(x, LARGEST[dtype])).permute(1, 2, 0, 3)
        check(out[:n], None, reference(q[:n], *(x.cuda().float() for x in model), [position] * batch, SCALE), f"{n} at {position}")
    back = [torch.zeros((155, batch, hkv, D), dtype=dtype, device="cuda") for _ in range(2)]
    cache.read(0, 0, *back)
    for got, want in zip(back, model):
        assert torch.equal(got.cpu().double(), want[:, :, :155].permute(2, 0, 1, 3))


def test_refusals():
    t = Setup(40, F16, 8, 2, 2, 8, 64)
    E = ellm_amd.EllmError

    def refused(call, error=E):
        with pytest.raises(error):
            call()

    def made(**over):
        a = dict(q=t.q, k=t.codes[0], v=t.codes[1], scales=t.scales, strides=t.codes[0].stride(), cap=64)
        a.update(over)
        return ellm_amd.Attention(a["q"], a["k"], a["v"], torch.zeros_like(a["q"]), 2, 8, 2, D, a["strides"], SCALE,
                                  sequence_capacity=a["cap"], kv_scales=a["scales"])

    refused(lambda: made(scales=(t.scales[0][:-1].clone(), t.scales[1])), ValueError)
    refused(lambda: made(scales=[s.view(torch.uint8) for s in t.scales]), TypeError)
    refused(lambda: made(k=t.codes[0].view(torch.uint8)), TypeError)
    refused(lambda: made(q=t.q.float()), TypeError)
    refused(lambda: made(strides=(2 * 64 * D, 64 * D, 64, 1)))
    refused(lambda: made(cap=65), ValueError)
    refused(lambda: t.op.run(60, 8, 2))
    refused(lambda: t.op.run(0, 9, 2))
    refused(lambda: t.op.run(0, 1, 3))
    refused(lambda: t.op.set_scores(cap=30.0))
    refused(lambda: t.op.set_shared_prefix(torch.zeros((2, 4, D), dtype=F16, device="cuda"), torch.zeros((2, 4, D), dtype=F16, device="cuda")))
    refused(lambda: t.op.run_noalloc(3, 2), ValueError)
    # a cache and an operator that do not belong together
    cache, op, q, out, *_ = _step(F16, False)
    x, rope = torch.zeros((1, 5, 4, D), dtype=F16, device="cuda"), rope_table(700, F16).cuda()
    cache.append_norm_rope_with_attention(1, op, 3, x, x, rope)
    refused(lambda: cache.append_norm_rope_with_attention(0, op, 3, x, x, rope))   # another layer
    wide = ellm_amd.KVCache(2, 5, 4, 700, CODE[F16])
    refused(lambda: wide.append_norm_rope_with_attention(1, op, 3, x, x, rope))
    kt, vt = wide.layer_tensors(1, F16)
    plain = ellm_amd.Attention(q, kt, vt, out, 5, 16, 4, D, wide.layer(1)[2], SCALE)
    refused(lambda: cache.append_norm_rope_with_attention(1, plain, 3, x, x, rope))
    # a projection writes 16-bit rows
    w = torch.zeros((16 * D, 64), dtype=F16, device="cuda")
    proj = ellm_amd.MatMul3(torch.zeros((1, 5, 64), dtype=F16, device="cuda"), w, q, w, kt, w, vt, rope, D, 5, 16, 4, wide.layer(1)[2], 700)
    refused(lambda: proj.run_with_attention(op, 3, 5))
    assert proj.attention_path(plain, 5) in (0, 1)
    torch.cuda.synchronize()
