"""Steps over caches in 8 bits where one launch writes the new rows and attends over them: the cache bit for bit as the write
alone leaves it, and the attention of the cache as it then stands."""
import ctypes
import math

import pytest
import torch

import ellm_amd
from e4m3_util import CODE, D, LARGEST, hold, rope_table, rows, values
from shaped_util import check, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = 1.0 / math.sqrt(D)


class Layer:
    """A cache whose rows are random codes (no NaN among them) and scales 2^-9 .. 2^-6, and a handle over it."""

    def __init__(self, seed, dtype, hq, hkv, capacities, uniform=False, scale=SCALE, layers=1, interval=1):
        self.dtype, self.hq, self.hkv, self.caps, self.uniform, self.layers = dtype, hq, hkv, capacities, uniform, layers
        batch = len(capacities)
        if uniform:
            self.cache = ellm_amd.KVCache(layers, batch, hkv, capacities[0], CODE[dtype], e4m3=True)
        else:
            self.cache = ellm_amd.KVCache.ragged(layers, capacities, hkv, CODE[dtype], e4m3=True)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for codes, byte in self.tensors():
            codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, device="cuda").to(torch.uint8))
            codes[(codes & 127) == 127] = 0
            byte.copy_(torch.randint(118, 122, byte.shape, generator=gen, device="cuda").to(torch.uint8))
        view = self.cache.layer_e4m3(layers - 1)
        k, v, ks, vs = self.cache.layer_e4m3_tensors(layers - 1)
        self.q = torch.randn((interval, batch, hq, D), generator=gen, device="cuda").to(dtype)
        self.out, self.lse = torch.full_like(self.q, 7.0), torch.full(self.q.shape[:3], 7.0, device="cuda")
        self.op = ellm_amd.Attention(self.q, k, v, self.out, batch, hq, hkv, D, view.strides, scale, lse=self.lse,
                                     sequence_capacity=max(capacities), max_position_interval=interval,
                                     seq_table=None if uniform else view, kv_scales=(ks, vs))
        self.scale = scale

    def tensors(self):
        k, v, ks, vs = (t.view(torch.uint8) for t in self.cache.layer_e4m3_tensors(self.layers - 1))
        return (k, ks), (v, vs)

    def plane(self, s):
        """K and V of sequence s as the cache holds them, [1, heads, capacity, 128] in 32 bits (exact)."""
        at = sum(self.caps[:s])
        part = (lambda t: t[s]) if self.uniform else (lambda t: t[:, at:at + self.caps[s]])
        return [values(part(c), part(b)).float()[None] for c, b in self.tensors()]

    def check(self, positions, what=""):
        torch.cuda.synchronize()
        for s, p in enumerate(positions):
            k, v = self.plane(s)
            n = p + self.q.shape[0]
            want = reference(self.q[:, s:s + 1], k[:, :, :n], v[:, :, :n], [p], self.scale)
            check(self.out[:, s:s + 1], self.lse[:, s:s + 1], want, f"{what} sequence {s}")


def _new(seed, batch, hkv, dtype, tokens=1):
    gen = torch.Generator().manual_seed(seed)
    return [rows(gen, (tokens, batch, hkv), dtype, 0.5).cuda() for _ in range(2)]


def _same_bits(a, b):
    torch.cuda.synchronize()
    return all(torch.equal(x, y) for m, n in zip(a.tensors(), b.tensors()) for x, y in zip(m, n))


CASES = [
    (4, 1, [1], [0]),                                    # the first token
    (8, 8, [3, 1, 40], [0, 0, 0]),
    (5, 1, [33, 34, 32, 65], [32, 33, 31, 64]),          # the new key begins a chunk, or ends one
    (40, 2, [400, 129, 1, 300], [399, 128, 0, 7]),       # twenty heads a group
    (16, 1, [6000], [5777]),                             # many workgroups to a plane
    (17, 1, [6000, 40], [5999, 39]),
    (64, 8, [3000, 100, 7], [2999, 5, 6]),
    (8, 4, [9000 - 200 * i for i in range(16)], [8990 - 500 * i for i in range(16)]),   # shares of different planes
    (32, 4, [9000] * 16, [8999] * 16),
    (40, 2, [9000] * 9, [8700, 31, 0, 8999, 8000, 1, 8992, 8991, 100]),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,capacities,positions", CASES)
def test_a_step_with_positions_of_their_own(dtype, hq, hkv, capacities, positions):
    batch, most = len(capacities), max(positions)
    step, apart = (Layer(50, dtype, hq, hkv, capacities, layers=2) for _ in range(2))
    k, v = _new(51, batch, hkv, dtype)
    rope = rope_table(most + 1, dtype).cuda()
    at = torch.tensor(positions, dtype=torch.int32, device="cuda")
    step.cache.append_norm_rope_with_attention(1, step.op, 0, k, v, rope, positions=at, max_position=most)
    apart.cache.append_norm_rope(1, 0, k, v, rope, positions=at, max_position=most)
    assert _same_bits(step, apart)
    step.check(positions)


def test_the_cases_reach_both_kernels():
    paths = {Layer(50, F16, hq, hkv, capacities).op.ragged_path(max(positions), len(capacities))
             for hq, hkv, capacities, positions in CASES}
    assert paths == {0, 1}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,position", [(4, 1, 1, 0), (8, 2, 3, 31), (8, 2, 3, 32), (34, 2, 2, 1000), (16, 1, 1, 5999),
                                                   (64, 8, 16, 3000)])
def test_a_step_at_one_position(dtype, hq, hkv, batch, position):
    step, apart = (Layer(52, dtype, hq, hkv, [position + 2] * batch, uniform=True) for _ in range(2))
    k, v = _new(53, batch, hkv, dtype)
    rope = rope_table(position + 1, dtype).cuda()
    step.cache.append_norm_rope_with_attention(0, step.op, position, k, v, rope)
    apart.cache.append_norm_rope(0, position, k, v, rope)
    assert _same_bits(step, apart)
    step.check([position] * batch)


@pytest.mark.parametrize("batch,position", [(3, 100), (16, 8999)])
def test_new_rows_that_are_not_finite(batch, position):
    """They read as NaN from then on, in their own sequence and group of heads only."""
    hq, hkv = 8, 4
    step, apart = (Layer(54, BF16, hq, hkv, [9000] * batch, uniform=True) for _ in range(2))
    k, v = _new(55, batch, hkv, BF16)
    k[0, 0, 1, 5], v[0, 2, 3, 100] = float("inf"), float("nan")
    rope = rope_table(position + 1, BF16).cuda()
    step.cache.append_norm_rope_with_attention(0, step.op, position, k, v, rope)
    apart.cache.append_norm_rope(0, position, k, v, rope)
    assert _same_bits(step, apart)
    bad = torch.zeros(1, batch, hq, dtype=torch.bool, device="cuda")
    bad[0, 0, 2:4] = bad[0, 2, 6:8] = True
    assert torch.equal(torch.isnan(step.out).all(dim=-1), bad) and torch.equal(torch.isnan(step.out).any(dim=-1), bad)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,batch,keys", [(8, 2, 2, 200), (17, 1, 3, 700), (8, 4, 8, 9000)])
def test_what_sees_a_row_that_is_nan_has_no_log_sum(dtype, hq, hkv, batch, keys):
    """A key or a value row whose scale is NaN: both results of single tokens that see it are NaN, as a chunk's are; and of a step
    that writes such a row."""
    t = Layer(59, dtype, hq, hkv, [keys] * batch, uniform=True)
    bad, group = keys // 2 + 5, hq // hkv
    first = [keys - 1 - 7 * i for i in range(batch)]
    first[1] = bad - 1   # does not see it
    at = torch.tensor(first, dtype=torch.int32, device="cuda")
    sees = torch.zeros(t.out.shape[:3], dtype=torch.bool, device="cuda")
    sees[0, 0, :group] = True
    t.op.run_ragged(at, keys - 1, batch)
    torch.cuda.synchronize()
    out, lse = t.out.clone(), t.lse.clone()
    t.check(first)
    for _, byte in t.tensors():
        was = byte[:2, 0, bad].clone()
        byte[:2, 0, bad] = 255
        t.op.run_ragged(at, keys - 1, batch)
        torch.cuda.synchronize()
        assert torch.equal(torch.isnan(t.lse), sees) and torch.equal(torch.isnan(t.out).all(dim=-1), sees)
        assert torch.equal(t.out[~sees], out[~sees]) and torch.equal(t.lse[~sees], lse[~sees])
        byte[:2, 0, bad] = was
    k, v = _new(62, batch, hkv, dtype)
    v[0, 0, 0, 77] = float("inf")
    t.cache.append_norm_rope_with_attention(0, t.op, 0, k, v, rope_table(keys, dtype).cuda(), positions=at, max_position=keys - 1)
    torch.cuda.synchronize()
    assert torch.equal(torch.isnan(t.lse), sees) and torch.equal(torch.isnan(t.out).all(dim=-1), sees)


def test_rows_behind_the_last_sequence_stay():
    step = Layer(56, F16, 8, 2, [50] * 4, uniform=True)
    before = [t.clone() for pair in step.tensors() for t in pair]
    k, v = _new(57, 2, 2, F16)
    step.cache.append_norm_rope_with_attention(0, step.op, 20, k, v, rope_table(21, F16).cuda(), batch_size=2)
    torch.cuda.synchronize()
    assert (step.out[:, 2:] == 7.0).all() and (step.lse[:, 2:] == 7.0).all()
    for was, now in zip(before, (t for pair in step.tensors() for t in pair)):
        assert torch.equal(was[2:], now[2:]) and torch.equal(was[:, :, :20], now[:, :, :20])
        assert torch.equal(was[:, :, 21:], now[:, :, 21:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.07, 1e-40])
@pytest.mark.parametrize("interval,batch,keys", [(1, 2, 100), (1, 16, 9000), (20, 2, 60), (40, 1, 300)])
def test_scales_of_zero_and_below(dtype, scale, interval, batch, keys):
    t = Layer(58, dtype, 8, 4, [keys] * batch, uniform=True, scale=scale, interval=interval)
    first = keys - interval - (1 if interval == 1 else 0)   # (a last chunk that is not whole)
    if interval == 1:
        t.op.run_ragged(torch.full((batch,), first, dtype=torch.int32, device="cuda"), first, batch)
    else:
        t.op.run(first, interval, batch)
    t.check([first] * batch)


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-42, -1e-42])
@pytest.mark.parametrize("interval,batch,keys", [(1, 2, 100), (1, 8, 9000), (20, 2, 60), (40, 1, 2040), (96, 2, 4200), (200, 1, 2500)])
def test_scales_that_large_products_do_not_feel(scale, interval, batch, keys):
    """Products of up to 2^124 under a scale of (nearly) zero: every key that is seen weighs the same."""
    t = Layer(63, BF16, 8, 4, [keys] * batch, uniform=True, scale=scale, interval=interval)
    t.tensors()[0][1].copy_(torch.where(t.tensors()[0][1] > 119, 178, 177))   # keys 2^50 and 2^51 times their codes
    t.q.copy_(torch.where(t.q > 0, 2.0 ** 57, -2.0 ** 57))
    first = keys - interval - (1 if interval == 1 else 0)
    if interval == 1:
        t.op.run_ragged(torch.full((batch,), first, dtype=torch.int32, device="cuda"), first, batch)
    else:
        t.op.run(first, interval, batch)
    t.check([first] * batch)


def test_two_recorded_steps_of_one_handle():
    """Recorded twice with different rows to write, replayed in turn with eager runs between: each as the eager call."""
    dtype, caps = BF16, [9000] * 16
    step, eager = (Layer(60, dtype, 8, 4, caps) for _ in range(2))
    rope = rope_table(9000, dtype).cuda()
    at = torch.tensor([8000 - 450 * i for i in range(16)], dtype=torch.int32, device="cuda")
    moving = [at.clone(), at.clone() + 1]
    new = [_new(61 + i, 16, 4, dtype) for i in range(2)]
    stream, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(stream), ellm_amd.StepGraph(stream) as graph:
            step.cache.append_norm_rope_with_attention(0, step.op, 0, *new[i], rope, positions=moving[i], max_position=8999, stream=stream)
            ellm_amd.positions_advance(moving[i], 2, stream=stream)
        graphs.append(graph)
    stream.synchronize()
    for turn in range(6):
        graphs[turn % 2].launch(stream)
        stream.synchronize()
        eager.cache.append_norm_rope_with_attention(0, eager.op, 0, *new[turn % 2], rope, positions=at + turn, max_position=8999)
        torch.cuda.synchronize()
        assert torch.equal(step.out, eager.out) and torch.equal(step.lse, eager.lse)
        assert _same_bits(step, eager)
        step.op.run_ragged(at, 8999, 16)   # eager work of the same handle and workspace in between
        torch.cuda.synchronize()
    for graph in graphs:
        graph.close()


def test_on_a_stream_of_the_callers():
    """Rows that arrive late on a side stream: the write and the run wait for them there."""
    step, apart = (Layer(64, F16, 8, 2, [700] * 3, uniform=True) for _ in range(2))
    k, v = _new(65, 3, 2, F16)
    rope = rope_table(700, F16).cuda()
    late_k, late_v = torch.zeros_like(k), torch.zeros_like(v)
    stream = torch.cuda.Stream()
    work = torch.randn(2048, 2048, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(20):
            work = torch.mm(work, work).clamp(-1, 1)
        late_k.copy_(k), late_v.copy_(v)
        step.cache.append_norm_rope_with_attention(0, step.op, 600, late_k, late_v, rope)   # (the current stream)
    stream.synchronize()
    apart.cache.append_norm_rope(0, 600, k, v, rope)
    assert _same_bits(step, apart)
    step.check([600] * 3)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_several_tokens_that_are_clamped_to_one_row_leave_the_last(dtype):
    t = Layer(66, dtype, 2, 2, [4, 30, 9])
    before = [[x.clone() for x in pair] for pair in t.tensors()]
    k, v = _new(67, 3, 2, dtype, tokens=5)
    rope = rope_table(30, dtype)
    at = torch.tensor([2, 20, 25], dtype=torch.int32)
    t.cache.append_norm_rope(0, 0, k, v, rope.cuda(), positions=at.cuda(), max_position=25)
    torch.cuda.synchronize()
    written = {0: [(2, 0), (3, 4)], 1: [(20 + i, i) for i in range(5)], 2: [(8, 4)]}   # sequence -> (row, token)
    start = [0, 4, 34]
    codes, byte = t.tensors()[1]
    want_codes, want_byte = before[1]
    c, b = hold(v.cpu(), LARGEST[dtype])
    for s, pairs in written.items():
        for row, token in pairs:
            want_codes[:, start[s] + row], want_byte[:, start[s] + row] = c[token, s].cuda(), b[token, s].cuda()
    assert torch.equal(codes, want_codes) and torch.equal(byte, want_byte)
    codes, byte = t.tensors()[0]   # the keys: only those rows changed, and none is a mixture
    alone = Layer(66, dtype, 2, 2, [4, 30, 9])
    for token in range(5):         # one token a call, in order
        alone.cache.append_norm_rope(0, 0, k[token:token + 1], v[token:token + 1], rope.cuda(), positions=(at + token).cuda(),
                                     max_position=29)
    assert _same_bits(t, alone)


def test_rows_read_onto_one_another_are_refused():
    cache = ellm_amd.KVCache(1, 3, 2, 8, CODE[F16], e4m3=True)
    flat = torch.zeros(40 * D, dtype=F16, device="cuda")

    def views(strides, shape=(4, 3, 2)):
        return [flat.as_strided((*shape, D), (*strides, 1)) for _ in range(2)]

    for strides in ((D, D, D), (6 * D, 2 * D, D // 2), (3 * D, 2 * D, D), (D, 4 * D, 4 * D)):
        with pytest.raises(ellm_amd.EllmError):
            cache.read(0, 0, *views(strides))
    cache.read(0, 0, *views((D, 8 * D, 4 * D)))
    cache.read(0, 0, *views((5, 3, D), (1, 1, 2)))   # (strides of axes of length one mean nothing)
    torch.cuda.synchronize()


def test_positions_past_a_sequences_capacity_write_its_last_row():
    caps, at = [3, 40, 9], [30, 39, 9]
    step, apart = (Layer(68, BF16, 8, 2, caps) for _ in range(2))
    k, v = _new(69, 3, 2, BF16)
    rope = rope_table(40, BF16).cuda()
    where = torch.tensor(at, dtype=torch.int32, device="cuda")
    step.cache.append_norm_rope_with_attention(0, step.op, 0, k, v, rope, positions=where, max_position=39)
    apart.cache.append_norm_rope(0, 0, k, v, rope, positions=where, max_position=39)
    assert _same_bits(step, apart)
    step.check([min(p, c - 1) for p, c in zip(at, caps)])


@pytest.mark.parametrize("interval,first", [(1, 299), (1, 256), (40, 250), (3, 290)])
def test_rows_as_far_apart_as_the_handle_takes(interval, first):
    """Rows 2^24 codes apart: offsets of codes pass 2^32 inside a plane, and in the middle of a tile."""
    hkv, hq, n, pitch = 2, 8, 300, 1 << 24
    gen = torch.Generator(device="cuda").manual_seed(70)
    codes = torch.empty(n * pitch, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n * pitch // D, dtype=torch.uint8, device="cuda")
    planes, scale_planes, held = [], [], []
    for at in (0, 1024):   # keys and values of a position in the same stretch
        plane = codes.as_strided((1, hkv, n, D), (n * pitch, 256, pitch, 1), at)
        plane.copy_(torch.randint(0, 120, plane.shape, generator=gen, device="cuda").to(torch.uint8))
        byte = scales.as_strided((1, hkv, n), (n * pitch // D, 2, pitch // D), at // D)
        byte.copy_(torch.randint(118, 122, byte.shape, generator=gen, device="cuda").to(torch.uint8))
        planes.append(codes[at:].view(torch.float8_e4m3fn))
        scale_planes.append(scales[at // D:].view(torch.float8_e8m0fnu))
        held.append(values(plane, byte).float())
    q = torch.randn((interval, 1, hq, D), generator=gen, device="cuda").to(F16)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device="cuda")
    op = ellm_amd.Attention(q, *planes, out, 1, hq, hkv, D, (n * pitch, 256, pitch, 1), SCALE, lse=lse, sequence_capacity=n,
                            kv_scales=scale_planes)
    op.run(first, interval, 1)
    torch.cuda.synchronize()
    check(out, lse, reference(q, *held, [first], SCALE))


def test_a_layer_with_projections():
    """Two layers whose projections write 16-bit rows into one buffer that all layers share, from there into each layer's cache in
    8 bits; attention over that cache; output projection and residual.  A prompt in two chunks, then single tokens."""
    dtype, batch, hq, hkv, hidden, capacity, layers = F16, 3, 8, 2, 256, 128, 2
    gen = torch.Generator(device="cuda").manual_seed(71)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    rope = rope_table(capacity, dtype).cuda()
    cache = ellm_amd.KVCache(layers, batch, hkv, capacity, CODE[dtype], e4m3=True)
    k_rows, v_rows = (torch.zeros((capacity, batch, hkv, D), dtype=dtype, device="cuda") for _ in range(2))
    shared = (hkv * D, D, batch * hkv * D, 1)   # (sequence, head, position) strides of that buffer
    x = torch.zeros((32, batch, hidden), dtype=dtype, device="cuda")
    q = torch.zeros((32, batch, hq, D), dtype=dtype, device="cuda")
    att, out = torch.zeros_like(q), torch.zeros_like(x)
    stack = []
    for layer in range(layers):
        wq, wk, wv = (normal(n * D, hidden, scale=hidden ** -0.5) for n in (hq, hkv, hkv))
        wo = normal(hidden, hq * D, scale=(hq * D) ** -0.5)
        k, v, ks, vs = cache.layer_e4m3_tensors(layer)
        stack.append((ellm_amd.MatMul3(x, wq, q, wk, k_rows, wv, v_rows, rope, D, batch, hq, hkv, shared, capacity),
                      ellm_amd.Attention(q, k, v, att, batch, hq, hkv, D, cache.layer_e4m3(layer).strides, SCALE,
                                         sequence_capacity=capacity, kv_scales=(ks, vs)),
                      ellm_amd.MatMulAdd(att.view(32, batch, hq * D), wo, x, out), wo, (k, v, ks, vs)))
    for first, n in ellm_amd.schedule_calls(0, 52, 32, 55):
        for layer, (project, attend, finish, wo, (k, v, ks, vs)) in enumerate(stack):
            x[:n] = normal(n, batch, hidden)
            project.run(first, n, batch)
            cache.append(layer, first, k_rows[first:first + n], v_rows[first:first + n])
            attend.run(first, n, batch)
            finish.run(0, n, batch)
            torch.cuda.synchronize()
            for got, byte, rows_ in ((k, ks, k_rows), (v, vs, v_rows)):
                codes, want_byte = hold(rows_[first:first + n].cpu(), LARGEST[dtype])
                assert torch.equal(byte.view(torch.uint8)[:, :, first:first + n].cpu(), want_byte.permute(1, 2, 0))
                assert torch.equal(got.view(torch.uint8)[:, :, first:first + n].cpu(), codes.permute(1, 2, 0, 3))
            planes = [values(c.view(torch.uint8), b.view(torch.uint8)).float() for c, b in ((k, ks), (v, vs))]
            check(att[:n], None, reference(q[:n], *planes, [first] * batch, SCALE), f"layer {layer}, {n} at {first}")
            a, w = att[:n].reshape(-1, hq * D).double(), wo.double()
            want = a @ w.T + x[:n].reshape(-1, hidden).double()
            # the result rounded once, and a binary32 sum of hq * 128 products and the residual
            bound = 2.0 ** -11 * want.abs() + (hq * D + 1) * 2.0 ** -24 * (a.abs() @ w.abs().T + x[:n].reshape(-1, hidden).double().abs())
            assert ((out[:n].reshape(-1, hidden).double() - want).abs() <= bound * (1 + 2.0 ** -10)).all()


@pytest.mark.parametrize("batch,longest", [(65, 4100), (257, 1030), (300, 900), (1024, 260)])
def test_many_sequences_of_different_lengths(batch, longest):
    """More sequences than a wave has lanes, up to the most that a launch deals evenly: lengths from one key on."""
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(1, longest + 1, (batch,), generator=gen).tolist()
    lengths[0], lengths[-1], lengths[batch // 2] = longest, 1, longest
    step, apart = (Layer(72, BF16, 2, 1, [longest] * batch, uniform=True) for _ in range(2))
    assert step.op.ragged_path(longest - 1, batch) == 1
    positions = [n - 1 for n in lengths]
    at = torch.tensor(positions, dtype=torch.int32, device="cuda")
    k, v = _new(73, batch, 1, BF16)
    rope = rope_table(longest, BF16).cuda()
    step.cache.append_norm_rope_with_attention(0, step.op, 0, k, v, rope, positions=at, max_position=longest - 1)
    apart.cache.append_norm_rope(0, 0, k, v, rope, positions=at, max_position=longest - 1)
    assert _same_bits(step, apart)
    step.check(positions)
    step.op.run_ragged(at, longest - 1, batch)   # the same keys, all of the cache now
    step.check(positions)


def test_strides_past_any_address_are_refused():
    cache = ellm_amd.KVCache(1, 3, 2, 8, CODE[F16], e4m3=True)
    out = torch.zeros(64 * D, dtype=F16, device="cuda")
    lib = ellm_amd.load_library()
    for strides in ((1 << 62, 2 * D, D), (1 << 63, 2 * D, D), (2 * D, 1 << 61, D), ((1 << 64) - 8, 2 * D, D)):
        steps = (ctypes.c_size_t * 3)(*strides)
        assert lib.ellm_kv_read_e4m3(cache._handle, 0, 0, 0, 8, 3, out.data_ptr(), out.data_ptr(), steps, None) == 1


def test_scales_laid_out_otherwise_than_their_rows_are_refused():
    codes = torch.zeros((2, 3, 40, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros((2, 3, 40), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    q = torch.zeros((1, 2, 3, D), dtype=F16, device="cuda")
    out = torch.zeros_like(q)
    turned = scales.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e8m0fnu)
    for ks, vs in ((turned, scales), (scales, turned)):
        with pytest.raises(ValueError):
            ellm_amd.Attention(q, codes, codes, out, 2, 3, 3, D, codes.stride(), SCALE, kv_scales=(ks, vs))
    ellm_amd.Attention(q, codes, codes, out, 2, 3, 3, D, codes.stride(), SCALE, kv_scales=(scales, scales.flatten()))
