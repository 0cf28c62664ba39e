"""Caches in 8 bits: what is written, code for code, what is read back, and what is refused."""
import gc
import weakref

import pytest
import torch

import ellm_amd
from e4m3_util import CODE, D, GRID, LARGEST, hold, norm_rope, rope_table, rows, values

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
EPS = 1e-6


def _bytes(cache, layer=0):
    torch.cuda.synchronize()
    return [t.view(torch.uint8).cpu() for t in cache.layer_e4m3_tensors(layer)]


def _fill(cache, layers=1, byte=0x5a):
    """Codes and scales that no write in these tests produces in whole rows."""
    for n in range(layers):
        for t in cache.layer_e4m3_tensors(n):
            t.view(torch.uint8).fill_(byte)


def _want(x, dtype):
    """[tokens, sequences, heads, 128] -> codes and scale bytes [sequences, heads, tokens, ...]"""
    codes, byte = hold(x, LARGEST[dtype])
    return codes.permute(1, 2, 0, 3), byte.permute(1, 2, 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,batch,pitch,heads,start,capacity", [
    (1, 1, 1, 1, 0, 1), (1, 3, 5, 4, 6, 7), (17, 2, 2, 1, 0, 40), (64, 1, 1, 8, 63, 127), (333, 3, 4, 5, 20, 353), (5, 9, 9, 3, 1, 11),
])
def test_append_holds_every_row_as_defined(dtype, tokens, batch, pitch, heads, start, capacity):
    gen = torch.Generator().manual_seed(tokens * 7 + heads)
    k, v = (rows(gen, (tokens, pitch, heads), dtype, 3.0) for _ in range(2))
    cache = ellm_amd.KVCache(2, max(batch, 2), heads, capacity, CODE[dtype], e4m3=True)
    _fill(cache, 2)
    cache.append(1, start, k.cuda(), v.cuda(), batch_size=batch)
    got = _bytes(cache, 1)
    for x, codes, byte in ((k, got[0], got[2]), (v, got[1], got[3])):
        want_codes, want_byte = (torch.full_like(t, 0x5a) for t in (codes, byte))
        c, b = _want(x[:, :batch], dtype)
        want_codes[:batch, :, start:start + tokens], want_byte[:batch, :, start:start + tokens] = c, b
        assert torch.equal(byte, want_byte)
        assert torch.equal(codes, want_codes)   # rows around it are as they were
    assert all((t == 0x5a).all() for t in _bytes(cache, 0))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_at_the_borders_of_the_format(dtype):
    """Every code, every midpoint between two codes and its neighbours in the type, at scales from the smallest to the largest;
    the largest finite values; zeros of either sign; rows that are zero but for one element."""
    mid = (GRID[1:] + GRID[:-1]) / 2
    step = torch.finfo(dtype).eps
    line = torch.cat([GRID, mid, mid * (1 + step), mid * (1 - step), -mid])
    line = line[torch.isfinite(line.to(dtype))]
    line = torch.cat([line, torch.zeros(-len(line) % (D - 1), dtype=torch.float64)]).view(-1, D - 1)
    line = torch.cat([line, torch.full((len(line), 1), 448.0, dtype=torch.float64)], dim=1)   # (scale 1)
    exponents = (-18, -8, 0, 7) if dtype == F16 else (-118, -30, 0, 7, 60, 119)
    x = torch.cat([(line * 2.0 ** e).to(dtype) for e in exponents])
    top = torch.finfo(dtype).max
    more = torch.zeros(8, D, dtype=dtype)
    more[0], more[1, 5], more[2, :2], more[3, 9] = top, top, torch.tensor([-top, top * 0.97]), torch.finfo(dtype).tiny
    more[4, 127], more[5] = torch.finfo(dtype).smallest_normal / 4, -0.0
    more[6, 0], more[6, 1] = 57344.0 if dtype == F16 else 1.75 * 2.0 ** 127, 1.0
    more[7, 0] = 1.0
    x = torch.cat([x, more])
    x = torch.cat([x, torch.zeros(-len(x) % 4, D, dtype=dtype)]).view(-1, 1, 4, D)
    cache = ellm_amd.KVCache(1, 1, 4, len(x), CODE[dtype], e4m3=True)
    cache.append(0, 0, x.cuda(), (-x).cuda())
    k, v, ks, vs = _bytes(cache)
    for got, got_byte, rows_ in ((k, ks, x), (v, vs, -x)):
        codes, byte = _want(rows_, dtype)
        assert torch.equal(got_byte, byte)
        assert torch.equal(got & 127, codes & 127)
        assert torch.equal(got[(codes & 127) != 0], codes[(codes & 127) != 0])
    out = [torch.empty_like(x, device="cuda") for _ in range(2)]
    cache.read(0, 0, *out)
    torch.cuda.synchronize()
    assert torch.equal(out[0].cpu().double(), values(k, ks).permute(2, 0, 1, 3).to(dtype).double())
    assert torch.isfinite(out[0]).all() and torch.equal(out[0], -out[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_a_row_that_is_not_finite_reads_as_nan(dtype, what):
    gen = torch.Generator().manual_seed(3)
    k, v = (rows(gen, (5, 2, 3), dtype) for _ in range(2))
    k[2, 1, 0, 77], v[4, 0, 2, 0] = what, what
    cache = ellm_amd.KVCache(1, 2, 3, 8, CODE[dtype], e4m3=True)
    cache.append(0, 1, k.cuda(), v.cuda())
    kc, vc, ks, vs = _bytes(cache)
    assert int(ks[1, 0, 3]) == 255 and (ks == 255).sum() == 1 and not kc[1, 0, 3].any()
    assert int(vs[0, 2, 5]) == 255 and (vs == 255).sum() == 1 and not vc[0, 2, 5].any()
    out = [torch.empty_like(k, device="cuda") for _ in range(2)]
    cache.read(0, 1, *out)
    for got, x in zip(out, (k, v)):
        want = torch.isfinite(x).all(dim=-1)
        assert torch.equal(torch.isnan(got.cpu()), ~want[..., None].expand_as(x))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,batch,heads,start,ragged", [
    (1, 1, 1, 0, False), (40, 2, 4, 25, False), (1, 5, 8, 0, True), (1, 70, 3, 0, True), (3, 4, 2, 0, True),
])
def test_append_norm_rope(dtype, tokens, batch, heads, start, ragged):
    """The row that goes to 8 bits is the 32-bit result of the formulas, rounded once."""
    gen = torch.Generator().manual_seed(tokens + heads)
    k, v = (rows(gen, (tokens, batch, heads), dtype, 2.0) for _ in range(2))
    capacity = 90
    first = torch.randint(0, capacity - tokens, (batch,), generator=gen) if ragged else torch.full((batch,), start)
    rope = rope_table(capacity, dtype)
    cache = ellm_amd.KVCache(1, batch, heads, capacity, CODE[dtype], e4m3=True)
    _fill(cache)
    most = capacity - tokens
    more = dict(positions=first.int().cuda(), max_position=most) if ragged else {}
    cache.append_norm_rope(0, start, k.cuda(), v.cuda(), rope.cuda(), eps=EPS, **more)
    at = first[None] + torch.arange(tokens)[:, None]
    got = _bytes(cache)
    for x, codes, byte in ((norm_rope(k, rope, at, EPS), got[0], got[2]), (v, got[1], got[3])):
        want_codes, want_byte = (torch.full_like(t, 0x5a) for t in (codes, byte))
        c, b = _want(x, dtype)
        for s in range(batch):
            want_codes[s, :, at[:, s]], want_byte[s, :, at[:, s]] = c[s], b[s]
        assert torch.equal(byte, want_byte)
        assert torch.equal(codes, want_codes)


def test_positions_past_their_bound_are_clamped_to_it():
    gen = torch.Generator().manual_seed(5)
    k = rows(gen, (1, 3, 2), F16)
    cache = ellm_amd.KVCache(1, 3, 2, 16, CODE[F16], e4m3=True)
    positions = torch.tensor([2, 9, -1], dtype=torch.int32, device="cuda")   # (-1: 2^32 - 1)
    cache.append_norm_rope(0, 0, k.cuda(), k.cuda(), rope_table(16, F16).cuda(), positions=positions, max_position=7)
    byte = _bytes(cache)[3]
    assert torch.equal((byte != 0).any(dim=1).nonzero(), torch.tensor([[0, 2], [1, 7], [2, 7]]))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_caches_with_a_capacity_for_each_sequence(dtype):
    """The same rows as a cache with one capacity, and nothing beside them."""
    caps, heads = [5, 130, 1, 77], 3
    gen = torch.Generator().manual_seed(6)
    cache = ellm_amd.KVCache.ragged(2, caps, heads, CODE[dtype], e4m3=True)
    _fill(cache, 2)
    rope = rope_table(130, dtype)
    first = torch.tensor([4, 100, 0, 900], dtype=torch.int32)   # (the last is clamped to its sequence's end)
    k, v = (rows(gen, (1, 4, heads), dtype) for _ in range(2))
    cache.append_norm_rope(1, 0, k.cuda(), v.cuda(), rope.cuda(), eps=EPS, positions=first.cuda(), max_position=129)
    got = _bytes(cache, 1)
    start = [sum(caps[:i]) for i in range(4)]
    at = torch.tensor([[4, 100, 0, 129]])
    where = [start[0] + 4, start[1] + 100, start[2], start[3] + 76]
    for x, codes, byte in ((norm_rope(k, rope, at, EPS), got[0], got[2]), (v, got[1], got[3])):
        want_codes, want_byte = (torch.full_like(t, 0x5a) for t in (codes, byte))
        c, b = _want(x, dtype)
        for s in range(4):
            want_codes[:, where[s]], want_byte[:, where[s]] = c[s, :, 0], b[s, :, 0]
        assert torch.equal(byte, want_byte) and torch.equal(codes, want_codes)
    assert all((t == 0x5a).all() for t in _bytes(cache, 0))
    # rows back, from the second sequence on
    k, v = (rows(gen, (60, 2, heads), dtype) for _ in range(2))
    with pytest.raises(ellm_amd.EllmError):
        cache.append(0, 0, k.cuda(), v.cuda())   # (past the first sequence's end)
    view = cache.layer_e4m3(0, 1)
    assert view.capacities == caps[1:] and view.strides[1] == sum(caps) * D
    for s, n in ((1, 130), (3, 77)):
        x = [rows(gen, (n, 1, heads), dtype) for _ in range(2)]
        flat = cache.layer_e4m3_tensors(0)
        for name in range(2):
            codes, byte = _want(x[name], dtype)
            flat[name].view(torch.uint8)[:, start[s]:start[s] + n] = codes[0].cuda()
            flat[2 + name].view(torch.uint8)[:, start[s]:start[s] + n] = byte[0].cuda()
        out = [torch.empty((n - 1, 1, heads, D), dtype=dtype, device="cuda") for _ in range(2)]
        cache.read(0, 1, *out, first_sequence=s)
        for got_, want in zip(out, x):
            assert torch.equal(got_.cpu().double(), values(*hold(want[1:], LARGEST[dtype])))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", ["append", "planes", "spread"])
def test_read_into_any_strides(dtype, layout):
    gen = torch.Generator().manual_seed(8)
    tokens, batch, heads, start = 37, 3, 5, 4
    x = [rows(gen, (64, 4, heads), dtype) for _ in range(2)]
    cache = ellm_amd.KVCache(2, 4, heads, 64, CODE[dtype], e4m3=True)
    cache.append(1, 0, *(t.cuda() for t in x))
    if layout == "append":
        whole = [torch.full((tokens, batch, heads, D), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        out = whole
    elif layout == "planes":
        whole = [torch.full((batch, heads, 50, D), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        out = [t.permute(2, 0, 1, 3)[:tokens] for t in whole]
    else:
        whole = [torch.full((tokens, 2 * batch, heads + 1, D + 8), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        out = [t[:, ::2, :heads, :D] for t in whole]
    cache.read(1, start, *out, first_sequence=1)
    torch.cuda.synchronize()
    for got, want, all_ in zip(out, x, whole):
        want = values(*hold(want[start:start + tokens, 1:1 + batch], LARGEST[dtype]))
        assert torch.equal(got.cpu().double(), want)
        assert int((all_ == 7.0).sum()) >= all_.numel() - got.numel()   # nothing beside the rows


def test_tensors_of_a_layer_keep_the_cache():
    gen = torch.Generator().manual_seed(9)
    x = rows(gen, (4, 1, 2), F16).cuda()
    cache = ellm_amd.KVCache(1, 1, 2, 4, CODE[F16], e4m3=True)
    cache.append(0, 0, x, x)
    kept = cache.layer_e4m3_tensors(0)[1].view(torch.uint8)[:, :, 1:]
    want = kept.clone()
    cache_alive = weakref.ref(cache)
    del cache
    gc.collect()
    assert cache_alive() is not None
    assert torch.equal(kept, want)


def test_refusals():
    cache = ellm_amd.KVCache(1, 2, 3, 8, CODE[F16], e4m3=True)
    plain = ellm_amd.KVCache(1, 2, 3, 8, CODE[F16])
    x = torch.zeros((4, 2, 3, D), dtype=F16, device="cuda")
    out = [torch.zeros_like(x) for _ in range(2)]

    def refused(call, error=ellm_amd.EllmError):
        with pytest.raises(error):
            call()

    refused(lambda: cache.layer(0))
    refused(lambda: cache.layer_ragged(0))
    refused(lambda: plain.layer_e4m3(0))
    refused(lambda: plain.read(0, 0, *out))
    refused(lambda: cache.layer_e4m3(1))
    refused(lambda: cache.layer_e4m3(0, 2))
    refused(lambda: cache.append(0, 5, x, x))                        # 5 + 4 > 8
    refused(lambda: cache.append(0, 0, x.bfloat16(), x.bfloat16()), TypeError)
    refused(lambda: cache.append(0, 0, x.cpu(), x.cpu()), TypeError)
    refused(lambda: cache.append_norm_rope(0, 0, x, x, torch.zeros((3, D), dtype=F16, device="cuda")))   # short table
    refused(lambda: cache.read(0, 5, *out))
    refused(lambda: cache.read(0, 0, *out, first_sequence=1))        # sequences 1 and 2 of 2
    refused(lambda: cache.read(0, 0, out[0].bfloat16(), out[1].bfloat16()), TypeError)
    refused(lambda: cache.read(0, 0, out[0][:, :, :2], out[1][:, :, :2]), ValueError)
    refused(lambda: cache.read(0, 0, out[0], out[1].transpose(0, 1).contiguous().transpose(0, 1)), ValueError)
    refused(lambda: cache.read(0, 0, *(t.transpose(2, 3).contiguous().transpose(2, 3) for t in out)), ValueError)
    refused(lambda: cache.read(0, 0, *(t[:1, :1].expand(4, 2, 3, D) for t in out)))   # rows onto one another
    cache.read(0, 0, *(t[:0] for t in out))
    cache.read(0, 7, *(t[:1] for t in out))
    torch.cuda.synchronize()
    assert not out[0].any()   # a cache that nothing was written to reads as zeros
