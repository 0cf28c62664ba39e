"""What a handle with shaped scores or a shared prefix keeps, refuses and allocates."""
import gc
import weakref

import pytest
import torch

import ellm_amd
from shaped_util import D, slopes_of
from test_gpu_shaped_scores import F16, SCALE, Setup, _u32

pytestmark = pytest.mark.gpu


def test_the_call_without_a_handle_is_refused_while_scores_or_a_prefix_are_set():
    """It reads the description alone, so it would compute the plain operator."""
    t = Setup(81, F16, 8, 2, 2, 1, 64, prefix=16)
    t.op.run(40, 1, 2)
    torch.cuda.synchronize()
    plain = t.out.clone()

    def taken():
        t.out.fill_(7.0)
        t.op.run_noalloc(40, 2)
        torch.cuda.synchronize()
        return torch.equal(t.out, plain)

    assert taken()
    for on, off in ((lambda: t.op.set_scores(cap=30.0), t.op.set_scores), (lambda: t.op.set_scores(window=5), t.op.set_scores),
                    (lambda: t.op.set_scores(slopes=slopes_of(8)), t.op.set_scores),
                    (lambda: t.op.set_shared_prefix(*t.prefix), t.op.set_shared_prefix)):
        on()
        t.out.fill_(7.0)
        with pytest.raises(ValueError):
            t.op.run_noalloc(40, 2)
        torch.cuda.synchronize()
        assert (t.out == 7.0).all()
        off()
        assert taken()


def test_arguments_that_the_c_types_would_change():
    """A window past 64 bits is a window past every key; a cap that 32 bits hold as zero, or a view of fewer slopes than
    heads in a longer buffer, is refused and nothing of it stays."""
    t = Setup(82, F16, 8, 2, 2, 1, 64)
    for window in (1 << 32, (1 << 64) + 5, 1 << 100):
        t.op.set_scores(window=window)
        t.op.run(40, 1, 2)
        t.check(t.want([40, 40]), f"window {window}")
    t.op.set_scores()
    for bad in (dict(cap=1e-50), dict(cap=-1e-60), dict(slopes=slopes_of(16)[:7])):
        with pytest.raises(ValueError):
            t.op.set_scores(**bad)
        assert t.op.ragged_path(40, 2) != 2
    t.op.set_scores(slopes=slopes_of(16)[:8])
    t.op.run(40, 1, 2)
    t.check(t.want([40, 40], slopes=slopes_of(16)[:8]), "the first of a longer buffer")


def test_setters_that_set_nothing_take_no_room():
    """A handle that never had scores or a prefix keeps its memory when they are set to none; the first that sets
    anything takes the room for partial results once."""
    t = Setup(83, F16, 32, 4, 4, 64, 128, prefix=16)
    gc.collect()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    t.op.set_scores()
    t.op.set_shared_prefix()
    t.op.set_shared_prefix(*t.prefix, 0)
    assert torch.cuda.mem_get_info()[0] == free
    t.op.set_scores(cap=30.0)
    after = torch.cuda.mem_get_info()[0]
    assert 0 < free - after <= 80 << 20
    t.op.set_shared_prefix(*t.prefix)
    t.op.set_scores()
    t.op.set_shared_prefix()
    assert torch.cuda.mem_get_info()[0] == after
    t.op.run(3, 64, 4)
    torch.cuda.synchronize()


@pytest.mark.parametrize("way", ["step", "chunk", "append", "projection"])
def test_a_recorded_graph_keeps_the_tensors_it_was_recorded_with(way):
    """Set, record, set something else with no other reference to the first tensors, allocate over whatever was freed,
    replay: the recorded call's results, and the tensors live until the graph is closed."""
    hq, hkv, batch, cap, prefix, at = 8, 2, 3, 64, 40, 33
    n = 4 if way == "chunk" else 1
    t = Setup(84, F16, hq, hkv, batch, 4, cap, prefix=prefix)
    op, stream = t.op, torch.cuda.Stream()
    rope = torch.zeros((128, D), dtype=F16, device="cuda")
    rope[:, 0::2] = 1.0
    if way == "append":
        cache = ellm_amd.KVCache(1, batch, hkv, cap, ellm_amd.DTYPE_F16)
        kt, vt = cache.layer_tensors(0, F16)
        kt.copy_(t.k)
        vt.copy_(t.v)
        op = ellm_amd.Attention(t.q, kt, vt, t.out, batch, hq, hkv, D, cache.layer(0)[2], SCALE, lse=t.lse, sequence_capacity=cap)
        rows = [torch.randn((1, batch, hkv, D), device="cuda").to(F16) for _ in range(2)]
    elif way == "projection":
        x = torch.randn((1, batch, 1024), device="cuda").to(F16)
        w = [(torch.randn((h * D, 1024), device="cuda") / 32).to(F16) for h in (hq, hkv, hkv)]
        proj = ellm_amd.MatMul3(x, w[0], t.q, w[1], t.k, w[2], t.v, rope, D, batch, hq, hkv, t.k.stride(), cap)
    if way in ("step", "chunk"):
        begin = [[max(0, p - 20) for p in range(cap)]] * batch
        kept = [slopes_of(hq), _u32(begin, cap)]
        op.set_scores(cap=20.0, slopes=kept[0], key_begin=kept[1])
    else:
        kept = [slopes_of(hq), *t.prefix]
        op.set_scores(cap=20.0, slopes=kept[0])
        op.set_shared_prefix(kept[1], kept[2])
    torch.cuda.synchronize()
    with ellm_amd.StepGraph(stream) as g:
        if way == "append":
            cache.append_norm_rope_with_attention(0, op, at, *rows, rope, stream=stream)
        elif way == "projection":
            proj.run_with_attention(op, at, batch, stream=stream)
        else:
            op.run(at, n, batch, stream=stream)
    g.launch()
    stream.synchronize()
    want = t.out.clone(), t.lse.clone()
    alive = [weakref.ref(x) for x in kept]
    del kept
    t.prefix = None
    op.set_shared_prefix()
    op.set_scores(slopes=torch.zeros(hq, device="cuda"))
    gc.collect()
    assert all(r() is not None for r in alive)
    filler = [torch.full((1 << n,), float("nan"), device="cuda") for n in range(3, 14) for _ in range(4)]
    for _ in range(3):
        t.out[:n].fill_(7.0)
        torch.cuda.synchronize()
        g.launch()
        stream.synchronize()
        assert torch.equal(t.out, want[0]) and torch.equal(t.lse, want[1])
    g.close()
    gc.collect()
    assert all(r() is None for r in alive)
    del filler
