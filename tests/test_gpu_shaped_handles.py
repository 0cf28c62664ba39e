"""What a handle with shaped scores or a shared prefix keeps, refuses and allocates."""
import gc

import pytest
import torch

import ellm_amd
from shaped_util import slopes_of
from test_gpu_shaped_scores import F16, Setup

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
