"""Chunks over planes in 8 bits (ellm_amd/csrc/prefill.hip), without a GPU: what the compiler makes of the conversions, and that
the GPU tests reach every kernel."""
import re

import pytest

import plan_probe
from test_build_invariants import _listing
from test_gpu_e4m3_chunks import CASES


@pytest.mark.parametrize("name", ["prefill.hip", "decode.hip", "decode_balanced.hip"])
def test_conversions_take_scales_that_were_loaded(name, tmp_path):
    """Codes are converted with a scale that a load brought, never with a constant: a constant there is what the compiler puts
    in the place of a register that nothing has set (the tile of zeros ahead of a walk's first one has no scales; converted
    with a leftover of all ones in its low byte it would be a tile of NaN)."""
    found = re.findall(r"v_cvt_scalef32_pk_b?f16_fp8 v\d+, (\S+), (\S+)", _listing(name, tmp_path))
    assert len(found) > 100
    assert [f for f in found if not re.fullmatch(r"v\d+", f[1])] == []


def test_the_cases_reach_every_kernel():
    """Those of prefill.hip that are built for 8 bits: short prompts of one and two row blocks, the streaming kernel of four, eight
    and twelve waves, the ping-pong kernels of both instructions, also where 16-bit rows would go straight into LDS."""
    for (hq, hkv, batch, start, tokens), (kernel, which, split) in CASES.items():
        for bf16 in (False, True):
            call = (batch, batch, hq, hkv, start, tokens)
            found, number, n_split, _ = plan_probe.chunk_plan(*call, bf16=bf16)
            form = plan_probe.chunk_form(*call, bf16=bf16) if found == "pingpong" else number
            assert (found, form, n_split > 1) == (kernel, which, split), call
    assert set(CASES.values()) == {("short", n, False) for n in (1, 2)} | {("stream", n, s) for n in (4, 8, 12) for s in (False, True)} | {
        ("pingpong", f, s) for f in ("registers", "wide") for s in (False, True)} | {("pingpong", "direct", False)}
