"""Chunks over planes in 8 bits (ellm_amd/csrc/prefill.hip), without a GPU: what the compiler makes of the conversions."""
import re

import pytest

from test_build_invariants import _listing


@pytest.mark.parametrize("name", ["prefill.hip", "decode.hip", "decode_balanced.hip"])
def test_conversions_take_scales_that_were_loaded(name, tmp_path):
    """Codes are converted with a scale that a load brought, never with a constant: a constant there is what the compiler puts
    in the place of a register that nothing has set (the tile of zeros ahead of a walk's first one has no scales; converted
    with a leftover of all ones in its low byte it would be a tile of NaN)."""
    found = re.findall(r"v_cvt_scalef32_pk_b?f16_fp8 v\d+, (\S+), (\S+)", _listing(name, tmp_path))
    assert len(found) > 100
    assert [f for f in found if not re.fullmatch(r"v\d+", f[1])] == []
