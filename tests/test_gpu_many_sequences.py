"""Single-token steps over more sequences than a workgroup has lanes, up to the most whose keys a launch deals evenly."""
import math

import pytest
import torch

import ellm_amd
from shaped_util import check, reference

pytestmark = pytest.mark.gpu
D, SCALE = 128, 1.0 / math.sqrt(128)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,longest", [(65, 4100), (257, 1030), (300, 900), (1024, 260)])
def test_lengths_from_one_key_on(dtype, batch, longest):
    gen = torch.Generator(device="cuda").manual_seed(batch)
    k, v = (torch.randn((batch, 1, longest, D), generator=gen, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn((1, batch, 2, D), generator=gen, device="cuda").to(dtype)
    out, lse = torch.full_like(q, 7.0), torch.full((1, batch, 2), 7.0, device="cuda")
    op = ellm_amd.Attention(q, k, v, out, batch, 2, 1, D, k.stride(), SCALE, lse=lse)
    lengths = torch.randint(1, longest + 1, (batch,), generator=torch.Generator().manual_seed(batch)).tolist()
    lengths[0], lengths[-1], lengths[batch // 2] = longest, 1, longest
    first = [n - 1 for n in lengths]
    assert op.ragged_path(longest - 1, batch) == 1
    op.run_ragged(torch.tensor(first, dtype=torch.int32, device="cuda"), longest - 1, batch)
    torch.cuda.synchronize()
    check(out, lse, reference(q, k, v, first, SCALE))
    op.run_ragged(torch.tensor(first[::-1], dtype=torch.int32, device="cuda"), longest - 1, batch)
    torch.cuda.synchronize()
    check(out, lse, reference(q, k, v, first[::-1], SCALE))
