"""Chunks over planes in 8 bits, each of the kernels that they run on (test_e4m3_chunk_kernels.py has it that the list below
reaches every one of them): against the definition in 64 bits, with rows apart from one another, anything behind the last key
and between the rows, and rows whose scale is NaN."""
import math

import pytest
import torch

import ellm_amd
from e4m3_util import D, values
from shaped_util import check, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = 1.0 / math.sqrt(D)

# (query heads, K/V heads, sequences, cached positions, tokens): (kernel, waves, row blocks or form, whether keys are split)
CASES = {
    (17, 1, 2, 300, 33): ("short", 1, False),
    (8, 8, 24, 450, 2): ("short", 2, False),
    (40, 2, 12, 31, 24): ("short", 2, False),
    (5, 1, 1, 1500, 3): ("stream", 4, True),
    (24, 2, 130, 700, 2): ("stream", 4, False),
    (16, 1, 1, 2000, 9): ("stream", 8, True),
    (16, 1, 130, 450, 16): ("stream", 8, False),
    (17, 1, 1, 4100, 16): ("stream", 12, True),
    (40, 2, 64, 450, 16): ("stream", 12, False),
    (17, 1, 3, 2000, 40): ("pingpong", "registers", True),
    (17, 1, 12, 2000, 24): ("pingpong", "registers", False),
    (17, 1, 12, 4100, 24): ("pingpong", "direct", False),   # planned for tiles straight into LDS: 8 bits take registers
    (17, 1, 1, 2000, 40): ("pingpong", "wide", True),
    (40, 2, 8, 200, 96): ("pingpong", "wide", False),
}


class Chunk:
    """Planes of random codes and scales 2^-9 .. 2^-6, `gap` rows apart; NaN codes and scales between the rows and behind the
    chunk's last key."""

    def __init__(self, seed, dtype, shape, gap):
        hq, hkv, batch, self.start, tokens = shape
        gen = torch.Generator(device="cuda").manual_seed(seed)
        keys = self.start + tokens
        rows = keys + 5
        self.codes, self.scales, self.values, self.bytes = [], [], [], []
        for _ in range(2):
            codes = torch.full((batch, hkv, rows, gap, D), 0x7f, dtype=torch.uint8, device="cuda")
            scale = torch.full((batch, hkv, rows, gap), 255, dtype=torch.uint8, device="cuda")
            own = torch.randint(0, 256, (batch, hkv, keys, D), generator=gen, device="cuda").to(torch.uint8)
            own[(own & 127) == 127] = 0
            byte = torch.randint(118, 122, (batch, hkv, keys), generator=gen, device="cuda").to(torch.uint8)
            at = gap // 2
            codes[:, :, :keys, at], scale[:, :, :keys, at] = own, byte
            self.codes.append(codes[..., at, :].view(torch.float8_e4m3fn))
            self.scales.append(scale.view(-1)[at:].view(torch.float8_e8m0fnu))
            self.bytes.append(scale[..., at])
            self.values.append(values(own, byte).float())   # (exact)
        self.q = torch.randn((tokens, batch, hq, D), generator=gen, device="cuda").to(dtype)
        self.out, self.lse = torch.full_like(self.q, 7.0), torch.full(self.q.shape[:3], 7.0, device="cuda")
        self.op = ellm_amd.Attention(self.q, *self.codes, self.out, batch, hq, hkv, D, self.codes[0].stride(), SCALE, lse=self.lse,
                                     sequence_capacity=rows, kv_scales=self.scales)

    def run(self):
        self.out.fill_(7.0), self.lse.fill_(7.0)
        self.op.run(self.start, self.q.shape[0], self.q.shape[1])
        torch.cuda.synchronize()

    def want(self):
        return reference(self.q, *self.values, [self.start] * self.q.shape[1], SCALE)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", CASES)
def test_every_kernel(dtype, shape):
    t = Chunk(60, dtype, shape, 1)
    t.run()
    check(t.out, t.lse, t.want())
    first = t.out.clone(), t.lse.clone()
    t.run()
    assert torch.equal(t.out, first[0]) and torch.equal(t.lse, first[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", CASES)
def test_rows_apart_and_rows_that_are_nan(dtype, shape):
    """A key or a value row whose scale is NaN, halfway through the new tokens: what sees it is NaN, the rest as without it."""
    hq, hkv, batch, start, tokens = shape
    t = Chunk(61, dtype, shape, 3)
    t.run()
    want = t.want()
    check(t.out, t.lse, want)
    for which in (0, 1):
        bad, seq, head = tokens // 2, batch - 1, hkv - 1
        was = t.bytes[which][seq, head, start + bad].clone()
        t.bytes[which][seq, head, start + bad] = 255
        t.run()
        sees = torch.zeros(t.out.shape[:3], dtype=torch.bool, device="cuda")
        sees[bad:, seq, head * (hq // hkv):] = True
        assert torch.isnan(t.out[sees]).all() and torch.isnan(t.lse[sees]).all()
        t.out[sees], t.lse[sees] = want[0][sees].to(dtype), want[1][sees].float()
        check(t.out, t.lse, want, ("key", "value")[which])
        t.bytes[which][seq, head, start + bad] = was
