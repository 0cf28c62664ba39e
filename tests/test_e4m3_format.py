"""The 8-bit row format and what the C ABI refuses about it, without a GPU."""
import ctypes

import pytest
import torch

import ellm_amd
from e4m3_util import D, GRID, LARGEST, hold, scales_of, values
from ellm_amd import _lib

OK, INVALID, UNSUPPORTED, OUT_OF_RANGE, HIP, NO_DEVICE = range(6)


def test_grid_is_the_e4m3_type():
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), GRID)


def test_rows_are_held_as_the_type_rounds():
    """hold() against torch's own conversion of the scaled values (exact in 32 bits)."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((2000, D), generator=gen) * torch.randn((2000, 1), generator=gen).mul_(4).exp_()
    codes, byte = hold(x, LARGEST[torch.bfloat16])
    want = torch.ldexp(x.double(), 127 - byte.int()[:, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(codes, want)
    err = (values(codes, byte) - x.double()).abs()
    scale = torch.pow(2.0, byte.double() - 127)[:, None]
    assert (err <= torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)).all()


@pytest.mark.parametrize("top,byte", [(448.0, 127), (448.25, 128), (224.0, 126), (1.75, 119), (1.0, 119), (0.0, 1),
                                      (2.0 ** -133, 1), (float("inf"), 255), (float("nan"), 255)])
def test_scales(top, byte):
    x = torch.zeros(1, D)
    x[0, 77] = -top
    assert int(scales_of(x)) == byte


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_is_read_back_fits_the_type(dtype):
    """Every finite value of the type as a row's largest, and its neighbourhood: what its row holds is a finite value of the type."""
    bits = torch.arange(0x8000, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype)
    x = x[torch.isfinite(x)]
    row = torch.stack([x, x / 2, -x * 0.9375, x / 64, x / 500, x / 1000] + [torch.zeros_like(x)] * 122, dim=-1)
    back = values(*hold(row, LARGEST[dtype]))
    assert torch.isfinite(back).all()
    if dtype == torch.float16:
        assert torch.equal(back.to(dtype).double(), back)
    else:   # (binary32 and bfloat16 end at 2^-126, below it a row's smallest codes are cut)
        normal = row[:, 0].double() >= 2.0 ** -100
        assert torch.equal(back[normal].to(dtype).double(), back[normal])


def _desc(**over):
    d = _lib.AttnDesc()
    d.q = d.k = d.v = d.out = 0x1000
    d.batch_size, d.attention_head_num, d.kv_head_num, d.head_size = 2, 8, 2, 128
    for i, s in enumerate(over.pop("kv_strides", (2 * 64 * 128, 64 * 128, 128, 1))):
        d.kv_strides[i] = s
    d.inverse_sqrt_head, d.dtype = 0.088, _lib.DTYPE_F16
    d.sequence_capacity, d.max_position_interval = 64, 16
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,scales,status", [
    ({}, (None, 0x1000), INVALID),
    ({}, (0x1000, None), INVALID),
    (dict(k=0x1008), (0x1000, 0x1000), INVALID),
    (dict(head_size=64, kv_strides=(64 * 64 * 2, 64 * 64, 64, 1)), (0x1000, 0x1000), UNSUPPORTED),
    (dict(dtype=_lib.DTYPE_F32), (0x1000, 0x1000), UNSUPPORTED),
    (dict(kv_strides=(2 * 64 * 136, 64 * 136, 136, 1)), (0x1000, 0x1000), INVALID),    # no whole row apart
    (dict(kv_strides=(2 * 64 * 128 + 8, 64 * 128, 128, 1)), (0x1000, 0x1000), INVALID),
    (dict(kv_strides=(2 * 64 * 128, 64 * 128 + 64, 128, 1)), (0x1000, 0x1000), INVALID),
    (dict(attention_head_num=7), (0x1000, 0x1000), INVALID),
])
def test_create_refuses(over, scales, status):
    lib = ellm_amd.load_library()
    h = ctypes.c_void_p(1)
    assert lib.ellm_attn_create_e4m3(ctypes.byref(_desc(**over)), *scales, None, ctypes.byref(h)) == status
    assert not h.value and lib.ellm_last_error_string()


def test_null_arguments():
    lib = ellm_amd.load_library()
    c, h = ctypes.c_void_p(), ctypes.c_void_p()
    strides, steps = (ctypes.c_size_t * 4)(), (ctypes.c_size_t * 3)()
    p = [ctypes.c_void_p() for _ in range(4)]
    assert lib.ellm_attn_create_e4m3(None, 0x1000, 0x1000, None, ctypes.byref(h)) == INVALID
    assert lib.ellm_attn_create_e4m3(ctypes.byref(_desc()), 0x1000, 0x1000, None, None) == INVALID
    assert lib.ellm_kv_create_e4m3(None, ctypes.byref(c)) == INVALID
    assert lib.ellm_kv_create_ragged_e4m3(None, ctypes.byref(c)) == INVALID
    assert lib.ellm_kv_layer_e4m3(None, 0, 0, *(ctypes.byref(x) for x in p), ctypes.byref(strides), None) == INVALID
    assert lib.ellm_kv_read_e4m3(None, 0, 0, 0, 1, 1, None, None, ctypes.byref(steps), None) == INVALID


@pytest.mark.parametrize("desc,status", [
    ((1, 1, 1, 64, 16, 0), UNSUPPORTED), ((1, 1, 1, 128, 16, 2), INVALID), ((0, 1, 1, 128, 16, 0), INVALID),
    ((1, 1, 0, 128, 16, 0), INVALID), ((1, 1, 1, 128, 0, 0), INVALID), ((1, 1 << 20, 1, 128, 16, 0), UNSUPPORTED),
    ((1 << 60, 60000, 60000, 128, 1 << 20, 0), UNSUPPORTED),
])
def test_cache_refuses(desc, status):
    lib = ellm_amd.load_library()
    c = ctypes.c_void_p()
    d = _lib.KvDesc(*desc)
    assert lib.ellm_kv_create_e4m3(ctypes.byref(d), ctypes.byref(c)) == status and not c.value
