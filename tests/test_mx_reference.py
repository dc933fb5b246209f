"""The MXFP4 codec that the GPU tests are held to, against its definition by hand."""

import math

import torch

from mx_reference import VALUES, decode, encode, nearest, scale_bytes


def test_scale_is_the_rounded_exponent_less_two():
    top = torch.tensor([1.0, 1.7499, 1.75, 2.0, 6.99, 7.0, 8.0, 2.0**-123, 2.0**-124, 0.0,
                        3.3e38, math.inf], dtype=torch.float64)
    want = [125, 125, 126, 126, 127, 128, 128, 2, 0, 0, 252, 255]
    assert scale_bytes(top).tolist() == want


def test_codes_are_the_nearest_halves_to_even():
    x = torch.tensor([0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 6.9, -0.75, -5.0],
                     dtype=torch.float64)
    got = nearest(x, torch.tensor(127))
    assert got.tolist() == [0.0, 0.5, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, -1.0, -4.0]


def test_packing():
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :16] = torch.cat((VALUES, -VALUES))
    codes, byte = encode(x)
    assert byte.tolist() == [[127]]
    assert codes[0, :8].tolist() == [0x10, 0x32, 0x54, 0x76, 0x98, 0xba, 0xdc, 0xfe]
    assert torch.equal(decode(codes, byte), x)


def test_every_byte_decodes_to_what_it_stands_for():
    codes = torch.arange(256, dtype=torch.uint8).view(16, 16)
    got = decode(codes, torch.full((16, 1), 130, dtype=torch.uint8))
    for i in range(256):
        for j, c in enumerate((i & 15, i >> 4)):
            e, m = c >> 1 & 3, c & 1
            v = m / 2 if e == 0 else (1 + m / 2) * 2.0**(e - 1)
            assert got[i // 16, 2 * (i % 16) + j] == (-v if c & 8 else v) * 8.0
    assert torch.isnan(decode(codes, torch.full((16, 1), 255, dtype=torch.uint8))).all()


def test_blocks_out_of_the_ordinary():
    x = torch.zeros(4, 32, dtype=torch.float64)
    x[0, 3] = math.nan
    x[1, 5] = -math.inf
    x[2, 7] = 2.0**-124
    x[3] = torch.linspace(-3.38e38, 3.38e38, 32, dtype=torch.float64)
    codes, byte = encode(x)
    assert byte[:, 0].tolist() == [255, 255, 0, 252] and not codes[:3].any()
    assert torch.isfinite(decode(codes, byte)[2:]).all()
