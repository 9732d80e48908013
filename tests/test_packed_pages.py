"""Pages in 4 bits on the host: layout, refusals, and the kernels' layout read from their header."""
import re
from pathlib import Path

import pytest
import torch

from leone_b200.cache import packed

CSRC = Path(packed.__file__).parent.parent / "csrc"


@pytest.mark.parametrize("d", [16, 32, 64, 96, 128, 192, 256, 512])
@pytest.mark.parametrize("values", [False, True])
def test_pack_and_unpack(d, values):
    g = torch.Generator().manual_seed(d)
    shape = (3, 2, 32)
    codes = torch.randint(0, 16, shape + (d,), generator=g, dtype=torch.uint8)
    s, z = torch.randn((2,) + shape + (packed.groups(d),), generator=g).to(torch.bfloat16).unbind(0)
    pool = packed.pack_pages(codes, s, z, values)
    assert pool.dtype == torch.uint8 and pool.shape == shape + (packed.row_bytes(d),) and pool.is_contiguous()
    back = packed.unpack_pages(pool, d, values)
    for got, want in zip(back, (codes, s, z)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("d", [32, 64, 128, 192, 256])
@pytest.mark.parametrize("values", [False, True])
def test_a_token_owns_its_bytes(d, values):
    # a token's write must touch no other token's bytes, and every place of a unit is used once
    places = packed._places(d, values)
    assert sorted(places.flatten().tolist()) == list(range(packed.UNIT * d // 8))


def test_words_follow_the_documented_places():
    # keys: word (g, i) at (i / 2) * 2 G + 2 g + i % 2; values: rows and words as the header's comment has them
    k, v = packed._places(128, False), packed._places(128, True)
    for t in range(16):
        row = (t & 8) | ((t & 7) >> 1) | ((t & 1) << 2)
        for g in range(2):
            for i in range(8):
                assert int(k[t, 8 * g + i]) == 16 * t + (i // 2) * 4 + 2 * g + i % 2
                assert int(v[t, 8 * g + i]) == 16 * row + ((2 * i + g) ^ (8 * ((row >> 1) & 1)))


def test_nibbles():
    codes = torch.zeros((1, 1, 16, 32), dtype=torch.uint8)
    codes[0, 0, 0, :8] = torch.arange(1, 9)
    zero = torch.zeros((1, 1, 16, 1))
    word = int(packed.pack_pages(codes, zero, zero, False).view(torch.int32)[0, 0, 0, 0]) & 0xFFFFFFFF
    assert word == 0x86427531                    # elements 0, 2, 4, 6 in the low half, 1, 3, 5, 7 in the high one


@pytest.mark.parametrize("d", [0, 4, 20, 72, 144 + 8, 176, 520])
def test_dims_that_cannot_be_held(d):
    assert not packed.dim_ok(d)
    with pytest.raises(ValueError):
        packed._check_pool(16, d)


def test_refusals():
    codes = torch.zeros((1, 1, 24, 64), dtype=torch.uint8)
    with pytest.raises(ValueError, match="multiple of 16"):
        packed.pack_pages(codes, torch.zeros(1, 1, 24, 1), torch.zeros(1, 1, 24, 1), False)
    with pytest.raises(ValueError, match="scales"):
        packed.pack_pages(codes[:, :, :16], torch.zeros(1, 1, 16, 2), torch.zeros(1, 1, 16, 2), False)
    with pytest.raises(ValueError, match="uint8"):
        packed.unpack_pages(torch.zeros((1, 1, 16, 35), dtype=torch.uint8), 64, False)


def test_header_and_host_agree():
    text = (CSRC / "cache4.cuh").read_text()
    assert re.search(r"kUnit = 16\b", text) and re.search(rf"kMaxDim = {packed.MAX_DIM}\b", text)
    assert "return (d + 63) / 64;" in text and "return d / 2 + 4 * groups(d);" in text
