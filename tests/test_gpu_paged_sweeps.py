"""The paged cache's quantising over whole ranges: every mantissa a scale can come from, every pair of 16-bit mantissas."""
from __future__ import annotations

import pytest
import torch

from paged_reference import LARGEST
from test_gpu_paged import BF16, E4M3, F16, F32, INT8, loaded  # noqa: F401

pytestmark = pytest.mark.gpu


def nearest(y, kind):
    """y (float64) rounded to the nearest value of the type, ties to even: 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    if kind == INT8:
        return torch.round(y)
    _, power = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (power - 1).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def stored(x, kind):
    """(codes as float64, scales) of the rows x[tokens, heads, dim] in the key pages and in the value pages, which hold -x."""
    from autosage_b200 import paged

    tokens, heads, dim = x.shape
    page = 64
    assert tokens % page == 0
    pools = [torch.zeros(tokens // page, page, heads, dim, device="cuda").to(kind) for _ in range(2)]
    scales = [torch.zeros(tokens // page, heads, page, device="cuda") for _ in range(2)]
    paged.paged_cache_write(torch.arange(tokens, device="cuda"), x, -x, *pools, key_scales=scales[0], value_scales=scales[1])
    return ([p.view(tokens, heads, dim).float().double() for p in pools], [s.transpose(1, 2).reshape(tokens, heads) for s in scales])


@pytest.mark.parametrize("power", [-79, -1, 0, 88])
@pytest.mark.parametrize("kind", [E4M3, INT8], ids=str)
def test_the_scale_of_every_float32_mantissa(kind, power):
    """The scale is max|x| / Q rounded once, and max|x| is stored as Q; the ends of the range that is computed in float32 among them."""
    x = (torch.arange(1 << 23, device="cuda", dtype=torch.int32) | (127 + power) << 23).view(torch.float32).view(-1, 8, 1)
    codes, scales = stored(x, kind)
    # (a 24-bit number over one of 9 bits is never within 2^-34 of the middle between two float32 numbers: float64 decides)
    exact = (x.double() / LARGEST[kind]).float().squeeze(-1)
    assert torch.equal(scales[0], exact) and torch.equal(scales[1], exact)
    assert bool((codes[0] == LARGEST[kind]).all()) and bool((codes[1] == -LARGEST[kind]).all())


@pytest.mark.parametrize("cache", [E4M3, INT8], ids=str)
@pytest.mark.parametrize("kind, bits", [(F16, 10), (BF16, 7)], ids=["float16", "bfloat16"])
def test_the_codes_of_every_pair_of_16_bit_mantissas(kind, bits, cache):
    """Every largest value of a binade with every smaller one of 21 binades, whether the scale is exact, rounded up or rounded down."""
    count = 1 << bits
    mantissas = 1 + torch.arange(count, device="cuda").double() / count
    values = torch.ldexp(mantissas.repeat(21, 1), 14 - torch.arange(21, device="cuda").view(-1, 1)).view(-1)
    rows = -(-values.numel() // 255)
    others = torch.zeros(rows * 255, dtype=torch.float64, device="cuda")
    others[:values.numel()] = values
    seen = set()
    for part in torch.arange(count, device="cuda").split(64):
        tops = (mantissas[part] * 2.0 ** 14).view(-1, 1, 1)
        smaller = others.view(1, rows, 255).expand(part.numel(), rows, 255)
        x = torch.cat((tops.expand(-1, rows, 1), torch.where(smaller <= tops, smaller, torch.zeros_like(smaller))), 2)
        given = x.to(kind)
        assert torch.equal(given.double(), x)
        codes, scales = stored(given, cache)
        scale = (tops.view(-1, 1) / LARGEST[cache]).float().expand(-1, rows)
        seen |= set(torch.sign(tops.view(-1) - scale[:, 0].double() * LARGEST[cache]).tolist())
        # (x is a multiple of its last place, and so is the border times the scale: float64's quotient lies on a border if the true one does)
        exact = nearest(x / scale.double().unsqueeze(-1), cache)
        for got, sign in zip(codes, (1, -1)):
            assert torch.equal(got, sign * exact)
        assert torch.equal(scales[0], scale) and torch.equal(scales[1], scale)
    assert seen == {-1.0, 0.0, 1.0}


@pytest.mark.parametrize("cache", [E4M3, INT8], ids=str)
def test_float32_quotients_beside_the_borders(cache):
    """Rows whose other values are the float32 numbers at, just below and just above each border between codes, for some 4,000 scales."""
    gen = torch.Generator().manual_seed(70)
    values = torch.arange(127, dtype=torch.uint8).view(E4M3).double() if cache == E4M3 else torch.arange(128).double()
    middle = ((values[1:] + values[:-1]) / 2).cuda()
    tops = torch.cat((torch.exp2(torch.linspace(-70, 80, 4032)).float() * (1 + torch.rand(4032, generator=gen)),
                      torch.ldexp(torch.full((64,), LARGEST[cache]), torch.arange(-32, 32)))).cuda()
    scale = (tops.double() / LARGEST[cache]).float()
    border = middle.view(1, -1) * scale.double().view(-1, 1)
    near = border.float()
    x = torch.cat((tops.view(-1, 1), near, torch.nextafter(near, torch.zeros_like(near))), 1).unsqueeze(1)
    x = torch.where(x <= tops.view(-1, 1, 1), x, torch.zeros_like(x))[..., :256].contiguous()
    codes, scales = stored(x, cache)
    assert torch.equal(scales[0].view(-1), scale)
    # (a quotient of two 24-bit numbers that is not on a border of at most 9 bits is 2^-40 of itself away from it)
    exact = nearest(x.double() / scale.double().view(-1, 1, 1), cache)
    assert torch.equal(codes[0], exact) and torch.equal(codes[1], -exact)
