"""Paged attention over values at the ends of their range: infinite ones, and finite ones that a weight above 1 would make
infinite on the way."""
from __future__ import annotations

import pytest
import torch

from test_gpu_paged import BF16, E4M3, F16, F32, INT8, TYPES, Case, loaded  # noqa: F401

pytestmark = pytest.mark.gpu

INF = float("inf")


def weights(case):
    """log2 of the smallest softmax weight of the case, by float64."""
    least = 0.0
    for r, n in enumerate(case.lengths.tolist()):
        t = torch.arange(n)
        k = case.exact[0][case.col[case.crow[r] + t // case.page], t % case.page]
        q = case.query[r].double().view(case.kv, -1, case.dim)
        s = torch.log_softmax(torch.einsum("hgd,thd->hgt", q, k) * case.scale, -1)
        least = min(least, s.min().item() / 0.6931471805599453)
    return least


def place(case, row, token):
    return int(case.col[case.crow[row] + token // case.page]), token % case.page


@pytest.mark.parametrize("spread", [1.0, 8.0])
@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, F16)], ids=str)
@pytest.mark.parametrize("shape", [(4, 2, 64, 16), (32, 2, 128, 16), (12, 1, 256, 24), (4, 2, 100, 16)], ids=str)
def test_an_infinite_value_makes_its_feature_infinite(shape, kinds, spread):
    """Every weight is above 0, so a feature with an infinity is that infinity, with both of them NaN, and the others are what
    they were, in every head of the group and nowhere else; whatever the tile of the token and the rounding of its weight."""
    case = Case(shape, kinds, [130, 90, 1, 5000], seed=60, spread=spread)
    assert weights(case) > -126                                    # float32 holds them all
    exact, exact_lse, slack, lse_slack, total = case.expected()
    values = case.pages[1].clone()
    group = case.heads // case.kv
    wanted = {}
    for row, token, head, feature, value in [(0, 0, 0, 5, INF), (0, 77, case.kv - 1, 6, -INF), (0, 129, 0, 7, INF),
                                             (1, 3, 0, 0, INF), (1, 60, 0, 0, INF), (1, 61, 0, 1, INF), (1, 62, 0, 1, -INF),
                                             (1, 89, 0, 2, float("nan")), (2, 0, 0, 9, -INF),
                                             *[(3, 611 * i, 0, i, INF if i % 2 else -INF) for i in range(8)], (3, 4999, 0, 20, INF)]:
        values[(*place(case, row, token), head, feature)] = value
        for h in range(head * group, (head + 1) * group):
            wanted[row, h, feature] = wanted.get((row, h, feature), 0.0) + value
    out, lse = case.run(value_pages=values)
    for at, value in wanted.items():
        got = out[at].item()
        assert got == value or (value != value and got != got), (at, value, got)
        exact[at] = 0.0
        out[at] = 0.0
    case.check((out, lse), (exact, exact_lse, slack, lse_slack, total))


@pytest.mark.parametrize("kinds", [k for k in TYPES if k[1] in (E4M3, INT8)], ids=str)
@pytest.mark.parametrize("shape", [(4, 2, 64, 16), (24, 2, 128, 16)], ids=str)
def test_an_infinite_value_scale(shape, kinds):
    """value = code * scale: infinite by the sign of the code, NaN for a code of 0; the other head and the other rows are what they were."""
    case = Case(shape, kinds, [130, 90, 1, 5000], seed=61)
    exact, exact_lse, slack, lse_slack, total = case.expected()
    group = case.heads // case.kv
    scales = case.scales[1].clone()
    codes = case.pages[1].float().cpu()
    out = {}
    for row, token in ((0, 33), (3, 4321)):
        page, at = place(case, row, token)
        scales[page, 0, at] = INF
        exact[row, :group] = codes[page, at, 0].double() * INF
        slack[row, :group] = total[row, :group] = 0.0
    out, lse = case.run(value_scales=scales)
    special = ~torch.isfinite(exact)
    assert torch.equal(out.cpu().double()[special].nan_to_num(nan=7.0), exact[special].nan_to_num(nan=7.0))
    exact[special] = 0.0
    out[special.cuda()] = 0.0
    case.check((out, lse), (exact, exact_lse, slack, lse_slack, total))


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F32, E4M3), (BF16, E4M3), (BF16, INT8), (F32, INT8)], ids=str)
@pytest.mark.parametrize("shape", [(4, 2, 64, 16), (24, 2, 128, 16), (4, 2, 100, 16), (6, 1, 256, 7)], ids=str)
def test_large_values_whose_scores_rise(shape, kinds):
    """The value of the highest score is near the largest number, and scores have risen by less than a factor of 2^6 before: no weight
    above 1 may make it infinite."""
    case = Case(shape, kinds, [65, 200, 700, 1, 9000], seed=62)
    case.query = torch.zeros_like(case.query)
    case.query[:, :, 0] = 1
    case.scale = 1.0
    gen = torch.Generator().manual_seed(63)
    scores = -30 * torch.rand(case.pages[0].shape[:3], generator=gen) - 20
    size = torch.ones(scores.shape)
    for row, n in enumerate(case.lengths.tolist()):
        for t, score in ((0, 0.0), (64, 3.4), (128, 6.9), (8000, 7.1)):   # every fourth tile is of the same ring
            if t < n:
                scores[place(case, row, t)] = score
        size[place(case, row, next(t for t in (8000, 128, 64, 0) if t < n))] = 2.0 ** 123
    if case.scales[0] is None:
        keys, values = torch.zeros(case.pages[0].shape), case.pages[1].cpu().float().nan_to_num(0.0).clamp(-4, 4)
        keys[..., 0] = scores
        pools = [keys.to(case.cache), (values * size.unsqueeze(-1)).to(case.cache)]
        case.exact = [x.double() for x in pools]
    else:
        keys = torch.zeros(case.pages[0].shape)
        keys[..., 0] = 64
        values = case.pages[1].cpu().float().nan_to_num(0.0)
        pools = [keys.to(case.cache), case.pages[1].cpu()]
        scales = [scores / 64, size * (2.0 ** -6 if kinds[1] == E4M3 else 2.0 ** -4)]
        case.scales = [s.transpose(1, 2).contiguous().cuda() for s in scales]
        case.exact = [k.double() * s.double().unsqueeze(-1) for k, s in zip((keys, values), scales)]
    case.pages = [x.cuda() for x in pools]
    expected = case.expected()
    assert bool((expected[0].abs().amax(-1) < 2.0 ** 127).all()) and expected[0].abs().max() > 2.0 ** 122
    case.check(case.run(), expected)


@pytest.mark.parametrize("kinds", [k for k in TYPES if k[1] in (E4M3, INT8)], ids=str)
@pytest.mark.parametrize("power, key_power, rest", [(127, -110, 17), (126, -110, 16), (-126, 110, -16), (-14, 12, 0), (60, -61, 0)], ids=str)
def test_queries_at_the_ends_of_their_range(kinds, power, key_power, rest):
    """Query features of 2^power or more beside key scales that bring the scores back to where they always are."""
    if kinds[0] == F16 and abs(power) > 15:
        power, key_power, rest = (15, -16, 0) if power > 0 else (-14, 12, 0)
    case = Case((8, 2, 64, 16), kinds, [200, 33, 700], seed=64)
    size = case.query.double().abs().amax(-1, keepdim=True)
    unit = torch.full_like(size, 1.9 * 2.0 ** power)
    case.query = (case.query.double() / size * unit).to(kinds[0])
    assert bool(torch.isfinite(case.query).all())
    case.scales[0] = case.scales[0] * 2.0 ** key_power
    case.exact[0] = case.exact[0] * 2.0 ** key_power
    case.scale = 2.0 ** -rest
    case.check(case.run(), case.expected())


@pytest.mark.parametrize("kinds", [k for k in TYPES if k[1] in (E4M3, INT8)], ids=str)
def test_a_key_of_zeros_scores_0_whatever_its_scale(kinds):
    case = Case((8, 2, 64, 16), kinds, [40], seed=65)
    page, at = place(case, 0, 17)
    if kinds[0] != F16:
        case.query = case.query * 2.0 ** 70
        case.scales[0] = case.scales[0] * 2.0 ** -70
        case.exact[0] = case.exact[0] * 2.0 ** -70
    case.pages[0].view(torch.uint8)[page, at] = 0
    case.exact[0][page, at] = 0
    case.scales[0][page, :, at] = 2.0 ** 100
    case.check(case.run(), case.expected())
