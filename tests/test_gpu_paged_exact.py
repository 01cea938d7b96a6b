"""Paged attention where every token's share of the answer is known exactly."""
from __future__ import annotations

import pytest
import torch

from paged_reference import HALF_STEP, LARGEST
from test_gpu_paged import BF16, E4M3, F16, F32, INT8, TYPES, Case, loaded  # noqa: F401

pytestmark = pytest.mark.gpu


def counted(shape, kinds, lengths, block=16, **options):
    """A case whose query is 0, so that all weights are 1, and whose value rows are 1 in feature (position // block) % dim and
    0 elsewhere: output feature f is the share of the row's tokens that belong to f, the log-sum-exp log n."""
    case = Case(shape, kinds, lengths, **options)
    case.query = torch.zeros_like(case.query)
    place, feature = [], []
    for r, n in enumerate(lengths):
        t = torch.arange(n)
        place.append(case.col[case.crow[r] + t // case.page] * case.page + t % case.page)
        feature.append(t // block % case.dim)
    place, feature = torch.cat(place), torch.cat(feature)
    one = 64.0 if case.cache in LARGEST else 1.0                 # a code that both 8-bit types hold, with a scale of 2^-6
    rows = torch.zeros(place.numel(), case.kv, case.dim)
    rows[torch.arange(place.numel()), :, feature] = one
    values = case.pages[1].cpu()
    flat = values.reshape(-1, case.kv, case.dim)
    if values.element_size() == 1:
        flat.view(torch.uint8)[place] = rows.to(values.dtype).view(torch.uint8)
    else:
        flat[place] = rows.to(values.dtype)
    case.pages[1] = flat.view(values.shape).cuda()
    if case.scales[1] is not None:
        case.scales[1] = torch.full_like(case.scales[1], 2.0 ** -6)
    case.block = block
    return case


def shares(case, window=None):
    out = torch.zeros(len(case.lengths), case.dim, dtype=torch.float64)
    n = case.lengths.clone()
    for r, length in enumerate(case.lengths.tolist()):
        t = torch.arange(max(0, length - window) if window else 0, length)
        n[r] = t.numel()
        if t.numel():
            out[r] = torch.bincount(t // case.block % case.dim, minlength=case.dim).double() / t.numel()
    return out, torch.log(n.double())


def check(case, got, window=None):
    exact, exact_lse = shares(case, window)
    out, lse = got[0].double().cpu(), got[1].double().cpu()
    # weights of 1 and their sums are whole numbers below 2^24, whatever pieces they are joined from: what is left is the
    # rounding of 1 / n, of the product with it, and of the answer to its type
    limit = (2.0 ** -23 + HALF_STEP[case.kind] * (1 + 2.0 ** -22)) * exact
    assert bool(((out - exact.unsqueeze(1)).abs() <= limit.unsqueeze(1)).all())
    # log2 (one unit in the last place), the factor ln 2 and its product
    assert torch.equal(lse == float("-inf"), (exact_lse == float("-inf")).unsqueeze(1).expand_as(lse))
    fine = torch.isfinite(exact_lse)
    assert bool(((lse - exact_lse.unsqueeze(1)).abs()[fine] <= 2.0 ** -22 * exact_lse.unsqueeze(1)[fine]).all())


@pytest.mark.parametrize("kinds", TYPES, ids=str)
@pytest.mark.parametrize("lengths", [[1, 60001, 1], [40000], [5000] * 10, [4000, 3000, 1, 0, 2500, 7001] * 3, [300] * 200,
                                     [2000 + 37 * r for r in range(24)], [64] * 7, list(range(130))], ids=lambda n: f"{len(n)}x{max(n)}")
def test_every_token_counts_once(lengths, kinds):
    """Wherever shares end and pieces are joined, no tile is lost or taken twice."""
    case = counted((4, 2, 64, 16), kinds, lengths, seed=50)
    check(case, case.run())
    check(case, case.run(window=777), window=777)


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, E4M3), (F32, INT8)], ids=str)
@pytest.mark.parametrize("shape", [(24, 1, 128, 24), (16, 1, 256, 64), (3, 3, 100, 7)], ids=str)
def test_every_token_counts_once_in_other_heads(shape, kinds):
    case = counted(shape, kinds, [30011, 900, 0, 17], seed=51)
    check(case, case.run())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, INT8)], ids=str)
def test_more_items_than_ctas_on_one_walk(kinds):
    """Each CTA walks through many whole items, some with rows that see nothing between them."""
    lengths = [17 * (r % 13) for r in range(3000)]
    case = counted((6, 3, 64, 16), kinds, lengths, seed=52)
    check(case, case.run())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, INT8)], ids=str)
def test_a_crow_whose_rows_overlap_past_2_to_the_32_entries(kinds):
    """No table, and no answer: every second row lists all columns, 2^32 entries and some 65,000 of the list together.  The call ends,
    and the next one is right."""
    from autosage_b200 import paged

    rows, n, page = 65534, 4096, 1024
    assert (rows // 2 * (n * page // 64 + 3) * 2) % 2 ** 32 < 2 ** 17 < 2 ** 32 < rows // 2 * (n * page // 64 + 3) * 2
    case = counted((4, 2, 64, 16), kinds, [700, 3], seed=53)
    pools = dict(key_pages=torch.zeros(4, page, 2, 64, device="cuda").to(case.cache),
                 value_pages=torch.zeros(4, page, 2, 64, device="cuda").to(case.cache))
    if case.cache in LARGEST:
        pools.update(key_scales=torch.ones(4, 2, page, device="cuda"), value_scales=torch.ones(4, 2, page, device="cuda"))
    crow = torch.tensor([0, n], device="cuda").repeat(rows // 2 + 1)[:rows + 1]
    lengths = torch.full((rows,), n * page, device="cuda")
    out = paged.csr_paged_attention(crow, torch.arange(n, device="cuda") % 4, lengths,
                                    torch.zeros(rows, 4, 64, device="cuda").to(case.kind), **pools)
    torch.cuda.synchronize()
    assert out.shape == (rows, 4, 64)
    check(case, case.run())


def on_four_pages(kinds, lengths, rows_of_values, dim=64, page=1024, kv=2):
    """A call whose rows list the same four pages over and over: long rows from little memory.  Queries and keys are such that
    all weights are 1.  rows_of_values: [4 * page, dim], of values that the type of the pages holds times 2^-6."""
    from autosage_b200 import paged

    kind, cache = kinds
    counts = torch.tensor([-(-n // page) for n in lengths])
    crow = torch.zeros(len(lengths) + 1, dtype=torch.long)
    torch.cumsum(counts, 0, out=crow[1:])
    col = torch.cat([torch.arange(int(c)) % 4 for c in counts])
    values = rows_of_values.view(4, page, 1, dim).expand(4, page, kv, dim)
    scales = {}
    if cache in LARGEST:
        scales = dict(key_scales=torch.ones(4, kv, page, device="cuda"), value_scales=torch.full((4, kv, page), 2.0 ** -6, device="cuda"))
        values = values * 64
    values = values.to(cache).contiguous().cuda()
    keys = torch.ones(4, page, kv, dim, device="cuda").to(cache)
    out, lse = paged.csr_paged_attention(crow.cuda(), col.cuda(), torch.tensor(lengths).cuda(),
                                         torch.zeros(len(lengths), 2 * kv, dim, device="cuda", dtype=kind), keys, values,
                                         return_lse=True, **scales)
    return out.double().cpu(), lse.double().cpu()


@pytest.mark.parametrize("kinds", TYPES, ids=str)
@pytest.mark.parametrize("lengths", [[2 ** 20 + 77] * 40 + [5, 0, 9000] + [700001] * 3, [3 * 2 ** 20 + 1, 1, 2 ** 21],
                                     [70000 + 1111 * (r % 13) for r in range(900)]], ids=lambda n: f"{len(n)}x{max(n)}")
def test_pieces_of_many_legs(lengths, kinds):
    """Items of many legs, whole in a CTA, cut once or running through several: every token counts once."""
    marks = torch.zeros(4096, 64)
    marks[torch.arange(4096), torch.arange(4096) // 16 % 64] = 1
    out, lse = on_four_pages(kinds, lengths, marks)
    n = torch.tensor(lengths)
    whole = torch.bincount(torch.arange(4096) // 16 % 64, minlength=64)
    exact = torch.stack([(whole * (m // 4096) + torch.bincount(torch.arange(m % 4096) // 16 % 64, minlength=64)).double() / max(m, 1)
                         for m in lengths])
    limit = (2.0 ** -23 + HALF_STEP[kinds[0]] * (1 + 2.0 ** -22)) * exact     # as in check()
    assert bool(((out - exact.unsqueeze(1)).abs() <= limit.unsqueeze(1)).all())
    some = n > 0
    assert bool(((lse - torch.log(n.double()).unsqueeze(1))[some].abs() <= 2.0 ** -22 * torch.log(n.double())[some].unsqueeze(1)).all())


@pytest.mark.parametrize("kinds", TYPES, ids=str)
def test_a_million_equal_tokens(kinds):
    """The mean of equal values is the value, however many there are in one accumulator's way: 1200 rows of 2^20 tokens, more items
    than CTAs, so that each CTA adds up whole rows."""
    value = 85 / 64 if kinds[1] != E4M3 else 88 / 64                 # held by every type (with the scale of 2^-6 by the 8-bit ones)
    out, lse = on_four_pages(kinds, [2 ** 20] * 1200, torch.full((4096, 64), value), kv=1)
    # sums of a leg, cut off on the tensor cores (2 x 128 of 2^-23 of them) or rounded on the FMA pipe (1024 of 2^-24), one rounding a
    # leg when it is added to those before (128 legs of 8192 tokens, 256 of 4096), then 1 / n, the product and the type's rounding
    error = 2.0 ** -14 + 2.0 ** -16 + 2.0 ** -23 if kinds[1] == F32 else 2.0 ** -15 + 2.0 ** -17 + 2.0 ** -23
    if kinds[0] == F32:
        assert bool(((out - value).abs() <= (error + 2.0 ** -24) * value).all())
    else:
        assert error < HALF_STEP[kinds[0]] / 2 and bool((out == value).all())    # nothing else lies as near
    assert bool(((lse - torch.log(torch.tensor(2.0 ** 20).double())).abs() <= 2.0 ** -22 * 14).all())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, INT8)], ids=str)
def test_a_workspace_that_is_too_small_is_refused(kinds, monkeypatch):
    """By the library, before anything is launched; the next call is right."""
    from autosage_b200 import _native

    case = counted((4, 2, 64, 16), kinds, [3000, 5], seed=54)
    check(case, case.run())
    whole = _native._scratch_on
    for cut, message in ((lambda w: w[:4096], "smaller than"), (lambda w: w[128:], "256-byte aligned"),
                         (lambda w: w[:0], "null")):
        monkeypatch.setattr(_native, "_scratch_on", lambda *of: cut(whole(*of)))
        with pytest.raises(RuntimeError, match=message):
            case.run()
    monkeypatch.setattr(_native, "_scratch_on", whole)
    check(case, case.run())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16)], ids=str)
def test_another_operator_of_another_thread_on_the_same_stream(kinds, monkeypatch):
    """An SpMM that builds its plan in the stream's scratch at every call, between the launches of the attention's calls."""
    import threading

    import autosage_b200

    monkeypatch.setenv("AUTOSAGE_PLAN_CACHE", "0")
    case = counted((4, 1, 64, 16), kinds, [9000, 40, 7000], seed=55)
    fixed = dict(crow=case.crow.cuda(), col=case.col.cuda(), lengths=case.lengths.cuda(), query=case.query.cuda())
    gen = torch.Generator().manual_seed(56)
    degrees = torch.randint(0, 40, (3000,), generator=gen)
    crow = torch.cat((torch.zeros(1, dtype=torch.long), degrees.cumsum(0))).cuda()
    col = torch.randint(0, 3000, (int(degrees.sum()),), generator=gen).cuda()
    val, x = torch.ones(col.numel(), device="cuda"), torch.randn(3000, 64, generator=gen).cuda()
    wanted, sums = case.run(**fixed), autosage_b200.spmm_csr(crow, col, val, x)
    check(case, wanted)
    answers, others = [], []

    def attend():
        with torch.no_grad():
            answers.extend(case.run(**fixed) for _ in range(200))

    def aggregate():
        with torch.no_grad():
            others.extend(autosage_b200.spmm_csr(crow, col, val, x) for _ in range(200))

    threads = [threading.Thread(target=work) for work in (attend, aggregate)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert len(answers) == len(others) == 200
    assert all(torch.equal(out, wanted[0]) and torch.equal(lse, wanted[1]) for out, lse in answers)
    assert all(torch.equal(y, sums) for y in others)
