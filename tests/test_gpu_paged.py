"""The paged cache and its attention on the GPU against the float64 restatement in ``paged_reference.py``."""
from __future__ import annotations

import pytest
import torch

from helpers import misaligned_copy
from paged_reference import HALF_STEP, LARGEST, attention, quantise

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3, INT8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, E4M3), (BF16, E4M3), (F16, E4M3), (F32, INT8), (BF16, INT8), (F16, INT8)]
# query heads, key heads, features, page size
SHAPES = [(1, 1, 1, 1), (4, 4, 64, 16), (32, 8, 128, 16), (20, 4, 96, 24), (12, 3, 40, 7), (6, 2, 113, 5), (16, 1, 256, 64),
          (16, 1, 192, 32), (24, 1, 100, 1), (40, 2, 72, 128), (2, 2, 32, 3), (36, 2, 128, 16), (3, 1, 8, 16)]
LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0, 700]


@pytest.fixture(scope="module", autouse=True)
def loaded():
    import autosage_b200

    assert torch.cuda.is_available()
    assert autosage_b200.load_native(), autosage_b200.ops.native_load_error()


def codes(x, kind):
    """8-bit pages of x [n, page, heads, dim] with scales [n, heads, page], and the float64 values that they stand for."""
    value, scale = quantise(x.double(), kind)
    stored = value.to(torch.int8) if kind == INT8 else value.float().to(E4M3)
    return stored, scale.transpose(1, 2).float().contiguous(), value * scale.unsqueeze(-1)


class Case:
    """Random pages, a shuffled page table and a query; everything that no row may see holds NaN."""

    def __init__(self, shape, kinds, lengths, seed=0, reserve=1, spread=1.0, layout="token"):
        self.heads, self.kv, self.dim, self.page = shape
        self.kind, self.cache = kinds
        gen = torch.Generator().manual_seed(seed)
        self.lengths = torch.tensor(lengths, dtype=torch.long)
        counts = (self.lengths + self.page - 1) // self.page + reserve
        self.crow = torch.zeros(len(lengths) + 1, dtype=torch.long)
        torch.cumsum(counts, 0, out=self.crow[1:])
        n = int(self.crow[-1]) + 2
        self.col = torch.randperm(n, generator=gen)[:int(self.crow[-1])]
        self.query = torch.randn(len(lengths), self.heads, self.dim, generator=gen).to(self.kind)
        self.scale = spread * self.dim ** -0.5
        used = torch.zeros(n * self.page, dtype=torch.bool)
        for r, length in enumerate(lengths):
            t = torch.arange(length)
            used[self.col[self.crow[r] + t // self.page] * self.page + t % self.page] = True
        used = used.view(n, self.page)
        self.pages, self.scales, self.exact = [], [], []
        for _ in range(2):
            x = torch.randn(n, self.page, self.kv, self.dim, generator=gen).to(self.kind if self.cache in LARGEST else self.cache)
            scale = None
            if self.cache in LARGEST:
                stored, scale, exact = codes(x, self.cache)
                scale = torch.where(used.unsqueeze(1), scale, torch.full_like(scale, float("nan")))
                if self.cache == E4M3:
                    stored.view(torch.uint8)[~used] = 0x7F
            else:
                stored, exact = x, x.double()
                stored[~used] = float("nan")
            if layout == "head":      # pages with the heads outside the tokens
                stored = stored.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            self.pages.append(stored.cuda())
            self.scales.append(None if scale is None else scale.cuda())
            self.exact.append(exact)

    def run(self, window=None, lse=True, query=None, **change):
        from autosage_b200 import paged

        for name in ("crow", "col", "lengths"):
            if name not in change:                                # (nothing is copied inside a capture)
                change[name] = getattr(self, name).cuda()
        call = dict(query=self.query.cuda() if query is None else query, key_pages=self.pages[0], value_pages=self.pages[1],
                    key_scales=self.scales[0], value_scales=self.scales[1], scale=self.scale, window=window, return_lse=lse)
        call.update(change)
        return paged.csr_paged_attention(**call)

    def expected(self, window=None, crow=None, col=None, lengths=None):
        return attention(self.crow if crow is None else crow, self.col if col is None else col,
                         self.lengths if lengths is None else lengths, self.query.double(), *self.exact, self.page, self.scale, window)

    def check(self, got, expected):
        out, lse = got
        exact, exact_lse, slack, lse_slack, spread = expected
        out, lse = out.double().cpu(), lse.double().cpu()
        # with a 16-bit query the weights go to the tensor cores as two pieces of the storage type (2^-16 of a weight at
        # most is lost); then the result, itself off by the slack, is rounded once, by a fixed step below the normal range
        if self.kind != F32:
            slack = slack + 2.0 ** -16 * spread
        bound = slack + HALF_STEP[self.kind] * (exact.abs() + slack) + torch.finfo(self.kind).tiny
        worst = ((out - exact).abs() / bound).max().item()
        assert worst <= 1, f"out: error / bound = {worst:.3f}"
        assert torch.equal(lse == float("-inf"), exact_lse == float("-inf"))
        fine = torch.isfinite(exact_lse)
        off = (lse - exact_lse).abs()[fine] / (lse_slack + 2.0 ** -23 * exact_lse.abs())[fine]
        assert off.numel() == 0 or off.max().item() <= 1, f"lse: error / bound = {off.max().item():.3f}"


@pytest.mark.parametrize("kinds", TYPES, ids=lambda k: str(k[0])[6:] + "-" + str(k[1])[6:])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention(shape, kinds):
    case = Case(shape, kinds, LENGTHS)
    case.check(case.run(), case.expected())
    case.check(case.run(window=50), case.expected(window=50))


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, INT8)], ids=str)
def test_attention_with_a_window_and_without_a_reserve(kinds):
    case = Case((8, 2, 64, 16), kinds, LENGTHS, seed=1, reserve=0)
    for window in (1, 16, 17, 64, 100000):
        case.check(case.run(window=window), case.expected(window=window))


@pytest.mark.parametrize("kinds", TYPES, ids=str)
def test_one_long_row_is_split_and_joined(kinds):
    """One row shared by every CTA of the GPU, beside rows of one token: the pieces are joined in order, twice alike."""
    case = Case((4, 1, 64, 16), kinds, [1, 60001, 1], seed=2, spread=3.0)
    first = case.run()
    case.check(first, case.expected())
    again = case.run()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, INT8)], ids=str)
def test_shared_rows_of_every_size(kinds):
    """Rows cut into two pieces, into dozens and into hundreds, one call after another on one workspace."""
    cases = [Case((2, 1, 64, 16), kinds, lengths, seed=30 + i) for i, lengths in enumerate(
        ([5000] * 10, [4000, 3000, 1, 0, 2500, 7001] * 3, [300] * 200, [40000], [2000 + 37 * r for r in range(24)], [64] * 7))]
    expected = [case.expected() for case in cases]
    first = [case.run() for case in cases]
    for case, got, exact in zip(cases, first, expected):
        case.check(got, exact)
    for case, got in zip(reversed(cases), reversed(first)):
        again = case.run()
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (BF16, E4M3)], ids=str)
def test_many_short_rows(kinds):
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 90, (2500,), generator=gen)
    lengths[torch.rand(2500, generator=gen) < 0.5] = 0          # a padded batch: runs of empty rows
    lengths[600:1400] = 0
    case = Case((4, 2, 32, 8), kinds, lengths.tolist(), seed=3)
    case.check(case.run(), case.expected())


@pytest.mark.parametrize("kinds", [(F32, F32), (F16, F16), (BF16, INT8)], ids=str)
def test_all_rows_empty_and_no_rows_at_all(kinds):
    case = Case((4, 2, 32, 8), kinds, [0, 0, 0], seed=4)
    out, lse = case.run()
    assert out.abs().max() == 0 and bool((lse == float("-inf")).all())
    none = dict(crow=torch.zeros(1, dtype=torch.long, device="cuda"), col=torch.zeros(0, dtype=torch.long, device="cuda"),
                lengths=torch.zeros(0, dtype=torch.long, device="cuda"), query=case.query[:0].cuda())
    out, lse = case.run(**none)
    assert out.shape == (0, 4, 32) and lse.shape == (0, 4)
    # rows, but not a single page
    empty = dict(crow=torch.zeros(4, dtype=torch.long, device="cuda"), col=none["col"],
                 key_pages=case.pages[0][:0], value_pages=case.pages[1][:0])
    if case.scales[0] is not None:
        empty.update(key_scales=case.scales[0][:0], value_scales=case.scales[1][:0])
    out, lse = case.run(**empty)
    assert out.abs().max() == 0 and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("kinds", TYPES, ids=str)
def test_holes_short_tables_and_lengths_past_the_pages(kinds):
    """Ids outside the pages mask their tokens (a row may consist of nothing else); a length past the row's pages is cut;
    crow past the columns too."""
    case = Case((6, 3, 64, 16), kinds, [200, 64, 40, 33, 500], seed=5)
    col = case.col.clone()
    n = case.pages[0].size(0)
    col[case.crow[0] + 1] = -1
    col[case.crow[0] + 4:case.crow[0] + 9] = n                   # a whole unit of tokens and more
    col[case.crow[1]:case.crow[2]] = -7                          # row 1 sees nothing
    col[case.crow[4] + 30] = 2 ** 40
    case.check(case.run(col=col.cuda()), case.expected(col=col))
    # the reserve pages hold NaN: rows may not be read past their lengths, but lengths may point past the table
    case = Case((6, 3, 64, 16), kinds, [208, 64], seed=6, reserve=0)
    lengths = torch.tensor([100000, -3])
    case.check(case.run(lengths=lengths.cuda()), case.expected(lengths=torch.tensor([208, 0])))
    crow = case.crow.clone()
    crow[-1] += 1000
    case.check(case.run(crow=crow.cuda()), case.expected())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, INT8)], ids=str)
def test_rows_may_share_pages(kinds):
    """A common prefix: two rows list the same pages."""
    case = Case((4, 2, 64, 16), kinds, [160, 160], seed=7, reserve=0)
    col = case.col.clone()
    col[10:17] = col[0:7]
    case.check(case.run(col=col.cuda()), case.expected(col=col))


@pytest.mark.parametrize("kinds", TYPES, ids=str)
def test_keys_and_values_in_pages_of_different_strides(kinds):
    case = Case((8, 2, 64, 16), kinds, [33, 0, 257, 64], seed=19)
    expected = case.expected()
    turned = case.pages[1].transpose(1, 2).contiguous().transpose(1, 2)
    case.check(case.run(value_pages=turned), expected)
    both = torch.stack(case.pages, 1) if case.pages[0].element_size() > 1 else \
        torch.stack([p.view(torch.uint8) for p in case.pages], 1).view(case.pages[0].dtype)
    case.check(case.run(key_pages=both[:, 0], value_pages=both[:, 1]), expected)   # [pages, 2, page, heads, dim]
    case.check(case.run(window=2 ** 70), expected)


@pytest.mark.parametrize("kinds", [(F32, E4M3), (BF16, E4M3), (F16, INT8), (BF16, INT8)], ids=str)
def test_scales_of_either_sign_and_other_sizes(kinds):
    """Scales are the caller's: negative ones, zeros, keys and values whose tokens differ by 2^8 in size."""
    case = Case((8, 2, 64, 16), kinds, [200, 33, 700], seed=20)
    gen = torch.Generator().manual_seed(21)
    for w in range(2):
        factor = torch.exp2(torch.randint(-8, 1, case.scales[w].shape, generator=gen).float())
        factor[torch.rand(factor.shape, generator=gen) < 0.3] *= -1
        factor[torch.rand(factor.shape, generator=gen) < 0.05] = 0
        case.scales[w] = case.scales[w] * factor.cuda()
        case.exact[w] = case.exact[w] * factor.double().transpose(1, 2).unsqueeze(-1)
    case.check(case.run(), case.expected())


@pytest.mark.parametrize("kinds", [(F32, E4M3), (BF16, E4M3), (F16, INT8), (BF16, INT8), (F32, INT8)], ids=str)
def test_a_zero_value_takes_all_the_weight_of_large_ones(kinds):
    """The first token of a row has a value scale of 0 and outweighs the others, whose values are large, by some 2^900."""
    case = Case((8, 2, 64, 16), kinds, [200, 33, 700], seed=23)
    case.query = case.query.abs()
    first = case.col[case.crow[:-1]]
    codes = case.pages[0].view(torch.uint8)
    codes[first, 0] = codes[first, 0] & 0x7F if case.cache == E4M3 else case.pages[0][first, 0].abs().view(torch.uint8)
    case.scales[0][first, :, 0] *= 128
    case.scales[1] *= 2.0 ** 17
    case.scales[1][first, :, 0] = 0
    case.exact[0][first, 0] = case.exact[0][first, 0].abs() * 128
    case.exact[1] *= 2.0 ** 17
    case.exact[1][first, 0] = 0
    expected = case.expected()
    assert expected[0].abs().max() < 1e-60                        # (float64 holds what float32 cannot)
    case.check(case.run(), expected)


@pytest.mark.parametrize("kind", [F32, BF16, F16], ids=str)
def test_a_nan_code_is_a_nan(kind):
    case = Case((4, 2, 64, 16), (kind, E4M3), [100, 70], seed=22)
    page, place = int(case.col[case.crow[0] + 1]), 3
    keys = case.pages[0].clone()
    keys.view(torch.uint8)[page, place, 1, 5] = 0x7F
    out, lse = case.run(key_pages=keys)
    assert bool(torch.isnan(out[0, 2:]).all()) and bool(torch.isnan(lse[0, 2:]).all())
    assert bool(torch.isfinite(out[0, :2]).all()) and bool(torch.isfinite(out[1]).all())
    values = case.pages[1].clone()
    values.view(torch.uint8)[page, place, 0, 9] = 0xFF
    out, lse = case.run(value_pages=values)
    assert bool(torch.isnan(out[0, :2, 9]).all()) and int(torch.isnan(out).sum()) == 2 and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("kinds", [(BF16, BF16), (F32, F32)], ids=str)
def test_two_threads_on_one_stream(kinds):
    """Calls of two host threads on the same stream share its workspace; their launches do not interleave."""
    import threading

    cases = [Case((4, 1, 64, 16), kinds, lengths, seed=40 + i) for i, lengths in enumerate(([9000], [100, 7000, 3]))]
    wanted = [case.run() for case in cases]
    calls = []
    for case in cases:
        fixed = dict(crow=case.crow.cuda(), col=case.col.cuda(), lengths=case.lengths.cuda(), query=case.query.cuda())
        calls.append(lambda case=case, fixed=fixed: case.run(**fixed))
    results = [[], []]

    def work(i):
        with torch.no_grad():
            for _ in range(200):
                results[i].append(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for got, exact in zip(results, wanted):
        assert len(got) == 200 and all(torch.equal(out, exact[0]) and torch.equal(lse, exact[1]) for out, lse in got)


def test_writing_counts_as_a_change_in_place():
    from autosage_b200 import paged

    pages = [torch.zeros(2, 8, 1, 64, device="cuda") for _ in range(2)]
    before = [p._version for p in pages]
    x = torch.ones(1, 1, 64, device="cuda")
    paged.paged_cache_write(torch.tensor([3], device="cuda"), x, x, *pages)
    assert all(p._version > v for p, v in zip(pages, before))
    with torch.inference_mode():
        pages = [torch.zeros(2, 8, 1, 64, device="cuda") for _ in range(2)]
        paged.paged_cache_write(torch.tensor([3], device="cuda"), x, x, *pages)
        assert pages[0][0, 3].min().item() == 1


@pytest.mark.parametrize("kinds", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(8, 2, 128, 16), (5, 5, 48, 12)], ids=str)
def test_layouts(shape, kinds):
    """Heads outside the tokens; a query cut out of a wider projection; 32-bit indices; rows that no vector load fits."""
    case = Case(shape, kinds, [33, 0, 257, 64], seed=8, layout="head")
    assert case.pages[0].stride(1) < case.pages[0].stride(2)
    expected = case.expected()
    wide = torch.randn(4, case.heads + 3, case.dim).to(case.kind).cuda()
    wide[:, 2:2 + case.heads] = case.query.cuda()
    case.check(case.run(query=wide[:, 2:2 + case.heads]), expected)
    case.check(case.run(query=case.query.cuda().transpose(0, 1).contiguous().transpose(0, 1)), expected)
    case.check(case.run(query=case.query.cuda().transpose(1, 2).contiguous().transpose(1, 2)), expected)   # strided features
    case.check(case.run(crow=case.crow.int().cuda(), col=case.col.int().cuda(), lengths=case.lengths.int().cuda()), expected)
    shifted = dict(key_pages=misaligned_copy(case.pages[0].contiguous()), value_pages=misaligned_copy(case.pages[1].contiguous()))
    case.check(case.run(**shifted), expected)
    case.check(case.run(query=misaligned_copy(case.query.cuda())), expected)
    only_values = dict(value_pages=shifted["value_pages"])
    case.check(case.run(**only_values), expected)
    if case.scales[0] is not None:
        tokens_first = [s.transpose(1, 2).contiguous().transpose(1, 2) for s in case.scales]
        case.check(case.run(key_scales=tokens_first[0], value_scales=tokens_first[1]), expected)


def test_the_answer_needs_no_lse_and_no_scale():
    case = Case((4, 2, 64, 16), (F32, F32), [50, 3], seed=9)
    assert torch.equal(case.run(lse=False), case.run()[0])
    case.scale = 1.0
    case.check(case.run(scale=None), case.expected())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (F16, E4M3)], ids=str)
def test_infinities_and_large_scores(kinds):
    """Scores of some hundreds (weights of single tokens), -inf keys beside finite ones, NaN keys."""
    case = Case((4, 2, 64, 16), kinds, [130, 90], seed=10, spread=40.0)
    case.check(case.run(), case.expected())
    if case.scales[0] is not None:
        return
    page, place = case.col[case.crow[0]], 3
    flat = case.query.clone()
    flat[0] = flat[0].abs() + 0.5                                 # every score of this key is -inf
    pages = case.pages[0].clone()
    pages[page, place] = float("-inf")
    out, lse = case.run(query=flat.cuda(), key_pages=pages)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    pages[page, place] = float("nan")
    out, lse = case.run(query=flat.cuda(), key_pages=pages)
    assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(lse[0]).all()) and bool(torch.isfinite(out[1]).all())
    only = Case((4, 2, 64, 16), kinds, [1], seed=11)
    pages = only.pages[0].clone()
    pages[only.col[0], 0] = float("nan")                          # nothing but a NaN is not an empty row
    assert bool(torch.isnan(only.run(key_pages=pages)[0]).all())


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (BF16, INT8)], ids=str)
def test_offsets_past_32_bits(kinds):
    """Pages so far apart that their offsets need more than 32 bits (in elements)."""
    case = Case((4, 2, 64, 16), kinds, [33, 31], seed=12, reserve=0)
    top = int(case.col.max())                                     # the last page that a row sees
    page, kv, dim = case.pages[0].shape[1:]
    step = (2 ** 32 // top + 64) // 64 * 64
    assert top * step >= 2 ** 32
    far = []
    for pages in case.pages:
        store = torch.empty(top * step + page * kv * dim, dtype=torch.uint8 if pages.element_size() == 1 else pages.dtype,
                            device="cuda").view(pages.dtype)
        view = store.as_strided((top + 1, page, kv, dim), (step, kv * dim, dim, 1))
        view.copy_(pages[:top + 1])
        far.append(view)
    scales = dict(key_scales=None, value_scales=None)
    if case.scales[0] is not None:
        scales = dict(key_scales=case.scales[0][:top + 1], value_scales=case.scales[1][:top + 1])
    case.check(case.run(key_pages=far[0], value_pages=far[1], **scales), case.expected())
    from autosage_b200 import paged

    slots = (case.col[:1] * page).cuda() + torch.arange(5).cuda()
    slots[4] = int(case.col[case.col.argmax()]) * page
    key, value = paged.paged_cache_read(slots, *far, dtype=F32, **scales)
    for got, exact in ((key, case.exact[0]), (value, case.exact[1])):
        wanted = exact.reshape(-1, kv, dim)[slots.cpu()]
        assert bool(((got.cpu().double() - wanted).abs() <= 2.0 ** -24 * wanted.abs()).all())
    paged.paged_cache_write(slots[4:], key[4:].to(case.kind), value[4:].to(case.kind), *far, **scales)
    again = paged.paged_cache_read(slots, *far, dtype=F32, **scales)
    assert torch.equal(again[0][:4], key[:4])
    if kinds[1] != INT8:
        assert torch.equal(again[0], key) and torch.equal(again[1], value)


@pytest.mark.parametrize("kinds", [(F32, F32), (BF16, BF16), (BF16, E4M3)], ids=str)
def test_capture_and_replay_with_new_lengths(kinds):
    """A captured call goes by what the table, lengths and query hold at each replay; two captured graphs and an eager
    call on other streams do not disturb one another."""
    case = Case((8, 2, 64, 16), kinds, [500, 40, 0, 129], seed=13)
    lengths, query = case.lengths.cuda(), case.query.cuda()
    crow, col = case.crow.cuda(), case.col.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        case.run(lengths=lengths, query=query, crow=crow, col=col)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(case.run(lengths=lengths, query=query, crow=crow, col=col))
        graphs.append(graph)
    new = torch.tensor([3, 40, 0, 65])
    lengths.copy_(new)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = case.run(lengths=lengths, query=query, crow=crow, col=col)
    torch.cuda.synchronize()
    for got in (*results, eager):
        case.check(got, case.expected(lengths=new))


def test_a_wanted_gradient_is_refused():
    case = Case((4, 2, 64, 16), (F32, F32), [20], seed=14)
    query = case.query.cuda().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        case.run(query=query)
    with torch.no_grad():
        case.check(case.run(query=query), case.expected())


def test_debug_checks_refuse_a_bad_table(monkeypatch):
    from autosage_b200 import paged

    monkeypatch.setenv("AUTOSAGE_CHECK_INDICES", "1")
    case = Case((4, 2, 64, 16), (F32, F32), [20, 40], seed=15)
    case.check(case.run(), case.expected())
    for change, message in ((dict(lengths=torch.tensor([20, 4000]).cuda()), "lengths must lie"),
                            (dict(crow=torch.tensor([0, 5, 3]).cuda()), "crow must run"),
                            (dict(col=case.col.cuda() + 100), "page ids")):
        with pytest.raises(RuntimeError, match=message):
            case.run(**change)
    tokens = torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="same slot"):
        paged.paged_cache_write(torch.tensor([4, 4], device="cuda"), tokens, tokens, case.pages[0].clone(), case.pages[1].clone())
    paged.paged_cache_write(torch.tensor([-1, -1], device="cuda"), tokens, tokens, case.pages[0].clone(), case.pages[1].clone())


# ------------------------------------------------------------------------------------------- the cache
def tokens_for(kind, count, heads, dim, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(2, count, heads, dim, generator=gen)
    x[:, 0] *= 1e-30 if kind != F16 else 1e-6
    if count > 4:
        x[:, 1] *= 1e4
        x[:, 2] = 0
        x[:, 3] = torch.arange(dim) - dim / 2 + 0.5               # many quotients on or next to a border between codes
        x[:, 4] = torch.round(x[:, 4] * 8) / 8
    return x.to(kind)


@pytest.mark.parametrize("kinds", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (70, 8, 128, 16), (33, 3, 100, 7), (9, 2, 113, 5), (40, 1, 256, 64), (17, 5, 24, 1),
                                   (64, 4, 64, 32), (5, 2, 192, 16)], ids=str)
def test_write_then_read(shape, kinds):
    """Codes and scales equal those of the float64 definition, whatever was there before; nothing else is touched."""
    from autosage_b200 import paged

    count, heads, dim, page = shape
    kind, cache = kinds
    x = tokens_for(kind, count, heads, dim, seed=count + dim)
    n = count // page + 3
    gen = torch.Generator().manual_seed(dim)
    slots = torch.randperm(n * page, generator=gen)[:count]
    if count > 8:
        slots[5], slots[6], slots[7], slots[8] = -1, n * page, 2 ** 45, -2 ** 60
    kept = (slots >= 0) & (slots < n * page)
    before = torch.randint(0, 100, (n, page, heads, dim), generator=gen, dtype=torch.int64)
    for layout in ("plain", "heads outside", "cut out", "shifted"):
        pools, scales = [], []
        for _ in range(2):
            pool = before.to(torch.uint8).view(E4M3).cuda() if cache == E4M3 else before.to(cache).cuda()
            if layout == "heads outside":
                pool = pool.transpose(1, 2).contiguous().transpose(1, 2)
            if layout == "shifted":
                pool = misaligned_copy(pool.view(torch.uint8)).view(E4M3) if cache == E4M3 else misaligned_copy(pool)
            pools.append(pool)
            scales.append(torch.full((n, heads, page), 7.0, device="cuda") if cache in LARGEST else None)
        given = x.cuda()
        if layout == "cut out":
            wide = torch.zeros(2, count, heads + 2, dim, dtype=kind, device="cuda")
            wide[:, :, 1:1 + heads] = given
            given = wide[:, :, 1:1 + heads]
        paged.paged_cache_write(slots.cuda(), given[0], given[1], pools[0], pools[1], key_scales=scales[0], value_scales=scales[1])
        wanted_dtype = F32 if cache in LARGEST else cache
        back = paged.paged_cache_read(slots.cuda(), pools[0], pools[1], key_scales=scales[0], value_scales=scales[1])
        for w in range(2):
            pool = pools[w].cpu()
            flat = (pool.float() if cache in LARGEST else pool).double().reshape(n * page, heads, dim)
            untouched = torch.ones(n * page, dtype=torch.bool)
            untouched[slots[kept]] = False
            was = (before.to(torch.uint8).view(E4M3).float() if cache == E4M3 else before).double().reshape(n * page, heads, dim)
            assert torch.equal(flat[untouched], was[untouched])
            assert back[w].dtype == wanted_dtype and back[w][(~kept).cuda()].abs().sum() == 0
            if cache not in LARGEST:
                assert torch.equal(flat[slots[kept]], x[w][kept].double())
                assert torch.equal(back[w].cpu()[kept], x[w][kept])
                continue
            value, scale = quantise(x[w].double(), cache)
            held = scales[w].cpu().double().transpose(1, 2).reshape(n * page, heads)
            assert torch.equal(held[slots[kept]], scale[kept]) and bool((held[untouched] == 7).all())
            assert torch.equal(flat[slots[kept]], value[kept])
            assert torch.equal(back[w].cpu()[kept], (value.float() * scale.float().unsqueeze(-1))[kept])


@pytest.mark.parametrize("cache", [E4M3, INT8], ids=str)
def test_rows_at_the_ends_of_the_range(cache):
    """The smallest and largest float32 magnitudes, scales that are subnormal or vanish, infinities and NaN."""
    from autosage_b200 import paged

    gen = torch.Generator().manual_seed(1)
    base = torch.randn(12, 1, 64, generator=gen)
    factors = [2.0 ** -149, 2.0 ** -140, 2.0 ** -130, 2.0 ** -120, 2.0 ** -100, 2.0 ** -91, 2.0 ** -80, 2.0 ** 80, 2.0 ** 98, 2.0 ** 125, 1, 1]
    x = (base.double() * torch.tensor(factors).double().view(-1, 1, 1)).float()
    x[10, 0, 9], x[11, 0, 60] = float("inf"), float("nan")
    pools = [torch.zeros(12, 1, 1, 64, device="cuda").to(cache) for _ in range(2)]
    scales = [torch.zeros(12, 1, 1, device="cuda") for _ in range(2)]
    slots = torch.arange(12).cuda()
    paged.paged_cache_write(slots, x.cuda(), x.cuda(), *pools, key_scales=scales[0], value_scales=scales[1])
    value, scale = quantise(x[:10].double(), cache)
    assert torch.equal(scales[0].cpu().view(-1)[:10].double(), scale.view(-1))
    assert torch.equal(pools[0].cpu().float().view(12, 64)[:10].double(), value.view(10, 64))
    back = paged.paged_cache_read(slots, *pools, key_scales=scales[0], value_scales=scales[1])
    assert bool(torch.isnan(back[0][10:]).all()) and bool(torch.isfinite(back[0][:10]).all())


@pytest.mark.parametrize("cache", [F32, BF16, F16, E4M3, INT8], ids=str)
@pytest.mark.parametrize("kind", [F32, BF16, F16], ids=str)
def test_read_in_another_type_and_the_same_slot_twice(kind, cache):
    from autosage_b200 import paged

    case = Case((2, 2, 64, 8), (kind if cache in LARGEST else cache, cache), [80], seed=16, reserve=0)
    slots = torch.tensor([3, 3, -1, 70, 3])
    slots[[0, 1, 3, 4]] = case.col[slots[[0, 1, 3, 4]] // 8] * 8 + slots[[0, 1, 3, 4]] % 8
    key, value = paged.paged_cache_read(slots.cuda(), *case.pages, key_scales=case.scales[0], value_scales=case.scales[1], dtype=kind)
    for got, exact in ((key, case.exact[0]), (value, case.exact[1])):
        wanted = exact.reshape(-1, 2, 64)[slots.clamp_min(0)]
        wanted[2] = 0
        assert got.dtype == kind
        # the product with the scale is rounded to float32 and then to the type
        bound = (HALF_STEP[kind] + 2.0 ** -24) * wanted.abs() + torch.finfo(kind).tiny
        assert bool(((got.double().cpu() - wanted).abs() <= bound).all())
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[4])
    none = paged.paged_cache_read(slots[:0].cuda(), *case.pages, key_scales=case.scales[0], value_scales=case.scales[1])
    assert none[0].shape == (0, 2, 64)


def test_write_and_read_are_captured_and_replayed():
    from autosage_b200 import paged

    x = torch.randn(2, 6, 2, 64).bfloat16().cuda()
    slots = torch.arange(6).cuda() * 3
    pools = [torch.zeros(4, 8, 2, 64, device="cuda").to(E4M3) for _ in range(2)]
    scales = dict(key_scales=torch.zeros(4, 2, 8, device="cuda"), value_scales=torch.zeros(4, 2, 8, device="cuda"))
    paged.paged_cache_write(slots, x[0], x[1], *pools, **scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.paged_cache_write(slots, x[0], x[1], *pools, **scales)
        key, value = paged.paged_cache_read(slots, *pools, **scales)
    x.copy_(torch.randn_like(x))
    slots.copy_(torch.arange(6) * 5 + 1)
    graph.replay()
    for got, given in ((key, x[0]), (value, x[1])):
        code, scale = quantise(given.double().cpu(), E4M3)
        assert torch.equal(got.cpu(), code.float() * scale.float().unsqueeze(-1))


# --------------------------------------------------------------------------- together, as they are used
def test_answering_token_by_token_equals_the_whole_pattern():
    """One float32 head: the rows that csr_attention_forward gives for the causal pattern, one at a time from a cache."""
    import autosage_b200
    from autosage_b200 import paged

    n, dim, page = 150, 64, 16
    gen = torch.Generator().manual_seed(17)
    q, k, v = (torch.randn(n, dim, generator=gen).cuda() for _ in range(3))
    counts = torch.arange(1, n + 1)
    crow = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0))).cuda()
    col = torch.cat([torch.arange(c) for c in counts.tolist()]).cuda()
    whole, _ = autosage_b200.csr_attention_forward(crow, col, q, k, v, scale=dim ** -0.5, fused=True)
    pages = torch.randperm(-(-n // page), generator=gen)
    pools = [torch.full((pages.numel(), page, 1, dim), float("nan"), device="cuda") for _ in range(2)]
    table, row = pages.cuda(), torch.tensor([0, pages.numel()]).cuda()
    slots = (pages[torch.arange(n) // page] * page + torch.arange(n) % page).cuda()
    prompt = 100
    paged.paged_cache_write(slots[:prompt], k[:prompt, None], v[:prompt, None], *pools)
    for t in range(prompt, n):
        paged.paged_cache_write(slots[t:t + 1], k[t:t + 1, None], v[t:t + 1, None], *pools)
        out = paged.csr_paged_attention(row, table, torch.tensor([t + 1]).cuda(), q[t:t + 1, None], *pools, scale=dim ** -0.5)
        # the paged row is within its bound of the float64 value, the whole-pattern row within the project's
        # (1e-5 of the value and 1e-5 sqrt(tokens))
        seen = torch.arange(t + 1)
        exact, _, slack, _, _ = attention(torch.tensor([0, 1]), torch.tensor([0]), torch.tensor([t + 1]), q[t:t + 1, None].cpu().double(),
                                          k[seen].cpu().double().view(1, -1, 1, dim), v[seen].cpu().double().view(1, -1, 1, dim), t + 1,
                                          dim ** -0.5, None)
        bound = slack + (HALF_STEP[F32] + 1e-5) * exact.abs() + 1e-5 * (t + 1) ** 0.5
        assert bool(((out - whole[t]).cpu().abs() <= bound).all())
    back = paged.paged_cache_read(slots, *pools)
    assert torch.equal(back[0][:, 0], k) and torch.equal(back[1][:, 0], v)


@pytest.mark.parametrize("cache", [BF16, E4M3, INT8], ids=str)
def test_a_batch_is_written_read_and_attended(cache):
    """A ragged batch: prompts, then steps, with a padded row; two halves of a row joined by their log-sum-exp."""
    from autosage_b200 import paged

    gen = torch.Generator().manual_seed(18)
    heads, kv, dim, page, pages_per_row = 8, 2, 128, 16, 6
    lengths = [0, 77, 5, 32]
    rows = len(lengths)
    col = torch.randperm(rows * pages_per_row, generator=gen)
    crow = torch.arange(rows + 1) * pages_per_row
    kind = cache if cache not in LARGEST else torch.uint8
    pools = [torch.full((rows * pages_per_row, page, kv, dim), 255 if kind == torch.uint8 else float("nan"), dtype=kind,
                        device="cuda").view(cache) for _ in range(2)]
    scales = {}
    if cache in LARGEST:
        scales = {name: torch.full((rows * pages_per_row, kv, page), float("nan"), device="cuda") for name in ("key_scales", "value_scales")}

    def slot(r, t):
        return col[crow[r] + t // page] * page + t % page

    history = [torch.zeros(2, 0, kv, dim).bfloat16() for _ in lengths]
    for step in range(4):
        new, slots = [], []
        for r, n in enumerate(lengths):
            count = 1 if step else n
            if r == 0:
                count = 1 if step else 0                         # the padded row: a token that goes nowhere
            x = torch.randn(2, count, kv, dim, generator=gen).bfloat16()
            at = torch.arange(history[r].size(1), history[r].size(1) + count)
            slots.append(slot(r, at) if r else torch.full((count,), -1))
            new.append(x)
            if r:
                history[r] = torch.cat((history[r], x), 1)
        x = torch.cat(new, 1).cuda()
        paged.paged_cache_write(torch.cat(slots).cuda(), x[0], x[1], *pools, **scales)
        now = torch.tensor([h.size(1) for h in history])
        query = torch.randn(rows, heads, dim, generator=gen).bfloat16()
        case = Case.__new__(Case)
        case.kind = BF16
        case.query = query
        case.crow, case.col, case.lengths, case.page, case.scale = crow, col, now, page, dim ** -0.5
        case.exact = []
        for w in range(2):
            full = torch.zeros(rows * pages_per_row, page, kv, dim, dtype=torch.float64)
            for r in range(rows):
                t = torch.arange(int(now[r]))
                h = history[r][w].double()
                if cache in LARGEST:
                    code, scale = quantise(h, cache)
                    h = code * scale.unsqueeze(-1)
                full.view(-1, kv, dim)[slot(r, t)] = h
            case.exact.append(full)
        call = dict(key_pages=pools[0], value_pages=pools[1], scale=case.scale, return_lse=True, **scales)
        whole = paged.csr_paged_attention(crow.cuda(), col.cuda(), now.cuda(), query.cuda(), **call)
        expected = case.expected()
        case.check(whole, expected)
        # row 1 in two parts: its first two pages, and the rest
        parts = [paged.csr_paged_attention(torch.tensor([0, 2]).cuda(), col[crow[1]:crow[1] + 2].cuda(), torch.tensor([2 * page]).cuda(),
                                           query[1:2].cuda(), **call),
                 paged.csr_paged_attention(torch.tensor([0, 4]).cuda(), col[crow[1] + 2:crow[2]].cuda(), (now[1:2] - 2 * page).cuda(),
                                           query[1:2].cuda(), **call)]
        lse = torch.logaddexp(parts[0][1], parts[1][1])
        joined = sum(out.float() * torch.exp(part - lse).unsqueeze(-1) for out, part in parts)
        # each part and the whole carry one bf16 rounding and the error of their softmax, the parts' bounded by the whole's
        # (they have fewer tokens); the weights of the parts are exp of differences of three such log-sum-exps
        slack, lse_slack = expected[2][1].max().item() + 2.0 ** -16 * expected[4][1].max().item(), expected[3][1].max().item()
        largest = max(p[0].float().abs().max().item() for p in parts)
        lse_limit = 3 * lse_slack + 3 * 2.0 ** -23 * lse.abs().max().item()
        assert (lse - whole[1][1:2]).abs().max().item() <= lse_limit
        assert (joined - whole[0][1:2].float()).abs().max().item() <= 3 * HALF_STEP[BF16] * largest + 3 * slack + 2 * lse_limit * largest
