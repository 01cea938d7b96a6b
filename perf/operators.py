"""The paged cache and its attention: what is measured.

Three operators: `paged_cache_write` (keys and values of new tokens into the pages of a cache, quantised to 8
bits on the way where the cache holds 8), `paged_cache_read` (tokens out of the pages again) and
`csr_paged_attention` (one new token of every sequence attends to the tokens of its pages; the page table is
a CSR pattern, row = sequence, column = page).  `own` chooses between the plain forms below and the calls that
a user makes of `autosage_b200.paged`.
"""
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}
LARGEST_CODE = {"e4m3": 448.0, "int8": 127.0}


# --------------------------------------------------------------------------------------------- cases
def listed():
    attend = dict(op="attend", window=0, lse=False)
    return [
        # the first answer of a chat with one user: latency is all that counts
        dict(attend, name="attend_one_short", type="bf16", cache="bf16", sequences=1, longest=37, heads=32, kv_heads=8,
             dim=128, page=16),
        # one user far into a long document: a single row has to fill the GPU
        dict(attend, name="attend_one_long", type="bf16", cache="bf16", sequences=1, longest=131072, heads=32,
             kv_heads=8, dim=128, page=16, lse=True),
        # an ordinary serving batch, ragged, the largest case
        dict(attend, name="attend_batch_f16", type="f16", cache="f16", sequences=64, longest=8192, heads=32, kv_heads=8,
             dim=128, page=16),
        # the framework's own type, a key and value head for each query head, with the log-sum-exp that joins parts
        dict(attend, name="attend_batch_f32", type="f32", cache="f32", sequences=24, longest=4096, heads=8, kv_heads=8,
             dim=64, page=32, lse=True),
        # a batch of long contexts on an 8-bit cache
        dict(attend, name="attend_batch_e4m3", type="bf16", cache="e4m3", sequences=48, longest=16384, heads=32,
             kv_heads=4, dim=128, page=64),
        # odd sizes: five query heads to a key head, 96 features, pages that no tile divides
        dict(attend, name="attend_odd_int8", type="f16", cache="int8", sequences=13, longest=5001, heads=20, kv_heads=4,
             dim=96, page=24, lse=True),
        # many sequences, one shared key head, wide features, only the last 1024 tokens seen
        dict(attend, name="attend_window_bf16", type="bf16", cache="bf16", sequences=192, longest=2500, heads=16,
             kv_heads=1, dim=256, page=64, window=1024),
        # one decoding step's tokens written and read back
        dict(name="store_step_e4m3", op="store", type="bf16", cache="e4m3", tokens=64, kv_heads=8, dim=128, page=16),
        # a prompt of many tokens
        dict(name="store_prompt_e4m3", op="store", type="bf16", cache="e4m3", tokens=32768, kv_heads=8, dim=128, page=16),
        # the framework's own type on an 8-bit cache, odd sizes
        dict(name="store_odd_int8", op="store", type="f32", cache="int8", tokens=5003, kv_heads=5, dim=100, page=24),
        # no quantising: a cache in the type of the model
        dict(name="store_prompt_f16", op="store", type="f16", cache="f16", tokens=8192, kv_heads=8, dim=64, page=32),
        # a long prefix taken out of an 8-bit cache, to be used by another program
        dict(name="read_prefix_int8", op="read", type="bf16", cache="int8", tokens=65536, kv_heads=8, dim=128, page=64),
    ]


def _log_uniform(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "store", "read"])
    kind = rng.choice(["f32", "bf16", "f16"])
    cache = rng.choice([kind, "e4m3", "int8"])
    dim = rng.choice([32, 40, 64, 64, 80, 96, 100, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([1, 7, 16, 16, 24, 32, 64, 128])
    if op != "attend":
        return dict(op=op, type=kind, cache=cache, tokens=_log_uniform(rng, 1, 30000), kv_heads=kv_heads, dim=dim, page=page)
    group = rng.choice([1, 2, 3, 4, 5, 8, 8, 12, 16])
    most = 9e8 / (2 * kv_heads * dim * BYTES[kind])       # tokens, half of them seen where lengths are ragged
    sequences = _log_uniform(rng, 1, 200)
    longest = _log_uniform(rng, 1, max(1, min(65536, int(most / sequences))))
    return dict(op=op, type=kind, cache=cache, sequences=sequences, longest=longest, heads=kv_heads * group,
                kv_heads=kv_heads, dim=dim, page=page, window=rng.choice([0, 0, 0, max(1, longest // 3)]),
                lse=rng.random() < 0.5)


def _lengths(case):
    """Tokens of each sequence: fixed by the case, so that its work is known; one row is the longest, others
    lie anywhere below, and a batch has a row that has just begun and one that is empty (a padded batch)."""
    rows, longest = case["sequences"], case["longest"]
    rng = random.Random(rows * 1000003 + longest)
    lengths = [longest] + [rng.randint(1, longest) for _ in range(rows - 1)]
    if rows >= 8:
        lengths[-1], lengths[-2] = 0, 1
    return lengths


# -------------------------------------------------------------------------------------------- inputs
def _quantised(x, cache):
    """(codes, scales) of x[..., dim]: one scale for each row of `dim` features, held in 32 bits.  The quotients
    are formed in 64: many lie next to the border between two codes, and 32 bits would move them onto it."""
    largest = x.float().abs().amax(-1)
    scales = largest / torch.full_like(largest, LARGEST_CODE[cache])   # a divisor on the host would be inverted first
    y = x.double() / scales.double().unsqueeze(-1)
    y = torch.where(scales.unsqueeze(-1) > 0, y, torch.zeros_like(y)).clamp(-LARGEST_CODE[cache], LARGEST_CODE[cache])
    if cache == "int8":
        return y.round().to(torch.int8), scales
    exponent = ((y.abs().view(torch.int64) >> 52) - 1023).clamp_min(-6).double()       # 3 bits behind the leading one,
    step = torch.exp2(exponent - 3)                                                     # none below 2^-9
    return (torch.round(y / step) * step).float().to(torch.float8_e4m3fn), scales


def _roughly_quantised(x, cache):
    """The same for pages that are only read: a code on the wrong side of a border is an input like another."""
    scales = x.float().abs().amax(-1) / LARGEST_CODE[cache]
    y = (x.float() / scales.unsqueeze(-1)).clamp(-LARGEST_CODE[cache], LARGEST_CODE[cache])
    return (y.round() if cache == "int8" else y).to(DTYPES[cache]), scales


def _filled_pages(pages, case, generator):
    """Key or value pages [pages, page, kv_heads, dim] with every slot in use, and scales [pages, kv_heads, page]."""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    quantised = case["cache"] in LARGEST_CODE
    kind = torch.bfloat16 if quantised else DTYPES[case["cache"]]
    x = torch.randn(shape, device="cuda", dtype=kind, generator=generator)
    x *= torch.rand(case["kv_heads"], case["dim"], device="cuda", generator=generator).to(kind) + 0.5   # features differ in size
    if not quantised:
        return x, None
    codes = torch.empty(shape, device="cuda", dtype=DTYPES[case["cache"]])
    scales = torch.empty(pages, case["kv_heads"], case["page"], device="cuda")
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, pages, step):
        part, scale = _roughly_quantised(x[at:at + step], case["cache"])
        codes[at:at + step] = part
        scales[at:at + step] = scale.transpose(1, 2)
    return codes, scales


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    state = dict(case=dict(case))
    if case["op"] == "attend":
        lengths = _lengths(case)
        rng.shuffle(lengths)
        counts = [-(-n // page) + rng.randint(0, 1) for n in lengths]     # some rows have a page in reserve
        crow = [0]
        for n in counts:
            crow.append(crow[-1] + n)
        pages = crow[-1] + 3
        state["crow"] = torch.tensor(crow, device="cuda")
        state["lengths"] = torch.tensor(lengths, device="cuda")
        state["col"] = torch.randperm(pages, device="cuda", generator=generator)[:crow[-1]].contiguous()
        state["key_pages"], state["key_scales"] = _filled_pages(pages, case, generator)
        state["value_pages"], state["value_scales"] = _filled_pages(pages, case, generator)
        # the query as a slice of the projection that made query, key and value in one product
        projected = torch.randn(case["sequences"], case["heads"] + 2 * kv_heads, dim, device="cuda",
                                generator=generator).to(DTYPES[case["type"]])
        state["query"] = projected[:, :case["heads"]]
        state["scale"] = 1.5 * dim ** -0.5
        return state
    tokens = case["tokens"]
    pages = -(-tokens // page) + 5
    order = torch.randperm(pages, device="cuda", generator=generator)
    position = torch.arange(tokens, device="cuda")
    slots = order[position // page] * page + position % page
    slots[torch.rand(tokens, device="cuda", generator=generator) < 0.02] = -1      # padding among the tokens
    state["slots"] = slots
    if case["op"] == "read":
        state["key_pages"], state["key_scales"] = _filled_pages(pages, case, generator)
        state["value_pages"], state["value_scales"] = _filled_pages(pages, case, generator)
        return state
    projected = torch.randn(tokens, 4 * kv_heads, dim, device="cuda", generator=generator).to(DTYPES[case["type"]])
    state["key"], state["value"] = projected[:, 2 * kv_heads:3 * kv_heads], projected[:, 3 * kv_heads:]
    for name in ("key", "value"):
        state[name + "_pages"] = torch.zeros(pages, page, kv_heads, dim, device="cuda").to(DTYPES[case["cache"]])
        state[name + "_scales"] = torch.zeros(pages, kv_heads, page, device="cuda") if case["cache"] in LARGEST_CODE else None
    return state


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "attend":
        return _plain_attention(state, case)
    if case["op"] == "store":
        for name in ("key", "value"):
            _plain_write(state["slots"], state[name], state[name + "_pages"], state[name + "_scales"], case)
    out = {name: _plain_read(state["slots"], state[name + "_pages"], state[name + "_scales"], DTYPES[case["type"]])
           for name in ("key", "value")}
    if case["op"] == "store" and case["cache"] in LARGEST_CODE:
        out["key_scales"], out["value_scales"] = state["key_scales"], state["value_scales"]
    return out


def _run_own(state, case):
    from autosage_b200 import paged

    scales = dict(key_scales=state["key_scales"], value_scales=state["value_scales"])
    if case["op"] == "attend":
        out = paged.csr_paged_attention(state["crow"], state["col"], state["lengths"], state["query"], state["key_pages"],
                                        state["value_pages"], scale=state["scale"], window=case["window"] or None,
                                        return_lse=case["lse"], **scales)
        return dict(zip(("out", "lse"), out)) if case["lse"] else {"out": out}
    if case["op"] == "store":
        paged.paged_cache_write(state["slots"], state["key"], state["value"], state["key_pages"], state["value_pages"], **scales)
    key, value = paged.paged_cache_read(state["slots"], state["key_pages"], state["value_pages"], dtype=DTYPES[case["type"]],
                                        **scales)
    out = {"key": key, "value": value}
    if case["op"] == "store" and case["cache"] in LARGEST_CODE:
        out["key_scales"], out["value_scales"] = state["key_scales"], state["value_scales"]
    return out


def _plain_write(slots, x, pages, scales, case):
    page = pages.size(1)
    kept = slots >= 0
    at, x = slots[kept], x[kept]
    if scales is None:
        pages[at // page, at % page] = x
        return
    codes, scale = _quantised(x, case["cache"])
    pages.view(torch.uint8)[at // page, at % page] = codes.view(torch.uint8)
    scales[at // page, :, at % page] = scale


def _plain_read(slots, pages, scales, kind):
    page = pages.size(1)
    at = slots.clamp_min(0)
    x = pages.view(torch.uint8)[at // page, at % page].view(pages.dtype) if pages.element_size() == 1 else pages[at // page, at % page]
    x = x.float()
    if scales is not None:
        x = x * scales[at // page, :, at % page].unsqueeze(-1)
    return torch.where((slots >= 0).view(-1, 1, 1), x, torch.zeros_like(x)).to(kind)


def _plain_attention(state, case):
    crow, col, lengths, query = state["crow"], state["col"], state["lengths"], state["query"]
    page, kv_heads, dim = case["page"], case["kv_heads"], case["dim"]
    rows, heads = query.size(0), query.size(1)
    first = max(0, case["longest"] - case["window"]) if case["window"] else 0     # columns no row can see are left out ...
    seen = case["longest"] - first
    begin = (lengths - case["window"]).clamp_min(0) if case["window"] else torch.zeros_like(lengths)
    position = begin.view(-1, 1) + torch.arange(seen, device=query.device)        # ... by counting from each row's first token
    valid = position < lengths.view(-1, 1)
    place = (crow[:-1].view(-1, 1) + position // page).clamp_max(max(col.numel() - 1, 0))
    slots = torch.where(valid, col[place] * page + position % page, torch.full_like(position, -1)).view(-1)
    key = _plain_read(slots, state["key_pages"], state["key_scales"], torch.float32).view(rows, seen, kv_heads, dim)
    scores = torch.matmul(query.float().reshape(rows, kv_heads, heads // kv_heads, dim), key.permute(0, 2, 3, 1)) * state["scale"]
    del key
    scores = scores.masked_fill(~valid.view(rows, 1, 1, seen), float("-inf"))
    peak = scores.amax(-1, keepdim=True)
    peak = torch.where(peak == float("-inf"), torch.zeros_like(peak), peak)       # a row that sees nothing
    weights = torch.exp(scores - peak)
    total = weights.sum(-1, keepdim=True)
    value = _plain_read(slots, state["value_pages"], state["value_scales"], torch.float32).view(rows, seen, kv_heads, dim)
    out = torch.matmul(weights, value.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
    out = {"out": out.reshape(rows, heads, dim).to(query.dtype)}
    if case["lse"]:
        out["lse"] = (torch.log(total) + peak).reshape(rows, heads)
    return out


# ------------------------------------------------------------------------------------- work and truth
def work(case):
    row = case["dim"] * BYTES[case["cache"]] + (4 if case["cache"] in LARGEST_CODE else 0)
    if case["op"] == "attend":
        seen = sum(min(n, case["window"] or n) for n in _lengths(case))
        outer = case["sequences"] * case["heads"] * (2 * case["dim"] * BYTES[case["type"]] + (4 if case["lse"] else 0))
        return {"bytes": 2 * seen * case["kv_heads"] * row + outer + 8 * (seen // case["page"]) + 16 * case["sequences"],
                "flops": 4 * seen * case["heads"] * case["dim"]}
    rows = 2 * case["tokens"] * case["kv_heads"]
    through = rows * (case["dim"] * BYTES[case["type"]] + row)
    return {"bytes": (2 * through if case["op"] == "store" else through) + 8 * case["tokens"],
            "flops": rows * case["dim"] * (4 if case["op"] == "store" else 1)}


def _nearest_code(y, cache):
    """y rounded to the values that a code stands for, ties to even, in 64 bits."""
    if cache == "int8":
        return torch.round(y).clamp(-127, 127)
    y = y.clamp(-448, 448)
    _, power = torch.frexp(y)                                   # |y| = m 2^power, m in [1/2, 1)
    step = torch.ldexp(torch.ones_like(y), (power - 1).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _tokens64(state, name, page_ids, offsets):
    pages, scales = state[name + "_pages"], state[name + "_scales"]
    flat = pages.view(-1, *pages.shape[2:])
    index = page_ids * pages.size(1) + offsets
    x = (flat.view(torch.uint8)[index].view(pages.dtype) if pages.element_size() == 1 else flat[index])
    x = (x.float() if pages.element_size() == 1 else x).double()
    return x if scales is None else x * scales.transpose(1, 2).reshape(-1, pages.size(2))[index].double().unsqueeze(-1)


def exact(case, seed):
    state = prepare(case, seed)
    page = case["page"]
    if case["op"] == "attend":
        query = state["query"].double()
        out = torch.zeros_like(query)
        lse = torch.full(query.shape[:2], float("-inf"), dtype=torch.float64, device=query.device)
        crow, lengths, group = state["crow"].tolist(), state["lengths"].tolist(), case["heads"] // case["kv_heads"]
        for b, n in enumerate(lengths):
            t = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device=query.device)
            if t.numel() == 0:
                continue
            ids = state["col"][crow[b] + t // page]
            q = query[b].view(case["kv_heads"], group, -1)
            scores = torch.einsum("hgd,thd->hgt", q, _tokens64(state, "key", ids, t % page)) * state["scale"]
            lse[b] = torch.logsumexp(scores, -1).reshape(-1)
            out[b] = torch.einsum("hgt,thd->hgd", torch.softmax(scores, -1), _tokens64(state, "value", ids, t % page)).reshape(out[b].shape)
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    slots, quantised, answer = state["slots"], case["cache"] in LARGEST_CODE, {}
    kept = slots >= 0
    for name in ("key", "value"):
        if case["op"] == "read":
            x = _tokens64(state, name, slots.clamp_min(0) // page, slots.clamp_min(0) % page)
        else:
            x = state[name].double()
            if quantised:
                scale = (x.abs().amax(-1) / LARGEST_CODE[case["cache"]]).float()       # held in 32 bits
                held = state[name + "_scales"].double()
                held[slots[kept] // page, :, slots[kept] % page] = scale[kept].double()
                wide = scale.double().unsqueeze(-1)
                x = _nearest_code(x / wide, case["cache"]) * wide
        answer[name] = x * kept.view(-1, 1, 1)
        if case["op"] == "store" and quantised:
            answer[name + "_scales"] = held
    return answer
