"""Float64 restatement of the paged cache and its attention, on the CPU, one row at a time, and the error that
the kernels may make."""
from __future__ import annotations

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # of a rounding, relative


def e4m3_values() -> torch.Tensor:
    """The 127 magnitudes of the 8-bit float, ascending."""
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest_code_value(y: torch.Tensor, kind: torch.dtype) -> torch.Tensor:
    """y (float64) rounded to the nearest value of the type, ties to the even code, by comparing with all of them."""
    if kind == torch.int8:
        return torch.round(y).clamp(-127, 127)
    values = e4m3_values()
    middle = (values[1:] + values[:-1]) / 2
    size = y.abs()
    below = torch.searchsorted(middle, size)                       # first border >= size: that code, unless a tie goes up
    tie = (below < middle.numel()) & (middle[below.clamp_max(middle.numel() - 1)] == size)
    code = below + (tie & (below % 2 == 1)).long()
    return torch.copysign(values[code], y)


def quantise(x: torch.Tensor, kind: torch.dtype):
    """(values of the codes, scales) of x[..., dim], float64 in, scales as held in float32."""
    scale = (x.abs().amax(-1).float() / torch.tensor(LARGEST[kind])).double()
    y = torch.where(scale.unsqueeze(-1) > 0, x / scale.unsqueeze(-1), torch.zeros_like(x))
    return nearest_code_value(y, kind), scale


def attention(crow, col, lengths, query, key, value, page_size, scale, window):
    """key / value: [n_pages, page, heads, dim] float64.  Returns out, lse, the bound on the error of out before it is
    rounded, the bound on that of lse, and sum_t p_t |v_t|."""
    rows, n_heads, dim = query.shape
    kv_heads, n_pages = key.size(2), key.size(0)
    group = n_heads // kv_heads
    out = torch.zeros(rows, n_heads, dim, dtype=torch.float64)
    lse = torch.full((rows, n_heads), float("-inf"), dtype=torch.float64)
    slack = torch.zeros_like(out)
    lse_slack = torch.zeros_like(lse)
    spread = torch.zeros_like(out)
    eps = 2.0 ** -24
    for r in range(rows):
        n = min(int(lengths[r]), (int(crow[r + 1]) - int(crow[r])) * page_size)
        t = torch.arange(max(0, n - window) if window else 0, n)
        ids = col[crow[r] + t // page_size] if n else t
        seen = (ids >= 0) & (ids < n_pages)
        ids, place = ids[seen], (t % page_size)[seen]
        if ids.numel() == 0:
            continue
        k, v = key[ids, place], value[ids, place]                  # [tokens, kv heads, dim]
        q = query[r].view(kv_heads, group, dim)
        s = torch.einsum("hgd,thd->hgt", q, k) * scale
        p = torch.softmax(s, -1)
        out[r] = torch.einsum("hgt,thd->hgd", p, v).reshape(n_heads, dim)
        lse[r] = torch.logsumexp(s, -1).reshape(n_heads)
        # score: dim products added in float32, the tensor core truncating each sum (two half steps), and the
        # factors scale * log2(e), the key scale and the running maximum: eight more roundings of |s| or less
        size = torch.einsum("hgd,thd->hgt", q.abs(), k.abs()).amax(-1) * abs(scale)
        # (8-bit pages: the query is held to 2^-24 of its largest feature, rounded to half of that)
        score = (2 * dim + 8) * eps * size + eps / 2 * (q.abs().amax(-1, keepdim=True) * k.abs().sum(-1).t().unsqueeze(1)).amax(-1) * abs(scale)
        # weight: twice the score error (it and the sum), the exponential, the running factors of the sums
        count = ids.numel()
        relative = 2 * score + (2 * count + 32) * eps
        part = torch.einsum("hgt,thd->hgd", p, v.abs())
        spread[r] = part.reshape(n_heads, dim)
        slack[r] = (2 * relative.unsqueeze(-1) * part).reshape(n_heads, dim)
        lse_slack[r] = (score + (count + 16) * eps).reshape(n_heads)
    return out, lse, slack, lse_slack, spread
