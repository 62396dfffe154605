"""The paged operators in 64 bits on the CPU, from their formulas, one sequence and head at a time."""
import math

import torch

E4M3 = torch.tensor([(-1.0 if b & 128 else 1.0) * (math.nan if (b & 127) == 127 else
                     (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10) if b >> 3 & 15 else (b & 7) * 2.0 ** -9) for b in range(256)], dtype=torch.float64)


def values(bytes_):
    return E4M3[bytes_.long()]


def rounded(x):
    """Nearest e4m3 value, ties to even, saturating; NaN stays."""
    x = x.clamp(-448, 448)
    _, e = torch.frexp(x.abs())
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def pow2_scale(amax: float) -> float:
    if amax == 0:
        return 2.0 ** -126
    m, e = math.frexp(amax / 448)
    return max(2.0 ** (e - 1 if m == 0.5 else e), 2.0 ** -126)


def norm_rope(x, w, cos, sin, positions, pair_axis, eps=1e-6):
    """x [tokens, heads, d]; positions [axes, tokens]; float64."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + w.double())
    if cos is None:
        return x
    half = cos.shape[1]
    axis = torch.zeros(half, dtype=torch.long) if pair_axis is None else pair_axis.long()
    where = positions.long()[axis].T
    c, s = (t.double()[where, torch.arange(half)][:, None] for t in (cos, sin))
    y = x.clone()
    y[..., :half] = x[..., :half] * c - x[..., half:2 * half] * s
    y[..., half:2 * half] = x[..., half:2 * half] * c + x[..., :half] * s
    return y


def append_rows(x, pool, scale, ids, page, pos):
    """Append float64 rows x [n, h, d] of one sequence at slot `pos` to pool values [n_pages, h, page, d] (float64, in units of
    the scale) and scale [n_pages, h], in place."""
    n, heads, _ = x.shape
    at = 0
    while at < n:
        index, fill = divmod(pos + at, page)
        m = min(page - fill, n - at)
        pid = int(ids[index])
        for h in range(heads):
            a = x[at:at + m, h]
            finite = torch.where(torch.isfinite(a), a.abs(), torch.zeros_like(a))
            s, old = pow2_scale(float(finite.max())), float(scale[pid, h])
            if fill and s > old:
                pool[pid, h, :fill] = rounded(pool[pid, h, :fill] * (old / s))
            elif fill:
                s = old
            scale[pid, h] = s
            pool[pid, h, fill:fill + m] = rounded(a / s)
        at += m


def attention(q, k_pool, v_pool, k_scale, v_scale, ids, length, *, softmax_scale=None, causal=False):
    """q [n, h_q, d] of one sequence against its first `length` tokens; pools of bytes [n_pages, h, page, d].  Returns the
    float64 result and the largest |v| that each (row, head) sees."""
    n, h_q, d = q.shape
    heads, page = k_pool.shape[1], k_pool.shape[2]
    out, big = torch.zeros(n, h_q, d, dtype=torch.float64), torch.zeros(n, h_q, dtype=torch.float64)
    if length == 0:
        return out, big
    ids = ids[:-(-length // page)].long()
    for h in range(heads):
        k, v = ((values(pool[ids, h]) * s[ids, h].double()[:, None, None]).reshape(-1, d)[:length]
                for pool, s in ((k_pool, k_scale), (v_pool, v_scale)))
        for j in range(h * h_q // heads, (h + 1) * h_q // heads):
            a = q[:, j].double() @ k.T * (d ** -0.5 if softmax_scale is None else softmax_scale)
            seen = torch.ones(n, length, dtype=torch.bool)
            if causal:
                seen = torch.arange(length)[None, :] <= (length - n + torch.arange(n))[:, None]
            a = a.masked_fill(~seen, -math.inf)
            out[:, j] = torch.softmax(a, -1).nan_to_num(0.0) @ v
            big[:, j] = (v.abs().amax(-1)[None, :] * seen).amax(-1)
    return out, big


# An attention result is rounded once to bf16 (half a step: 2^-8 of the value), its probabilities to f16 (half a step: 2^-11
# each, so at most 2^-11 of the largest |v|), the query's split and the fp32 sums stay below another 2^-11 of it.
def assert_attention(got, ref, big, what=""):
    got, off = got.double(), (got.double() - ref).abs()
    limit = ref.abs() * 2.0 ** -8 + big[..., None] * 2.0 ** -10
    assert torch.isfinite(got).all(), what
    assert (off <= limit).all(), (what, float((off - limit).max()), float(off.max()))


def random_cache(gen, n_layers, n_pages, h_kv, page, d, pow2=True):
    """Random finite bytes and scales."""
    b = torch.randint(0, 256, (2, n_layers, n_pages, h_kv, page, d), generator=gen, dtype=torch.uint8)
    b = torch.where((b & 127) >= 0x70, b & 0x8F | 0x30, b)          # keep |value| below 128: scores of ordinary size
    s = torch.rand(2, n_layers, n_pages, h_kv, generator=gen) * 0.02 + 0.002
    if pow2:
        s = torch.exp2(torch.floor(torch.log2(s)))
    return b[0].contiguous(), b[1].contiguous(), s[0].contiguous(), s[1].contiguous()


def random_table(gen, lens, page, width, n_pages):
    """Distinct pages for every sequence, -1 beyond its last one."""
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    perm, at = torch.randperm(n_pages, generator=gen).to(torch.int32), 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = perm[at:at + m]
        at += m
    assert at <= n_pages
    return table
