"""What the operators of the paged FP8 cache are measured on: their cases, inputs, plain forms and exact values.

Three operators (``op`` of a case):

``append``   paged_rope_append: optional RMS norm of the query and key heads, rotary embedding (positions on one or three
             axes), quantise-and-append of the key and the value into pages with one power-of-two scale per (page, head).
``decode``   paged_decode_attention: one query token per sequence against the cache.
``prefill``  paged_prefill_attention: many query tokens per sequence against the cache, causal from its end, or not causal.

A page pool is [n_layers, n_pages, h_kv, page, head_dim] e4m3 bytes with fp32 scales [n_layers, n_pages, h_kv]; the page
table [batch, max_pages] places a sequence's pages anywhere in the pool.
"""
import importlib
import math

import torch

own = False

E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def _case(op, name=None, layers=1, batch=1, h_q=40, h_kv=8, d=128, page=64, lens="1", qlens="1", **more):
    c = {"op": op, "layers": layers, "batch": batch, "h_q": h_q, "h_kv": h_kv, "d": d, "page": page, "lens": lens, "qlens": qlens}
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    # lens: tokens in the cache (append: before the call; decode and prefill: those attended, the new ones included);
    # qlens: new tokens of each sequence.  "a:b" = drawn between a and b for every sequence, one number = the same for all.
    return [
        # one layer of one user's chat: a single token, all latency
        _case("append", "append 1 token", lens="511", qlens="1", rot=128, axes=1, norm=False),
        # a decode step of all 64 layers of a batch at ragged depths
        _case("append", "append 64 layers x 16 tokens", layers=64, batch=16, lens="1024:16384", qlens="1", rot=128, axes=1, norm=False),
        # prompts with pictures among the text: three position axes, a quarter of the head rotated, head norms, odd lengths
        _case("append", "append ragged prompts, 3 axes", batch=6, h_q=24, h_kv=4, d=256, lens="0:700", qlens="1:2500", rot=64, axes=3, norm=True),
        # one long prompt in one piece
        _case("append", "append 32768-token prompt", lens="0", qlens="32768", rot=128, axes=1, norm=False, page=128),
        # one layer of one user's chat: all latency
        _case("decode", "decode 1 x 512", lens="512"),
        # many short chats in small pages
        _case("decode", "decode 128 short, page 16", batch=128, lens="0:600", page=16),
        # a busy server: one layer, ragged lengths
        _case("decode", "decode 32 ragged to 16384", batch=32, lens="1:16384"),
        # a whole step's attention of one 8192-token chat: 64 layers in one call
        _case("decode", "decode 64 layers x 8192", layers=64, lens="8192"),
        # long documents, heads of 256
        _case("decode", "decode 8 x 65536, heads 256", batch=8, h_q=24, h_kv=4, d=256, lens="60001:65536", page=128),
        # a few guessed tokens of each chat to be verified
        _case("prefill", "prefill 8 x 4 on 4096", batch=8, lens="3000:4500", qlens="2:6", causal=True),
        # encoder states of another length, seen by every query token
        _case("prefill", "cross 4 x 300 on 1500", batch=4, h_q=24, h_kv=4, d=256, lens="1500", qlens="200:400", causal=False),
        # a long prompt in one piece
        _case("prefill", "prefill 8192 causal", lens="8192", qlens="8192", causal=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    h_q, h_kv, d = rng.choice([(40, 8, 128), (24, 4, 256), (8, 1, 128), (5, 1, 128), (16, 16, 128), (10, 2, 256), (10, 2, 128), (7, 1, 256)])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        batch = _log(rng, 1, 64)
        one = rng.random() < 0.5
        q = 1 if one else _log(rng, 2, 32768 // batch)
        layers = _log(rng, 1, 64) if one else 1
        return _case(op, None, layers, batch, h_q, h_kv, d, page, "0:%d" % _log(rng, 1, 8192), "1" if one else "1:%d" % q,
                     rot=rng.choice([0, d // 4, d // 2, d]), axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.5)
    if op == "decode":
        layers = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        batch = _log(rng, 1, 128)
        # the whole call stays below the largest listed case's cache bytes
        top = max(2, min(65536, (1 << 30) // (layers * batch * h_kv * d * 2)))
        hi = _log(rng, 2, top)
        return _case(op, None, layers, batch, h_q, h_kv, d, page, "%d:%d" % (rng.choice([0, 1, max(1, hi // 2), hi]), hi))
    batch = _log(rng, 1, 16)
    q = _log(rng, 2, max(2, 4096 // batch))
    # visible pairs x heads below those of the largest listed case
    kv = max(q, _log(rng, q, max(q + 1, min(32768, (1 << 30) // (h_q * d // 128 * batch * q)))))
    return _case(op, None, 1, batch, h_q, h_kv, d, page, "%d:%d" % (max(1, kv // 2), kv), "%d:%d" % (max(1, q // 2), q), causal=rng.random() < 0.75)


def _between(text, n, salt):
    """The lengths of a case: the same for every seed (sizes belong to the case, values to the seed)."""
    a, _, b = text.partition(":")
    if not b:
        return [int(a)] * n
    a, b = int(a), int(b)
    return [a + ((i * 2654435761 + salt * 40503 + 12345) % 1000003) % (b - a + 1) for i in range(n)]


def _lengths(case):
    lens, q = _between(case["lens"], case["batch"], 1), _between(case["qlens"], case["batch"], 2)
    return lens, q


# ------------------------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _pow2_scale(amax):
    """Smallest power of two s with amax / s <= 448 (never below 2^-126)."""
    m, e = torch.frexp(amax)                                 # amax = m * 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9)                 # 448 = 0.875 * 2^9
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e.clamp(min=-126)), torch.full_like(amax, 2.0 ** -126))


def _pages_of(lens, page):
    return [(n + page - 1) // page for n in lens]


def prepare(case, seed):
    lens, qlens = _lengths(case)
    op, page, d, h_q, h_kv, layers, batch = (case[k] for k in ("op", "page", "d", "h_q", "h_kv", "layers", "batch"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = [n + q for n, q in zip(lens, qlens)] if op == "append" else lens
    need = _pages_of(full, page)
    width, total = max(max(need), 1), sum(need) + 3          # a few pages of the pool belong to nobody
    perm = torch.randperm(total, generator=g, device="cuda", dtype=torch.int64).to(torch.int32).cpu()
    table = torch.full((batch, width), -1, dtype=torch.int32)
    held = torch.zeros(total, dtype=torch.int64)             # tokens that each page of the pool holds
    at = 0
    for b in range(batch):
        mine = perm[at:at + need[b]]
        table[b, :need[b]] = mine
        held[mine.long()] = (lens[b] - page * torch.arange(need[b])).clamp(0, page)
        at += need[b]
    table = table.cuda()

    # the cache as earlier appends left it; slots that hold no token hold what their last owner left, NaN patterns too
    k_pages = torch.empty(layers, total, h_kv, page, d, dtype=torch.uint8, device="cuda")
    v_pages = torch.empty_like(k_pages)
    k_scale = torch.empty(layers, total, h_kv, device="cuda")
    v_scale = torch.empty_like(k_scale)
    empty = torch.arange(page, device="cuda")[None, :] >= held.cuda()[:, None]                   # [total, page]
    for layer in range(layers):
        for pool, scale in ((k_pages, k_scale), (v_pages, v_scale)):
            x = _randn(g, total, h_kv, page, d)
            x *= torch.exp(0.3 * _randn(g, total, h_kv, 1, 1))                                   # pages of different loudness
            s = _pow2_scale(x.abs().amax(dim=(2, 3)))
            by = (x / s[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            pool[layer] = torch.where(empty[:, None, :, None], torch.full_like(by, 0x7F), by)
            scale[layer] = s

    n = sum(qlens)
    starts = torch.tensor([sum(qlens[:i]) for i in range(batch + 1)], dtype=torch.int32, device="cuda")
    state = {"case": {k: v for k, v in case.items() if k != "name"}, "n": n, "q_start": starts, "table": table, "k_pages": k_pages,
             "v_pages": v_pages, "k_scale": k_scale, "v_scale": v_scale, "max_q": max(qlens), "max_len": max(full),
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "q": _randn(g, layers, n, h_q, d).to(torch.bfloat16)}
    if op == "append":
        rot = case["rot"]
        state["k"] = _randn(g, layers, n, h_kv, d).to(torch.bfloat16)
        state["v"] = (_randn(g, layers, n, h_kv, d) * torch.exp(0.5 * _randn(g, 1, n, 1, 1))).to(torch.bfloat16)
        rows = max(full) + 1
        freq = 10000.0 ** (-torch.arange(0, rot // 2, device="cuda", dtype=torch.float64) * 2 / max(rot, 1))
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), torch.tensor(qlens, device="cuda"))
        slot = torch.arange(n, device="cuda") - starts[seq].long() + state["lens"][seq].long()
        if case["axes"] == 1:
            state["positions"], state["pair_axis"] = None, None
        else:                                                # pictures: height and width lag behind the running position
            state["positions"] = torch.stack([slot, slot - slot % 7, slot - slot % 5]).to(torch.int32).contiguous()
            state["pair_axis"] = (torch.arange(max(rot // 2, 1), device="cuda") % 3).to(torch.int32)
        if case["norm"]:
            state["qw"] = (0.1 * _randn(g, layers, d)).to(torch.bfloat16)
            state["kw"] = (0.1 * _randn(g, layers, d)).to(torch.bfloat16)
        else:
            state["qw"] = state["kw"] = None
        state["q_out"] = torch.empty_like(state["q"])
        state["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        state["out"] = torch.empty_like(state["q"])
        if own:                                              # the handle that a program keeps: scratch for split sequences
            pkg = importlib.import_module("qwen38-5080_b200")
            shape = pkg.make_paged_shape(h_q, k_pages, v_pages, k_scale, table)
            state["workspace"] = pkg.PagedWorkspace(shape, k_pages.device, max_seq_len=max(full), q_tokens=n if op == "prefill" else None)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_append(state) if op == "append" else _plain_decode(state) if op == "decode" else _plain_prefill(state)


def _own(state):
    pkg = importlib.import_module("qwen38-5080_b200")
    c, s = state["case"], state
    cache = (s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"])
    if c["op"] == "append":
        q = pkg.paged_rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], *cache, s["lens"],
                                  q_start=None if c["qlens"] == "1" else s["q_start"], positions=s["positions"], pair_axis=s["pair_axis"],
                                  q_norm_weight=s["qw"], k_norm_weight=s["kw"], advance=False, status=s["status"], q_out=s["q_out"])
        return {"q": q, "k": s["k_pages"].view(torch.float8_e4m3fn), "v": s["v_pages"].view(torch.float8_e4m3fn),
                "ks": s["k_scale"], "vs": s["v_scale"]}
    if c["op"] == "decode":
        return pkg.paged_decode_attention(s["q"], *cache, s["lens"], workspace=s["workspace"], out=s["out"])
    return pkg.paged_prefill_attention(s["q"], s["q_start"], *cache, s["lens"], workspace=s["workspace"], causal=c["causal"], out=s["out"])


# ---- plain forms: elementary torch operations in 32 bits, rounded once
def _norm_rope(x, w, cos, sin, rot, eps=1e-6):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * (1.0 + w.float()[:, None, None, :])
    if not rot:
        return x
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    cos, sin = cos[None, :, None, :], sin[None, :, None, :]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def _plain_append(s):
    c = s["case"]
    page, rot, n = c["page"], c["rot"], s["n"]
    tok = torch.arange(n, device="cuda")
    seq = torch.bucketize(tok, s["q_start"][1:].long(), right=True)
    slot = tok - s["q_start"].long()[seq] + s["lens"].long()[seq]
    pid = s["table"].long()[seq, slot // page]
    row = slot % page
    cos = sin = None
    if rot:
        pos = slot[None, :] if s["positions"] is None else s["positions"].long()
        axis = torch.zeros(rot // 2, dtype=torch.long, device="cuda") if s["pair_axis"] is None else s["pair_axis"].long()[:rot // 2]
        at = pos.T[:, axis]                                  # [n, rot/2]
        cos, sin = s["cos"].gather(0, at), s["sin"].gather(0, at)
    q = _norm_rope(s["q"], s["qw"], cos, sin, rot).to(torch.bfloat16)
    k = _norm_rope(s["k"], s["kw"], cos, sin, rot)
    _plain_store(s, k, s["k_pages"], s["k_scale"], pid, row)
    _plain_store(s, s["v"].float(), s["v_pages"], s["v_scale"], pid, row)
    return {"q": q, "k": s["k_pages"].view(torch.float8_e4m3fn), "v": s["v_pages"].view(torch.float8_e4m3fn), "ks": s["k_scale"], "vs": s["v_scale"]}


def _plain_store(s, x, pool, scale, pid, row):
    page = s["case"]["page"]
    layers, total, h_kv = scale.shape
    amax = torch.full((layers, total, h_kv), -1.0, device="cuda")
    amax.scatter_reduce_(1, pid[None, :, None].expand(layers, -1, h_kv), x.abs().amax(-1), "amax")
    new = _pow2_scale(amax.clamp(min=0))
    # the page a sequence was in the middle of: its rows follow the scale when that grows
    fill = s["lens"].long() % page
    col = (s["lens"].long() // page).clamp(max=s["table"].shape[1] - 1)
    mid = (fill > 0) & (s["q_start"][1:] > s["q_start"][:-1])
    cur = s["table"].long().gather(1, col[:, None])[:, 0]
    cur, fill = cur[mid], fill[mid]
    old = scale[:, cur].clone()
    grown = torch.maximum(old, new[:, cur])
    rows = pool[:, cur].view(torch.float8_e4m3fn).float()
    again = (rows * (old / grown)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = (torch.arange(page, device="cuda")[None, :] < fill[:, None])[None, :, None, :, None] & (grown > old)[..., None, None]
    pool[:, cur] = torch.where(keep, again, pool[:, cur])
    scale.copy_(torch.where(amax >= 0, new, scale))
    scale[:, cur] = grown
    by = (x / scale[:, pid][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    pool[:, pid, :, row] = by.transpose(0, 1)


def _gathered(s):
    """K and V of every sequence, dequantised, [layers, batch, h_kv, width * page, d]."""
    table = s["table"].long().clamp(min=0)
    k = s["k_pages"][:, table].view(torch.float8_e4m3fn).float() * s["k_scale"][:, table][..., None, None]
    v = s["v_pages"][:, table].view(torch.float8_e4m3fn).float() * s["v_scale"][:, table][..., None, None]
    return k.transpose(2, 3).flatten(3, 4), v.transpose(2, 3).flatten(3, 4)


def _plain_decode(s):
    c = s["case"]
    k, v = _gathered(s)
    seen = torch.arange(k.shape[3], device="cuda")[None, :] < s["lens"][:, None]                 # [batch, tokens]
    q = s["q"].float().view(c["layers"], c["batch"], c["h_kv"], c["h_q"] // c["h_kv"], c["d"])
    a = torch.matmul(q, k.masked_fill_(~seen[None, :, None, :, None], 0).transpose(3, 4)) * c["d"] ** -0.5
    a = a.masked_fill(~seen[None, :, None, None, :], -math.inf)
    p = torch.exp(a - a.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p, v.masked_fill_(~seen[None, :, None, :, None], 0)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.to(torch.bfloat16).view_as(s["q"])


def _plain_prefill(s):
    c = s["case"]
    b, h_kv, group, d, mq = c["batch"], c["h_kv"], c["h_q"] // c["h_kv"], c["d"], s["max_q"]
    k, v = _gathered(s)
    k, v = k[0], v[0]
    seen = torch.arange(k.shape[2], device="cuda")[None, :] < s["lens"][:, None]
    k.masked_fill_(~seen[:, None, :, None], 0)
    v.masked_fill_(~seen[:, None, :, None], 0)
    qlen = (s["q_start"][1:] - s["q_start"][:-1]).long()
    at = torch.arange(mq, device="cuda")[None, :]
    real = at < qlen[:, None]
    tok = (s["q_start"][:-1].long()[:, None] + at).clamp(max=s["n"] - 1)
    q = s["q"][0].float()[tok].view(b, mq, h_kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, h_kv, group * mq, d)
    a = torch.matmul(q, k.transpose(2, 3)).view(b, h_kv, group, mq, -1).mul_(d ** -0.5)
    mask = seen[:, None, :].expand(-1, mq, -1)
    if c["causal"]:
        last = s["lens"].long()[:, None] - qlen[:, None] + at
        mask = mask & (torch.arange(k.shape[2], device="cuda")[None, None, :] <= last[:, :, None])
    a.masked_fill_(~mask[:, None, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = a.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(a.view(b, h_kv, group * mq, -1), v).view(b, h_kv, group, mq, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, mq, c["h_q"], d)
    return o[real].to(torch.bfloat16)[None]


# ------------------------------------------------------------------------------------------------ work
def work(case):
    lens, qlens = _lengths(case)
    d, h_q, h_kv, layers, n = case["d"], case["h_q"], case["h_kv"], case["layers"], sum(qlens)
    if case["op"] == "append":
        pages = sum((a + q + case["page"] - 1) // case["page"] - a // case["page"] for a, q in zip(lens, qlens) if q)
        table = n * case["rot"] * 4                          # cos and sin of each token's position
        return {"bytes": layers * n * d * (h_q * 4 + 2 * h_kv * 3) + layers * pages * h_kv * 2 * 4 + table,
                "flops": layers * n * (h_q + h_kv) * (3 * case["rot"] + (4 * d if case["norm"] else 0)) + layers * n * h_kv * 2 * d}
    if case["op"] == "decode":
        return {"bytes": layers * (sum(lens) * h_kv * d * 2 + n * h_q * d * 4 + sum(_pages_of(lens, case["page"])) * h_kv * 8),
                "flops": layers * sum(lens) * h_q * d * 4}
    pairs = sum(q * a - (q * (q - 1) // 2 if case["causal"] else 0) if a >= q or not case["causal"] else a * (a + 1) // 2 for a, q in zip(lens, qlens))
    return {"bytes": sum(lens) * h_kv * d * 2 + n * h_q * d * 4 + sum(_pages_of(lens, case["page"])) * h_kv * 8, "flops": 4 * d * h_q * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definition
def _e4m3_round(x):
    """Nearest e4m3 value (ties to even) of float64 numbers within +-448."""
    _, e = torch.frexp(x.abs())
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _e4m3_value(by):
    """Float64 value of e4m3 bytes, from sign, exponent and mantissa."""
    i = by.to(torch.int64)
    sign, e, m = 1.0 - 2.0 * (i >> 7), (i >> 3) & 15, (i & 7).double()
    v = torch.where(e > 0, torch.ldexp(8 + m, e - 10), torch.ldexp(m, torch.full_like(e, -9)))
    return torch.where((i & 127) == 127, torch.full_like(v, math.nan), sign * v)


def exact(case, seed):
    s = prepare(case, seed)
    lens, qlens = _lengths(case)
    return _exact_append(case, s, lens, qlens) if case["op"] == "append" else _exact_attention(case, s, lens, qlens)


def _exact_append(c, s, lens, qlens):
    page, rot, d = c["page"], c["rot"], c["d"]
    freq_cos, freq_sin = s["cos"].double(), s["sin"].double()
    q_out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    pools = {"k": s["k_pages"].view(torch.float8_e4m3fn).clone(), "v": s["v_pages"].view(torch.float8_e4m3fn).clone()}
    scales = {"k": s["k_scale"].double(), "v": s["v_scale"].double()}
    start = 0

    def turned(x, w, at):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
        y = x.clone()
        if rot:
            where = at[axes].T                                # [tokens, rot / 2]
            cos, sin = freq_cos[where, pairs][:, None, :], freq_sin[where, pairs][:, None, :]
            y[..., :rot // 2] = x[..., :rot // 2] * cos - x[..., rot // 2:rot] * sin
            y[..., rot // 2:rot] = x[..., rot // 2:rot] * cos + x[..., :rot // 2] * sin
        return y

    pairs = torch.arange(rot // 2, device="cuda")
    axes = torch.zeros_like(pairs) if s["pair_axis"] is None else s["pair_axis"].long()[:rot // 2]
    table = s["table"].tolist()
    for b, q in enumerate(qlens):
        sl = slice(start, start + q)
        slot = torch.arange(lens[b], lens[b] + q, device="cuda")
        at = slot[None] if s["positions"] is None else s["positions"][:, sl].long()
        for layer in range(c["layers"]):
            w = (None, None) if s["qw"] is None else (s["qw"][layer], s["kw"][layer])
            for i in range(0, q, 4096):
                part = slice(start + i, min(start + i + 4096, start + q))
                q_out[layer, part] = turned(s["q"][layer, part], w[0], at[:, i:i + 4096])
            for name, x in (("k", turned(s["k"][layer, sl], w[1], at)), ("v", s["v"][layer, sl].double())):
                first = lens[b] // page * page
                pad = torch.zeros(-(-(lens[b] + q) // page) * page - first, c["h_kv"], d, dtype=torch.float64, device="cuda")
                pad[lens[b] - first:lens[b] - first + q] = x
                blocks = pad.view(-1, page, c["h_kv"], d)
                ids = torch.tensor(table[b][first // page:first // page + len(blocks)], device="cuda")
                amax = blocks.abs().amax(dim=(1, 3))                                             # [pages, h_kv]
                m, e = torch.frexp(amax / 448)
                new = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)).clamp(min=2.0 ** -126)
                held = lens[b] - first
                if held:
                    before = scales[name][layer, ids[0]]
                    new[0] = torch.maximum(new[0], before)
                scales_new = new
                vals = (blocks / scales_new[:, None, :, None]).clamp(-448, 448)
                got = _e4m3_round(vals)
                kept = pools[name][layer, ids]                                                   # [pages, h_kv, page, d]
                got = got.permute(0, 2, 1, 3).to(torch.float32).to(torch.float8_e4m3fn)
                mask = torch.zeros(len(blocks) * page, dtype=torch.bool, device="cuda")
                mask[held:held + q] = True
                mask = mask.view(-1, 1, page, 1)
                kept_v, got_v = kept.view(torch.uint8), got.view(torch.uint8)
                if held:
                    old_rows = _e4m3_value(kept_v[0, :, :held]) * (before / new[0])[:, None, None]
                    moved = _e4m3_round(old_rows).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
                    grew = (new[0] > before)[:, None, None]
                    kept_v[0, :, :held] = torch.where(grew, moved, kept_v[0, :, :held])
                pools[name].view(torch.uint8)[layer, ids] = torch.where(mask, got_v, kept_v)
                scales[name][layer, ids] = new
        start += q
    return {"q": q_out, "k": pools["k"], "v": pools["v"], "ks": scales["k"], "vs": scales["v"]}


def _exact_attention(c, s, lens, qlens):
    d, h_kv, group, page = c["d"], c["h_kv"], c["h_q"] // c["h_kv"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    table = s["table"].tolist()
    start = 0
    for b, nq in enumerate(qlens):
        if lens[b] == 0:
            start += nq
            continue
        ids = torch.tensor(table[b][:(lens[b] + page - 1) // page], dtype=torch.long, device="cuda")
        for layer in range(c["layers"]):
            k = _e4m3_value(s["k_pages"][layer, ids]) * s["k_scale"][layer, ids].double()[:, :, None, None]
            v = _e4m3_value(s["v_pages"][layer, ids]) * s["v_scale"][layer, ids].double()[:, :, None, None]
            k = k.transpose(0, 1).reshape(h_kv, -1, d)[:, :lens[b]]
            v = v.transpose(0, 1).reshape(h_kv, -1, d)[:, :lens[b]]
            for i in range(0, nq, 512):
                m = min(512, nq - i)
                part = slice(start + i, start + i + m)
                q = s["q"][layer, part].double().view(m, h_kv, group, d)
                a = torch.einsum("mhgd,htd->hgmt", q, k) / math.sqrt(d)
                if c["op"] == "prefill" and c["causal"]:
                    last = lens[b] - nq + i + torch.arange(m, device="cuda")
                    a = a.masked_fill(torch.arange(lens[b], device="cuda")[None, :] > last[:, None], -math.inf)
                p = torch.softmax(a, -1).nan_to_num(0.0)
                out[layer, part] = torch.einsum("hgmt,htd->mhgd", p, v).reshape(m, h_kv * group, d)
        start += nq
    return out
