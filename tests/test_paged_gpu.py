"""GPU tests of the paged FP8 cache against plain implementations in 64 bits (paged_ref.py)."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

HEADS = [(40, 8, 128), (24, 4, 256), (8, 1, 128), (3, 3, 128), (7, 1, 256)]


def _run_attention(pkg, dev, case, *, causal=None, qlens=None, seed=0, offset=0, hint=None, softmax_scale=None, spare_pages=2):
    """Decode (qlens None) or prefill of ragged sequences; compares every sequence with the 64-bit form."""
    n_layers, (h_q, h_kv, d), page, lens = case
    g = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lens)) + spare_pages
    n_pages = sum(-(-n // page) for n in lens) + 3
    kb, vb, ks, vs = ref.random_cache(g, n_layers, n_pages, h_kv, page, d, pow2=seed % 2 == 0)
    table = ref.random_table(g, lens, page, width, n_pages)
    # slots behind the last token and pages of nobody: NaN bytes, NaN scales
    nobody = sorted(set(range(n_pages)) - set(table[table >= 0].tolist()))
    kb[:, nobody], vb[:, nobody], ks[:, nobody], vs[:, nobody] = 0x7F, 0xFF, float("nan"), float("inf")
    for b, n in enumerate(lens):
        if n % page:
            kb[:, table[b, n // page], :, n % page:] = 0x7F
            vb[:, table[b, n // page], :, n % page:] = 0xFF
    n = sum(qlens) if qlens is not None else len(lens)
    tail = 3 if qlens is not None else 0                    # rows behind the last sequence
    q = torch.randn(n_layers, n + tail, h_q, d, generator=g).to(torch.bfloat16)
    shape = pkg.make_paged_shape(h_q, kb, vb, ks, table)
    ws = pkg.PagedWorkspace(shape, dev, max_seq_len=hint, q_tokens=None if qlens is None else n + tail)
    up = [t.to(dev) for t in (kb, vb, ks, vs, table)]
    out = torch.full_like(q, 7.0).to(dev)
    seq_len = torch.tensor(lens, dtype=torch.int32, device=dev) - offset
    if qlens is None:
        for _ in range(2):                                  # the second launch finds the workspace as the first left it
            got = pkg.paged_decode_attention(q.to(dev), *up, seq_len, workspace=ws, seq_len_offset=offset, out=out, softmax_scale=softmax_scale)
    else:
        starts = torch.tensor([sum(qlens[:i]) for i in range(len(qlens) + 1)], dtype=torch.int32, device=dev)
        for _ in range(2):
            got = pkg.paged_prefill_attention(q.to(dev), starts, *up, seq_len, workspace=ws, causal=causal, out=out, softmax_scale=softmax_scale)
    torch.cuda.synchronize()
    assert ws.read_status() == 0
    got = got.cpu()
    assert (got[:, n:] == 7.0).all(), "rows behind the last sequence were written"
    at = 0
    for b, length in enumerate(lens):
        m = 1 if qlens is None else qlens[b]
        for layer in range(n_layers):
            want, big = ref.attention(q[layer, at:at + m], kb[layer], vb[layer], ks[layer], vs[layer], table[b], length, causal=bool(causal),
                                      softmax_scale=softmax_scale)
            ref.assert_attention(got[layer, at:at + m], want, big, (case, b, layer))
        at += m
    return got


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_decode_lengths(pkg, cuda_device, heads, page):
    """Empty, one token, ends inside and at the end of pages and tiles, all in one batch."""
    _run_attention(pkg, cuda_device, (1, heads, page, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 511, 1000]), seed=page)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_decode_layers_and_long(pkg, cuda_device, page):
    _run_attention(pkg, cuda_device, (3, (10, 2, 128), page, [5000, 1, 2049]), seed=page + 1)


def test_decode_length_hint_too_small_or_absent_and_offset(pkg, cuda_device):
    for hint in (None, 1, 700, 5000):
        _run_attention(pkg, cuda_device, (1, (5, 1, 128), 64, [3000, 64, 1]), seed=3, hint=hint, offset=1)
    _run_attention(pkg, cuda_device, (1, (24, 4, 256), 32, [777, 5]), seed=4, softmax_scale=0.3)


def test_decode_only_empty_sequences(pkg, cuda_device):
    got = _run_attention(pkg, cuda_device, (2, (40, 8, 128), 64, [0, 0, 0]), seed=5)
    assert (got == 0).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads", HEADS)
def test_prefill_ragged(pkg, cuda_device, heads, causal):
    """Whole prompts, chunks on a prefix, single tokens, no token at all, fewer cached tokens than queries, nothing cached."""
    lens, qlens = [130, 300, 64, 5, 1, 20, 0, 257], [130, 40, 1, 0, 1, 33, 4, 129]
    _run_attention(pkg, cuda_device, (1, heads, 64, lens), qlens=qlens, causal=causal, seed=11)


@pytest.mark.parametrize("page", [16, 32, 128])
def test_prefill_pages_and_layers(pkg, cuda_device, page):
    _run_attention(pkg, cuda_device, (2, (10, 2, 128), page, [401, 33]), qlens=[77, 33], causal=True, seed=page)


@pytest.mark.parametrize("heads", [(5, 1, 128), (7, 1, 256)])
def test_prefill_few_rows_on_a_long_cache(pkg, cuda_device, heads):
    _run_attention(pkg, cuda_device, (1, heads, 64, [6000, 4097]), qlens=[3, 5], causal=True, seed=21)


def test_scores_far_from_zero_and_queries_of_any_size(pkg, cuda_device):
    """One key far above the rest; queries beyond the range of f16 and below it; all-zero queries."""
    g = torch.Generator().manual_seed(9)
    h_q, h_kv, d, page = 8, 1, 128, 64
    for size, scale in ((1e6, 1e-7), (1e-9, 1e8), (0.0, 1.0), (30.0, 0.1)):
        kb, vb, ks, vs = ref.random_cache(g, 1, 5, h_kv, page, d)
        q = (torch.randn(1, 4, h_q, d, generator=g) * size).to(torch.bfloat16)
        table = torch.tensor([[4, 0, 2]], dtype=torch.int32)
        up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
        shape = pkg.make_paged_shape(h_q, kb, vb, ks, table)
        lens = torch.tensor([150], dtype=torch.int32, device=cuda_device)
        want, big = ref.attention(q[0], kb[0], vb[0], ks[0], vs[0], table[0], 150, softmax_scale=scale)
        out = pkg.paged_prefill_attention(q.to(cuda_device), torch.tensor([0, 4], dtype=torch.int32, device=cuda_device), *up, lens, causal=False,
                                          softmax_scale=scale, workspace=pkg.PagedWorkspace(shape, cuda_device, q_tokens=4))
        ref.assert_attention(out[0].cpu(), want, big, ("prefill", size))
        out = pkg.paged_decode_attention(q[:, :1].contiguous().to(cuda_device), *up, lens, softmax_scale=scale,
                                         workspace=pkg.PagedWorkspace(shape, cuda_device))
        ref.assert_attention(out[0].cpu(), want[:1], big[:1], ("decode", size))


def test_bad_page_numbers_are_reported_and_skipped(pkg, cuda_device):
    """A page number outside the pool inside the valid length: the status says so, its tokens are not attended."""
    g = torch.Generator().manual_seed(2)
    kb, vb, ks, vs = ref.random_cache(g, 1, 4, 1, 64, 128)
    q = torch.randn(1, 1, 5, 128, generator=g).to(torch.bfloat16)
    for bad in (-1, 4, 1 << 30):
        table = torch.tensor([[2, bad, 1]], dtype=torch.int32)
        up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
        shape = pkg.make_paged_shape(5, kb, vb, ks, table)
        lens = torch.tensor([160], dtype=torch.int32, device=cuda_device)
        # the same tokens without the hole: 64 of page 2, then 32 of page 1
        want, big = ref.attention(q[0], kb[0], vb[0], ks[0], vs[0], torch.tensor([2, 1]), 96)
        ws = pkg.PagedWorkspace(shape, cuda_device)
        out = pkg.paged_decode_attention(q.to(cuda_device), *up, lens, workspace=ws)
        ref.assert_attention(out[0].cpu(), want, big, "decode")
        assert ws.read_status() == pkg._lib.STATUS_BAD_PAGE
        ws = pkg.PagedWorkspace(shape, cuda_device, q_tokens=1)
        out = pkg.paged_prefill_attention(q.to(cuda_device), torch.tensor([0, 1], dtype=torch.int32, device=cuda_device), *up, lens, workspace=ws)
        ref.assert_attention(out[0].cpu(), want, big, "prefill")
        assert ws.read_status() == pkg._lib.STATUS_BAD_PAGE


def test_lengths_outside_the_table_are_reported(pkg, cuda_device):
    g = torch.Generator().manual_seed(2)
    kb, vb, ks, vs = ref.random_cache(g, 1, 4, 1, 64, 128)
    q = torch.randn(1, 2, 5, 128, generator=g).to(torch.bfloat16)
    table = torch.tensor([[2, 1], [0, 3]], dtype=torch.int32)
    up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
    ws = pkg.PagedWorkspace(pkg.make_paged_shape(5, kb, vb, ks, table), cuda_device)
    out = pkg.paged_decode_attention(q.to(cuda_device), *up, torch.tensor([1000, -3], dtype=torch.int32, device=cuda_device), workspace=ws).cpu()
    want, big = ref.attention(q[0, :1], kb[0], vb[0], ks[0], vs[0], table[0], 128)
    ref.assert_attention(out[0, :1], want, big)
    assert (out[0, 1] == 0).all()
    assert ws.read_status() == pkg._lib.STATUS_LEN_OVER_CAP | pkg._lib.STATUS_LEN_NEGATIVE


# ---------------------------------------------------------------------------------------------- append
def _append_case(pkg, dev, heads, page, pos, qlens, *, rot, axes=1, norm=False, n_layers=1, seed=0, one=False, specials=False):
    h_q, h_kv, d = heads
    g = torch.Generator().manual_seed(seed)
    batch, n = len(pos), sum(qlens)
    width = max(-(-(p + m) // page) for p, m in zip(pos, qlens)) + 1
    n_pages = sum(-(-(p + m) // page) for p, m in zip(pos, qlens)) + 2
    kb, vb, ks, vs = ref.random_cache(g, n_layers, n_pages, h_kv, page, d)
    table = ref.random_table(g, [p + m for p, m in zip(pos, qlens)], page, width, n_pages)
    tail = 0 if one else 2
    q = torch.randn(n_layers, n + tail, h_q, d, generator=g).to(torch.bfloat16)
    k = torch.randn(n_layers, n + tail, h_kv, d, generator=g).to(torch.bfloat16)
    v = (torch.randn(n_layers, n + tail, h_kv, d, generator=g) * torch.exp(3 * torch.randn(1, n + tail, h_kv, 1, generator=g))).to(torch.bfloat16)
    if specials:
        v[0, 0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0])
        v[0, 1] = 0
    qw = (0.1 * torch.randn(n_layers, d, generator=g)).to(torch.bfloat16) if norm else None
    kw = (0.1 * torch.randn(n_layers, d, generator=g)).to(torch.bfloat16) if norm else None
    slots = torch.tensor([p + i for p, m in zip(pos, qlens) for i in range(m)] + [0] * tail)
    cos = sin = positions = pair_axis = None
    at = slots[None]
    if rot:
        cos, sin = pkg.rope_tables(int(slots.max()) + 1, rot, device="cpu")
        if axes > 1:
            at = torch.stack([slots // (a + 1) for a in range(axes)])
            positions = at.to(torch.int32)
            pair_axis = torch.randint(0, axes, (rot // 2,), generator=g).to(torch.int32)
    starts = torch.tensor([sum(qlens[:i]) for i in range(batch + 1)], dtype=torch.int32)
    d_ = lambda t: None if t is None else t.to(dev)  # noqa: E731
    up = [d_(t) for t in (kb, vb, ks, vs, table)]
    status, seq_pos = torch.zeros(1, dtype=torch.int32, device=dev), torch.tensor(pos, dtype=torch.int32, device=dev)
    q_out = torch.full_like(q, 7.0).to(dev)
    pkg.paged_rope_append(d_(q), d_(k), d_(v), d_(cos), d_(sin), *up, seq_pos, q_start=None if one else d_(starts), positions=d_(positions),
                          pair_axis=d_(pair_axis), q_norm_weight=d_(qw), k_norm_weight=d_(kw), status=status, q_out=q_out)
    torch.cuda.synchronize()
    assert status.item() == 0 and seq_pos.cpu().tolist() == [p + m for p, m in zip(pos, qlens)]
    q_out = q_out.cpu()
    assert (q_out[:, n:] == 7.0).all(), "query rows behind the last sequence were written"
    used = torch.zeros(n_pages, page, dtype=torch.bool)
    for layer in range(n_layers):
        want = ref.norm_rope(q[layer, :n], None if qw is None else qw[layer], cos, sin, at[:, :n], pair_axis)
        # bf16: half a step 2^-8 of the value; fp32 arithmetic: a few 2^-24 of the row
        assert ((q_out[layer, :n].double() - want).abs() <= want.abs() * 2.0 ** -8 + want.abs().amax(-1, keepdim=True) * 2.0 ** -20).all()
        for which, x, pool, scale, got_b, got_s in (("k", k, kb, ks, up[0], up[2]), ("v", v, vb, vs, up[1], up[3])):
            rows = x[layer, :n].double()
            if which == "k":
                rows = ref.norm_rope(k[layer, :n], None if kw is None else kw[layer], cos, sin, at[:, :n], pair_axis)
            vals, sc = ref.values(pool[layer]), scale[layer].double().clone()
            for b in range(batch):
                ref.append_rows(rows[starts[b]:starts[b + 1]], vals, sc, table[b], page, pos[b])
                used[[int(table[b, s // page]) for s in range(pos[b], pos[b] + qlens[b])], [s % page for s in range(pos[b], pos[b] + qlens[b])]] = True
            got_v, got_sc = ref.values(got_b[layer].cpu()), got_s[layer].cpu().double()
            assert torch.equal(got_sc, sc), which
            if which == "v" or (not rot and not norm):       # no arithmetic before the rounding: the same numbers
                assert torch.equal(torch.nan_to_num(got_v, 999.0), torch.nan_to_num(vals, 999.0)), which
            else:                                            # fp32 arithmetic may sit on the other side of a rounding border
                near = (got_v - vals).abs() <= vals.abs() * 2.0 ** -3 + 2.0 ** -9
                assert near.all() and (got_v != vals).double().mean() < 1e-4
    return up


@pytest.mark.parametrize("heads,rot,axes,norm", [((40, 8, 128), 128, 1, False), ((24, 4, 256), 64, 3, True), ((5, 1, 128), 0, 1, True),
                                                 ((8, 1, 256), 256, 2, False), ((3, 3, 128), 16, 4, True), ((10, 2, 128), 48, 1, False)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_prompts(pkg, cuda_device, heads, rot, axes, norm, page):
    pos, qlens = [0, 5, 63, 64, 0, 17, 130], [70, 1, 2, 129, 0, 300, 7]
    _append_case(pkg, cuda_device, heads, page, pos, qlens, rot=rot, axes=axes, norm=norm, seed=page + rot, n_layers=2 if page == 32 else 1)


@pytest.mark.parametrize("heads,rot,axes,norm", [((40, 8, 128), 128, 1, False), ((24, 4, 256), 64, 3, True), ((5, 1, 128), 0, 1, False)])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_append_one_token_each(pkg, cuda_device, heads, rot, axes, norm, page):
    pos = [0, 1, 15, 16, 63, 64, 127, 128, 129, 1000]
    _append_case(pkg, cuda_device, heads, page, pos, [1] * len(pos), rot=rot, axes=axes, norm=norm, seed=page, n_layers=3, one=True)
    _append_case(pkg, cuda_device, heads, page, pos, [1] * len(pos), rot=rot, axes=axes, norm=norm, seed=page)


@pytest.mark.parametrize("one", [True, False])
def test_append_infinities_nan_and_zero_rows(pkg, cuda_device, one):
    _append_case(pkg, cuda_device, (5, 1, 128), 64, [0, 0, 70], [1, 1, 1], rot=0, one=one, specials=True, seed=1)


def test_token_by_token_equals_one_piece(pkg, cuda_device):
    """A page's scale only grows, by powers of two: token by token the scales are those of the whole prompt, and the bytes too
    but for values that became subnormal on the way (rounded again: at most one subnormal step, 2^-9 of the scale)."""
    g = torch.Generator().manual_seed(5)
    h_kv, d, page, n = 2, 128, 32, 75
    k = (torch.randn(n, h_kv, d, generator=g) * torch.exp(1.5 * torch.randn(n, h_kv, 1, generator=g))).to(torch.bfloat16).to(cuda_device)
    table = torch.tensor([[3, 0, 4]], dtype=torch.int32, device=cuda_device)
    res = []
    for pieces in ([n], [1] * n, [10, 1, 1, 40, 23]):
        kp = torch.zeros(1, 5, h_kv, page, d, dtype=torch.uint8, device=cuda_device)
        vp, ks = torch.zeros_like(kp), torch.full((1, 5, h_kv), 1e30, device=cuda_device)
        vs, pos, status, at = ks.clone(), torch.zeros(1, dtype=torch.int32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device), 0
        for m in pieces:
            part = k[at:at + m].contiguous()
            pkg.paged_rope_append(None, part, part, None, None, kp, vp, ks, vs, table, pos, status=status,
                                  q_start=None if m == 1 and at % 2 else torch.tensor([0, m], dtype=torch.int32, device=cuda_device))
            at += m
        assert status.item() == 0 and pos.item() == n
        assert torch.equal(kp, vp) and torch.equal(ks, vs)
        res.append((ref.values(kp[0].cpu()), ks[0].cpu()))
    for vals, sc in res[1:]:
        assert torch.equal(sc, res[0][1])
        assert ((vals - res[0][0]).abs() <= 2.0 ** -9).all()


def test_append_reports_capacity_pages_and_positions(pkg, cuda_device):
    L = pkg._lib
    dev, h_kv, d, page = cuda_device, 2, 128, 16

    def call(pos, qlens, table, one=False, n_positions=64, positions=None):
        kp = torch.full((1, 4, h_kv, page, d), 0x11, dtype=torch.uint8, device=dev)
        vp, ks = kp.clone(), torch.ones(1, 4, h_kv, device=dev)
        vs, status = ks.clone(), torch.zeros(1, dtype=torch.int32, device=dev)
        seq_pos = torch.tensor(pos, dtype=torch.int32, device=dev)
        n = sum(qlens)
        x = torch.ones(n, h_kv, d, dtype=torch.bfloat16, device=dev)
        cos, sin = pkg.rope_tables(n_positions, 128, device=dev)
        starts = torch.tensor([sum(qlens[:i]) for i in range(len(qlens) + 1)], dtype=torch.int32, device=dev)
        pkg.paged_rope_append(x, x, x, cos, sin, kp, vp, ks, vs, torch.tensor(table, dtype=torch.int32, device=dev), seq_pos, status=status,
                              q_start=None if one else starts, positions=positions)
        torch.cuda.synchronize()
        return status.item(), seq_pos.cpu().tolist(), vp.cpu()

    for one in (True, False):
        st, pos, vp = call([32, 3], [1, 1], [[0, 1], [2, 3]], one=one)           # the first sequence is full
        assert st == L.STATUS_POS_AT_CAPACITY and pos == [32, 4]
        assert (vp[0, [0, 1, 3]] == 0x11).all() and (vp[0, 2, :, 3] != 0x11).all()
        for bad in (-1, 4, 1 << 30):
            st, pos, vp = call([16, 3], [1, 1], [[0, bad], [2, 3]], one=one)
            assert st == L.STATUS_BAD_PAGE and (vp[0, [0, 1, 3]] == 0x11).all()
        st, pos, vp = call([-1, 3], [1, 1], [[0, 1], [2, 3]], one=one)
        assert st & ~L.STATUS_BAD_POSITION == (L.STATUS_POS_AT_CAPACITY if one else 0) and pos == [-1, 4] and (vp[0, [0, 1, 3]] == 0x11).all()
    st, pos, vp = call([30], [5], [[1, 2]])                                       # two fit, three do not
    assert st == L.STATUS_POS_AT_CAPACITY and pos == [30] and (vp[0, 2, :, 14:] != 0x11).all() and (vp[0, [0, 1, 3]] == 0x11).all()
    far = torch.tensor([0, 64, -1], dtype=torch.int32, device=dev)
    st, pos, vp = call([0], [3], [[1, 2]], positions=far)
    assert st == L.STATUS_BAD_POSITION and pos == [3]


# ---------------------------------------------------------------------------------------------- together
def _dense_attention(q, k, v, causal_from):
    """float64 attention of q [n, h_q, d] at positions causal_from.. over k, v [t, h_kv, d]."""
    n, h_q, d = q.shape
    rep = h_q // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    a = torch.einsum("nhd,thd->hnt", q, k) * d ** -0.5
    a = a.masked_fill(torch.arange(k.shape[0])[None, None, :] > (causal_from + torch.arange(n))[None, :, None], float("-inf"))
    return torch.einsum("hnt,thd->nhd", torch.softmax(a, -1), v)


def test_serving_run(pkg, cuda_device):
    """Prompts, decode steps captured in a graph, a sequence that ends and its pages taken by another: the cache class against
    64-bit attention over the bf16 keys and values.  The cache keeps 4 significant bits: a key or value is off by at most
    2^-4 of itself; compared by cosine, which random errors of that size leave above 0.998."""
    dev, layers, slots, h_q, h_kv, d, page = cuda_device, 2, 3, 10, 2, 128, 16
    c = pkg.PagedFP8Cache(layers, slots, h_q, h_kv, d, n_pages=30, max_pages=12, page_size=page, device=dev, max_prompt_tokens=150)
    cos, sin = pkg.rope_tables(256, 128, device=dev)
    g = torch.Generator().manual_seed(0)
    hist = [[torch.zeros(layers, 0, h_kv, d, dtype=torch.float64)] * 2 for _ in range(slots)]
    mk = lambda n, h: torch.randn(layers, n, h, d, generator=g).to(torch.bfloat16)  # noqa: E731

    def check(q, k, v, out, lens):
        at = 0
        for b, n in enumerate(lens):
            if n == 0:
                continue
            before = hist[b][0].shape[1]
            pos = torch.arange(before, before + n)[None]
            for i, x in ((0, torch.stack([ref.norm_rope(k[l, at:at + n], None, cos.cpu(), sin.cpu(), pos, None) for l in range(layers)])),
                         (1, v[:, at:at + n].double())):
                hist[b][i] = torch.cat([hist[b][i], x], 1)
            for l in range(layers):
                qr = ref.norm_rope(q[l, at:at + n], None, cos.cpu(), sin.cpu(), pos, None)
                want = _dense_attention(qr, hist[b][0][l], hist[b][1][l], before)
                got = out[l, at:at + n].cpu().double()
                assert torch.cosine_similarity(got.flatten(), want.flatten(), dim=0) > 0.998
            at += n

    def prompt(lens):
        q, k, v = mk(sum(lens), h_q), mk(sum(lens), h_kv), mk(sum(lens), h_kv)
        out = c.prefill(q.to(dev), k.to(dev), v.to(dev), cos, sin, lens)
        check(q, k, v, out, lens)

    prompt([50, 7, 90])
    prompt([0, 20, 5])                                     # a second piece on top of the first
    buf = [mk(slots, h).to(dev) for h in (h_q, h_kv, h_kv)]
    out = torch.empty(layers, slots, h_q, d, dtype=torch.bfloat16, device=dev)
    for b in range(slots):
        c.reserve(b, 40)
    step = lambda: c.step(*buf, cos, sin, out=out, count=False)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    pos0 = c.seq_pos.clone()
    with torch.cuda.stream(s):
        step()                                             # warm-up; its token is written again by the first replay
    torch.cuda.current_stream().wait_stream(s)
    c.seq_pos.copy_(pos0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):
        q, k, v = mk(slots, h_q), mk(slots, h_kv), mk(slots, h_kv)
        for t, x in zip(buf, (q, k, v)):
            t.copy_(x)
        graph.replay()
        c.host_len = [x + 1 for x in c.host_len]
        check(q, k, v, out, [1, 1, 1])
    torch.cuda.synchronize()
    assert c.seq_pos.cpu().tolist() == c.host_len and c.read_status() == 0
    c.release(1)
    hist[1] = [torch.zeros(layers, 0, h_kv, d, dtype=torch.float64)] * 2
    prompt([1, 60, 0])                                     # another sequence in the freed slot, on used pages
    assert c.read_status() == 0


def test_other_stream_and_bits_stay_the_same(pkg, cuda_device):
    """Calls on a side stream, twenty times: the same bits (partial results are joined in a fixed order)."""
    g = torch.Generator().manual_seed(1)
    kb, vb, ks, vs = ref.random_cache(g, 1, 200, 2, 64, 128)
    table = torch.randperm(200, generator=g).to(torch.int32).view(2, 100)
    up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
    q = torch.randn(1, 2, 10, 128, generator=g).to(torch.bfloat16).to(cuda_device)
    starts, lens = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device), torch.tensor([6400, 3333], dtype=torch.int32, device=cuda_device)
    shape = pkg.make_paged_shape(10, kb, vb, ks, table)
    wd, wp = pkg.PagedWorkspace(shape, cuda_device), pkg.PagedWorkspace(shape, cuda_device, q_tokens=2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a = [pkg.paged_decode_attention(q, *up, lens, workspace=wd) for _ in range(20)]
        b = [pkg.paged_prefill_attention(q, starts, *up, lens, workspace=wp) for _ in range(20)]
    s.synchronize()
    assert all(torch.equal(x, a[0]) for x in a) and all(torch.equal(x, b[0]) for x in b)
    for i, n in enumerate([6400, 3333]):
        want, big = ref.attention(q[0, i:i + 1].cpu(), kb[0], vb[0], ks[0], vs[0], table[i], n)
        ref.assert_attention(a[0][0, i:i + 1].cpu(), want, big)
        ref.assert_attention(b[0][0, i:i + 1].cpu(), want, big)


@pytest.mark.parametrize("causal", [True, False])
def test_prefill_enough_rows_for_the_whole_gpu(pkg, cuda_device, causal):
    """As many query tiles as make every thread block take two of them (heads of 128), with blocks that have one tile, a full
    pair, or a pair whose second tile has one token."""
    _run_attention(pkg, cuda_device, (1, (40, 8, 128), 64, [700, 1000, 26, 80, 25]), qlens=[700, 333, 26, 51, 25], causal=causal, seed=31)
    _run_attention(pkg, cuda_device, (1, (16, 16, 128), 32, [600, 129]), qlens=[600, 129], causal=causal, seed=32)


def _spare(pairs, d, page):
    """Table columns that make the largest possible call a large one, whatever the lengths are."""
    return max(1100 * 128 // d, 133000 * 128 // (d * pairs)) // page + 2


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_decode_lengths_in_a_wide_table(pkg, cuda_device, heads, page):
    """Empty, one token, ends inside and at the end of pages and tiles, far below what the table could hold."""
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 300, 511, 1000]
    _run_attention(pkg, cuda_device, (1, heads, page, lens), seed=page, spare_pages=_spare(len(lens) * heads[1], heads[2], page))


@pytest.mark.parametrize("heads", [(8, 1, 128), (5, 1, 256), (20, 4, 128)])
def test_decode_one_long_sequence_and_layers(pkg, cuda_device, heads):
    """One pair on the whole GPU (many pieces to join); layers of a long and short sequences; equal short lengths."""
    _run_attention(pkg, cuda_device, (1, heads, 32, [20011]), seed=40, spare_pages=_spare(heads[1], heads[2], 32))
    _run_attention(pkg, cuda_device, (3, heads, 128, [7000, 1, 2049]), seed=41, spare_pages=_spare(9 * heads[1], heads[2], 128))
    _run_attention(pkg, cuda_device, (2, heads, 64, [320, 320, 320]), seed=42, spare_pages=_spare(6 * heads[1], heads[2], 64), hint=500000)
    _run_attention(pkg, cuda_device, (1, heads, 16, [0, 0]), seed=43, spare_pages=_spare(2 * heads[1], heads[2], 16))


def test_decode_more_sequences_than_one_block_can_list(pkg, cuda_device):
    lens = [i * 7 % 40 for i in range(2100)]
    _run_attention(pkg, cuda_device, (1, (3, 3, 128), 16, lens), seed=44, spare_pages=80)


def test_bad_page_numbers_in_a_wide_table(pkg, cuda_device):
    g = torch.Generator().manual_seed(2)
    kb, vb, ks, vs = ref.random_cache(g, 1, 4, 1, 16, 128)
    q = torch.randn(1, 2, 5, 128, generator=g).to(torch.bfloat16)
    for bad in (-1, 4, 1 << 30):
        table = torch.full((2, 5000), bad, dtype=torch.int32)
        table[0, :6] = torch.tensor([2, bad, 1, bad, bad, 3])     # the second sequence has bad pages only
        up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
        ws = pkg.PagedWorkspace(pkg.make_paged_shape(5, kb, vb, ks, table), cuda_device)
        lens = torch.tensor([90, 300], dtype=torch.int32, device=cuda_device)
        out = pkg.paged_decode_attention(q.to(cuda_device), *up, lens, workspace=ws).cpu()
        want, big = ref.attention(q[0, :1], kb[0], vb[0], ks[0], vs[0], torch.tensor([2, 1, 3]), 42)
        ref.assert_attention(out[0, :1], want, big, bad)
        assert (out[0, 1] == 0).all()
        assert ws.read_status() == pkg._lib.STATUS_BAD_PAGE


def test_ragged_batch_launched_many_times(pkg, cuda_device):
    """Launches back to back, eager and as one graph: no wait runs out, and the bits stay the same."""
    g = torch.Generator().manual_seed(6)
    lens = [(i * 613) % 3000 + 1 for i in range(32)]
    kb, vb, ks, vs = ref.random_cache(g, 1, 900, 8, 64, 128)
    table = torch.randint(0, 900, (32, 256), generator=g).to(torch.int32)
    q = torch.randn(1, 32, 40, 128, generator=g).to(torch.bfloat16).to(cuda_device)
    up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    shape = pkg.make_paged_shape(40, kb, vb, ks, table)
    ws, outs = [pkg.PagedWorkspace(shape, cuda_device) for _ in range(2)], [torch.empty_like(q) for _ in range(2)]
    for i in range(4000):
        pkg.paged_decode_attention(q, *up, n, workspace=ws[i % 2], out=outs[i % 2])
    first = outs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(8):
            pkg.paged_decode_attention(q, *up, n, workspace=ws[i % 2], out=outs[i % 2])
    for _ in range(500):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, outs[0]) and torch.equal(first, outs[1])
    assert [w.read_status() for w in ws] == [0, 0]
    for b in (0, 7, 31):
        want, big = ref.attention(q[0, b:b + 1].cpu(), kb[0], vb[0], ks[0], vs[0], table[b], lens[b])
        ref.assert_attention(first[0, b:b + 1].cpu(), want, big)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 128])
def test_prefill_a_few_tokens_each(pkg, cuda_device, heads, causal, page):
    """A handful of new tokens per sequence, none for some, many for one; fewer cached tokens than new ones."""
    lens, qlens = [130, 300, 64, 5, 1, 20, 0, 257, 1100, 17], [1, 2, 1, 0, 1, 3, 2, 4, 1, 2]
    _run_attention(pkg, cuda_device, (2, heads, page, lens), qlens=qlens, causal=causal, seed=51)
    lens, qlens = [700, 31, 0, 9, 16, 2, 64, 128, 500, 12, 33, 1], [15, 1, 0, 0, 0, 0, 1, 1, 1, 1, 1, 1]
    _run_attention(pkg, cuda_device, (1, heads, page, lens), qlens=qlens, causal=causal, seed=52)


@pytest.mark.parametrize("heads", [(5, 1, 128), (40, 8, 128), (4, 2, 256), (8, 1, 256)])
def test_prefill_a_few_tokens_on_long_caches(pkg, cuda_device, heads):
    """Few sequences: the keys are cut into pieces, which do not all have tokens."""
    _run_attention(pkg, cuda_device, (1, heads, 64, [6000, 4097, 40]), qlens=[2, 1, 2], causal=True, seed=53)
    _run_attention(pkg, cuda_device, (1, heads, 32, [33, 9001]), qlens=[1, 1], causal=True, seed=54, hint=20000)
    _run_attention(pkg, cuda_device, (1, heads, 16, [257]), qlens=[2], causal=False, seed=55, hint=100)


def test_workspaces_serve_calls_of_any_shape(pkg, cuda_device):
    """One workspace for calls that are laid out differently in it, in turn: short and long tables, few and many sequences."""
    g = torch.Generator().manual_seed(8)
    kb, vb, ks, vs = ref.random_cache(g, 1, 300, 2, 64, 128)
    up = [t.to(cuda_device) for t in (kb, vb, ks, vs)]
    cases = []
    for batch, lens, width in ((1, [700], 11), (2, [3000, 5000], 2000), (4, [900, 1000, 64, 1], 16), (3, [9000, 1, 130], 1500), (70, [200] * 70, 4)):
        table = torch.zeros(batch, width, dtype=torch.int32)
        table[:, :min(width, 150)] = torch.randint(0, 300, (batch, min(width, 150)), generator=g).to(torch.int32)
        for h_q in (2, 10):
            q = torch.randn(1, batch, h_q, 128, generator=g).to(torch.bfloat16)
            cases.append((q, table, lens, pkg.make_paged_shape(h_q, kb, vb, ks, table)))
    wd, wp = (pkg.PagedWorkspace(cases[0][3], cuda_device, q_tokens=n) for n in (None, 70))
    for turn in range(3):
        for q, table, lens, _ in cases:
            n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
            starts = torch.arange(len(lens) + 1, dtype=torch.int32, device=cuda_device)
            a = pkg.paged_decode_attention(q.to(cuda_device), *up, table.to(cuda_device), n, workspace=wd).cpu()
            b = pkg.paged_prefill_attention(q.to(cuda_device), starts, *up, table.to(cuda_device), n, workspace=wp).cpu()
            for i in sorted({0, len(lens) - 1, len(lens) // 2}):
                want, big = ref.attention(q[0, i:i + 1], kb[0], vb[0], ks[0], vs[0], table[i], lens[i])
                ref.assert_attention(a[0, i:i + 1], want, big, ("decode", turn, lens))
                ref.assert_attention(b[0, i:i + 1], want, big, ("prefill", turn, lens))
    assert wd.read_status() == 0 and wp.read_status() == 0


def test_as_many_sequences_as_one_block_can_list(pkg, cuda_device):
    lens = [i * 11 % 50 for i in range(2048)]
    _run_attention(pkg, cuda_device, (1, (8, 1, 256), 16, lens), seed=46, spare_pages=80)


def test_pages_beyond_two_gigabytes(pkg, cuda_device):
    """The last pages of a large pool: appended to, then read by every attention kernel."""
    g = torch.Generator().manual_seed(12)
    h_q, h_kv, d, page, n_pages = 40, 8, 128, 64, 34000
    kb, vb = (torch.zeros(1, n_pages, h_kv, page, d, dtype=torch.uint8, device=cuda_device) for _ in range(2))
    ks, vs = (torch.ones(1, n_pages, h_kv, device=cuda_device) for _ in range(2))
    lens, width = [300, 129, 1], 600
    table = torch.full((3, width), -1, dtype=torch.int32)
    at = n_pages - 1
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b, i], at = at, at - 1
    low = at + 1                                            # the pages used are [low, n_pages)
    k, v = (torch.randn(1, sum(lens), h_kv, d, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2))
    starts = torch.tensor([0, 300, 429, 430], dtype=torch.int32, device=cuda_device)
    pos, status = torch.zeros(3, dtype=torch.int32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    up = (kb, vb, ks, vs, table.to(cuda_device))
    pkg.paged_rope_append(None, k, v, None, None, *up, pos, q_start=starts, status=status)
    assert pos.tolist() == lens and status.item() == 0
    small = [t[:, low:].cpu() for t in (kb, vb, ks, vs)]
    for b, n in enumerate(lens):                            # the bytes are the new tokens', to half a step of e4m3
        rows = torch.cat([small[0][0, table[b, i] - low].permute(1, 0, 2) for i in range(-(-n // page))])[:n]
        scale = torch.stack([small[2][0, table[b, i // page] - low] for i in range(n)])[:, :, None].double()
        want = k[0, starts[b]:starts[b] + n].cpu().double()
        assert ((ref.values(rows) * scale - want).abs() <= want.abs() * 2.0 ** -4 + scale * 2.0 ** -10).all()
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    q = torch.randn(1, 3, h_q, d, generator=g).to(torch.bfloat16)
    many = torch.randn(1, 200, h_q, d, generator=g).to(torch.bfloat16)
    shape = pkg.make_paged_shape(h_q, kb, vb, ks, table)
    wp = pkg.PagedWorkspace(shape, cuda_device, q_tokens=200)
    first = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda_device)
    got = [pkg.paged_decode_attention(q.to(cuda_device), *up, n, workspace=pkg.PagedWorkspace(shape, cuda_device, max_seq_len=most)) for most in (300, 38400)]
    got.append(pkg.paged_prefill_attention(q.to(cuda_device), first, *up, n, workspace=wp))
    rows = torch.tensor([0, 100, 199, 200], dtype=torch.int32, device=cuda_device)
    out = pkg.paged_prefill_attention(many.to(cuda_device), rows, *up, n, workspace=wp, causal=False).cpu()
    for b, length in enumerate(lens):
        ids = torch.where(table[b] >= 0, table[b] - low, table[b])
        want, big = ref.attention(q[0, b:b + 1], small[0][0], small[1][0], small[2][0], small[3][0], ids, length)
        for i, x in enumerate(got):
            ref.assert_attention(x[0, b:b + 1].cpu(), want, big, (i, b))
        a, z = rows[b].item(), rows[b + 1].item()
        want, big = ref.attention(many[0, a:z], small[0][0], small[1][0], small[2][0], small[3][0], ids, length)
        ref.assert_attention(out[0, a:z], want, big, ("many", b))


def test_captured_calls_follow_lengths_and_share_workspaces(pkg, cuda_device):
    """Two graphs over the same workspaces, replayed in turn with other lengths and queries: many rows, few rows, one row."""
    g = torch.Generator().manual_seed(15)
    h_q, h_kv, d, page = 10, 2, 128, 32
    kb, vb, ks, vs = ref.random_cache(g, 1, 400, h_kv, page, d)
    table = torch.randperm(400, generator=g)[:360].to(torch.int32).view(2, 180)
    up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
    shape = pkg.make_paged_shape(h_q, kb, vb, ks, table)
    wd, wp = pkg.PagedWorkspace(shape, cuda_device), pkg.PagedWorkspace(shape, cuda_device, q_tokens=90)
    n = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    q1, few, many = (torch.zeros(1, m, h_q, d, dtype=torch.bfloat16, device=cuda_device) for m in (2, 5, 90))
    s_few, s_many = torch.zeros(3, dtype=torch.int32, device=cuda_device), torch.zeros(3, dtype=torch.int32, device=cuda_device)
    outs = [torch.empty_like(t) for t in (q1, few, many)]

    def calls():
        pkg.paged_decode_attention(q1, *up, n, workspace=wd, out=outs[0])
        pkg.paged_prefill_attention(few, s_few, *up, n, workspace=wp, out=outs[1])
        pkg.paged_prefill_attention(many, s_many, *up, n, workspace=wp, out=outs[2])
    calls()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            calls()
            calls()
    for turn, (lens, a, b) in enumerate([([5000, 33], [0, 4, 5], [0, 80, 90]), ([70, 5760], [0, 0, 5], [0, 1, 90]), ([0, 1], [0, 2, 3], [0, 45, 46])]):
        qs = [torch.randn(t.shape, generator=g).to(torch.bfloat16) for t in (q1, few, many)]
        for dst, src in zip((q1, few, many, n, s_few, s_many), (*qs, torch.tensor(lens), torch.tensor(a), torch.tensor(b))):
            dst.copy_(src)
        for o in outs:
            o.fill_(7.0)
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        for q, starts, out in zip(qs, ([0, 1, 2], a, b), outs):
            out = out.cpu()
            assert (out[0, starts[2]:] == 7.0).all()
            for i in range(2):
                rows = slice(starts[i], starts[i + 1])
                want, big = ref.attention(q[0, rows], kb[0], vb[0], ks[0], vs[0], table[i], lens[i], causal=q is not qs[0])
                ref.assert_attention(out[0, rows], want, big, (turn, i, starts))
    assert wd.read_status() == 0 and wp.read_status() == 0


def test_pools_strided_over_layers(pkg, cuda_device):
    """Every other layer of a larger pool, keys and values at different strides: appended to and attended; the layers between stay."""
    g = torch.Generator().manual_seed(17)
    h_q, h_kv, d, page, lens = 10, 2, 128, 32, [100, 45]
    kb = torch.full((4, 9, h_kv, page, d), 0x11, dtype=torch.uint8, device=cuda_device)
    vb = torch.full((6, 9, h_kv, page, d), 0x22, dtype=torch.uint8, device=cuda_device)
    ks, vs = (torch.ones(2, 9, h_kv, device=cuda_device) for _ in range(2))
    table = torch.full((2, 700), -1, dtype=torch.int32)
    table[0, :4], table[1, :2] = torch.tensor([8, 1, 5, 0]), torch.tensor([3, 7])
    pools = (kb[::2], vb[::3], ks, vs, table.to(cuda_device))
    q, k, v = (torch.randn(2, sum(lens), h, d, generator=g).to(torch.bfloat16).to(cuda_device) for h in (h_q, h_kv, h_kv))
    starts = torch.tensor([0, 100, 145], dtype=torch.int32, device=cuda_device)
    pos, status = torch.zeros(2, dtype=torch.int32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    pkg.paged_rope_append(None, k, v, None, None, *pools, pos, q_start=starts, status=status)
    assert (kb[1::2] == 0x11).all() and (vb[[1, 2, 4, 5]] == 0x22).all() and status.item() == 0
    shape = pkg.make_paged_shape(h_q, *pools[:3], pools[4])
    n, first = torch.tensor(lens, dtype=torch.int32, device=cuda_device), torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device)
    wp, last = pkg.PagedWorkspace(shape, cuda_device, q_tokens=145), q[:, [99, 144]].contiguous()
    outs = [pkg.paged_decode_attention(last, *pools, n, workspace=pkg.PagedWorkspace(shape, cuda_device, max_seq_len=most)) for most in (100, 22400)]
    outs.append(pkg.paged_prefill_attention(last, first, *pools, n, workspace=wp))
    outs.append(pkg.paged_prefill_attention(q, starts, *pools, n, workspace=wp)[:, [99, 144]])
    for layer in range(2):
        kl, vl, sk, sv = kb[2 * layer].cpu(), vb[3 * layer].cpu(), ks[layer].cpu(), vs[layer].cpu()
        for b, length in enumerate(lens):
            want, big = ref.attention(last[layer, b:b + 1].cpu(), kl, vl, sk, sv, table[b], length)
            for i, out in enumerate(outs):
                ref.assert_attention(out[layer, b:b + 1].cpu(), want, big, (layer, b, i))


def test_python_calls_refuse_wrong_tensors(pkg, cuda_device):
    """Types, shapes, strides and devices that do not fit raise ValueError before anything is launched."""
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=cuda_device)
    bf, i32 = torch.bfloat16, torch.int32
    good = dict(q=z(2, 10, 128, t=bf), k=z(2, 2, 128, t=bf), v=z(2, 2, 128, t=bf), cos=z(64, 64), sin=z(64, 64), k_pages=z(6, 2, 16, 128, t=torch.uint8),
                v_pages=z(6, 2, 16, 128, t=torch.uint8), k_scale=z(6, 2), v_scale=z(6, 2), page_table=z(2, 3, t=i32), seq_pos=z(2, t=i32),
                q_start=torch.tensor([0, 1, 2], dtype=i32, device=cuda_device), status=z(1, t=i32))
    shape = pkg.make_paged_shape(10, good["k_pages"], good["v_pages"], good["k_scale"], good["page_table"])
    wd, wp = pkg.PagedWorkspace(shape, cuda_device), pkg.PagedWorkspace(shape, cuda_device, q_tokens=2)
    cache = ("k_pages", "v_pages", "k_scale", "v_scale", "page_table")

    def append(**kw):
        a = {**good, **kw}
        return pkg.paged_rope_append(a["q"], a["k"], a["v"], a["cos"], a["sin"], *(a[n] for n in cache), a["seq_pos"], q_start=a.get("q_start"),
                                     positions=a.get("positions"), pair_axis=a.get("pair_axis"), q_norm_weight=a.get("wq"), status=a["status"],
                                     q_out=a.get("q_out"), advance=False)

    def decode(**kw):
        a = {**good, **kw}
        return pkg.paged_decode_attention(a["q"], *(a[n] for n in cache), a["seq_pos"], workspace=a.get("ws", wd), out=a.get("out"))

    def prefill(**kw):
        a = {**good, **kw}
        return pkg.paged_prefill_attention(a["q"], a["q_start"], *(a[n] for n in cache), a["seq_pos"], workspace=a.get("ws", wp), out=a.get("out"))
    for call in (append, decode, prefill):
        call()
        for bad in (dict(q=z(2, 10, 128)), dict(q=z(2, 10, 256, t=bf)[..., ::2]), dict(q=z(2, 10, 64, t=bf)), dict(q=good["q"].cpu()), dict(seq_pos=z(3, t=i32)),
                    dict(seq_pos=z(2)), dict(k_scale=z(6, 3)), dict(v_scale=z(5, 2)), dict(k_scale=z(6, 2, t=bf)), dict(page_table=z(6, t=i32)),
                    dict(page_table=z(2, 3)), dict(v_pages=z(7, 2, 16, 128, t=torch.uint8)), dict(v_pages=z(6, 2, 16, 128)),
                    dict(k_pages=z(6, 16, 2, 128, t=torch.uint8).transpose(1, 2)), dict(page_table=good["page_table"].cpu()), dict(q=z(2, 128, t=bf))):
            with pytest.raises(ValueError):
                call(**bad)
        with pytest.raises((TypeError, AttributeError)):
            call(v_pages=None)
    for bad in (dict(k=z(2, 3, 128, t=bf)), dict(v=z(3, 2, 128, t=bf)), dict(k=None), dict(status=None), dict(sin=None), dict(sin=z(63, 64)), dict(cos=z(64)),
                dict(positions=z(3, t=i32)), dict(positions=z(2, 3, t=i32)), dict(pair_axis=z(63, t=i32)), dict(wq=z(127, t=bf)), dict(wq=z(128)),
                dict(q_out=z(2, 9, 128, t=bf)), dict(q_start=z(2, t=i32)), dict(q_start=None, k=z(1, 2, 128, t=bf), v=z(1, 2, 128, t=bf), q=z(1, 10, 128, t=bf))):
        with pytest.raises(ValueError):
            append(**bad)
    for call, other in ((decode, wp), (prefill, wd)):
        for bad in (dict(out=z(2, 9, 128, t=bf)), dict(out=z(2, 10, 128)), dict(ws=other), dict(ws=None)):
            with pytest.raises(ValueError):
                call(**bad)
    with pytest.raises(ValueError):
        prefill(q=z(3, 10, 128, t=bf))                       # more tokens than the workspace is for
    with pytest.raises(ValueError):
        decode(q=z(3, 10, 128, t=bf))
    torch.cuda.synchronize()
    assert good["status"].item() == 0 and wd.read_status() == 0 and wp.read_status() == 0
