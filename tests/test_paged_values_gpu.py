"""GPU tests of the paged operators on values at the edges of their types: all of them zero, far apart, loud, quiet, NaN.  Every
attention kernel is reached (FORMS), and compared with the 64-bit form of paged_ref.py."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

# name: heads, query tokens of each sequence (None: decode), longest sequence that the host names
FORMS = {
    "one token, short": ((5, 1, 128), None, 1), "one token, short, heads of 256": ((7, 1, 256), None, 1),
    "one token, long": ((5, 1, 128), None, None), "one token, long, heads of 256": ((7, 1, 256), None, None),
    "few rows": ((5, 1, 128), 2, None), "few rows, heads of 256": ((7, 1, 256), 2, None),
    "a tile": ((5, 1, 128), 20, None), "two tiles": ((64, 8, 128), 32, None), "tiles, heads of 256": ((7, 1, 256), 30, None),
}
PAGE = 16
TWO_TILES = 640   # rows of a call, those of nobody among them, that make the tile kernel's thread blocks take two tiles each


def _cache(g, form, lens):
    """Random pools, scales and table for sequences of these lengths, in a table wide enough for the kernel that streams long caches."""
    (_, h_kv, d), m, _ = FORMS[form]
    need = sum(-(-n // PAGE) for n in lens)
    spare = max(1100 * 128 // d, 133000 * 128 // (d * len(lens) * h_kv)) // PAGE + 2 if m is None else 1
    kb, vb, ks, vs = ref.random_cache(g, 1, need + 1, h_kv, PAGE, d)
    table = ref.random_table(g, lens, PAGE, max(-(-n // PAGE) for n in lens) + spare, need + 1)
    return kb, vb, ks, vs, table


def _queries(g, form, lens):
    (h_q, _, d), m, _ = FORMS[form]
    return torch.randn(1, len(lens) * (m or 1), h_q, d, generator=g).to(torch.bfloat16)


def _attend(pkg, dev, form, cache, lens, q, causal=False):
    """The call of a form; a list with every sequence's rows."""
    (h_q, _, _), m, longest = FORMS[form]
    up = [t.to(dev) for t in cache]
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    rows = q.shape[1]
    if form == "two tiles":
        q = torch.cat([q, torch.zeros(1, max(0, TWO_TILES - rows), *q.shape[2:], dtype=q.dtype)], 1)
    shape = pkg.make_paged_shape(h_q, *cache[:3], cache[4])
    ws = pkg.PagedWorkspace(shape, dev, max_seq_len=longest, q_tokens=m and q.shape[1])
    if m is None:
        out = pkg.paged_decode_attention(q.to(dev), *up, n, workspace=ws)
    else:
        starts = torch.arange(len(lens) + 1, dtype=torch.int32, device=dev) * m
        out = pkg.paged_prefill_attention(q.to(dev), starts, *up, n, workspace=ws, causal=causal)
    torch.cuda.synchronize()
    assert ws.read_status() == 0
    return list(out[0, :rows].cpu().split(m or 1))


def _want(form, cache, b, length, q, causal=False):
    kb, vb, ks, vs, table = cache
    m = FORMS[form][1] or 1
    return ref.attention(q[0, b * m:(b + 1) * m], kb[0], vb[0], ks[0], vs[0], table[b], length, causal=causal and FORMS[form][1] is not None)


def _compare(form, cache, lens, q, got, causal=False, slack=0.0):
    for b, n in enumerate(lens):
        want, big = _want(form, cache, b, n, q, causal)
        ref.assert_attention(got[b], want, big + slack * 2.0 ** 10, (form, b))


@pytest.mark.parametrize("form", FORMS)
def test_values_that_are_all_zero(pkg, cuda_device, form):
    """Zero values as the append stores them, with the smallest scale there is: zeros, not NaN."""
    g = torch.Generator().manual_seed(1)
    lens = [300, 40, 129]
    cache = _cache(g, form, lens)
    (_, h_kv, d), _, _ = FORMS[form]
    up = [t.to(cuda_device) for t in cache]
    k = torch.randn(1, sum(lens), h_kv, d, generator=g).to(torch.bfloat16).to(cuda_device)
    starts = torch.tensor([0, 300, 340, 469], dtype=torch.int32, device=cuda_device)
    pos, status = torch.zeros(3, dtype=torch.int32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    pkg.paged_rope_append(None, k, torch.zeros_like(k), None, None, *up, pos, q_start=starts, status=status)
    assert status.item() == 0 and pos.tolist() == lens
    for rows in _attend(pkg, cuda_device, form, [t.cpu() for t in up], lens, _queries(g, form, lens), causal=True):
        assert (rows == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_values_that_are_zero_in_one_piece_of_the_keys(pkg, cuda_device, form):
    """A long sequence, cut into pieces of 512 keys by the tile kernels: the values of the second 512 are zero."""
    g = torch.Generator().manual_seed(2)
    cache = _cache(g, form, [2000])
    ids = cache[4][0, 512 // PAGE:1024 // PAGE].long()
    cache[1][:, ids], cache[3][:, ids] = 0, 2.0 ** -126
    q = _queries(g, form, [2000])
    _compare(form, cache, [2000], q, _attend(pkg, cuda_device, form, cache, [2000], q))


@pytest.mark.parametrize("form", FORMS)
def test_rows_that_see_nothing_beside_loud_values(pkg, cuda_device, form):
    """Fewer cached tokens than queries: the first rows of a tile see nothing, the others values of 10^8."""
    g = torch.Generator().manual_seed(3)
    m = FORMS[form][1] or 1
    lens = [max(1, m - 7 + b) for b in range(8)]
    cache = _cache(g, form, lens)
    cache[3].mul_(2.0 ** 33)
    q = _queries(g, form, lens)
    got = _attend(pkg, cuda_device, form, cache, lens, q, causal=True)
    _compare(form, cache, lens, q, got, causal=True)
    for rows, n in zip(got, lens):
        assert (rows[:max(0, m - n)] == 0).all()


def _far_key(cache, b, index, jump, d):
    """Key `index` of sequence b gets a score of about `jump` with queries near 1; the rest of its page scores 0."""
    kb, _, ks, _, table = cache
    page, row = int(table[b, index // PAGE]), index % PAGE
    kb[0, page], ks[0, page] = 0, 0.125
    byte = torch.tensor(jump / d ** 0.5 / 0.125).to(torch.float8_e4m3fn).view(torch.uint8)
    kb[0, page, :, row] = byte


@pytest.mark.parametrize("jump", [60.0, 100.0, 200.0, 400.0])
@pytest.mark.parametrize("form", FORMS)
def test_a_key_far_above_the_rest(pkg, cuda_device, form, jump):
    """One key of the second 128 scores far above all others: at each of 16 neighbouring places, a sequence each."""
    g = torch.Generator().manual_seed(4)
    lens = [300 + b for b in range(16)]
    cache = _cache(g, form, lens)
    for b in range(16):
        _far_key(cache, b, 192 + b, jump, FORMS[form][0][2])
    q = (1 + 0.1 * _queries(g, form, lens).float()).to(torch.bfloat16)
    _compare(form, cache, lens, q, _attend(pkg, cuda_device, form, cache, lens, q))


@pytest.mark.parametrize("form", FORMS)
def test_scores_that_grow_along_the_sequence(pkg, cuda_device, form):
    """Keys that get louder with every page: the running reference of every row moves many times."""
    g = torch.Generator().manual_seed(5)
    lens = [900, 333]
    cache = _cache(g, form, lens)
    for b, n in enumerate(lens):
        for i in range(-(-n // PAGE)):
            cache[2][:, cache[4][b, i]] = 2.0 ** (-9 + 8 * i * PAGE // 900)
    q = _queries(g, form, lens)
    for causal in (False, True):
        _compare(form, cache, lens, q, _attend(pkg, cuda_device, form, cache, lens, q, causal), causal)


@pytest.mark.parametrize("form", FORMS)
def test_a_key_that_is_nan(pkg, cuda_device, form):
    """A NaN in a key that is seen makes the row NaN, wherever it stands; one that is hidden does nothing."""
    g = torch.Generator().manual_seed(6)
    lens = [300] * 16
    cache = _cache(g, form, lens)
    for b in range(16):
        cache[0][0, cache[4][b, 12], :, b, 5] = 0x7F
    for rows in _attend(pkg, cuda_device, form, cache, lens, _queries(g, form, lens)):
        assert torch.isnan(rows).all()
    if FORMS[form][1] is None:
        return
    cache, m = _cache(g, form, lens), FORMS[form][1]
    q = _queries(g, form, lens)
    clean = _attend(pkg, cuda_device, form, cache, lens, q, causal=True)
    for b in range(16):
        cache[0][0, cache[4][b, 299 // PAGE], :, 299 % PAGE, b] = 0xFF
    for rows, before in zip(_attend(pkg, cuda_device, form, cache, lens, q, causal=True), clean):
        assert torch.equal(rows[:m - 1], before[:m - 1]) and torch.isnan(rows[m - 1]).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lens", [[300, 40], [2000, 1]])
def test_a_query_that_is_nan(pkg, cuda_device, form, lens):
    """A row whose query has a NaN is NaN; its neighbours are what they are without it."""
    g = torch.Generator().manual_seed(7)
    cache = _cache(g, form, lens)
    q = _queries(g, form, lens)
    row = min(3, (FORMS[form][1] or 1) - 1)
    q[0, row, 2, 17] = float("nan")
    got = _attend(pkg, cuda_device, form, cache, lens, q)
    assert torch.isnan(got[0][row, 2]).all()
    got[0][row, 2], q[0, row, 2] = 0, 0
    want, big = _want(form, cache, 0, lens[0], q)
    want[row, 2] = 0
    ref.assert_attention(got[0], want, big, form)
    want, big = _want(form, cache, 1, lens[1], q)
    ref.assert_attention(got[1], want, big, form)


@pytest.mark.parametrize("exponent", [-149, -140, -127, -126, -118, -110])
@pytest.mark.parametrize("form", FORMS)
def test_quiet_values(pkg, cuda_device, form, exponent):
    """V scales down to the smallest positive number.  Results may be subnormal bf16: half a step of those is 2^-134."""
    g = torch.Generator().manual_seed(8)
    lens = [300, 40]
    cache = _cache(g, form, lens)
    cache[3].fill_(2.0 ** exponent)
    q = _queries(g, form, lens)
    _compare(form, cache, lens, q, _attend(pkg, cuda_device, form, cache, lens, q), slack=2.0 ** -134)


@pytest.mark.parametrize("lens", [[300, 40], [2000, 1]])
@pytest.mark.parametrize("form", FORMS)
def test_loud_values(pkg, cuda_device, form, lens):
    """Values up to 2^119, near the largest bf16: the weighted sums stay within fp32."""
    g = torch.Generator().manual_seed(9)
    cache = _cache(g, form, lens)
    cache[3].fill_(2.0 ** 112)
    q = _queries(g, form, lens)
    _compare(form, cache, lens, q, _attend(pkg, cuda_device, form, cache, lens, q))


@pytest.mark.parametrize("exponent", [-149, -127])
@pytest.mark.parametrize("form", FORMS)
def test_quiet_keys(pkg, cuda_device, form, exponent):
    """K scales down to the smallest positive number: every visible key weighs the same."""
    g = torch.Generator().manual_seed(10)
    lens = [300, 40]
    cache = _cache(g, form, lens)
    cache[2].fill_(2.0 ** exponent)
    q = _queries(g, form, lens)
    _compare(form, cache, lens, q, _attend(pkg, cuda_device, form, cache, lens, q))


@pytest.mark.parametrize("below", [10, 20, 30, 45])
@pytest.mark.parametrize("form", FORMS)
def test_quiet_values_beside_loud_ones(pkg, cuda_device, form, below):
    """All the weight lies on a key whose page's V scale is 2^-below of the others': it is held to 2^-31 of the largest scale."""
    g = torch.Generator().manual_seed(11)
    lens = [300, 290]
    cache = _cache(g, form, lens)
    cache[3].fill_(1.0)
    for b in range(2):
        _far_key(cache, b, 100 + b, 150.0, FORMS[form][0][2])
        cache[3][0, cache[4][b, 100 // PAGE]] = 2.0 ** -below
    q = (1 + 0.1 * _queries(g, form, lens).float()).to(torch.bfloat16)
    for b, (rows, n) in enumerate(zip(_attend(pkg, cuda_device, form, cache, lens, q), lens)):
        want, _ = _want(form, cache, b, n, q)
        off = (rows.double() - want).abs()
        # bf16: half a step 2^-9 of the value; p of the one key that counts in f16: 2^-12 of it
        assert (off <= want.abs() * (2.0 ** -9 + 2.0 ** -11) + 2.0 ** -30).all(), (b, float(off.max()))
