"""Packed calls whose sequences cannot be what q_start or seq_pos say: skipped, reported, and nothing else touched."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

# q_start of three sequences and 40 tokens (spread over layers below), and which sequences are skipped
RANGES = [([0, 10, 5, 40], [1]), ([-1, 10, 30, 40], [0]), ([0, 10, 30, 41], [2]), ([0, 50, 30, 40], [0, 1]), ([50, 10, 30, 40], [0]), ([0, 10, 30, 1 << 30], [2]),
          ([-(1 << 31), 10, 30, 40], [0])]


@pytest.mark.parametrize("starts,skipped", RANGES)
def test_append_reports_ranges_that_do_not_fit(pkg, cuda_device, starts, skipped):
    dev, page, d = cuda_device, 16, 128
    kp = torch.full((1, 12, 1, page, d), 0x11, dtype=torch.uint8, device=dev)
    vp, ks, vs = kp.clone(), torch.ones(1, 12, 1, device=dev), torch.ones(1, 12, 1, device=dev)
    table = torch.arange(12, dtype=torch.int32, device=dev).view(3, 4)
    pos, status = torch.tensor([3, 4, 5], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.ones(40, 1, d, dtype=torch.bfloat16, device=dev)
    pkg.paged_rope_append(None, x, x, None, None, kp, vp, ks, vs, table, pos, q_start=torch.tensor(starts, dtype=torch.int32, device=dev), status=status)
    assert status.item() == pkg._lib.STATUS_BAD_RANGE
    for b in range(3):
        n = 0 if b in skipped else starts[b + 1] - starts[b]
        assert pos[b].item() == 3 + b + n
        if n == 0:
            assert (kp[0, 4 * b:4 * b + 4] == 0x11).all() and (vp[0, 4 * b:4 * b + 4] == 0x11).all()


@pytest.mark.parametrize("rope", [False, True])
def test_append_reports_negative_positions_of_prompts(pkg, cuda_device, rope):
    dev, page, d = cuda_device, 16, 128
    kp = torch.full((1, 8, 1, page, d), 0x11, dtype=torch.uint8, device=dev)
    vp, ks, vs = kp.clone(), torch.ones(1, 8, 1, device=dev), torch.ones(1, 8, 1, device=dev)
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    cos, sin = pkg.rope_tables(64, d, device=dev) if rope else (None, None)
    x = torch.ones(25, 1, d, dtype=torch.bfloat16, device=dev)
    for pos, n, want in (([-1, 0], [20, 5], 1), ([0, -7], [20, 5], 1), ([-1, 0], [0, 25], 0)):
        at, status = torch.tensor(pos, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
        pkg.paged_rope_append(None, x, x, cos, sin, kp, vp, ks, vs, table, at, q_start=torch.tensor([0, n[0], 25], dtype=torch.int32, device=dev), status=status)
        assert status.item() == want * pkg._lib.STATUS_BAD_POSITION
        assert at.tolist() == [p if p < 0 else p + m for p, m in zip(pos, n)]


@pytest.mark.parametrize("starts,skipped", RANGES)
@pytest.mark.parametrize("heads", [(1, 1, 128), (8, 1, 128), (7, 1, 256)])
def test_prefill_reports_ranges_that_do_not_fit(pkg, cuda_device, heads, starts, skipped):
    """Rows of sequences that are skipped, and of nobody, stay; the others' are right as far as no other sequence claims them."""
    dev, page, (h_q, h_kv, d) = cuda_device, 16, heads
    g = torch.Generator().manual_seed(1)
    kb, vb, ks, vs = ref.random_cache(g, 1, 30, h_kv, page, d)
    lens = [100, 60, 200]
    table = ref.random_table(g, lens, page, 14, 30)
    up = [t.to(dev) for t in (kb, vb, ks, vs, table)]
    q = torch.randn(1, 40, h_q, d, generator=g).to(torch.bfloat16)
    ws = pkg.PagedWorkspace(pkg.make_paged_shape(h_q, kb, vb, ks, table), dev, q_tokens=40)
    out = torch.full_like(q, 7.0).to(dev)
    pkg.paged_prefill_attention(q.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), *up, torch.tensor(lens, dtype=torch.int32, device=dev),
                                workspace=ws, out=out)
    assert ws.read_status() == pkg._lib.STATUS_BAD_RANGE
    out, owners = out[0].cpu(), torch.zeros(40, dtype=torch.int32)
    for b in range(3):
        if b not in skipped:
            owners[starts[b]:starts[b + 1]] += 1
    assert (out[owners == 0] == 7.0).all()
    for b in range(3):
        a, z = starts[b], starts[b + 1]
        if b not in skipped and (owners[a:z] == 1).all():
            want, big = ref.attention(q[0, a:z], kb[0], vb[0], ks[0], vs[0], table[b], lens[b], causal=True)
            ref.assert_attention(out[a:z], want, big, (b, starts))


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("start", [48, 1000, (1 << 31) - 1, (1 << 31) - 8, (1 << 31) - 130])
def test_append_of_prompts_far_beyond_the_table(pkg, cuda_device, start, page):
    """Positions behind the last slot, up to the largest number there is: nothing read or stored for them, the neighbour's tokens are."""
    dev, d, m = cuda_device, 128, 5
    kp = torch.full((1, 8, 1, page, d), 0x11, dtype=torch.uint8, device=dev)
    vp, ks, vs = kp.clone(), torch.ones(1, 8, 1, device=dev), torch.ones(1, 8, 1, device=dev)
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)[:, :3 if page == 16 else 1].contiguous()
    start = max(start, table.shape[1] * page)
    x = torch.randn(2 * m, 1, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    cos, sin = pkg.rope_tables(64, d, device=dev)
    at, status = torch.tensor([3, start], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    q = x.expand(2 * m, 3, d).contiguous()
    pkg.paged_rope_append(q, x, x, cos, sin, kp, vp, ks, vs, table, at, q_start=torch.tensor([0, m, 2 * m], dtype=torch.int32, device=dev), status=status)
    off_the_tables = pkg._lib.STATUS_BAD_POSITION if start + m > 64 else 0
    assert status.item() == pkg._lib.STATUS_POS_AT_CAPACITY | off_the_tables and at.tolist() == [3 + m, start]
    assert (kp[0, 1:] == 0x11).all() and (vp[0, 1:] == 0x11).all()
    got = ref.values(vp[0, 0, 0, 3:3 + m].cpu()) * vs[0, 0, 0].item()
    assert ((got - x[:m, 0].cpu().double()).abs() <= x[:m, 0].cpu().double().abs() * 2.0 ** -4 + vs[0, 0, 0].item() * 2.0 ** -10).all()


@pytest.mark.parametrize("longest", [1, None])
def test_decode_lengths_beyond_31_bits(pkg, cuda_device, longest):
    """A length and an offset whose sum passes 2^31: over the capacity (all of it attended), not negative."""
    g = torch.Generator().manual_seed(2)
    kb, vb, ks, vs = ref.random_cache(g, 1, 8, 1, 16, 128)
    table = torch.randint(0, 8, (2, 9000), generator=g).to(torch.int32)
    q = torch.randn(1, 2, 5, 128, generator=g).to(torch.bfloat16)
    table[0], table[1] = table[0, 0], table[1, 0]           # every page the same: 144,000 slots like 16
    up = [t.to(cuda_device) for t in (kb, vb, ks, vs, table)]
    ws = pkg.PagedWorkspace(pkg.make_paged_shape(5, kb, vb, ks, table), cuda_device, max_seq_len=longest)
    n = torch.tensor([(1 << 31) - 3, 30 - (1 << 30)], dtype=torch.int32, device=cuda_device)
    out = pkg.paged_decode_attention(q.to(cuda_device), *up, n, workspace=ws, seq_len_offset=1 << 30).cpu()
    assert ws.read_status() == pkg._lib.STATUS_LEN_OVER_CAP
    for b, length in enumerate([16, 30]):
        want, big = ref.attention(q[0, b:b + 1], kb[0], vb[0], ks[0], vs[0], table[b], length)
        ref.assert_attention(out[0, b:b + 1], want, big, b)


def test_calls_refuse_tensors_whose_layers_are_not_first(pkg, cuda_device):
    """[n_tokens, n_layers, ..] has the right number of elements, and its rows would be read as other tokens' and layers'."""
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=cuda_device)  # noqa: E731
    layers, n, h_q, h_kv, d = 3, 2, 5, 1, 128
    cache = (z(layers, 4, h_kv, 16, d, t=torch.uint8), z(layers, 4, h_kv, 16, d, t=torch.uint8), z(layers, 4, h_kv, t=torch.float32),
             z(layers, 4, h_kv, t=torch.float32), torch.arange(4, dtype=torch.int32, device=cuda_device).view(n, 2))
    pos, status, starts = z(n, t=torch.int32), z(1, t=torch.int32), torch.arange(n + 1, dtype=torch.int32, device=cuda_device)
    shape = pkg.make_paged_shape(h_q, *cache[:3], cache[4])
    wd, wp = pkg.PagedWorkspace(shape, cuda_device), pkg.PagedWorkspace(shape, cuda_device, q_tokens=n)
    good, bad = (layers, n), (n, layers)

    def append(q=good, k=good, v=good, out=good):
        pkg.paged_rope_append(z(*q, h_q, d), z(*k, h_kv, d), z(*v, h_kv, d), None, None, *cache, pos, advance=False, status=status, q_out=z(*out, h_q, d))

    def decode(q=good, out=good):
        pkg.paged_decode_attention(z(*q, h_q, d), *cache, pos, workspace=wd, out=z(*out, h_q, d))

    def prefill(q=good, out=good):
        pkg.paged_prefill_attention(z(*q, h_q, d), starts, *cache, pos, workspace=wp, out=z(*out, h_q, d))
    for call, names in ((append, ("q", "k", "v", "out")), (decode, ("q", "out")), (prefill, ("q", "out"))):
        call()
        for name in names:
            with pytest.raises(ValueError):
                call(**{name: bad})
    torch.cuda.synchronize()
    assert status.item() == 0 and wd.read_status() == 0 and wp.read_status() == 0
