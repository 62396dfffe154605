"""Slots of the paged cache that come and go: idle ones, steps captured and replayed, pages handed out in between."""
import pytest
import torch

import paged_ref as ref


@pytest.mark.gpu
def test_append_leaves_idle_sequences_alone(pkg, cuda_device):
    """Position 0 and no page (-1): nothing stored, advanced or reported.  Any other missing page is reported, and stays too."""
    L, dev, h_q, h_kv, d, page = pkg._lib, cuda_device, 5, 1, 128, 16

    def call(pos, table, n_each=None):
        kp = torch.full((2, 4, h_kv, page, d), 0x11, dtype=torch.uint8, device=dev)
        vp, ks, vs = kp.clone(), torch.ones(2, 4, h_kv, device=dev), torch.ones(2, 4, h_kv, device=dev)
        status, seq_pos = torch.zeros(1, dtype=torch.int32, device=dev), torch.tensor(pos, dtype=torch.int32, device=dev)
        n = len(pos) if n_each is None else sum(n_each)
        x = torch.ones(2, n, h_kv, d, dtype=torch.bfloat16, device=dev)
        starts = None if n_each is None else torch.tensor([sum(n_each[:i]) for i in range(len(pos) + 1)], dtype=torch.int32, device=dev)
        cos, sin = pkg.rope_tables(64, d, device=dev)
        pkg.paged_rope_append(x.expand(2, n, h_q, d).contiguous(), x, x, cos, sin, kp, vp, ks, vs, torch.tensor(table, dtype=torch.int32, device=dev),
                              seq_pos, q_start=starts, status=status)
        return status.item(), seq_pos.tolist(), kp.cpu(), vp.cpu()

    st, pos, kp, vp = call([0, 3, 0], [[-1, -1], [2, 3], [-1, -1]])
    assert st == 0 and pos == [0, 4, 0]
    for pool in (kp, vp):
        assert (pool[:, [0, 1, 3]] == 0x11).all() and (pool[:, 2, :, :3] == 0x11).all() and (pool[:, 2, :, 3] != 0x11).all()
    for at, table in ((0, [[-2, -1], [2, 3]]), (0, [[4, -1], [2, 3]]), (16, [[0, -1], [2, 3]]), (16, [[0, 9], [2, 3]])):
        st, pos, kp, vp = call([at, 3], table)
        assert st == L.STATUS_BAD_PAGE and pos == [at, 4] and (kp[:, [0, 1, 3]] == 0x11).all()
    # packed: a page missing in the middle
    st, pos, kp, vp = call([10, 3], [[0, -1, 1], [2, 3, -1]], [30, 1])
    assert st == L.STATUS_BAD_PAGE and pos == [10, 4]
    st, pos, kp, vp = call([0, 3], [[-1], [2]], [0, 2])
    assert st == 0 and pos == [0, 5]


def _mk(g, layers, n, h, d):
    return torch.randn(layers, n, h, d, generator=g).to(torch.bfloat16)


def _check(c, q, out, lens_now, rows_of):
    """out against 64-bit attention over the cache as it is on the device, of sequences of these lengths."""
    pools = [t.cpu() for t in (c.k_pages, c.v_pages, c.k_scale, c.v_scale)]
    table = c.page_table.cpu()
    for b, (a, z) in enumerate(rows_of):
        for layer in range(c.n_layers):
            want, big = ref.attention(q[layer, a:z], *(p[layer] for p in pools), table[b], lens_now[b], causal=True)
            ref.assert_attention(out[layer, a:z].cpu(), want, big, (b, layer))


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_steps_with_a_released_slot_and_its_next_sequence(pkg, cuda_device, captured):
    dev, layers, slots, h_q, h_kv, d, page = cuda_device, 2, 3, 10, 2, 128, 16
    c = pkg.PagedFP8Cache(layers, slots, h_q, h_kv, d, n_pages=30, max_pages=12, page_size=page, device=dev, max_prompt_tokens=150)
    g = torch.Generator().manual_seed(0)

    def prompt(lens):
        q, k, v = _mk(g, layers, sum(lens), h_q, d), _mk(g, layers, sum(lens), h_kv, d), _mk(g, layers, sum(lens), h_kv, d)
        out = c.prefill(q.to(dev), k.to(dev), v.to(dev), None, None, lens)
        at = [sum(lens[:i]) for i in range(slots + 1)]
        _check(c, q, out, c.host_len, [(at[b], at[b + 1]) for b in range(slots)])

    prompt([50, 7, 90])
    for b in range(slots):
        c.reserve(b, 20)
    buf = [_mk(g, layers, slots, h, d).to(dev) for h in (h_q, h_kv, h_kv)]
    out = torch.empty_like(buf[0])
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph):
            c.step(*buf, None, None, out=out, count=False)
    c.release(1)
    want = [50, 0, 90]
    for turn in range(10):
        q = _mk(g, layers, slots, h_q, d)
        buf[0].copy_(q)
        for t in buf[1:]:
            t.copy_(_mk(g, layers, slots, h_kv, d))
        if captured:
            graph.replay()
        else:
            c.step(*buf, None, None, out=out)
        want = [want[0] + 1, 0, want[2] + 1]
        assert c.seq_pos.tolist() == want and c.read_status() == 0
        assert (out[:, 1] == 0).all()
        _check(c, q, out, want, [(b, b + 1) for b in range(slots)])
    if captured:
        c.host_len = list(want)
    assert c.host_len == want
    prompt([0, 60, 3])                                     # another sequence in the released slot
    assert c.seq_pos.tolist() == [60, 60, 103] and c.read_status() == 0


@pytest.mark.gpu
def test_pages_reserved_between_replays(pkg, cuda_device):
    """Capture counts nothing; replays are counted by `replayed`, so that `reserve` hands out the pages that the next ones need."""
    dev, layers, slots, h_q, h_kv, d, page = cuda_device, 1, 2, 5, 1, 128, 16
    c = pkg.PagedFP8Cache(layers, slots, h_q, h_kv, d, n_pages=20, max_pages=10, page_size=page, device=dev, max_prompt_tokens=64)
    g = torch.Generator().manual_seed(1)
    c.prefill(*(_mk(g, layers, 40, h, d).to(dev) for h in (h_q, h_kv, h_kv)), None, None, [30, 10])
    c.reserve(0, 2)
    c.reserve(1, 6)
    buf = [_mk(g, layers, slots, h, d).to(dev) for h in (h_q, h_kv, h_kv)]
    out, graph = torch.empty_like(buf[0]), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step(*buf, None, None, out=out)
    assert c.host_len == [30, 10] and [len(p) for p in c.pages] == [2, 1]
    want, q = [30, 10], None
    for turn in range(40):
        if turn in (2, 10, 25):                            # slot 0 is full after 2 more tokens
            with pytest.raises(ValueError, match="slot"):
                c.replayed(17)
            for b in range(slots):
                c.reserve(b, 17)
        c.replayed()
        q = _mk(g, layers, slots, h_q, d)
        for t, x in zip(buf, (q, _mk(g, layers, slots, h_kv, d), _mk(g, layers, slots, h_kv, d))):
            t.copy_(x)
        graph.replay()
        want = [x + 1 for x in want]
        assert c.seq_pos.tolist() == want == c.host_len and c.read_status() == 0
    _check(c, q, out, want, [(0, 1), (1, 2)])


def _host_side(pkg):
    """PagedFP8Cache without a device: what it keeps on the host, over CPU tensors."""
    c = object.__new__(pkg.PagedFP8Cache)
    c.slots, c.n_pages, c.max_pages, c.page_size, c.device = 3, 10, 6, 16, torch.device("cpu")
    c.page_table, c.seq_pos = torch.full((3, 6), -1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    c.host_len, c.pages, c.free = [0] * 3, [[] for _ in range(3)], list(range(9, -1, -1))
    return c


def test_replays_are_counted_against_the_reserved_pages(pkg):
    c = _host_side(pkg)
    c.reserve(0, 20)
    c.host_len[0] = 20
    c.reserve(2, 5)
    c.replayed(12)                                         # 32 tokens of 32; slot 1 is idle, slot 2 holds 12 of 16
    assert c.host_len == [32, 0, 12]
    with pytest.raises(ValueError, match="slot 0"):
        c.replayed()
    assert c.host_len == [32, 0, 12]
    c.reserve(0, 1)
    c.replayed(4)
    assert c.host_len == [36, 0, 16] and len(c.pages[0]) == 3
    with pytest.raises(ValueError, match="slot 2"):
        c.replayed()
    c.release(2)
    c.replayed()
    assert c.host_len == [37, 0, 0]


def test_a_refused_prompt_changes_nothing(pkg):
    """Lengths that are negative, and a call that the append refuses (here: the cache is on the CPU): no page stays handed out."""
    c = _host_side(pkg)
    c.workspace = c.prompt_workspace = type("Scratch", (), {"q_tokens": 100, "status": torch.zeros(1, dtype=torch.int32)})()
    c.k_pages = c.v_pages = torch.zeros(1, 10, 1, 16, 128, dtype=torch.uint8)
    c.k_scale = c.v_scale = torch.ones(1, 10, 1)
    c.reserve(0, 20)
    c.host_len[0] = 20
    before = ([list(p) for p in c.pages], list(c.free), c.page_table.clone(), list(c.host_len))
    q, k = torch.zeros(1, 30, 5, 128, dtype=torch.bfloat16), torch.zeros(1, 30, 1, 128, dtype=torch.bfloat16)
    for lens, what in (([40, -10, 0], "share"), ([20, 10, 0], "CUDA"), ([0, 0, 30], "CUDA")):
        with pytest.raises(ValueError, match=what):
            c.prefill(q, k, k, None, None, lens)
        assert (c.pages, c.free, c.host_len) == (before[0], before[1], before[3]) and torch.equal(c.page_table, before[2])
