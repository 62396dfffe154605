"""CPU tests of the paged cache: refusals of the C-ABI and of the Python calls, and the page allocator (nothing launches)."""
import ctypes

import pytest
import torch

A = 0x10000   # fake, aligned, never dereferenced: validation fails first


def _shape(pkg, **kw):
    base = dict(n_layers=1, batch=2, h_q=40, h_kv=8, head_dim=128, page_size=64, n_pages=100, max_pages=50,
                k_layer_stride=0, v_layer_stride=0, reserved=0, reserved2=0)
    base.update(kw)
    return pkg._lib.B200AttnPagedShape(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=96), "ERR_SHAPE"), (dict(head_dim=64), "ERR_SHAPE"), (dict(h_q=41), "ERR_SHAPE"), (dict(h_q=72), "ERR_SHAPE"),
    (dict(page_size=8), "ERR_SHAPE"), (dict(page_size=48), "ERR_SHAPE"), (dict(page_size=256), "ERR_SHAPE"), (dict(n_pages=0), "ERR_SHAPE"),
    (dict(max_pages=0), "ERR_SHAPE"), (dict(batch=0), "ERR_SHAPE"), (dict(n_layers=0), "ERR_SHAPE"), (dict(reserved=1), "ERR_SHAPE"),
    (dict(reserved2=1), "ERR_SHAPE"), (dict(n_layers=64, batch=1025), "ERR_SHAPE"), (dict(max_pages=1 << 26), "ERR_SHAPE"),
    (dict(n_pages=1 << 23), "ERR_SHAPE"), (dict(n_layers=2, k_layer_stride=16), "ERR_SHAPE"),
    (dict(k_layer_stride=100 * 8 * 64 * 128 + 8), "ERR_ALIGN"),
])
def test_bad_shapes_are_refused(pkg, kw, code):
    L, lib = pkg._lib, pkg._lib.lib()
    s, n = _shape(pkg, **kw), ctypes.c_size_t(0)
    want = getattr(L, code)
    assert lib.b200attn_paged_workspace_bytes(ctypes.byref(s), 0, 0, ctypes.byref(n)) == want
    assert lib.b200attn_paged_decode(ctypes.byref(s), A, A, A, A, A, A, A, 0, 0, 0.1, A, 1 << 40, A, A, None) == want
    assert lib.b200attn_paged_prefill(ctypes.byref(s), 4, A, A, A, A, A, A, A, A, 0, 1, 0.1, A, 1 << 40, A, A, None) == want
    assert lib.b200attn_paged_rope_append(ctypes.byref(s), None, 2, None, A, A, A, None, None, 1e-6, A, A, A, A, A, A, A, 0, A, None) == want


def test_bad_arguments_launch_nothing(pkg):
    L, lib = pkg._lib, pkg._lib.lib()
    s = ctypes.byref(_shape(pkg))

    def append(rope=None, n=2, qs=None, q=A, k=A, v=A, qo=A, eps=1e-6, kp=A, sc=A, table=A, pos=A, status=A, kw=None):
        return lib.b200attn_paged_rope_append(s, rope, n, qs, q, k, v, None, kw, ctypes.c_float(eps), qo, kp, A, sc, A, table, pos, 1, status, None)
    for bad in (dict(k=None), dict(v=None), dict(kp=None), dict(sc=None), dict(table=None), dict(pos=None), dict(status=None),
                dict(q=None), dict(qo=None)):
        assert append(**bad) == L.ERR_NULL, bad
    for bad in (dict(n=3), dict(n=-1), dict(n=-1, qs=A), dict(eps=-1.0), dict(eps=float("nan"))):
        assert append(**bad) == L.ERR_SHAPE, bad
    for bad in (dict(q=A + 8), dict(k=A + 2), dict(v=A + 8), dict(qo=A + 4), dict(kp=A + 8), dict(kw=A + 8)):
        assert append(**bad) == L.ERR_ALIGN, bad

    def rope(**kw):
        base = dict(cos=A, sin=A, positions=None, pair_axis=None, n_positions=10, n_axes=1, rotary_dim=128, reserved=0)
        base.update(kw)
        return ctypes.byref(L.B200AttnRope(**base))
    for bad in (dict(rotary_dim=0), dict(rotary_dim=8), dict(rotary_dim=24), dict(rotary_dim=144), dict(n_positions=0), dict(n_axes=0),
                dict(n_axes=5, positions=A), dict(n_axes=3), dict(reserved=1)):
        assert append(rope=rope(**bad)) == L.ERR_SHAPE, bad
    assert append(rope=rope(cos=None)) == L.ERR_NULL and append(rope=rope(sin=None)) == L.ERR_NULL
    assert append(rope=rope(cos=A + 4)) == L.ERR_ALIGN

    def decode(q=A, kp=A, ks=A, table=A, lens=A, most=0, ws=A, nbytes=1 << 40, out=A, status=A):
        return lib.b200attn_paged_decode(s, q, kp, A, ks, A, table, lens, 0, most, 0.1, ws, nbytes, out, status, None)
    for bad in ("q", "kp", "ks", "table", "lens", "out", "status"):
        assert decode(**{bad: None}) == L.ERR_NULL, bad
    assert decode(q=A + 8) == L.ERR_ALIGN and decode(ws=A + 8) == L.ERR_ALIGN and decode(most=-1) == L.ERR_CAPACITY

    def prefill(n=4, q=A, qs=A, kp=A, table=A, lens=A, most=0, out=A, status=A):
        return lib.b200attn_paged_prefill(s, n, q, qs, kp, A, A, A, table, lens, most, 1, 0.1, A, 1 << 40, out, status, None)
    for bad in ("q", "qs", "kp", "table", "lens", "out", "status"):
        assert prefill(**{bad: None}) == L.ERR_NULL, bad
    assert prefill(n=-1) == L.ERR_SHAPE and prefill(out=A + 2) == L.ERR_ALIGN and prefill(most=-5) == L.ERR_CAPACITY
    assert prefill(n=0) == L.OK                       # nothing to do, nothing launched


def test_too_small_a_workspace_is_refused(pkg):
    L, lib = pkg._lib, pkg._lib.lib()
    s = _shape(pkg)
    for q_tokens in (0, 64):
        n = ctypes.c_size_t(0)
        assert lib.b200attn_paged_workspace_bytes(ctypes.byref(s), q_tokens, 3000, ctypes.byref(n)) == 0
        if n.value == 0:
            continue
        if q_tokens == 0:
            rc = lib.b200attn_paged_decode(ctypes.byref(s), A, A, A, A, A, A, A, 0, 3000, 0.1, A, n.value - 1, A, A, None)
        else:
            rc = lib.b200attn_paged_prefill(ctypes.byref(s), q_tokens, A, A, A, A, A, A, A, A, 3000, 1, 0.1, A, n.value - 1, A, A, None)
        assert rc == L.ERR_WORKSPACE


def test_python_calls_refuse_what_they_cannot_take(pkg):
    kp = torch.zeros(10, 8, 64, 128, dtype=torch.uint8)
    sc, table, lens = torch.ones(10, 8), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    shape = pkg.make_paged_shape(40, kp, kp, sc, table)
    assert (shape.n_layers, shape.batch, shape.h_kv, shape.page_size, shape.n_pages, shape.max_pages) == (1, 1, 8, 64, 10, 4)
    with pytest.raises(ValueError, match="dense"):
        pkg.make_paged_shape(40, kp.transpose(1, 2), kp.transpose(1, 2), sc, table)
    with pytest.raises(ValueError, match="scales"):
        pkg.make_paged_shape(40, kp, kp, sc[:9], table)
    with pytest.raises(ValueError, match="uint8"):
        pkg.make_paged_shape(40, kp.float(), kp.float(), sc, table)
    q, k = torch.zeros(1, 40, 128, dtype=torch.bfloat16), torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.paged_rope_append(q, k, k, None, None, kp, kp, sc, sc, table, lens, status=lens)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.paged_decode_attention(q, kp, kp, sc, sc, table, lens, workspace=None)


class _Pages:
    """The host side of PagedFP8Cache over CPU tensors."""

    def __new__(cls, pkg, slots=3, n_pages=10, max_pages=6, page=16):
        c = object.__new__(pkg.PagedFP8Cache)
        c.slots, c.n_pages, c.max_pages, c.page_size, c.device = slots, n_pages, max_pages, page, torch.device("cpu")
        c.page_table = torch.full((slots, max_pages), -1, dtype=torch.int32)
        c.seq_pos = torch.zeros(slots, dtype=torch.int32)
        c.host_len, c.pages, c.free = [0] * slots, [[] for _ in range(slots)], list(range(n_pages - 1, -1, -1))
        return c


def test_pages_are_handed_out_once_and_come_back(pkg):
    c = _Pages(pkg)
    c.reserve(0, 17)
    c.reserve(1, 16)
    c.host_len[0] = 17
    c.reserve(0, 20)                                   # 17 cached + 20: three pages in all
    assert [len(p) for p in c.pages] == [3, 1, 0] and len(c.free) == 6
    assert c.page_table[0, :3].tolist() == c.pages[0] and c.page_table[0, 3:].tolist() == [-1] * 3
    assert len(set(c.pages[0] + c.pages[1] + c.free)) == 10
    with pytest.raises(ValueError, match="capacity"):
        c.reserve(2, 16 * 6 + 1)
    c.reserve(2, 16 * 6)
    before = (c.pages[1][:], c.free[:], c.page_table.clone())
    with pytest.raises(ValueError, match="free"):
        c.reserve(1, 17)                               # the pool is empty: refused, nothing changed
    assert (c.pages[1], c.free) == before[:2] and torch.equal(c.page_table, before[2])
    c.seq_pos[0] = 17
    c.release(0)
    assert len(c.free) == 3 and c.host_len[0] == 0 and int(c.seq_pos[0]) == 0 and c.page_table[0].tolist() == [-1] * 6
    c.reserve(1, 33)
    assert len(set(c.pages[1] + c.pages[2] + c.free)) == 10


def test_rope_tables_are_those_of_64_bits(pkg):
    cos, sin = pkg.rope_tables(1 << 17, 64, base=1e6, device="cpu")
    import math
    for pos, j in ((0, 0), (1, 5), (131071, 0), (131071, 31), (99999, 3)):
        a = pos * 1e6 ** (-2 * j / 64)
        assert abs(float(cos[pos, j]) - math.cos(a)) < 1e-7 and abs(float(sin[pos, j]) - math.sin(a)) < 1e-7


def test_softmax_scales_that_are_negative_or_not_finite_are_refused(pkg):
    L, lib = pkg._lib, pkg._lib.lib()
    s = ctypes.byref(_shape(pkg))
    for scale in (-0.1, float("nan"), float("inf"), float("-inf")):
        assert lib.b200attn_paged_decode(s, A, A, A, A, A, A, A, 0, 0, scale, A, 1 << 40, A, A, None) == L.ERR_SHAPE
        assert lib.b200attn_paged_prefill(s, 4, A, A, A, A, A, A, A, A, 0, 1, scale, A, 1 << 40, A, A, None) == L.ERR_SHAPE


def test_workspace_bytes_do_not_depend_on_the_batch_or_the_length(pkg):
    """Calls of different shapes may use a workspace in turn."""
    lib = pkg._lib.lib()

    def size(q_tokens, most, **kw):
        n = ctypes.c_size_t(0)
        assert lib.b200attn_paged_workspace_bytes(ctypes.byref(_shape(pkg, **kw)), q_tokens, most, ctypes.byref(n)) == 0
        return n.value
    for q_tokens in (0, 5):
        assert len({size(q_tokens, most, batch=b) for b in (1, 7, 900) for most in (0, 1, 100000)}) == 1


def test_things_that_are_not_tensors_are_refused(pkg):
    kp = torch.zeros(10, 8, 64, 128, dtype=torch.uint8)
    sc, table, lens = torch.ones(10, 8), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 40, 128, dtype=torch.bfloat16)
    binding = pkg._lib.paged_binding()
    for bad in ((3, kp), (q, "pages"), (q, None)):
        with pytest.raises(TypeError):
            binding.decode(bad[0], bad[1], kp, sc, sc, table, lens, 0, None, 0, None, 0, None, q, 0)
    with pytest.raises(ValueError, match="arguments"):
        binding.decode(q, kp)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.paged_prefill_attention(q, lens, kp, kp, sc, sc, table, lens, workspace=None)
