"""The paged kernels under the index-checking build, and with guard words round every buffer that they write (stand-ins for a
memory checker)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import paged_ref as ref
from test_paged_values_gpu import FORMS, TWO_TILES, _cache

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CHILD = r'''
import importlib, sys
sys.path.insert(0, "ROOT")
import pytest
assert importlib.import_module("qwen38-5080_b200")._lib.lib().b200attn_bounds_checked() == 1
sys.exit(pytest.main(["-x", "-q", "-m", "gpu", "-p", "no:warnings", "-p", "no:cacheprovider", "-k", "not launched_many_times",
                      *("ROOT/tests/test_paged_%s.py" % n for n in ("gpu", "values_gpu", "ranges_gpu", "slots"))]))
'''.replace("ROOT", str(ROOT))


def test_index_checking_build_stays_silent_over_the_paged_tests(cuda_device):
    """Every paged test reads the status word: a violation anywhere is a status that the test does not expect."""
    res = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, env=dict(os.environ, B200ATTN_BOUNDS="1"), timeout=1200)
    assert res.returncode == 0 and " passed" in res.stdout, res.stdout[-4000:] + res.stderr[-2000:]


class _Guarded:
    """A tensor between two stretches of a pattern."""

    def __init__(self, like, guard=4096):
        self.n, self.guard = like.numel() * like.element_size(), guard
        self.raw = torch.full((self.n + 2 * guard + 256,), 0xA5, dtype=torch.uint8, device=like.device)
        self.t = self.raw[guard:guard + self.n].view(like.dtype).view(like.shape)
        self.t.copy_(like)

    def intact(self):
        return bool((self.raw[:self.guard] == 0xA5).all()) and bool((self.raw[self.guard + self.n:] == 0xA5).all())


def _guard_scratch(ws):
    """The workspace's buffers between guards, initialised as the workspace was."""
    g = {"workspace": _Guarded(ws.buf), "status": _Guarded(ws.status)}
    ws.buf, ws.status = g["workspace"].t, g["status"].t
    return g


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("lens", [[0, 1, 15, 16, 17, 127, 128, 129], [2049, 33]])
def test_guard_words_of_the_attention(pkg, cuda_device, form, lens):
    (h_q, _, d), m, longest = FORMS[form]
    g = torch.Generator().manual_seed(1)
    cache = _cache(g, form, lens)
    up = [t.to(cuda_device) for t in cache]
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    rows = TWO_TILES if form == "two tiles" else len(lens) * (m or 1)
    q = torch.randn(1, rows, h_q, d, generator=g).to(torch.bfloat16).to(cuda_device)
    ws = pkg.PagedWorkspace(pkg.make_paged_shape(h_q, *cache[:3], cache[4]), cuda_device, max_seq_len=longest, q_tokens=m and rows)
    guards = _guard_scratch(ws)
    guards["out"] = _Guarded(torch.full_like(q, 7.0))
    for _ in range(2):
        if m is None:
            pkg.paged_decode_attention(q, *up, n, workspace=ws, out=guards["out"].t)
        else:
            starts = torch.arange(len(lens) + 1, dtype=torch.int32, device=cuda_device) * m
            pkg.paged_prefill_attention(q, starts, *up, n, workspace=ws, out=guards["out"].t)
    torch.cuda.synchronize()
    assert ws.read_status() == 0
    for name, x in guards.items():
        assert x.intact(), f"guard words of the {name} overwritten"


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", [(5, 1, 128), (7, 1, 256), (10, 2, 128)])
@pytest.mark.parametrize("one", [True, False])
def test_guard_words_of_the_append(pkg, cuda_device, heads, page, one):
    """The pool's first and last pages are in use; the table's capacity is used up to its last slot."""
    dev, (h_q, h_kv, d), layers = cuda_device, heads, 2
    g = torch.Generator().manual_seed(2)
    pos, new = ([0, page - 1, 2 * page - 1], [1, 1, 1]) if one else ([0, 5, 2 * page - 7], [2 * page, 1, 7])
    kb, vb, ks, vs = (_Guarded(t.to(dev)) for t in ref.random_cache(g, layers, 6, h_kv, page, d))
    table = torch.tensor([[0, 5], [1, 4], [2, 3]], dtype=torch.int32, device=dev)
    n = sum(new)
    q, k, v = (torch.randn(layers, n, h, d, generator=g).to(torch.bfloat16).to(dev) for h in (h_q, h_kv, h_kv))
    at, status = _Guarded(torch.tensor(pos, dtype=torch.int32, device=dev)), _Guarded(torch.zeros(1, dtype=torch.int32, device=dev))
    out = _Guarded(torch.empty_like(q))
    cos, sin = pkg.rope_tables(2 * page, d // 2, device=dev)
    w = torch.randn(layers, d, generator=g).to(torch.bfloat16).to(dev)
    starts = None if one else torch.tensor([sum(new[:i]) for i in range(4)], dtype=torch.int32, device=dev)
    pkg.paged_rope_append(q, k, v, cos, sin, kb.t, vb.t, ks.t, vs.t, table, at.t, q_start=starts, q_norm_weight=w, k_norm_weight=w, status=status.t, q_out=out.t)
    assert status.t.item() == 0 and at.t.tolist() == [a + m for a, m in zip(pos, new)]
    for name, x in (("keys", kb), ("values", vb), ("key scales", ks), ("value scales", vs), ("positions", at), ("status", status), ("queries", out)):
        assert x.intact(), f"guard words of the {name} overwritten"
