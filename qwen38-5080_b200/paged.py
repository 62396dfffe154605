"""The FP8 cache in pages: append with rotary positions on the way, attention of one or of many query tokens, and the
container that hands out pages.

The reference keeps one capacity-sized block per sequence (runner/model/static_cache.py:135-158); a batch of sequences of
very different lengths wants pages instead, and a prompt wants to be appended and attended without a bf16 copy of the
cache.  torch only owns memory and streams here; all arithmetic runs in libb200attn.so.

Layouts (n_layers may be dropped for a single layer):
    k_pages, v_pages uint8 / float8_e4m3fn [n_layers, n_pages, h_kv, page_size, head_dim], page_size 16, 32, 64 or 128
    k_scale, v_scale fp32  [n_layers, n_pages, h_kv]                a value is byte * scale
    page_table       int32 [batch, max_pages] on the device
    q, out           bf16  [n_layers, n_tokens, h_q, head_dim]       decode: n_tokens = batch
    k, v             bf16  [n_layers, n_tokens, h_kv, head_dim]
    q_start          int32 [batch + 1] on the device: sequence b owns tokens [q_start[b], q_start[b + 1])
    seq_len, seq_pos int32 [batch] on the device
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import B200AttnPagedShape, check

_BYTE_TYPES = (torch.uint8, torch.float8_e4m3fn)


def _call(k_pages, fn, *args) -> int:
    """fn(*args, stream) on the cache's device, which is made current for the call if it is not, and its current stream."""
    idx = k_pages.get_device()
    if idx < 0:
        raise ValueError("the cache must be on a CUDA device: there is no CPU path")
    if torch._C._cuda_getDevice() == idx:
        return fn(*args, torch._C._cuda_getCurrentRawStream(idx))
    with torch.cuda.device(idx):
        return fn(*args, torch._C._cuda_getCurrentRawStream(idx))


def make_paged_shape(h_q: int, k_pages, v_pages, k_scale, page_table) -> B200AttnPagedShape:
    """Geometry from the cache handles.  A 5-d pool may be strided over layers (dim 0) only."""
    dims = k_pages.shape
    if v_pages.shape != dims or len(dims) not in (4, 5):
        raise ValueError("k_pages and v_pages must have the same shape [n_layers, n_pages, h_kv, page_size, head_dim]")
    n = 1 if len(dims) == 4 else dims[0]
    n_pages, h_kv, page, d = dims[-4:]
    if k_pages.dtype not in _BYTE_TYPES or v_pages.dtype not in _BYTE_TYPES:
        raise ValueError("the cache must be uint8 / float8_e4m3fn")
    k_stride, v_stride, dense = k_pages.stride(), v_pages.stride(), (h_kv * page * d, page * d, d, 1)
    if k_stride[-4:] != dense or v_stride[-4:] != dense:
        raise ValueError("the cache must be dense within a layer")
    if k_scale.numel() != n * n_pages * h_kv:
        raise ValueError("scales must be [n_layers, n_pages, h_kv]")
    table = page_table.shape
    if len(table) != 2:
        raise ValueError("page_table must be [batch, max_pages]")
    return B200AttnPagedShape(n, table[0], h_q, h_kv, d, page, n_pages, table[1], k_stride[0] if n > 1 else 0, v_stride[0] if n > 1 else 0, 0, 0)


class PagedWorkspace:
    """Scratch of the attention calls, allocated once (before any graph capture): for decode, or with `q_tokens` for prefill
    calls of up to that many query tokens; calls of different shapes may use it in turn.  `max_seq_len`: an upper bound of the
    lengths (default: the table's capacity); it decides how the work is split.  Launches that may overlap on the device need workspaces of their own."""

    def __init__(self, shape: B200AttnPagedShape, device, *, max_seq_len: int | None = None, q_tokens: int | None = None):
        self.max_seq_len = int(max_seq_len or 0)
        self.q_tokens = int(q_tokens or 0)
        out = ctypes.c_size_t(0)
        with torch.cuda.device(device):
            check(_lib.lib().b200attn_paged_workspace_bytes(ctypes.byref(shape), self.q_tokens, self.max_seq_len, ctypes.byref(out)),
                  "b200attn_paged_workspace_bytes")
            self.nbytes = max(256, out.value)
            self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
            self.status = torch.zeros(1, dtype=torch.int32, device=device)
            check(_lib.lib().b200attn_workspace_init(self.buf.data_ptr(), self.nbytes, torch.cuda.current_stream().cuda_stream),
                  "b200attn_workspace_init")

    def read_status(self) -> int:
        """Device status bits (synchronises; not for use inside a captured step)."""
        return int(self.status.item())


def _scratch(w: PagedWorkspace | None):
    return (w.buf, w.nbytes, w.status, w.max_seq_len) if w is not None else (None, 0, None, 0)


def paged_rope_append(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, page_table, seq_pos, *, q_start=None,
                      positions=None, pair_axis=None, q_norm_weight=None, k_norm_weight=None, eps: float = 1e-6,
                      advance: bool = True, status: torch.Tensor, q_out: torch.Tensor | None = None):
    """Rotate queries and keys and quantise-and-append keys and values to the pages, all layers in one call; returns the rotated
    queries (None if `q` is None).

    Without `q_start`: one token per sequence.  `cos`, `sin`: fp32 tables [n_positions, rotary_dim / 2] (None: no rotation);
    a token's row is its slot in the sequence, or `positions` int32 [n_tokens] or [n_axes, n_tokens] with `pair_axis` int32
    [rotary_dim / 2] saying which axis turns which pair.  Norm weights bf16 [n_layers, head_dim]: RMS norm with weight 1 + w
    before the rotation.  `seq_pos`: tokens cached before the call, advanced afterwards if `advance` (a sequence whose tokens did not
    all find a page stays).  Capacity, bad pages and bad positions are reported in `status`.  Without `q_start`, a sequence at
    position 0 whose first page is -1 is idle: nothing is stored, advanced or reported."""
    if q is not None and q_out is None:
        q_out = torch.empty_like(q)
    rc = _call(k_pages, _lib.paged_binding().append, q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, page_table, seq_pos, q_start,
               positions, pair_axis, q_norm_weight, k_norm_weight, eps, advance, status, q_out)
    check(rc, "b200attn_paged_rope_append")
    return q_out if q is not None else None


def paged_decode_attention(q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, *, workspace: PagedWorkspace,
                           softmax_scale: float | None = None, seq_len_offset: int = 0, out: torch.Tensor | None = None):
    """Attention of one query token per sequence (q bf16 [n_layers, batch, h_q, head_dim]) over the first
    seq_len[b] + seq_len_offset tokens of its pages; bf16 with q's shape.  A sequence without tokens gives zeros."""
    if out is None:
        out = torch.empty_like(q)
    if workspace is not None and workspace.q_tokens:
        raise ValueError("the workspace must be one for decode, on the cache's device")
    rc = _call(k_pages, _lib.paged_binding().decode, q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, seq_len_offset,
               *_scratch(workspace), softmax_scale, out)
    check(rc, "b200attn_paged_decode")
    return out


def paged_prefill_attention(q, q_start, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, *, workspace: PagedWorkspace,
                            causal: bool = True, softmax_scale: float | None = None, out: torch.Tensor | None = None):
    """Attention of many query tokens per sequence (q bf16 [n_layers, n_tokens, h_q, head_dim], packed by `q_start`) over the
    first seq_len[b] tokens of its pages.  causal: a sequence's queries are its last tokens, each sees those up to itself;
    not causal: all (cross attention).  Rows that see nothing are zero; rows behind q_start[batch] are left as they were."""
    if out is None:
        out = torch.empty_like(q)
    rc = _call(k_pages, _lib.paged_binding().prefill, q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, q_start,
               workspace.q_tokens if workspace is not None else 0, causal, *_scratch(workspace), softmax_scale, out)
    check(rc, "b200attn_paged_prefill")
    return out


def rope_tables(n_positions: int, rotary_dim: int, base: float = 10000.0, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin fp32 [n_positions, rotary_dim / 2] of the angles pos * base^(-2 j / rotary_dim), computed in 64 bits."""
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / max(rotary_dim, 1))
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


class PagedFP8Cache:
    """A pool of pages for `slots` sequences, all layers: storage, page table, positions, and which pages are free.

    Pages are handed out on the host, ahead of the steps that need them (`reserve`); a decode step reads table and
    positions on the device and can be captured into a CUDA graph and replayed as long as pages are reserved.
    The host counts every sequence's tokens: `prefill` and `step` do, and `replayed` says how often a captured step is to run.
    A slot without pages is idle: steps, captured ones too, store nothing for it, leave its position at 0 and give zeros."""

    def __init__(self, n_layers: int, slots: int, h_q: int, h_kv: int, head_dim: int, n_pages: int, max_pages: int,
                 page_size: int = 64, device="cuda", max_prompt_tokens: int = 0):
        self.n_layers, self.slots, self.h_q, self.h_kv, self.head_dim = n_layers, slots, h_q, h_kv, head_dim
        self.n_pages, self.max_pages, self.page_size = n_pages, max_pages, page_size
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        pool = (n_layers, n_pages, h_kv, page_size, head_dim)
        self.k_pages = torch.zeros(pool, dtype=torch.uint8, device=self.device)
        self.v_pages = torch.zeros(pool, dtype=torch.uint8, device=self.device)
        self.k_scale = torch.ones(n_layers, n_pages, h_kv, device=self.device)
        self.v_scale = torch.ones(n_layers, n_pages, h_kv, device=self.device)
        self.page_table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=self.device)
        self.seq_pos = torch.zeros(slots, dtype=torch.int32, device=self.device)
        self.host_len = [0] * slots
        self.pages: list[list[int]] = [[] for _ in range(slots)]
        self.free = list(range(n_pages - 1, -1, -1))
        self.shape = make_paged_shape(h_q, self.k_pages, self.v_pages, self.k_scale, self.page_table)
        self.workspace = PagedWorkspace(self.shape, self.device)
        self.prompt_workspace = None
        if max_prompt_tokens:
            self.prompt_workspace = PagedWorkspace(self.shape, self.device, q_tokens=max_prompt_tokens)

    @property
    def status(self) -> torch.Tensor:
        return self.workspace.status

    def read_status(self) -> int:
        st = self.workspace.read_status()
        return st | self.prompt_workspace.read_status() if self.prompt_workspace is not None else st

    def reserve(self, slot: int, n_tokens: int) -> None:
        """Pages for `n_tokens` more tokens of a sequence; refuses, and changes nothing, if the pool or the table has no room."""
        need = -(-(self.host_len[slot] + n_tokens) // self.page_size)
        more = need - len(self.pages[slot])
        if need > self.max_pages:
            raise ValueError(f"capacity {self.max_pages * self.page_size} exceeded: {self.host_len[slot]} cached + {n_tokens}")
        if more > len(self.free):
            raise ValueError(f"{more} pages needed, {len(self.free)} free")
        if more > 0:
            first = len(self.pages[slot])
            self.pages[slot] += [self.free.pop() for _ in range(more)]
            self.page_table[slot, first:need] = torch.tensor(self.pages[slot][first:], dtype=torch.int32).to(self.device)

    def release(self, slot: int) -> None:
        """The sequence's pages go back to the pool (stream order: launches that read them come before)."""
        self.free += reversed(self.pages[slot])
        self.pages[slot] = []
        self.host_len[slot] = 0
        self.page_table[slot].fill_(-1)
        self.seq_pos[slot] = 0

    def prefill(self, q, k, v, cos, sin, lens, *, out=None, causal: bool = True, **rope) -> torch.Tensor:
        """New tokens of every sequence (lens[b] of them, 0 allowed; packed along the token dimension): rotated, appended and
        attended.  Returns bf16 [n_layers, n_tokens, h_q, head_dim].  `rope`: further arguments of `paged_rope_append`."""
        if len(lens) != self.slots or min(lens) < 0 or sum(lens) != q.shape[-3]:
            raise ValueError("lens must give every sequence's share of the tokens")
        if self.prompt_workspace is None or self.prompt_workspace.q_tokens < sum(lens):
            raise ValueError(f"max_prompt_tokens is too small for {sum(lens)} tokens")
        need = [-(-(a + n) // self.page_size) - len(p) for a, n, p in zip(self.host_len, lens, self.pages)]
        if sum(max(x, 0) for x in need) > len(self.free):
            raise ValueError(f"{sum(max(x, 0) for x in need)} pages needed, {len(self.free)} free")
        for a, n in zip(self.host_len, lens):
            if a + n > self.max_pages * self.page_size:
                raise ValueError(f"capacity {self.max_pages * self.page_size} exceeded: {a} cached + {n}")
        had = [len(p) for p in self.pages]
        for b, n in enumerate(lens):
            self.reserve(b, n)
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        q_start = torch.tensor(starts, dtype=torch.int32).to(self.device)
        try:
            qr = paged_rope_append(q, k, v, cos, sin, self.k_pages, self.v_pages, self.k_scale, self.v_scale, self.page_table,
                                   self.seq_pos, q_start=q_start, advance=True, status=self.status, **rope)
        except Exception:
            for b, n in reversed(list(enumerate(had))):    # the call was refused: a slot that was idle is idle
                self.free += reversed(self.pages[b][n:])
                del self.pages[b][n:]
                self.page_table[b, n:] = -1
            raise
        self.host_len = [a + n for a, n in zip(self.host_len, lens)]
        return paged_prefill_attention(qr, q_start, self.k_pages, self.v_pages, self.k_scale, self.v_scale, self.page_table,
                                       self.seq_pos, workspace=self.prompt_workspace, causal=causal, out=out)

    def _room(self, n: int) -> None:
        for b in range(self.slots):
            if self.pages[b] and self.host_len[b] + n > len(self.pages[b]) * self.page_size:
                raise ValueError(f"slot {b}: {len(self.pages[b])} pages reserved for {self.host_len[b]} cached + {n}")

    def _count(self, n: int) -> None:
        self.host_len = [x + n if p else x for x, p in zip(self.host_len, self.pages)]

    def replayed(self, n: int = 1) -> None:
        """Count `n` replays of a captured step, before they run; refuses, and counts nothing, if the pages reserved for a sequence
        do not hold them."""
        self._room(n)
        self._count(n)

    def step(self, q, k, v, cos, sin, *, out=None, count: bool = True, **rope) -> torch.Tensor:
        """One decode step of all slots that have pages: rotate, append, attend, advance (graph capturable; `reserve` first).  q, k
        and v hold a row for every slot; an idle slot's result is zero.  A step under capture does not run and is not counted
        (`replayed`); count=False: the caller counts this one too."""
        count = count and not torch.cuda.is_current_stream_capturing()
        if count:
            self._room(1)
        qr = paged_rope_append(q, k, v, cos, sin, self.k_pages, self.v_pages, self.k_scale, self.v_scale, self.page_table,
                               self.seq_pos, advance=True, status=self.status, **rope)
        if count:
            self._count(1)
        return paged_decode_attention(qr, self.k_pages, self.v_pages, self.k_scale, self.v_scale, self.page_table, self.seq_pos,
                                      workspace=self.workspace, out=out)


__all__ = ["PagedFP8Cache", "PagedWorkspace", "make_paged_shape", "paged_decode_attention", "paged_prefill_attention",
           "paged_rope_append", "rope_tables"]
