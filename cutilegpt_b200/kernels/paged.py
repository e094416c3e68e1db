"""Paged key/value cache: appending to it and attention over it (no reference counterpart).

``PagedKV`` describes a cache: keys and values in pages of ``page_size``
positions, a page table and a length per sequence, and optionally a prefix per
group of sequences (several samples of one prompt, requests behind one
instruction) whose pages all sequences of the group share.
``cutile_paged_kv_append`` writes the keys and values of new tokens into it,
with the position rotation on the way where a model has one;
``cutile_shared_prefix_attention`` lets the new tokens look at it.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib as L
from . import ops
from ._common import as_cuda, same_dtype


def _table(t, name: str, rows: int | None, device) -> torch.Tensor:
    t = as_cuda(t, name)
    if t.dtype != torch.int32 or t.device != device:
        raise ValueError(f"{name}: expected an int32 tensor on {device}, got {t.dtype} on {t.device}")
    if t.dim() != 2 or t.shape[1] == 0 or t.stride(1) != 1 or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name}: expected [{'n' if rows is None else rows}, pages >= 1] with contiguous rows, got "
                         f"shape {tuple(t.shape)} strides {t.stride()}")
    return t


def _lens(t, name: str, n: int, device) -> torch.Tensor:
    t = as_cuda(t, name)
    if t.dtype != torch.int32 or t.device != device or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {n} lengths on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t


class PagedKV:
    """A paged cache of one layer and the tables that say whose pages are whose.

    k_pages, v_pages   [n_pages, n_kv_head, page_size, head_dim], any page / head / slot strides (the
                       same for both), contiguous head_dim
    page_table         int32 [batch, max_pages]: the pages of each sequence's own positions
    seq_lens           int32 [batch]: own positions of each sequence, new tokens included; 0 = idle
    prefix_table       int32 [n_groups, max_prefix_pages], prefix_lens int32 [n_groups]: the prefix of
                       sequences b with b // (batch // n_groups) == group; its positions come first

    The tensors are used in place: a program changes tables and lengths in
    them between calls (or between replays of a captured graph). Entries
    behind a length are never read.
    """

    def __init__(self, k_pages, v_pages, page_table, seq_lens, prefix_table=None, prefix_lens=None):
        k_pages, v_pages = as_cuda(k_pages, "k_pages"), as_cuda(v_pages, "v_pages")
        same_dtype(k_pages, v_pages)
        L.dtype_code(k_pages.dtype)
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.numel() == 0:
            raise ValueError("PagedKV: k_pages and v_pages must share shape (n_pages, n_kv_head, page_size, head_dim), got "
                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        if k_pages.stride() != v_pages.stride() or (k_pages.shape[3] > 1 and k_pages.stride(3) != 1):
            raise ValueError("PagedKV: k_pages and v_pages must have the same strides and a contiguous head_dim, got "
                             f"{k_pages.stride()} and {v_pages.stride()}")
        dev = k_pages.device
        if v_pages.device != dev:
            raise ValueError(f"PagedKV: k_pages on {dev} but v_pages on {v_pages.device}")
        page_table = _table(page_table, "page_table", None, dev)
        seq_lens = _lens(seq_lens, "seq_lens", page_table.shape[0], dev)
        if (prefix_table is None) != (prefix_lens is None):
            raise ValueError("PagedKV: prefix_table and prefix_lens come together")
        if prefix_table is not None:
            prefix_table = _table(prefix_table, "prefix_table", None, dev)
            n = prefix_table.shape[0]
            prefix_lens = _lens(prefix_lens, "prefix_lens", n, dev)
            if n == 0 or page_table.shape[0] % n:
                raise ValueError(f"PagedKV: {n} prefixes do not divide {page_table.shape[0]} sequences")
        self._tensors = (k_pages, v_pages, page_table, seq_lens, prefix_table, prefix_lens)
        n_pages, heads, page, dim = k_pages.shape
        self.dtype, self.device = k_pages.dtype, dev
        self.batch, self.n_kv_head, self.head_dim = page_table.shape[0], heads, dim
        self._dtype_code = L.dtype_code(k_pages.dtype)
        s = L.PagedKvStruct()
        s.k_pages, s.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
        s.n_pages, s.kv_heads, s.page_size, s.head_dim = n_pages, heads, page, dim
        s.page_stride, s.head_stride, s.slot_stride = k_pages.stride()[:3]
        s.page_table, s.ld_page_table, s.max_pages = page_table.data_ptr(), page_table.stride(0), page_table.shape[1]
        if page_table.shape[0] <= 1:
            s.ld_page_table = max(s.ld_page_table, s.max_pages)
        s.seq_lens, s.batch = seq_lens.data_ptr(), page_table.shape[0]
        if prefix_table is not None:
            s.prefix_table, s.max_prefix_pages = prefix_table.data_ptr(), prefix_table.shape[1]
            s.ld_prefix_table = max(prefix_table.stride(0), s.max_prefix_pages) if n == 1 else prefix_table.stride(0)
            s.prefix_lens, s.n_groups = prefix_lens.data_ptr(), n
        self._struct = s
        self._ref = ctypes.byref(s)
        self._ws_bytes: dict[tuple[int, int], int] = {}

    k_pages = property(lambda self: self._tensors[0])
    v_pages = property(lambda self: self._tensors[1])
    page_table = property(lambda self: self._tensors[2])
    seq_lens = property(lambda self: self._tensors[3])
    prefix_table = property(lambda self: self._tensors[4])
    prefix_lens = property(lambda self: self._tensors[5])

    def workspace_bytes(self, n_head: int, tokens: int) -> int:
        """Workspace of cutile_shared_prefix_attention for queries (batch, n_head, tokens, head_dim): a
        function of the cache's sizes, the same at every length."""
        n = self._ws_bytes.get((n_head, tokens))
        if n is None:
            n = int(L.lib().gpt_attention_shared_prefix_workspace_size(tokens, n_head, self._ref, self._dtype_code))
            self._ws_bytes[(n_head, tokens)] = n
        return n


def _rows(t, name: str, kv: PagedKV, heads: int | None, tokens: int | None) -> torch.Tensor:
    """A (batch, heads, tokens, head_dim) tensor of the cache's type and device, head_dim contiguous."""
    if type(t) is not torch.Tensor:
        t = as_cuda(t, name)
    shape = t.shape
    b, h, n, d = shape if len(shape) == 4 else (-1, 0, 0, 0)
    if b != kv.batch or d != kv.head_dim or (heads is not None and h != heads) or (tokens is not None and n != tokens):
        raise ValueError(f"{name}: expected ({kv.batch}, {'n_head' if heads is None else heads}, "
                         f"{'tokens' if tokens is None else tokens}, {kv.head_dim}), got {tuple(shape)}")
    if t.dtype != kv.dtype or t.device != kv.device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, but the cache holds {kv.dtype} on {kv.device}")
    return t if t.stride(3) == 1 or d == 1 else t.contiguous()


def _out_rows(t, name: str, kv: PagedKV, heads: int, tokens: int) -> torch.Tensor:
    if type(t) is not torch.Tensor:
        t = as_cuda(t, name)
    if _rows(t, name, kv, heads, tokens) is not t:
        raise ValueError(f"{name}: head_dim must be contiguous")
    return t


def cutile_paged_kv_append(q, k, v, kv: PagedKV, cos_sin=None, interleaved: bool = False, q_out=None):
    """Keys and values of new tokens into the cache; returns the queries, rotated where cos_sin is given.

    q (batch, n_head, tokens, head_dim), k and v (batch, n_kv_head, tokens, head_dim), any strides with a
    contiguous head_dim (the parts of a fused projection are read in place). Token t of sequence b goes
    to own position seq_lens[b] - tokens + t; a negative one is padding and is skipped, one past the
    table is skipped and reported by the device error word. cos_sin float32 [n_pos, rot]: cosines, then
    sines, of the rot / 2 angles of each position; the first rot values of every query and key head are
    turned, in pairs (j, j + rot / 2) or, interleaved, (2j, 2j + 1), by the position counted from the start
    of the prefix. q_out may be q itself (same strides), and overlaps q in no other way; without cos_sin
    q is returned as it is and may be None.
    """
    k = _rows(k, "k", kv, kv.n_kv_head, None)
    tokens = k.shape[2]
    v = _rows(v, "v", kv, kv.n_kv_head, tokens)
    if cos_sin is None:
        if q_out is not None:
            raise ValueError("paged_kv_append: q_out needs a rotation (cos_sin)")
        ops.paged_kv_append(None, k, v, None, kv)
        return q
    q = _rows(q, "q", kv, None, tokens)
    if type(cos_sin) is not torch.Tensor:
        cos_sin = as_cuda(cos_sin, "cos_sin")
    table = cos_sin.shape
    if (len(table) != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or table[0] == 0 or table[1] % 2
            or not 0 < table[1] <= kv.head_dim or cos_sin.device != kv.device):
        raise ValueError(f"cos_sin: expected a contiguous float32 [n_pos, rot] table with even rot <= {kv.head_dim} on "
                         f"{kv.device}, got {cos_sin.dtype} {tuple(table)}")
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        q_out = _out_rows(q_out, "q_out", kv, q.shape[1], tokens)
        if (q_out.data_ptr() == q.data_ptr() and q.numel()
                and any(n > 1 and a != b for n, a, b in zip(q.shape, q.stride(), q_out.stride()))):
            raise ValueError(f"q_out: in q's memory it needs q's strides {q.stride()}, got {q_out.stride()}")
    ops.paged_kv_append(q, k, v, q_out, kv, cos_sin, interleaved)
    return q_out


def cutile_shared_prefix_attention(q, kv: PagedKV, scale: float | None = None, out=None, workspace=None) -> torch.Tensor:
    """softmax(scale q·kᵀ) v of each sequence's newest tokens over its group's prefix and its own positions.

    q (batch, n_head, tokens, head_dim), n_head a multiple of the cache's key heads (head h reads key head
    h // (n_head // n_kv_head)); token t of sequence b sees the prefix and its own positions 0 ..
    seq_lens[b] - tokens + t, and gives zeros where that is negative (padding, idle sequences). The prefix
    is read once for a block of its sequences' rows, 128 or 256 of a key head in bf16 with the usual sizes
    (see the C header), not once for a sequence. In bf16 the probabilities are rounded to bf16 for their
    product with the values. scale is 1/√head_dim by default. A new contiguous tensor is returned unless `out`
    (any strides, contiguous head_dim, no overlap with q) is given; `workspace` (uint8,
    kv.workspace_bytes(n_head, tokens)) is allocated unless given.
    """
    q = _rows(q, "q", kv, None, None)
    _, heads, tokens, dim = q.shape
    if heads == 0 or heads % kv.n_kv_head:
        raise ValueError(f"shared_prefix_attention: {heads} heads are no multiple of {kv.n_kv_head} key heads")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        out = _out_rows(out, "out", kv, heads, tokens)
        if out.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("out: must not be q's memory")
    if workspace is not None and type(workspace) is not torch.Tensor:
        workspace = as_cuda(workspace, "workspace")
    return ops.shared_prefix_attention(q, kv, out, dim ** -0.5 if scale is None else scale, workspace)
