"""A 4-bit paged key/value cache and the attention that reads it (fml_kv4_*,
fml_attention_kv4 in include/freeml_cuda.h).

One layer's cache is a uint8 tensor [pages, kv_heads, page_size, 5 * hd / 4]
(its bytes are laid out block by block, see the header); sequences live in
slots: `table` int32 [slots, max_pages] (page numbers, -1 where there is none),
`lens` int32 [slots].  `refs` int32 [pages] counts the slots that hold a page.
Page operations take every layer's pool at once, [layers, pages, ...], and OR
into `status` (int32 [1]) why a call could not be carried out; it then changes
nothing.  `KV4Cache` keeps these tensors together.
"""
from __future__ import annotations

import torch

from ._lib import FmlError, call, load

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # FML_TYPE_*
NO_PAGES, BAD_SLOT, ROW_FULL = 1, 2, 4                           # FML_KV4_*


def _check(cond, msg):
    if not cond:
        raise FmlError(1, "kv4", msg)


def _s():
    return torch.cuda.current_stream().cuda_stream


def _rows(t, heads, hd, what):
    """(pointer, row stride) of [rows, heads, hd] whose heads are dense."""
    s = t.stride()
    if t.dim() != 3 or not t.is_cuda or t.shape[1] != heads or t.shape[2] != hd or s[2] != 1 or (s[1] != hd and heads > 1):
        raise FmlError(1, "kv4", f"{what}: expected a CUDA tensor [rows, {heads}, {hd}] with dense heads")
    return t.data_ptr(), max(s[0], heads * hd) if t.shape[0] < 2 else s[0]


def _ints(t, what, dims=1):
    if t is None:
        return None
    if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.dim() != dims:
        raise FmlError(1, "kv4", f"{what}: expected a contiguous int32 CUDA tensor of {dims} dimension(s)")
    return t.data_ptr()


def _geometry(pool, hd):
    """(pages, kv_heads, page_size) of one layer's pool."""
    if pool.dtype != torch.uint8 or pool.dim() != 4 or not pool.is_cuda or not pool.is_contiguous() \
            or pool.shape[3] * 4 != hd * 5:
        raise FmlError(1, "kv4", f"pool: expected a contiguous uint8 CUDA tensor [pages, kv_heads, page_size, {hd * 5 // 4}]")
    return pool.shape[:3]


def empty_pool(layers, pages, kv_heads, page_size, head_dim, device="cuda"):
    """Zeroed pools of `layers` layers."""
    _check(int(load().fml_kv4_block_bytes(head_dim, page_size)) > 0, f"head_dim {head_dim}, page_size {page_size}")
    return torch.zeros(layers, pages, kv_heads, page_size, 5 * head_dim // 4, dtype=torch.uint8, device=device)


def append(pool, table, lens, k, v, starts, slot_ids=None):
    """Write each sequence's newest rows (fml_kv4_append): k, v [rows,
    kv_heads, hd]; rows starts[b] .. starts[b + 1] - 1 are entry b's last."""
    hd = k.shape[-1]
    pages, heads, page = _geometry(pool, hd)
    pk, ldk = _rows(k, heads, hd, "k")
    pv, ldv = _rows(v, heads, hd, "v")
    _check(k.dtype == v.dtype and k.dtype in TYPES and k.shape[0] == v.shape[0], "append: k and v differ, or their type")
    batch = starts.shape[0] - 1
    _check(slot_ids is None and batch <= table.shape[0] or slot_ids is not None and slot_ids.shape[0] == batch,
           "append: starts and slot_ids")
    call("fml_kv4_append", pool.data_ptr(), _ints(table, "table", 2), _ints(lens, "lens"), _ints(slot_ids, "slot_ids"),
         pk, pv, TYPES[k.dtype], _ints(starts, "starts"), batch, k.shape[0], ldk, ldv, pages, table.shape[0],
         table.shape[1], page, heads, hd, _s())


def read(k, v, pool, table, lens, starts, slot_ids=None):
    """The values that each sequence's newest rows stand for, into k and v
    (fml_kv4_read); rows as in append."""
    hd = k.shape[-1]
    pages, heads, page = _geometry(pool, hd)
    pk, ldk = _rows(k, heads, hd, "k")
    pv, ldv = _rows(v, heads, hd, "v")
    _check(k.dtype == v.dtype and k.dtype in TYPES and k.shape[0] == v.shape[0], "read: k and v differ, or their type")
    batch = starts.shape[0] - 1
    _check(slot_ids is None and batch <= table.shape[0] or slot_ids is not None and slot_ids.shape[0] == batch,
           "read: starts and slot_ids")
    call("fml_kv4_read", pk, pv, TYPES[k.dtype], pool.data_ptr(), _ints(table, "table", 2), _ints(lens, "lens"),
         _ints(slot_ids, "slot_ids"), _ints(starts, "starts"), batch, k.shape[0], ldk, ldv, pages, table.shape[0],
         table.shape[1], page, heads, hd, _s())


def attention_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size):
    return int(load().fml_attention_kv4_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size))


def attention(out, q, pool, table, lens, scale, slot_ids=None, workspace=None):
    """One query row per sequence over the cache (fml_attention_kv4): q, out
    [batch, heads, hd]; entry b sees its lens keys."""
    batch, heads, hd = q.shape
    pages, kv_heads, page = _geometry(pool, hd)
    pq, ldq = _rows(q, heads, hd, "q")
    po, ldo = _rows(out, heads, hd, "out")
    _check(out.shape[0] == batch and out.dtype == q.dtype and q.dtype in TYPES, "attention: q and out differ, or their type")
    _check(slot_ids is None and batch <= table.shape[0] or slot_ids is not None and slot_ids.shape[0] == batch,
           "attention: batch and slot_ids")
    slots, most = table.shape
    need = attention_workspace_bytes(batch, heads, kv_heads, hd, most, page)
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    call("fml_attention_kv4", po, pq, TYPES[q.dtype], ldo, ldq, pool.data_ptr(), _ints(table, "table", 2),
         _ints(lens, "lens"), _ints(slot_ids, "slot_ids"), batch, pages, slots, most, page, heads, kv_heads, hd,
         float(scale), None if workspace is None else workspace.data_ptr(),
         0 if workspace is None else workspace.numel() * workspace.element_size(), _s())


def _pages_workspace(pages, n, device, workspace):
    if workspace is None:
        workspace = torch.empty(int(load().fml_kv4_pages_workspace_bytes(pages, n)), dtype=torch.uint8, device=device)
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _layers(pool):
    if pool.dtype != torch.uint8 or pool.dim() != 5 or not pool.is_cuda or not pool.is_contiguous():
        raise FmlError(1, "kv4", "pool: expected a contiguous uint8 CUDA tensor [layers, pages, kv_heads, page_size, bytes]")
    page_bytes = pool.shape[2] * pool.shape[3] * pool.shape[4]
    return pool.data_ptr(), pool.shape[0], pool.shape[1] * page_bytes, page_bytes


def reserve(refs, table, lens, counts, page_size, status, slot_ids=None, workspace=None):
    """lens[slot] += counts[i], with pages for the new rows (fml_kv4_reserve)."""
    n, pages = counts.shape[0], refs.shape[0]
    _check(slot_ids is None and n <= table.shape[0] or slot_ids is not None and slot_ids.shape[0] == n,
           "reserve: counts and slot_ids")
    ws, p, size = _pages_workspace(pages, max(n, 1), refs.device, workspace)
    call("fml_kv4_reserve", _ints(refs, "refs"), _ints(table, "table", 2), _ints(lens, "lens"),
         _ints(slot_ids, "slot_ids"), _ints(counts, "counts"), n, pages, table.shape[0], table.shape[1], page_size,
         _ints(status, "status"), p, size, _s())


def fork(pool, refs, table, lens, parents, children, status, workspace=None):
    """Slot children[i] becomes a copy of slot parents[i] (fml_kv4_fork): full
    pages shared, a page in use copied in every layer of pool."""
    base, layers, stride, page_bytes = _layers(pool)
    n, pages = parents.shape[0], refs.shape[0]
    _check(children.shape[0] == n and pool.shape[1] == pages, "fork: parents and children, or pool and refs")
    ws, p, size = _pages_workspace(pages, max(n, 1), refs.device, workspace)
    call("fml_kv4_fork", base, layers, stride, page_bytes, _ints(refs, "refs"), _ints(table, "table", 2),
         _ints(lens, "lens"), _ints(parents, "parents"), _ints(children, "children"), n, pages, table.shape[0],
         table.shape[1], pool.shape[3], _ints(status, "status"), p, size, _s())


def free(refs, table, lens, slot_ids, status):
    """Give the slots' pages back (fml_kv4_free)."""
    call("fml_kv4_free", _ints(refs, "refs"), _ints(table, "table", 2), _ints(lens, "lens"), _ints(slot_ids, "slot_ids"),
         slot_ids.shape[0], refs.shape[0], table.shape[0], table.shape[1], _ints(status, "status"), _s())


def compact(pool, refs, table, workspace=None):
    """Move the used pages together, in every layer of pool (fml_kv4_compact)."""
    base, layers, stride, page_bytes = _layers(pool)
    pages = refs.shape[0]
    _check(pool.shape[1] == pages, "compact: pool and refs")
    ws, p, size = _pages_workspace(pages, 0, refs.device, workspace)
    call("fml_kv4_compact", base, layers, stride, page_bytes, _ints(refs, "refs"), _ints(table, "table", 2), pages,
         table.shape[0], table.shape[1], p, size, _s())


class KV4Cache:
    """The pools, tables, lengths and counts of one model's 4-bit cache.

    A step: reserve(counts); for each layer append(layer, k, v, starts) and
    attention(layer, out, q).  check() reads the status word (it waits)."""

    def __init__(self, layers, kv_heads, head_dim, pages, page_size=64, slots=1, max_pages=None, device="cuda"):
        self.page_size = page_size
        self.pool = empty_pool(layers, pages, kv_heads, page_size, head_dim, device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.table = torch.full((slots, max_pages or pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def reserve(self, counts, slot_ids=None):
        reserve(self.refs, self.table, self.lens, counts, self.page_size, self.status, slot_ids)

    def append(self, layer, k, v, starts, slot_ids=None):
        append(self.pool[layer], self.table, self.lens, k, v, starts, slot_ids)

    def read(self, layer, k, v, starts, slot_ids=None):
        read(k, v, self.pool[layer], self.table, self.lens, starts, slot_ids)

    def attention(self, layer, out, q, scale, slot_ids=None, workspace=None):
        attention(out, q, self.pool[layer], self.table, self.lens, scale, slot_ids, workspace)

    def fork(self, parents, children):
        fork(self.pool, self.refs, self.table, self.lens, parents, children, self.status)

    def free(self, slot_ids):
        free(self.refs, self.table, self.lens, slot_ids, self.status)

    def compact(self):
        compact(self.pool, self.refs, self.table)

    def check(self):
        """Raise if an operation since the last check could not be carried out."""
        bits = int(self.status.item())
        self.status.zero_()
        why = [text for bit, text in ((NO_PAGES, "no free pages"), (BAD_SLOT, "a bad slot"),
                                      (ROW_FULL, "a sequence longer than its table row")) if bits & bit]
        if why:
            raise FmlError(5, "KV4Cache", ", ".join(why))
