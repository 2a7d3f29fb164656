"""A 4-bit paged key/value cache and the attention that reads it (fml_kv4_*,
fml_attention_kv4 in include/freeml_cuda.h).

One layer's cache is a uint8 tensor [pages, kv_heads, page_size, 5 * hd / 4]
(its bytes are laid out block by block, see the header); sequences live in
slots: `table` int32 [slots, max_pages] (page numbers, -1 where there is none),
`lens` int32 [slots].  `refs` int32 [pages] counts the slots that hold a page.
Page operations take every layer's pool at once, [layers, pages, ...], and OR
into `status` (int32 [1]) why a call could not be carried out; it then changes
nothing.  `kept` int32 [slots], where it is passed to reserve and append, keeps
an append behind a refused reserve off the rows that are there.  `KV4Cache`
keeps these tensors together.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from ._lib import FmlError, call, load

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # FML_TYPE_*
NO_PAGES, BAD_SLOT, ROW_FULL = 1, 2, 4                           # FML_KV4_*


def reasons(bits):
    """A status word in words."""
    return ", ".join(text for bit, text in ((NO_PAGES, "no free pages"), (BAD_SLOT, "a bad slot"),
                                            (ROW_FULL, "a sequence longer than its table row")) if bits & bit)


def _refuse(msg):
    raise FmlError(1, "kv4", msg)


# The checks below run before every launch of a decode step: they are written
# to cost little (the smallest calls take less time on the GPU than on the host).

def _elsewhere(device, function, *args):
    """function(*args) where its tensors' GPU is not the current one: with it current."""
    if device < 0:
        _refuse("expected CUDA tensors")
    with torch.cuda.device(device):
        function(*args)


# torch.cuda.current_stream(device).cuda_stream builds a Stream object (3 us);
# where torch has the plain query, that is used (0.1 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _rows(t, heads, hd, what, device):
    """(pointer, row stride) of [rows, heads, hd] on `device` whose heads are dense."""
    if t.get_device() == device and t.dim() == 3:
        n, h, d = t.shape
        s0, s1, s2 = t.stride()
        if h == heads and d == hd and s2 == 1 and (s1 == hd or h == 1) and (n <= 1 or s0 < 1 << 32):
            return t.data_ptr(), s0 if n > 1 else h * d
    _refuse(f"{what}: expected a tensor [rows, {heads}, {hd}] on GPU {device} with dense heads, rows less than 2^32 apart")


def _ints(t, what, device, dims=1):
    if t is None:
        return None
    if t.dtype is torch.int32 and t.get_device() == device and t.dim() == dims and t.is_contiguous():
        return t.data_ptr()
    _refuse(f"{what}: expected a contiguous int32 tensor of {dims} dimension(s) on GPU {device}")


def _geometry(pool, hd):
    """(pages, kv_heads, page_size) of one layer's pool (on the current GPU: the caller has looked)."""
    if pool.dim() == 4 and pool.dtype is torch.uint8 and pool.is_contiguous():
        pages, heads, page, width = pool.shape
        if width * 4 == hd * 5:
            return pages, heads, page
    _refuse(f"pool: expected a contiguous uint8 CUDA tensor [pages, kv_heads, page_size, {hd * 5 // 4}]")


def _tables(table, lens, slot_ids, batch, what, device):
    """(table, slots, max_pages, lens, slot_ids) as the C ABI takes them."""
    at = _ints(table, "table", device, 2)
    slots, most = table.shape
    if lens.shape[0] != slots:
        _refuse(f"{what}: lens of {lens.shape[0]} slots, a table of {slots}")
    if slot_ids is None:
        if batch > slots:
            _refuse(f"{what}: {batch} entries, {slots} slots")
    elif slot_ids.shape[0] != batch:
        _refuse(f"{what}: {batch} entries, {slot_ids.shape[0]} slot_ids")
    return at, slots, most, _ints(lens, "lens", device), _ints(slot_ids, "slot_ids", device)


def empty_pool(layers, pages, kv_heads, page_size, head_dim, device="cuda"):
    """Zeroed pools of `layers` layers."""
    if not int(load().fml_kv4_block_bytes(head_dim, page_size)):
        _refuse(f"head_dim {head_dim}, page_size {page_size}")
    return torch.zeros(layers, pages, kv_heads, page_size, 5 * head_dim // 4, dtype=torch.uint8, device=device)


def _workspace(t, device):
    """(pointer, bytes) of a caller's workspace."""
    if t.get_device() == device and t.is_contiguous():
        return t.data_ptr(), t.numel() * t.element_size()
    _refuse(f"workspace: expected a contiguous tensor on GPU {device}")


def _new_rows(what, pool, table, lens, k, v, starts, slot_ids, device):
    """The arguments that append and read share."""
    hd = k.shape[-1]
    pages, heads, page = _geometry(pool, hd)
    pk, ldk = _rows(k, heads, hd, "k", device)
    pv, ldv = _rows(v, heads, hd, "v", device)
    kind, rows, batch = TYPES.get(k.dtype), k.shape[0], starts.shape[0] - 1
    if kind is None or v.dtype is not k.dtype or v.shape[0] != rows:
        _refuse(f"{what}: k and v differ, or their type")
    table, slots, most, lens, slot_ids = _tables(table, lens, slot_ids, batch, what, device)
    tail = (batch, rows, ldk, ldv, pages, slots, most, page, heads, hd, _raw_stream(device))
    return pool.data_ptr(), table, lens, slot_ids, pk, pv, kind, _ints(starts, "starts", device), tail


def _kept(kept, slots, device):
    if kept.shape[0] != slots:
        _refuse(f"kept of {kept.shape[0]} slots, a table of {slots}")
    return _ints(kept, "kept", device)


def append(pool, table, lens, k, v, starts, slot_ids=None, kept=None):
    """Write each sequence's newest rows (fml_kv4_append): k, v [rows,
    kv_heads, hd]; rows starts[b] .. starts[b + 1] - 1 are entry b's last.
    Behind a refused reserve these places hold older rows: pass the reserve's
    `kept`, or read its status in between."""
    slots, device = table.shape[0], pool.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, append, pool, table, lens, k, v, starts, slot_ids, kept)
    p, table, lens, slot_ids, pk, pv, kind, starts, tail = _new_rows("append", pool, table, lens, k, v, starts, slot_ids,
                                                                     device)
    if kept is None:
        call("fml_kv4_append", p, table, lens, slot_ids, pk, pv, kind, starts, *tail)
    else:
        call("fml_kv4_append_keeping", p, table, lens, slot_ids, _kept(kept, slots, device), pk, pv, kind, starts, *tail)


def read(k, v, pool, table, lens, starts, slot_ids=None):
    """The values that each sequence's newest rows stand for, into k and v
    (fml_kv4_read); rows as in append."""
    device = pool.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, read, k, v, pool, table, lens, starts, slot_ids)
    p, table, lens, slot_ids, pk, pv, kind, starts, tail = _new_rows("read", pool, table, lens, k, v, starts, slot_ids,
                                                                     device)
    call("fml_kv4_read", pk, pv, kind, p, table, lens, slot_ids, starts, *tail)


@lru_cache(maxsize=256)
def attention_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size):
    return int(load().fml_attention_kv4_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size))


def attention(out, q, pool, table, lens, scale, slot_ids=None, workspace=None):
    """One query row per sequence over the cache (fml_attention_kv4): q, out
    [batch, heads, hd]; entry b sees its lens keys."""
    device = pool.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, attention, out, q, pool, table, lens, scale, slot_ids, workspace)
    batch, heads, hd = q.shape
    pages, kv_heads, page = _geometry(pool, hd)
    pq, ldq = _rows(q, heads, hd, "q", device)
    po, ldo = _rows(out, heads, hd, "out", device)
    kind = TYPES.get(q.dtype)
    if kind is None or out.dtype is not q.dtype or out.shape[0] != batch:
        _refuse("attention: q and out differ, or their type")
    table, slots, most, lens, slot_ids = _tables(table, lens, slot_ids, batch, "attention", device)
    size, ws = 0, None
    if workspace is None:
        size = attention_workspace_bytes(batch, heads, kv_heads, hd, most, page)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
            ws = workspace.data_ptr()
    else:
        ws, size = _workspace(workspace, device)
    call("fml_attention_kv4", po, pq, kind, ldo, ldq, pool.data_ptr(), table, lens, slot_ids, batch, pages, slots, most,
         page, heads, kv_heads, hd, float(scale), ws, size, _raw_stream(device))


@lru_cache(maxsize=256)
def _pages_bytes(pages, n):
    return int(load().fml_kv4_pages_workspace_bytes(pages, n))


def _pages_workspace(refs, n, workspace):
    """(tensor, pointer, bytes); the tensor is held until the call is made."""
    if workspace is None:
        size = _pages_bytes(refs.shape[0], n)
        workspace = torch.empty(size, dtype=torch.uint8, device=refs.device)
        return workspace, workspace.data_ptr(), size
    return workspace, *_workspace(workspace, refs.get_device())


def _layers(pool, pages, device):
    """(pointer, layers, bytes from one to the next, bytes of a page, rows of a page)"""
    if pool.dim() == 5 and pool.dtype is torch.uint8 and pool.get_device() == device and pool.is_contiguous():
        layers, n, heads, page, width = pool.shape
        if n == pages:
            return pool.data_ptr(), layers, n * heads * page * width, heads * page * width, page
    _refuse(f"pool: expected a contiguous uint8 tensor [layers, {pages}, kv_heads, page_size, bytes] on GPU {device}")


def reserve(refs, table, lens, counts, page_size, status, slot_ids=None, workspace=None, kept=None):
    """lens[slot] += counts[i], with pages for the new rows (fml_kv4_reserve);
    kept: where an append with it may write (fml_kv4_reserve_keeping)."""
    n, pages, device = counts.shape[0], refs.shape[0], refs.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, reserve, refs, table, lens, counts, page_size, status, slot_ids, workspace, kept)
    table, slots, most, lens, slot_ids = _tables(table, lens, slot_ids, n, "reserve", device)
    hold, ws, size = _pages_workspace(refs, max(n, 1), workspace)
    refs, counts, status = _ints(refs, "refs", device), _ints(counts, "counts", device), _ints(status, "status", device)
    tail = (slot_ids, counts, n, pages, slots, most, page_size, status, ws, size, _raw_stream(device))
    if kept is None:
        call("fml_kv4_reserve", refs, table, lens, *tail)
    else:
        call("fml_kv4_reserve_keeping", refs, table, lens, _kept(kept, slots, device), *tail)


def fork(pool, refs, table, lens, parents, children, status, workspace=None):
    """Slot children[i] becomes a copy of slot parents[i] (fml_kv4_fork): full
    pages shared, a page in use copied in every layer of pool."""
    n, pages, device = parents.shape[0], refs.shape[0], refs.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, fork, pool, refs, table, lens, parents, children, status, workspace)
    base, layers, stride, page_bytes, page = _layers(pool, pages, device)
    if children.shape[0] != n:
        _refuse(f"fork: {n} parents, {children.shape[0]} children")
    table, slots, most, lens, _ = _tables(table, lens, None, 0, "fork", device)
    hold, ws, size = _pages_workspace(refs, max(n, 1), workspace)
    call("fml_kv4_fork", base, layers, stride, page_bytes, _ints(refs, "refs", device), table, lens,
         _ints(parents, "parents", device), _ints(children, "children", device), n, pages, slots, most, page,
         _ints(status, "status", device), ws, size, _raw_stream(device))


def free(refs, table, lens, slot_ids, status):
    """Give the slots' pages back (fml_kv4_free)."""
    n, device = slot_ids.shape[0], refs.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, free, refs, table, lens, slot_ids, status)
    table, slots, most, lens, slot_ids = _tables(table, lens, slot_ids, n, "free", device)
    call("fml_kv4_free", _ints(refs, "refs", device), table, lens, slot_ids, n, refs.shape[0], slots, most,
         _ints(status, "status", device), _raw_stream(device))


def compact(pool, refs, table, workspace=None):
    """Move the used pages together, in every layer of pool (fml_kv4_compact)."""
    pages, device = refs.shape[0], refs.get_device()
    if device < 0 or device != torch.cuda.current_device():
        return _elsewhere(device, compact, pool, refs, table, workspace)
    base, layers, stride, page_bytes, _ = _layers(pool, pages, device)
    hold, ws, size = _pages_workspace(refs, 0, workspace)
    call("fml_kv4_compact", base, layers, stride, page_bytes, _ints(refs, "refs", device),
         _ints(table, "table", device, 2), pages, table.shape[0], table.shape[1], ws, size, _raw_stream(device))


class KV4Cache:
    """The pools, tables, lengths and counts of one model's 4-bit cache.

    A step: reserve(counts); for each layer append(layer, k, v, starts) and
    attention(layer, out, q).  check() reads the status word (it waits); until it
    has told of a refused reserve, the rows that were there are not written."""

    def __init__(self, layers, kv_heads, head_dim, pages, page_size=64, slots=1, max_pages=None, device="cuda"):
        self.page_size = page_size
        self.pool = empty_pool(layers, pages, kv_heads, page_size, head_dim, device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.table = torch.full((slots, max_pages or pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.kept = torch.zeros(slots, dtype=torch.int32, device=device)

    def reserve(self, counts, slot_ids=None):
        reserve(self.refs, self.table, self.lens, counts, self.page_size, self.status, slot_ids, kept=self.kept)

    def append(self, layer, k, v, starts, slot_ids=None):
        append(self.pool[layer], self.table, self.lens, k, v, starts, slot_ids, self.kept)

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
        self.kept.zero_()
        if bits:
            raise FmlError(5, "KV4Cache", reasons(bits))
