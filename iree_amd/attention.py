"""The attention block of a language model on a cache held in 4 bits.

Thin wrappers of the entry points that include/iree_amd_uk.h describes under that
heading (formulas, layout, what is refused), and ``Kv4Cache``, which keeps a pool of
pages and the page tables of the sequences in it. As in ``ukernel``, tensors own the
device memory, sizes are given, strides default to tight, and work is enqueued on
torch's current stream; every tensor lies on the current device.
"""
import ctypes as C
import functools

import torch

from . import flags as F
from ._lib import load_library
from .ukernel import _check, _raw_stream, _stream

_ROW_TYPES = {F.ATTENTION_TYPE_F16: torch.float16, F.ATTENTION_TYPE_BF16: torch.bfloat16}


_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _device():
    # (-1 is what a CPU tensor says: it matches no device)
    try:
        return _get_device()
    except RuntimeError:
        return -2


def _tensor(t, dtype, name, device):
    """Address of a tensor of that type on the current device; None stays None."""
    if t is None:
        return None
    where = t.get_device()
    if where != device or where < 0:
        raise ValueError(f"{name} must be a tensor on the current CUDA (HIP) device")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    return t.data_ptr()


def _stream_on(stream, device):
    if stream is None and _raw_stream is not None:
        return _raw_stream(device)
    return _stream(stream)


def _row_type(flags):
    return _ROW_TYPES.get(flags & F.ATTENTION_TYPE_MASK)


def kv4_page_bytes(page_size, kv_heads, head_dim):
    """Bytes of one page of one layer. Needs no device."""
    out = C.c_int64(0)
    _check(load_library().iree_amd_uk_kv4_page_bytes(page_size, kv_heads, head_dim, C.byref(out)))
    return out.value


def qk_norm_rope(q, k, q_out, k_out, tokens, heads, kv_heads, head_dim, flags, *, q_weight=None, k_weight=None,
                 eps=1e-6, cos_sin=None, table_rows=0, rotary_dim=0, positions=None, q_stride0=None, k_stride0=None,
                 q_out_stride0=None, k_out_stride0=None, v=None, v_stride0=None, cache=None, pages=0,
                 page_stride=None, page_size=0, slots=None, stream=None):
    """RMS norm and rotation of every query and key head; with ``cache``, keys and values
    go into the 4-bit cache at ``slots`` in the same launch. ``q``, or ``k`` and ``v``, may
    be None, and with a cache ``k_out`` too."""
    rows, device = _row_type(flags), _device()
    if page_stride is None:
        page_stride = kv_heads * page_size * (head_dim + 8)
    q_row, kv_row = heads * head_dim, kv_heads * head_dim
    _check(load_library().iree_amd_uk_qk_norm_rope(
        _tensor(q, rows, "q", device), q_row if q_stride0 is None else q_stride0,
        _tensor(k, rows, "k", device), kv_row if k_stride0 is None else k_stride0,
        _tensor(v, rows, "v", device), kv_row if v_stride0 is None else v_stride0,
        _tensor(q_out, rows, "q_out", device), q_row if q_out_stride0 is None else q_out_stride0,
        _tensor(k_out, rows, "k_out", device), kv_row if k_out_stride0 is None else k_out_stride0,
        _tensor(q_weight, rows, "q_weight", device), _tensor(k_weight, rows, "k_weight", device), eps,
        _tensor(cos_sin, torch.float32, "cos_sin", device), table_rows, rotary_dim,
        _tensor(positions, torch.int32, "positions", device), _tensor(cache, None, "cache", device), pages,
        page_stride, page_size, _tensor(slots, torch.int64, "slots", device), tokens, heads, kv_heads, head_dim, flags,
        _stream_on(stream, device)))


def kv4_read(cache, pages, page_size, slots, k_out, v_out, rows, kv_heads, head_dim, flags, *, page_stride=None,
             k_out_stride0=None, v_out_stride0=None, stream=None):
    """The K and V rows that the cache holds at ``slots``; ``k_out`` or ``v_out`` may be None."""
    kind, row, device = _row_type(flags), kv_heads * head_dim, _device()
    if page_stride is None:
        page_stride = kv_heads * page_size * (head_dim + 8)
    _check(load_library().iree_amd_uk_kv4_read(
        _tensor(cache, None, "cache", device), pages, page_stride, page_size,
        _tensor(slots, torch.int64, "slots", device),
        _tensor(k_out, kind, "k_out", device), row if k_out_stride0 is None else k_out_stride0,
        _tensor(v_out, kind, "v_out", device), row if v_out_stride0 is None else v_out_stride0, rows, kv_heads, head_dim,
        flags, _stream_on(stream, device)))


def attention_kv4_workspace(tokens, batch, heads, kv_heads, head_dim, *, max_kv_len, window=0, sinks=0):
    """Bytes of workspace that ``attention_kv4`` of these sizes uses (0: none). ``max_kv_len``: the
    call's own, or ``max_pages * page_size`` for a call without one."""
    out = C.c_uint64(0)
    _check(load_library().iree_amd_uk_attention_kv4_workspace(
        tokens, batch, heads, kv_heads, head_dim, window, sinks, max_kv_len, C.byref(out)))
    return out.value


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device, tokens, batch, heads, kv_heads, head_dim, window, sinks, max_kv_len):
    # (it follows from the sizes and the device alone, and a decode step asks again and again)
    return attention_kv4_workspace(tokens, batch, heads, kv_heads, head_dim, max_kv_len=max_kv_len, window=window,
                                   sinks=sinks)


def attention_kv4(q, out, cache, pages, page_size, page_table, q_starts, kv_lens, tokens, batch, heads, kv_heads,
                  head_dim, max_pages, flags, *, scale, window=0, sinks=0, max_kv_len=None, page_stride=None,
                  page_table_stride=None, q_stride0=None, out_stride0=None, workspace=None, stream=None):
    """Attention of the query tokens of ``batch`` sequences over the paged 4-bit cache,
    causal, optionally with a sliding window and ``sinks`` first tokens that stay visible.
    ``max_kv_len``: the longest of ``kv_lens`` as far as the caller knows (None or 0: as many as the
    page table holds). Without a ``workspace`` the call takes one from torch's allocator for its own
    duration."""
    kind, row, device = _row_type(flags), heads * head_dim, _device()
    if page_stride is None:
        page_stride = kv_heads * page_size * (head_dim + 8)
    capacity = max_pages * page_size
    max_kv_len = min(max_kv_len or capacity, capacity)
    where = _tensor(q, kind, "q", device)
    if workspace is None and max_kv_len:
        nbytes = _workspace_bytes(device, tokens, batch, heads, kv_heads, head_dim, window, sinks, max_kv_len)
        if nbytes:
            workspace = _workspace(nbytes, stream)
    _check(load_library().iree_amd_uk_attention_kv4(
        where, row if q_stride0 is None else q_stride0,
        _tensor(out, kind, "out", device), row if out_stride0 is None else out_stride0,
        _tensor(cache, None, "cache", device), pages, page_stride, page_size,
        _tensor(page_table, torch.int32, "page_table", device),
        max_pages if page_table_stride is None else page_table_stride, max_pages,
        _tensor(q_starts, torch.int32, "q_starts", device), _tensor(kv_lens, torch.int32, "kv_lens", device), tokens,
        batch, heads, kv_heads, head_dim, scale, window, sinks, max_kv_len,
        _tensor(workspace, None, "workspace", device), 0 if workspace is None else workspace.nbytes, flags,
        _stream_on(stream, device)))


def _workspace(nbytes, stream):
    # (the allocator hands freed memory out again on the stream it was taken on)
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    if type(stream) is int:
        stream = torch.cuda.ExternalStream(stream)
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device="cuda")


def copy_pages(pool, pages, page_bytes, src, dst, *, page_stride=None, stream=None):
    """Page ``src[i]`` to page ``dst[i]`` inside a pool; ``src`` and ``dst`` are page
    numbers on the host (int32 CPU tensors, or sequences)."""
    src, dst, device = _host_pages(src), _host_pages(dst), _device()
    if src.numel() != dst.numel():
        raise ValueError("src and dst must have as many pages")
    _check(load_library().iree_amd_uk_copy_pages(
        _tensor(pool, None, "pool", device), pages, page_bytes, page_bytes if page_stride is None else page_stride,
        src.data_ptr(), dst.data_ptr(), src.numel(), _stream_on(stream, device)))


def _host_pages(v):
    if not isinstance(v, torch.Tensor):
        v = torch.tensor(list(v), dtype=torch.int32)
    if v.is_cuda or v.dtype != torch.int32 or not v.is_contiguous():
        raise ValueError("page numbers must be a contiguous int32 CPU tensor or a sequence")
    return v


class Kv4Cache:
    """A pool of pages of a 4-bit cache for ``layers`` layers, and the sequences in it.

    A page holds ``page_size`` tokens of every layer side by side, so one page number
    stands for all of them. The tables live on the host; ``tables`` makes the tensors
    that a step needs. Pages are counted: ``fork`` shares the full pages of a sequence
    and copies the last, partly filled one, so tokens are only ever appended to pages
    of one owner. All device work goes to torch's current stream; a program that uses
    several orders them itself.
    """

    def __init__(self, pages, page_size, layers, kv_heads, head_dim, device="cuda"):
        if pages < 0 or layers < 1 or kv_heads < 1:
            raise ValueError("pages, layers and kv_heads must be positive")
        self.page_size, self.layers, self.kv_heads, self.head_dim = page_size, layers, kv_heads, head_dim
        self.pages, self.layer_bytes = pages, kv4_page_bytes(page_size, kv_heads, head_dim)
        self.page_bytes = layers * self.layer_bytes
        self.buffer = torch.zeros(pages, self.page_bytes, dtype=torch.uint8, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._owners = [0] * pages
        self._tables, self._lens, self._next = {}, {}, 0

    def layer(self, index):
        """The cache of one layer: what the entry points take with ``page_stride=page_bytes``."""
        if not 0 <= index < self.layers:
            raise ValueError("no such layer")
        return self.buffer.view(-1)[index * self.layer_bytes:]

    def free_pages(self):
        return len(self._free)

    def length(self, sequence):
        return self._lens[sequence]

    def new(self):
        """An empty sequence."""
        self._next += 1
        self._tables[self._next], self._lens[self._next] = [], 0
        return self._next

    def _take(self):
        page = self._free.pop()
        self._owners[page] = 1
        return page

    def _give(self, page):
        if page < 0:
            return
        self._owners[page] -= 1
        if not self._owners[page]:
            self._free.append(page)

    def extend(self, sequences, counts):
        """Room for ``counts[i]`` more tokens of ``sequences[i]`` (each once); the slots of
        the new tokens, sequence by sequence, as the int64 tensor that ``qk_norm_rope``
        takes. Raises MemoryError, with nothing changed, when the pool has too few pages."""
        if len(sequences) != len(counts) or len(set(sequences)) != len(sequences) or any(n < 0 for n in counts):
            raise ValueError("every sequence once, with a count that is not negative")
        size = self.page_size
        need = [-(-(self._lens[s] + n) // size) - len(self._tables[s]) for s, n in zip(sequences, counts)]
        if sum(need) > len(self._free):
            raise MemoryError(f"{sum(need)} pages needed, {len(self._free)} free")
        slots = []
        for s, n, more in zip(sequences, counts, need):
            table, at = self._tables[s], self._lens[s]
            table.extend(self._take() for _ in range(more))
            slots.extend(table[t // size] * size + t % size for t in range(at, at + n))
            self._lens[s] = at + n
        return torch.tensor(slots, dtype=torch.int64).to(self.buffer.device)

    def fork(self, sequence):
        """A sequence with the same tokens: full pages are shared, the last one is copied if
        it is partly filled. Raises MemoryError when that needs a page and none is free."""
        table, length = list(self._tables[sequence]), self._lens[sequence]
        if length % self.page_size and table[-1] >= 0:
            if not self._free:
                raise MemoryError("1 page needed, 0 free")
            page = self._take()
            try:
                copy_pages(self.buffer, self.pages, self.page_bytes, [table[-1]], [page])
            except Exception:
                self._give(page)
                raise
            table[-1] = page
            shared = table[:-1]
        else:
            shared = table
        for page in shared:
            if page >= 0:
                self._owners[page] += 1
        self._next += 1
        self._tables[self._next], self._lens[self._next] = table, length
        return self._next

    def free(self, sequence):
        """Ends a sequence; pages that no other shares return to the pool."""
        del self._lens[sequence]
        for page in self._tables.pop(sequence):
            self._give(page)

    def drop(self, sequence, window, sinks=0):
        """Frees the pages of a sequence that no token from its next one on sees through a
        sliding window with ``sinks``; their entries of the table become -1."""
        if window < 1 or sinks < 0:
            raise ValueError("window must be positive and sinks not negative")
        first = self._lens[sequence] - window + 1      # the first token that the next one's window holds
        table = self._tables[sequence]
        for i in range(-(-sinks // self.page_size), max(0, first) // self.page_size):
            self._give(table[i])
            table[i] = -1

    def compact(self):
        """Moves the pages in use to the front of the pool; returns how many there are.
        The tables of every sequence follow (call ``tables`` again for a step)."""
        used = self.pages - len(self._free)
        src = [p for p in range(used, self.pages) if self._owners[p]]
        dst = [p for p in range(used) if not self._owners[p]]
        if src:
            copy_pages(self.buffer, self.pages, self.page_bytes, src, dst)
        moved = dict(zip(src, dst))
        for old, new in moved.items():
            self._owners[new], self._owners[old] = self._owners[old], 0
        for table in self._tables.values():
            table[:] = [moved.get(p, p) for p in table]
        self._free = list(range(self.pages - 1, used - 1, -1))
        return used

    def tables(self, sequences):
        """(page_table, kv_lens, max_pages) of a batch: int32 tensors on the device for
        ``attention_kv4``, the table as wide as the longest of them."""
        rows = [self._tables[s] for s in sequences]
        wide = max(map(len, rows), default=0)
        table = torch.tensor([r + [-1] * (wide - len(r)) for r in rows], dtype=torch.int32).reshape(len(rows), wide)
        lens = torch.tensor([self._lens[s] for s in sequences], dtype=torch.int32)
        return table.to(self.buffer.device), lens.to(self.buffer.device), wide
