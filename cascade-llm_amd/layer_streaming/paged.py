"""KV cache of several sequences in pages.

The reference's cache holds one request (``SimpleKVCache``, layer_streaming/
llama31.py:34-54).  Continuations of one prompt, or a batch of requests, keep
their keys and values in pages instead: runs of ``page_size`` positions that
a page table assigns to sequences.  ``fork`` shares a sequence's pages with
its copies, and a page is copied only when one of them writes to it.

The host decides which page holds what (this class); the device holds the
pages, the page table and the lengths, and the kernels of libcascade_hip
read them there: ``append`` (cascade_paged_append_bf16), ``attend``
(cascade_paged_decode_attention_bf16) and the copies of ``extend`` and
``compact`` (cascade_copy_pages).  Table, lengths and pools never move, so a
captured graph of a decode step serves every later step: ``extend`` makes room and
updates them in place.  It, and whatever else assigns pages, refuses to run
while a graph is captured: a replay would bring its pages back.

Work is enqueued on the current stream; calls on several streams have to be
ordered by the caller.
"""

import heapq
import operator

import torch

from . import _hip

__all__ = ["PagedKVCache"]


class PagedKVCache:
    """Pages of up to ``max_sequences`` sequences of up to ``max_length``
    positions.

    ``buffer``: bf16 [layers, 2 (K, V), num_pages, kv_heads, page_size,
    head_dim].  ``page_table`` (int32 [max_sequences, pages of one], -1 where
    there is no page) and ``lengths`` (int32 [max_sequences]) are on the
    device.  A sequence is named by its table row.  ``head_dim``: a multiple
    of 16 of up to 1024; ``attend`` takes 64 and 128.
    """

    def __init__(self, num_pages, max_sequences, max_length, layer_count=32,
                 num_kv_heads=8, head_dim=128, page_size=64, device=None):
        for name, value in (("num_pages", num_pages),
                            ("max_sequences", max_sequences),
                            ("max_length", max_length),
                            ("layer_count", layer_count),
                            ("num_kv_heads", num_kv_heads)):
            if int(value) < 1:
                raise ValueError("{} must be positive".format(name))
        page_size = int(page_size)
        if not 8 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two of 8 to 1024")
        if not 16 <= int(head_dim) <= 1024 or int(head_dim) % 16:
            raise ValueError("head_dim must be a multiple of 16 of 16 to 1024")
        self.num_pages = int(num_pages)
        self.max_sequences = int(max_sequences)
        self.page_size = page_size
        self.max_pages = -(-int(max_length) // page_size)
        self.max_length = int(max_length)
        self.layer_count = int(layer_count)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)
        self.device = torch.device("cuda" if device is None else device)
        self.buffer = torch.empty(
            (self.layer_count, 2, self.num_pages, self.num_kv_heads, page_size,
             self.head_dim), dtype=torch.bfloat16, device=self.device)
        self.device = self.buffer.device  # with its index: the current one may change
        self.page_table = torch.full((self.max_sequences, self.max_pages), -1,
                                     dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(self.max_sequences, dtype=torch.int32,
                                   device=self.device)
        self.error = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._pages = [None] * self.max_sequences  # page numbers, None: unused row
        self._lengths = [0] * self.max_sequences
        self._refs = [0] * self.num_pages
        self._free = list(range(self.num_pages))  # a heap: low pages first
        self._workspaces = []  # growing ones; a captured graph may hold any

    # ------------------------------------------------------------- sequences

    def add(self):
        """A new empty sequence; returns its table row."""

        for row, pages in enumerate(self._pages):
            if pages is None:
                self._pages[row] = []
                self._lengths[row] = 0
                return row
        raise RuntimeError("all {} sequences are in use".format(self.max_sequences))

    def length(self, row):
        self._of(row)
        return self._lengths[row]

    def pages(self, row):
        """Page numbers of a sequence, in order."""

        return list(self._of(row))

    @property
    def free_pages(self):
        return len(self._free)

    def extend(self, rows, count=1):
        """Make room for ``count`` more positions of each sequence of
        ``rows`` and advance its length by them (write them with ``append``
        at positions length - count .. length - 1).  A partly filled last
        page that other sequences share is copied first.  Raises without any
        change when a row or the pool is too small."""

        rows, count = [operator.index(row) for row in rows], int(count)
        self._outside_graph()
        if count < 1:
            raise ValueError("count must be positive")
        if not rows:
            return
        if len(set(rows)) != len(rows):
            raise ValueError("a sequence occurs twice")
        # pages to take, and shared last pages; of the sequences that share
        # one, the last to write in it may keep it
        needed, copies, writers = 0, [], {}
        for row in rows:
            pages, length = self._of(row), self._lengths[row]
            if length + count > self.max_length:
                raise RuntimeError("sequence {} would exceed {} positions".format(
                    row, self.max_length))
            needed += -(-(length + count) // self.page_size) - len(pages)
            if length % self.page_size:
                page = pages[-1]
                writers[page] = writers.get(page, 0) + 1
                if self._refs[page] - writers[page] >= 1:
                    copies.append(row)
                    needed += 1
        if needed > len(self._free):
            raise RuntimeError("{} pages needed, {} free".format(
                needed, len(self._free)))
        moves = []
        for row in copies:
            pages = self._pages[row]
            old, new = pages[-1], self._take()
            moves.append((old, new))
            self._refs[old] -= 1
            pages[-1] = new
        for row in rows:
            self._lengths[row] += count
            pages = self._pages[row]
            while len(pages) * self.page_size < self._lengths[row]:
                pages.append(self._take())
        self._copy(moves)
        self._publish(rows)

    def fork(self, row, count=1):
        """``count`` new sequences with the pages of ``row``; returns their
        rows.  Nothing is copied until one of them is extended."""

        self._outside_graph()
        pages = self._of(row)
        if sum(p is None for p in self._pages) < count:
            raise RuntimeError("all {} sequences are in use".format(self.max_sequences))
        out = []
        for _ in range(int(count)):
            new = self.add()
            self._pages[new] = list(pages)
            self._lengths[new] = self._lengths[row]
            for page in pages:
                self._refs[page] += 1
            out.append(new)
        if out:
            self._publish(out)
        return out

    def truncate(self, row, length):
        """Drop the positions of a sequence from ``length`` on."""

        self._outside_graph()
        pages = self._of(row)
        length = int(length)
        if not 0 <= length <= self._lengths[row]:
            raise ValueError("length {} is outside [0, {}]".format(
                length, self._lengths[row]))
        self._drop(row, -(-length // self.page_size))
        self._lengths[row] = length
        self._publish([row])

    def free(self, row):
        """End a sequence; pages that no other one holds become free."""

        self._outside_graph()
        self._of(row)
        self._drop(row, 0)
        self._lengths[row] = 0
        self._publish([row])
        self._pages[row] = None

    def compact(self):
        """Move the pages in use to the front of the pool (so that its tail
        can be given up, or copied out); returns how many moved."""

        self._outside_graph()
        used = [p for p in range(self.num_pages) if self._refs[p]]
        # a page at or behind `len(used)` moves into a free one before it:
        # no page is both a source and a destination
        holes = [p for p in range(len(used)) if not self._refs[p]]
        moved = dict(zip((p for p in used if p >= len(used)), holes))
        if not moved:
            return 0
        for old, new in moved.items():
            self._refs[new], self._refs[old] = self._refs[old], 0
        touched = []
        for row, pages in enumerate(self._pages):
            if pages and any(p in moved for p in pages):
                self._pages[row] = [moved.get(p, p) for p in pages]
                touched.append(row)
        self._free = list(range(len(used), self.num_pages))
        self._copy(list(moved.items()))
        self._publish(touched)
        return len(moved)

    def _of(self, row):
        if not 0 <= row < self.max_sequences or self._pages[row] is None:
            raise ValueError("there is no sequence {}".format(row))
        return self._pages[row]

    def _outside_graph(self):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages cannot be assigned while a graph is captured")

    def _take(self):
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, row, keep):
        for page in self._pages[row][keep:]:
            self._refs[page] -= 1
            if self._refs[page] == 0:
                heapq.heappush(self._free, page)
        del self._pages[row][keep:]

    def _upload(self, values, dtype=torch.int32):
        # pinned memory of torch's caching allocator, which holds it until
        # the copy behind it has run
        host = torch.tensor(values, dtype=dtype, pin_memory=self.device.type == "cuda")
        return host.to(self.device, non_blocking=True)

    def _copy(self, moves):
        if moves:
            _hip.copy_pages(self.buffer, self._upload(moves), error_flag=self.error)

    def _publish(self, rows):
        """Write the page numbers and lengths of ``rows`` to the device."""

        width = self.max_pages
        table = [self._pages[r] + [-1] * (width - len(self._pages[r])) for r in rows]
        data = self._upload([t + [self._lengths[r], r] for t, r in zip(table, rows)])
        at = data[:, -1].long()
        self.page_table.index_copy_(0, at, data[:, :width])
        self.lengths.index_copy_(0, at, data[:, width])

    # ------------------------------------------------------------- operators

    def k_pages(self, layer):
        return self.buffer[layer, 0]

    def v_pages(self, layer):
        return self.buffer[layer, 1]

    def append(self, layer, q, k, v, positions, rows=None, rope=None,
               interleaved=False, q_out=None):
        """``paged_append`` into one layer's pages."""

        return _hip.paged_append(
            q, k, v, positions, self.buffer[layer, 0], self.buffer[layer, 1],
            self.page_table, rows=rows, rope=rope, interleaved=interleaved,
            q_out=q_out, error_flag=self.error)

    def attend(self, layer, q, out, rows=None, scale=None, workspace=None,
               max_length=None):
        """``paged_decode_attention`` over one layer's pages (heads of 64 or
        128); ``scale`` defaults to head_dim ** -0.5, ``workspace`` to one
        that the cache keeps (give one of your own to calls that may
        overlap)."""

        if self.head_dim not in (64, 128):
            raise ValueError("attention takes heads of 64 or 128, these have {}".format(
                self.head_dim))
        limit = self.max_length if max_length is None else max_length
        if workspace is None:
            workspace = self._attention_workspace(q.shape[0], q.shape[1])
        return _hip.paged_decode_attention(
            q, self.buffer[layer, 0], self.buffer[layer, 1], self.page_table,
            self.lengths, out, workspace,
            self.head_dim ** -0.5 if scale is None else scale, rows=rows,
            max_length=limit, error_flag=self.error)

    def _attention_workspace(self, batch, q_heads):
        # for any limit that a call may give: what a table row holds, and the
        # operator takes
        limit = min(self.max_pages * self.page_size, 0x7fffffff - 64)
        need = _hip.paged_attention_workspace_bytes(
            max(batch, 1), q_heads, self.num_kv_heads, self.head_dim, limit)
        if not self._workspaces or self._workspaces[-1].numel() < need:
            self._workspaces.append(
                torch.empty(need, dtype=torch.uint8, device=self.device))
        return self._workspaces[-1]

    def load(self, row, kv_cache):
        """Copy the positions of a ``SimpleKVCache`` behind those of a
        sequence (a prompt that the executor has prefilled)."""

        count = kv_cache.sequence_length()
        if count == 0:
            return
        if kv_cache.buffer.device != self.buffer.device:
            raise ValueError("the caches live on {} and {}".format(
                kv_cache.buffer.device, self.buffer.device))
        if kv_cache.lengths != [count] * kv_cache.layer_count:
            raise ValueError("the layers of the cache differ in length")
        if (kv_cache.layer_count, kv_cache.num_kv_heads, kv_cache.head_dim) != (
                self.layer_count, self.num_kv_heads, self.head_dim):
            raise ValueError("the caches differ in layers, heads or head size")
        start = self.length(row)
        self.extend([row], count)
        positions = torch.arange(start, start + count, dtype=torch.int32,
                                 device=self.device)
        rows = torch.full_like(positions, row)
        for layer in range(self.layer_count):
            k, v = (kv_cache.buffer[layer, which, :, :count].transpose(0, 1)
                    for which in (0, 1))
            self.append(layer, None, k, v, positions, rows=rows)

    def check(self):
        """Raise if an operator met an index out of range (waits for the
        GPU)."""

        if int(self.error.item()):
            self.error.zero_()
            raise RuntimeError("a paged operator met a row, position, length or "
                               "page out of range")
