"""The owner of a paged cache's pages and the pools behind it, over s1_pages_* and s1_pages_copy.

A Pages object knows which page holds which tokens of which sequence; pools are the device
buffers [n_pages, page bytes] that share its page numbers (keys and values of every full-attention
layer; recurrent states and convolution tails can be another set). append, fork, truncate and compact
keep the tables and return the copies that have to run; `copy` queues them over all pools of a set.
"""
import ctypes as C

import numpy as np

from . import lib as L


class Pages:
    def __init__(self, n_pages, page_tokens, max_seqs, max_seq_pages):
        self.lib = L.load()
        self.n_pages, self.page_tokens = int(n_pages), int(page_tokens)
        self.max_seqs, self.max_seq_pages = int(max_seqs), int(max_seq_pages)
        self.handle = C.c_void_p()
        L.check(self.lib.s1_pages_create(self.n_pages, self.page_tokens, self.max_seqs, self.max_seq_pages, C.byref(self.handle)), "pages")

    def close(self):
        if self.handle:
            self.lib.s1_pages_destroy(self.handle)
            self.handle = None

    def _copies(self, call, cap, what):
        src, dst, n = np.zeros(max(cap, 1), np.int32), np.zeros(max(cap, 1), np.int32), C.c_int(0)
        L.check(call(src.ctypes.data, dst.ctypes.data, cap, C.byref(n)), what)
        return [(int(a), int(b)) for a, b in zip(src[:n.value], dst[:n.value])]

    def append(self, seq, tokens):
        """Room for `tokens` more tokens; the copies (source, destination) that must run before they are written."""
        return self._copies(lambda *a: self.lib.s1_pages_append(self.handle, seq, tokens, *a), 1, "pages append")

    def fork(self, source, to):
        L.check(self.lib.s1_pages_fork(self.handle, source, to), "pages fork")

    def truncate(self, seq, tokens=0):
        L.check(self.lib.s1_pages_truncate(self.handle, seq, tokens), "pages truncate")

    def compact(self):
        return self._copies(lambda *a: self.lib.s1_pages_compact(self.handle, *a), self.n_pages, "pages compact")

    def free_pages(self):
        return self.lib.s1_pages_free_count(self.handle)

    def table(self, seq=0, n=None):
        """(page table [n, max_seq_pages], tokens [n]) of the sequences from `seq` on, int32. s1_attention_paged goes by the
        table's size (whether there are windows, and how large the caches may be): give it the rows of a step's sequences,
        and the columns that the longest of them may come to fill."""
        n = self.max_seqs - seq if n is None else n
        table, tokens = np.empty((n, self.max_seq_pages), np.int32), np.empty(n, np.int32)
        L.check(self.lib.s1_pages_table(self.handle, seq, n, table.ctypes.data, self.max_seq_pages, tokens.ctypes.data), "pages table")
        return table, tokens


def copy(pools, n_pages, page_bytes, pairs, stream):
    """Queue copies (source page, destination page) over every pool (device pointers) on `stream`."""
    if not pairs:
        return
    ptrs = (C.c_void_p * len(pools))(*[p.value if isinstance(p, C.c_void_p) else p for p in pools])
    src, dst = (np.array([p[i] for p in pairs], np.int32) for i in (0, 1))
    L.check(L.load().s1_pages_copy(ptrs, len(pools), n_pages, page_bytes, src.ctypes.data, dst.ctypes.data, len(pairs), stream.handle),
            "page copies")
