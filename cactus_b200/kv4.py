"""Python handle over the 4-bit paged KV cache (include/cactus_b200_kv4.h).

Thin ctypes plumbing: sequence numbers, row counts and kept rows are host integers; keys, values,
queries and results are fp16 (log-sum-exps fp32) arrays in device memory, given as addresses or as
objects with ``data_ptr()``. Strides are in elements.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import CactusError, check, lib


def _addr(x):
    return None if x is None else x if isinstance(x, int) else x.data_ptr()


def _host(v):
    """A list of sequences, counts or rows as int32 values, none of them changed on the way."""
    a = np.asarray(v).reshape(-1)
    if a.size and (a.dtype.kind not in "iu" or int(a.min()) < -2 ** 31 or int(a.max()) >= 2 ** 31):
        raise CactusError(f"lists hold whole numbers of 32 bits: got {a.dtype} {a[:4]}")
    a = np.ascontiguousarray(a, np.int32)
    return a, a.ctypes.data_as(C.c_void_p)


def _seq(v):
    """One sequence number: ctypes would take the low 32 bits of a larger one."""
    return int(_host([v])[0][0])


def rope_table(theta: float, rotary_dim: int, positions: int, table, stream: int = 0):
    """Fills table [positions][rotary_dim / 2][2] (fp32, device) with the turns that rope_append takes."""
    check(lib().cactus_cuda_rope_table(theta, rotary_dim, positions, _addr(table), stream), "rope_table")


class KVCache4:
    def __init__(self, layers: int, q_heads: int, kv_heads: int, head_dim: int, num_pages: int, max_seqs: int,
                 max_context: int, max_tokens: int, group_size: int = 32, page_size: int = 64, device: int = 0):
        self._L = lib()
        self.layers, self.q_heads, self.kv_heads, self.head_dim = layers, q_heads, kv_heads, head_dim
        self.h = self._L.cactus_kv4_create(layers, q_heads, kv_heads, head_dim, group_size, page_size, num_pages,
                                           max_seqs, max_context, max_tokens, device)
        if not self.h:
            raise CactusError("cactus_kv4_create failed: " + self._L.cactus_cuda_last_error().decode(errors="replace"))

    def close(self):
        if self.h:
            self._L.cactus_kv4_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def begin(self, seqs, new_rows, stream: int = 0):
        """Room for new_rows[i] rows in sequence seqs[i]; the batch of the next append and attention calls."""
        (s, sp), (n, np_) = _host(seqs), _host(new_rows)
        if s.size != n.size:
            raise CactusError("begin: as many row counts as sequences are needed")
        check(self._L.cactus_kv4_begin(self.h, sp, np_, s.size, stream), "kv4_begin")

    def append(self, layer: int, keys, values, row_stride: int | None = None, stream: int = 0):
        check(self._L.cactus_kv4_append(self.h, layer, _addr(keys), _addr(values),
                                        row_stride or self.kv_heads * self.head_dim, stream), "kv4_append")

    def rope_append(self, layer: int, keys, values, table, positions: int, rotary_dim: int, queries=None, rotated=None,
                    q_weight=None, k_weight=None, eps: float = 1e-6, row_stride: int | None = None,
                    query_stride: int | None = None, rotated_stride: int | None = None, stream: int = 0):
        """Normalises and turns keys and queries at their positions, appends keys and values."""
        wide = self.q_heads * self.head_dim
        check(self._L.cactus_kv4_rope_append(self.h, layer, _addr(queries), query_stride or wide, _addr(rotated),
                                             rotated_stride or wide, _addr(keys), _addr(values),
                                             row_stride or self.kv_heads * self.head_dim, _addr(table), positions,
                                             rotary_dim, _addr(q_weight), _addr(k_weight), eps, stream),
              "kv4_rope_append")

    def attention(self, layer: int, queries, output, scale: float, lse=None, query_stride: int | None = None,
                  window: int = 0, causal: bool = True, stream: int = 0):
        check(self._L.cactus_kv4_attention(self.h, layer, _addr(queries),
                                           query_stride or self.q_heads * self.head_dim, _addr(output), _addr(lse),
                                           scale, window, int(causal), stream), "kv4_attention")

    def read(self, layer: int, seq: int, first: int, count: int, keys, values, stream: int = 0):
        check(self._L.cactus_kv4_read(self.h, layer, _seq(seq), first, count, _addr(keys), _addr(values), stream),
              "kv4_read")

    def fork(self, src, dst):
        """Sequences dst become copies of src (pages shared until they are written)."""
        (s, sp), (d, dp) = _host(src), _host(dst)
        if s.size != d.size:
            raise CactusError("fork: as many destinations as sources are needed")
        check(self._L.cactus_kv4_fork(self.h, sp, dp, s.size), "kv4_fork")

    def truncate(self, seq: int, length: int):
        check(self._L.cactus_kv4_truncate(self.h, _seq(seq), length), "kv4_truncate")

    def free(self, seqs):
        s, sp = _host(seqs)
        check(self._L.cactus_kv4_free(self.h, sp, s.size), "kv4_free")

    def compact(self, seqs, kept, stream: int = 0):
        """Sequence seqs[i] keeps its rows kept[i], in that order."""
        s, sp = _host(seqs)
        if s.size != len(kept):
            raise CactusError("compact: a list of rows for each sequence is needed")
        kept = [_host(k)[0] for k in kept]
        rows, rp = _host(np.concatenate(kept) if kept else [])
        offs, op = _host(np.concatenate([[0], np.cumsum([len(k) for k in kept], dtype=np.int64)]))
        check(self._L.cactus_kv4_compact(self.h, sp, rp, op, s.size, stream), "kv4_compact")

    def slide(self, seqs, sink: int, window: int, stream: int = 0):
        """Sequences keep their first `sink` rows and their last ones, `window` in all."""
        if sink < 0 or window < 0:
            raise CactusError("slide: sink and window must not be negative")
        kept = []
        for s in seqs:
            n = self.length(s)
            first = min(sink, window, n)
            kept.append(np.concatenate([np.arange(first), np.arange(max(first, n - (window - first)), n)]))
        self.compact(seqs, kept, stream)

    def length(self, seq: int) -> int:
        n = self._L.cactus_kv4_length(self.h, _seq(seq))
        if n < 0:
            check(n, "kv4_length")
        return n

    def info(self):
        out = (C.c_size_t * 4)()
        check(self._L.cactus_kv4_info(self.h, out), "kv4_info")
        return dict(zip(("pages", "free_pages", "page_bytes", "pool_bytes"), (int(v) for v in out)))
