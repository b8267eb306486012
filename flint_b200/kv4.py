"""A paged K/V cache of 4 bits a number (`fb_kv4_*` in include/flint_b200.h): appending with the position rotation, attention, moves.

`KvCache4` is the pool, the page table and the rotation's frequencies of a model whose layers share the table. The engine's own caches are bf16
tensors indexed by position (`DecodeEngine.kc`, reference: chat.py:68-69); this one holds a position and kv head in head_dim / 2 + 4 bytes each of K and V,
any number of sequences side by side. `DecodeEngine(..., kv_bits=4)` runs a model on it. There is no PyTorch arithmetic here: tensors are device memory handed to
the C ABI, calls are asynchronous on the current stream of the cache's GPU, and lengths given as device tensors are read when the kernels run, so a captured call
serves a sequence that grows. Two calls that write the same slots, or one that reads what another writes, are ordered by their streams, as with any tensor.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .engine import _ptr, _raw_stream

PAGE = 64                                                  # positions of a page
NO_SCRATCH = (1344, 64)                                    # positions of one sequence, and query rows of a kv head, up to which attention needs no scratch
Lengths = Union[int, torch.Tensor]


def rope_turns(head_dim: int, base: float, device) -> torch.Tensor:
    """Turns per position of the rotation pairs, base^(-2i / head_dim) / 2 pi, as whole multiples of 2^-64 in int64 [head_dim / 2]: times a position and modulo
    2^64 that is the angle, without the loss of a float at far positions."""
    turns = [round(base ** (-2.0 * i / head_dim) / (2.0 * math.pi) * 2.0 ** 64) for i in range(head_dim // 2)]
    return torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device)


def page_bytes(n_kv: int, head_dim: int) -> int:
    """Bytes of a page of one layer: 64 positions, K and V of all kv heads."""
    n = _lib.load().fb_kv4_page_bytes(n_kv, head_dim)
    if not n:
        raise ValueError(f"no 4-bit cache for {n_kv} kv heads of {head_dim}: head sizes are 64, 80 and 128")
    return n


class KvCache4:
    """`table` int32 [n_seq, pages a sequence may have], contiguous, on the GPU names the pages of every sequence; it stays the caller's, who may change its entries between
    calls. `pool` uint8 [n_layer, n_pages, n_kv, page bytes / n_kv] is allocated (zeroed) unless given. `rope_base` None: keys and queries come rotated."""

    def __init__(self, n_layer: int, n_pages: int, n_kv: int, head_dim: int, table: torch.Tensor, pool: Optional[torch.Tensor] = None,
                 rope_base: Optional[float] = None):
        self.lib = _lib.load()
        self.n_layer, self.n_pages, self.n_kv, self.head_dim = int(n_layer), int(n_pages), int(n_kv), int(head_dim)
        record = page_bytes(self.n_kv, self.head_dim) // self.n_kv
        self.device = table.device
        if self.device.type != "cuda":
            raise ValueError(f"the page table must be on the GPU that runs the kernels, not on {self.device}")
        # rows side by side: the kernels hold a length on the GPU against what a row has room for, and a wider step from row to row would let it into the next one
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[1] < 1 or not table.is_contiguous():
            raise ValueError("table must be contiguous int32 [n_seq, pages]")
        shape = (self.n_layer, self.n_pages, self.n_kv, record)
        if min(shape) < 1:
            raise ValueError(f"a pool of {shape} holds nothing")
        if pool is None:
            pool = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        if tuple(pool.shape) != shape or pool.dtype != torch.uint8 or not pool.is_contiguous() or pool.device != self.device or pool.data_ptr() % 16:
            raise ValueError(f"pool must be contiguous uint8 {shape} on {self.device}, 16-byte aligned")
        self.pool, self.table = pool, table
        self.layer_bytes = self.n_pages * self.n_kv * record
        self.freq = rope_turns(self.head_dim, float(rope_base), self.device) if rope_base is not None else None
        self._freq_ptr = _ptr(self.freq)
        self._status = torch.zeros(8, dtype=torch.int32, device=self.device)
        self._index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        self._ld = table.shape[1]
        self._n_seq = table.shape[0]
        self._f32 = torch.empty(0, dtype=torch.float32, device=self.device)
        # what every call says about the cache; a call copies it and adds its own (a call costs the host microseconds, as much as a short kernel)
        self._proto = bytes(_lib.Kv4Seqs(pool.data_ptr(), table.data_ptr(), None, None, self._status.data_ptr(), 0, self.n_pages, self.n_kv, self.head_dim,
                                         self._n_seq, self._ld, 0, self._index))

    # ------------------------------------------------------------------ plumbing
    @property
    def slots(self) -> int:
        """Positions that a sequence may have."""
        return self.table.shape[1] * PAGE

    def status(self):
        """Synchronises; (code, where, sequence) of the first call that met a page, length or path that cannot be since the last status(), code 0: none."""
        torch.cuda.synchronize(self.device)
        st = self._status.tolist()
        if st[0]:
            self._status.zero_()
        return {"code": st[0], "where": st[1], "sequence": st[2], "expected": st[4], "seen": st[5]}

    def check(self):
        st = self.status()
        if st["code"]:
            raise _lib.FlintError(st["code"], f"device status {st}")

    def _ints(self, t: torch.Tensor, n: int, what: str) -> int:
        if t.dtype is not torch.int32 or t.get_device() != self._index or not t.is_contiguous() or t.numel() != n:
            raise ValueError(f"{what} must be contiguous int32 [{n}] on {self.device}")
        return t.data_ptr()

    def _seqs(self, layer: int, n: int, cached: Lengths, start: Optional[torch.Tensor]) -> _lib.Kv4Seqs:
        if not 0 <= layer < self.n_layer:
            raise ValueError(f"layer {layer} of {self.n_layer}")
        s = _lib.Kv4Seqs.from_buffer_copy(self._proto)
        if layer:
            s.d_pool += layer * self.layer_bytes
        s.n_tokens = n
        if start is not None:
            s.d_start = self._ints(start, self._n_seq + 1, "start")
        elif self._n_seq > 1:
            raise ValueError(f"{self._n_seq} sequences: `start` says which tokens are whose")
        if isinstance(cached, torch.Tensor):
            s.d_cached = self._ints(cached, self._n_seq, "cached")
        else:
            if cached < 0 or cached + (n if start is None else 0) > self.slots:
                raise ValueError(f"{n} tokens behind {cached}: a sequence has {self.slots} slots")
            s.cached = cached
        return s

    def _rows(self, t: torch.Tensor, heads: Optional[int], what: str) -> Tuple[torch.Tensor, int, int, int]:
        """(t, its address, T, elements from token to token) of bf16 [T, heads, head_dim] as the kernels take it: heads adjacent, tokens a multiple of 16
        bytes apart (a copy where it is not so)."""
        shape = t.shape
        if t.dtype is not torch.bfloat16 or t.get_device() != self._index or len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{what} must be bf16 [T, {heads or 'heads'}, {self.head_dim}] on {self.device}")
        T, width, at = shape[0], shape[1] * self.head_dim, t.data_ptr()
        if t.is_contiguous() and not at & 15:
            return t, at, T, width
        ld, to_head, to_dim = t.stride()
        if T == 1:
            ld = width
        if to_dim != 1 or (shape[1] > 1 and to_head != self.head_dim) or ld % 8 or ld < width or at & 15:
            t = t.clone(memory_format=torch.contiguous_format)
            return t, t.data_ptr(), T, width
        return t, at, T, ld

    def _out(self, out: Optional[torch.Tensor], like: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int]:
        if out is None:
            out = torch.empty_like(like)                     # contiguous: its heads are adjacent
            return out, out.data_ptr(), like.shape[1] * self.head_dim
        got, at, _, ld = self._rows(out, like.shape[1], what)
        if got is not out or out.shape != like.shape:
            raise ValueError(f"{what} must be bf16 {tuple(like.shape)} with adjacent heads, tokens a multiple of 16 bytes apart")
        return out, at, ld

    # ------------------------------------------------------------------ launches (asynchronous on the current stream)
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, cached: Lengths, q: Optional[torch.Tensor] = None, start: Optional[torch.Tensor] = None,
               depth: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """New tokens k, v bf16 [T, n_kv, head_dim] into the slots behind the `cached` positions of their sequence (int, or int32 [n_seq] on the GPU), k rotated by
        its position on the way; returns q [T, heads, head_dim] rotated (in `q_out` if given, which may be q itself). start int32 [n_seq + 1]: tokens
        start[b] .. start[b+1] - 1 are sequence b's (needed with several sequences). depth int32 [T]: rotation position behind the cached ones, as for a
        tree's nodes; None: the token's place."""
        k, k_at, T, k_ld = self._rows(k, self.n_kv, "k")
        v, v_at, Tv, v_ld = self._rows(v, self.n_kv, "v")
        heads, q_at, q_ld, o_at, o_ld = 0, None, 0, None, 0
        if q is not None:
            q, q_at, Tq, q_ld = self._rows(q, None, "q")
            heads = q.shape[1]
            q_out, o_at, o_ld = self._out(q_out, q, "q_out")
        else:
            Tq, q_out = T, None
        if T != Tv or T != Tq:
            raise ValueError("q, k and v must have as many tokens")
        s = self._seqs(layer, T, cached, start)
        depth_ptr = None if depth is None else self._ints(depth, T, "depth")
        code = self.lib.fb_kv4_append(ctypes.byref(s), q_at, q_ld, k_at, k_ld, v_at, v_ld, heads, depth_ptr, self._freq_ptr, o_at, o_ld, _raw_stream(self._index))
        if code:
            _lib.check(code, "fb_kv4_append")
        return q_out

    def attend(self, layer: int, q: torch.Tensor, cached: Lengths, start: Optional[torch.Tensor] = None, amask: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, max_new: Optional[int] = None, max_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale * q K^T) V of the new tokens q bf16 [T, heads, head_dim], whose keys and values have been appended, over the cached positions and the new
        tokens of their own sequence: causal, or those with amask[m, j] != 0 (uint8 or bool [T, new tokens of a sequence], j counted from the sequence's first
        new token). max_new: no sequence has more new tokens (default: T); max_len: about the longest sequence, for cutting the work (default: what `cached`
        says, or all slots). A token that sees nothing gets zeros. Probabilities (times a row's s) are rounded to fp16, beyond 64 query rows a kv head keys and values too
        (bf16 in pages with very small or large values); scores and sums are fp32: include/flint_b200.h."""
        q, q_at, T, q_ld = self._rows(q, None, "q")
        heads = q.shape[1]
        if heads == 0 or heads % self.n_kv:
            raise ValueError(f"{heads} query heads do not share {self.n_kv} kv heads evenly")
        s = self._seqs(layer, T, cached, start)
        mask_at, mask_ld = None, 0
        if amask is not None:
            if amask.dtype not in (torch.uint8, torch.bool) or amask.get_device() != self._index or amask.dim() != 2 or amask.shape[0] != T or amask.shape[1] < 1:
                raise ValueError(f"amask must be uint8 or bool [{T}, new tokens of a sequence] on {self.device}")
            amask = amask.contiguous()
            mask_at, mask_ld = amask.data_ptr(), amask.shape[1]
            if start is None and mask_ld < T:
                raise ValueError(f"amask must have a column for each of the {T} new tokens")
        out, o_at, o_ld = self._out(out, q, "out")
        if max_new is None:
            max_new = T
        if max_len is None:
            max_len = self.slots if s.d_cached else min(self.slots, cached + max_new)
        if T and (max_new < 1 or max_len < 1):
            raise ValueError("max_new and max_len are at least 1")
        work_at, need, seqs = None, 0, ctypes.byref(s)
        if self._n_seq > 1 or max_len > NO_SCRATCH[0] or max_new * heads > NO_SCRATCH[1] * self.n_kv:
            need = self.lib.fb_kv4_attend_bytes(seqs, heads, max_new, max_len)
            if need:                                         # of the stream's own memory: calls on other streams and other captures have theirs
                work = torch.empty(need, dtype=torch.uint8, device=self.device)
                work_at = work.data_ptr()
        code = self.lib.fb_kv4_attend(seqs, q_at, q_ld, heads, max_new, max_len, mask_at, mask_ld, self.head_dim ** -0.5 if scale is None else scale, o_at, o_ld,
                                      work_at, need, _raw_stream(self._index))
        if code:
            _lib.check(code, "fb_kv4_attend")
        return out

    def read(self, layer: Optional[int], n: int, cached: Lengths, start: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """What n rows behind `cached` stand for (the tokens of an append with the same arguments; cached = 0: a sequence's first n): K and V, f32
        [n, n_kv, head_dim], or with layer None [n_layer, n, n_kv, head_dim]. Tokens that no sequence has: zeros."""
        s = self._seqs(layer or 0, n, cached, start)
        shape = (2, n, self.n_kv, self.head_dim) if layer is not None else (2, self.n_layer, n, self.n_kv, self.head_dim)
        k, v = self._f32.new_empty(shape).unbind(0)
        code = self.lib.fb_kv4_read(ctypes.byref(s), 1 if layer is not None else self.n_layer, self.layer_bytes, k.data_ptr(), v.data_ptr(), _raw_stream(self._index))
        if code:
            _lib.check(code, "fb_kv4_read")
        return k, v

    def _one(self, seq: int, cached: int) -> _lib.Kv4Seqs:
        if not 0 <= seq < self._n_seq:
            raise ValueError(f"sequence {seq} of {self._n_seq}")
        s = _lib.Kv4Seqs.from_buffer_copy(self._proto)
        s.d_table += 4 * seq * self._ld
        s.n_seq, s.cached, s.table_ld = 1, cached, self.table.shape[1]
        return s

    def compact(self, accept: torch.Tensor, pos: int, seq: int = 0):
        """Moves the accepted path's rows of sequence `seq` to slots pos + 1 .. in every layer, from `DecodeEngine.accept_tree`'s output (int32 [2 + nodes] on the
        GPU)."""
        if accept.numel() < 2:
            raise ValueError("accept must be int32 [2 + nodes]")
        s = self._one(seq, pos)
        _lib.check(self.lib.fb_kv4_compact(ctypes.byref(s), self.n_layer, self.layer_bytes, self._ints(accept, accept.numel(), "accept"), accept.numel() - 2,
                                           _raw_stream(self._index)), "fb_kv4_compact")

    def move(self, src, dst, seq: int = 0):
        """Slot dst[i] of sequence `seq` takes slot src[i], in order, in every layer."""
        if len(src) != len(dst):
            raise ValueError("src and dst must have as many slots")
        n = len(src)
        a = (ctypes.c_int32 * n)(*[int(x) for x in src])
        b = (ctypes.c_int32 * n)(*[int(x) for x in dst])
        s = self._one(seq, 0)
        _lib.check(self.lib.fb_kv4_move(ctypes.byref(s), self.n_layer, self.layer_bytes, a, b, n, _raw_stream(self._index)), "fb_kv4_move")
