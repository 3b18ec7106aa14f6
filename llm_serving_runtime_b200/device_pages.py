"""Pages of a paged cache on the device: copied, forked, freed, reserved, compacted.

    copy_pages([k_pool, v_pool], src_blocks, dst_blocks)        # e.g. copy-on-write

    pages = DevicePages(num_blocks, block_size, max_seqs, max_blocks_per_seq, device)
    pages.reserve(slots, n_tokens)             # room for tokens at the end of each slot
    pages.fork(parents, children, caches)      # children continue from their parents
    pages.free(slots)
    live = pages.compact(caches)               # live pages move to ids [0, live)
    out = paged_attention_decode(q, k, v, pages.block_tables[rows], ...)

``BlockRefAllocator`` (shared_blocks.py) keeps its books on the host and suits a
scheduler that lives there.  ``DevicePages`` keeps tables, lengths and counts in
device tensors, so a decode loop (a beam search, parallel sampling, a captured
graph) forks and frees without a host round trip.  Slot s holds ``seq_lens[s]``
tokens in pages ``block_tables[s, :ceil(len / block_size)]``, -1 behind them;
``ref_counts[p]`` is the number of table entries that hold page p.

A fork shares full pages and copies the one in use, so a page that two slots
hold is never appended to.  New pages are the lowest free ids in the order of the
arguments: results do not depend on timing.  The arguments (slots, parents,
children, numbers of tokens, block ids) are int32 tensors on the device; -1 is
padding.  Each call is a few kernels on the current stream, safe to capture.

Errors: a bad slot, a child that is not empty, a block written from two places
(IndexError) and a pool without enough free pages (RuntimeError) leave the slots
concerned as they were and raise at the next call, like the other kernels' errors
(``validate=True``: this call, synchronously; ``read_device_errors`` after a
captured replay of ``copy_pages``, ``DevicePages.read_errors`` of the others).

The reference copies pages one tensor at a time (``GpuKVBlockPool.copy_blocks``,
runtime/phase2/paged_kv_kernel.py:233-250) and allocates on the host
(runtime/phase2/kv_allocator.py); it has no counterpart of the rest.
"""

from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from . import _lib
from .paged_attention import (
    _VALIDATE_DEFAULT,
    _as_int32,
    _host,
    _host_words,
    _HostWord,
    _stream_ptr,
    _with_device,
    host_word,
)

__all__ = ["DevicePages", "copy_pages"]


def _view(t: torch.Tensor) -> _lib.PageViewArgs:
    """The pages t[i] of a cache as equal runs of bytes: dimensions that follow
    on from one another in memory (in any order) are one run, one more may be
    strided."""
    e = t.element_size()
    run, levels = 1, []  # contiguous elements; (size, stride) of what is not
    for stride, size in sorted(zip(t.stride()[1:], t.shape[1:])):
        if size == 1:
            continue
        if stride == 0:
            raise ValueError("the pages of a cache must not overlap")
        if not levels and stride == run:
            run *= size
        elif levels and stride == levels[-1][0] * levels[-1][1]:
            levels[-1] = (levels[-1][0] * size, levels[-1][1])
        else:
            levels.append((size, stride))
    if len(levels) > 1:
        raise ValueError(f"a page may have one strided dimension, got shape {tuple(t.shape)} with strides {t.stride()}")
    segments, stride = levels[0] if levels else (1, 0)
    # pages one after the other, or interleaved with one another's runs: no byte twice
    extent = run
    for step, size in sorted(((t.stride(0), t.shape[0]), (stride, segments))):
        if size > 1 and step < extent:
            raise ValueError("the pages of a cache must not overlap")
        extent += (size - 1) * step
    return _lib.PageViewArgs(t.data_ptr(), t.stride(0) * e, segments, stride * e, run * e)


def _views(caches: Sequence[torch.Tensor], num_blocks: int | None, device: torch.device | None):
    """(C array, count, num_blocks, device) of the caches, checked."""
    if len(caches) > _lib.PA_MAX_PAGE_VIEWS:
        raise ValueError(f"at most {_lib.PA_MAX_PAGE_VIEWS} caches in a call, got {len(caches)}")
    arr = (_lib.PageViewArgs * max(1, len(caches)))()
    for i, t in enumerate(caches):
        if t.dim() < 1 or not t.is_cuda:
            raise ValueError("caches must be CUDA tensors [num_blocks, ...]")
        device = t.device if device is None else device
        num_blocks = t.shape[0] if num_blocks is None else num_blocks
        if t.device != device or t.shape[0] != num_blocks:
            raise ValueError(f"caches must have {num_blocks} blocks on {device}, got {t.shape[0]} on {t.device}")
        if t.numel() > 0:
            arr[i] = _view(t)
    return arr, len(caches), num_blocks, device


def _ids(t: torch.Tensor, device: torch.device, name: str) -> torch.Tensor:
    t = _as_int32(t.reshape(-1), device, name)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _run(word: _HostWord, validate: bool | None, what: str, call) -> None:
    """One C call on the current stream, with the errors of the framework's kernels."""
    if validate is None:
        word.raise_landed()
    with _with_device(word.device):
        _lib.check(call(_stream_ptr(word.device)), what)
        word.finish(validate)


def copy_pages(caches: Sequence[torch.Tensor], src_blocks: torch.Tensor, dst_blocks: torch.Tensor, *,
               validate: bool | None = None) -> None:
    """cache[dst_blocks[i]] = cache[src_blocks[i]] for every pair and every cache
    ([num_blocks, ...] each, any element types; e.g. the K and V pools with all
    their layers, and an 8-bit cache's scales), in one kernel.

    Pairs with a negative id are padding.  A destination must be no other pair's
    source and be named once; pairs that break this are left out and flagged.
    """
    if not caches:
        raise ValueError("copy_pages needs a cache")
    if validate is None and not _VALIDATE_DEFAULT:
        word = _host_words.get(caches[0].device.index)
        if word is not None and _host.copy_pages(caches, src_blocks, dst_blocks, word.ptr):
            return
    arr, n_views, num_blocks, device = _views(caches, None, None)
    src, dst = _ids(src_blocks, device, "src_blocks"), _ids(dst_blocks, device, "dst_blocks")
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source blocks but {dst.numel()} destinations")
    if num_blocks == 0 and src.numel() > 0:
        raise ValueError("the caches have no blocks")
    if src.numel() == 0:
        return
    word = host_word(device)
    _run(word, validate, "pa_pages_copy",
         lambda stream: _lib.load().pa_pages_copy(arr, n_views, num_blocks, src.data_ptr(), dst.data_ptr(),
                                                  src.numel(), word.ptr, stream))


class DevicePages:
    """Tables, lengths and page counts of ``max_seqs`` sequence slots on a device.

    The tensors may be read at any time and rewritten between calls, as long as
    they stay consistent.  Calls that use one object must not overlap on the GPU,
    and a graph that captured some needs the object kept.  ``compact`` renames
    pages: copies of table rows made before it are void.
    """

    def __init__(self, num_blocks: int, block_size: int, max_seqs: int, max_blocks_per_seq: int,
                 device: torch.device | str = "cuda") -> None:
        for name, v in (("num_blocks", num_blocks), ("block_size", block_size), ("max_seqs", max_seqs),
                        ("max_blocks_per_seq", max_blocks_per_seq)):
            if v <= 0:
                raise ValueError(f"{name} must be positive, got {v}")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("DevicePages needs a CUDA device (no CPU fallback)")
        self._bind(torch.full((max_seqs, max_blocks_per_seq), -1, dtype=torch.int32, device=dev),
                   torch.zeros(max_seqs, dtype=torch.int32, device=dev),
                   torch.zeros(num_blocks, dtype=torch.int32, device=dev), block_size)

    @classmethod
    def from_tensors(cls, block_tables: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor, *,
                     block_size: int) -> "DevicePages":
        """Over the caller's own int32 tensors, which are used in place."""
        self = cls.__new__(cls)
        self._bind(block_tables, seq_lens, ref_counts, block_size)
        return self

    def _bind(self, block_tables, seq_lens, ref_counts, block_size) -> None:
        if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or not block_tables.is_cuda \
                or block_tables.stride(1) != 1 or 0 in block_tables.shape:
            raise ValueError("block_tables must be a CUDA int32 [max_seqs, max_blocks] with contiguous rows")
        if block_tables.shape[0] > 1 and block_tables.stride(0) < block_tables.shape[1]:
            raise ValueError("the rows of block_tables must not overlap")
        if not 0 < block_size <= 2**30:
            raise ValueError("block_size must be positive and at most 2^30")
        for name, t in (("seq_lens", seq_lens), ("ref_counts", ref_counts)):
            if t.dim() != 1 or t.dtype != torch.int32 or t.device != block_tables.device or not t.is_contiguous() \
                    or t.numel() == 0:
                raise ValueError(f"{name} must be a contiguous int32 vector on {block_tables.device}")
        if seq_lens.numel() != block_tables.shape[0]:
            raise ValueError("one length per row of block_tables")
        self.block_tables, self.seq_lens, self.ref_counts = block_tables, seq_lens, ref_counts
        self.block_size = int(block_size)
        self.device = block_tables.device
        words = _lib.load().pa_pages_scratch_words(self.max_seqs, self.num_blocks)
        self._scratch = torch.empty(words, dtype=torch.int32, device=self.device)
        # its own error word: two objects on two streams do not share one
        self._word = _HostWord(self.device)

    @property
    def max_seqs(self) -> int:
        return int(self.block_tables.shape[0])

    @property
    def num_blocks(self) -> int:
        return int(self.ref_counts.numel())

    def read_errors(self) -> int:
        """The PA_DEVERR_* bits of this object's calls so far, cleared.  Synchronises."""
        return self._word.take()

    def _args(self) -> _lib.PageTablesArgs:
        t = self.block_tables
        return _lib.PageTablesArgs(t.data_ptr(), max(t.stride(0), t.shape[1]), t.shape[0], t.shape[1],
                                   self.seq_lens.data_ptr(), self.ref_counts.data_ptr(), self.num_blocks,
                                   self.block_size, self._scratch.data_ptr(), self._word.ptr)

    def _call(self, what: str, validate: bool | None, *rest) -> None:
        args, fn = self._args(), getattr(_lib.load(), what)
        _run(self._word, validate, what, lambda stream: fn(ctypes.byref(args), *rest, stream))

    def _fast(self, op: int, validate: bool | None, a=None, b=None, caches=()):
        """The call in one step, when its arguments are the kernels' already; else None."""
        if validate is not None or _VALIDATE_DEFAULT:
            return None
        return _host.pages(op, self.block_tables, self.seq_lens, self.ref_counts, self.block_size, self._scratch,
                           self._word.ptr, a, b, caches)

    def _slots(self, t: torch.Tensor, name: str) -> torch.Tensor:
        t = _ids(t, self.device, name)
        if t.numel() > self.max_seqs:
            raise ValueError(f"{name}: at most {self.max_seqs} slots, got {t.numel()}")
        return t

    def free(self, slots: torch.Tensor, *, validate: bool | None = None) -> None:
        """Empty the slots; pages nobody holds any more are free.  A slot named twice
        is freed once, an empty one stays empty."""
        if self._fast(0, validate, slots):
            return
        slots = self._slots(slots, "slots")
        self._call("pa_pages_free", validate, slots.data_ptr(), slots.numel())

    def fork(self, parents: torch.Tensor, children: torch.Tensor, caches: Sequence[torch.Tensor] = (), *,
             validate: bool | None = None) -> None:
        """Each empty slot children[i] gets the tokens of parents[i]: the full pages are
        shared, the page in use is copied in every cache to the child's own."""
        if self._fast(1, validate, parents, children, caches):
            return
        parents, children = self._slots(parents, "parents"), self._slots(children, "children")
        if parents.numel() != children.numel():
            raise ValueError(f"{parents.numel()} parents but {children.numel()} children")
        arr, n, _, _ = _views(caches, self.num_blocks, self.device)
        self._call("pa_pages_fork", validate, parents.data_ptr(), children.data_ptr(), children.numel(), arr, n)

    def reserve(self, slots: torch.Tensor, n_tokens: torch.Tensor, *, validate: bool | None = None) -> None:
        """Slot slots[i] grows by n_tokens[i] tokens, with new pages where needed."""
        if self._fast(2, validate, slots, n_tokens):
            return
        slots, n_tokens = self._slots(slots, "slots"), _ids(n_tokens, self.device, "n_tokens")
        if slots.numel() != n_tokens.numel():
            raise ValueError(f"{slots.numel()} slots but {n_tokens.numel()} numbers of tokens")
        self._call("pa_pages_reserve", validate, slots.data_ptr(), n_tokens.data_ptr(), slots.numel())

    def compact(self, caches: Sequence[torch.Tensor] = (), *, out: torch.Tensor | None = None,
                validate: bool | None = None) -> torch.Tensor:
        """Move the live pages to ids [0, live) in every cache and in the tables; returns
        ``live`` as a device int32 [1] (``out`` when given)."""
        live = self._fast(3, validate, caches=caches) if out is None else None
        if live is not None:
            return live
        arr, n, _, _ = _views(caches, self.num_blocks, self.device)
        if out is None:
            out = torch.empty(1, dtype=torch.int32, device=self.device)
        elif out.dtype != torch.int32 or out.numel() != 1 or out.device != self.device:
            raise ValueError(f"out must be an int32 [1] on {self.device}")
        self._call("pa_pages_compact", validate, arr, n, out.data_ptr())
        return out
