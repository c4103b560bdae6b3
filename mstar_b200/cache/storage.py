"""Device memory of the cache: key/value pages and per-request state slots.

Run-order entries (caches) whose mixers have the same needs as to which keys
must stay (all of them, or a window) form a group; a group has one pool of page
ids and one block table per request, and each cache of the group has its own
tensor [pages, planes, kv_heads, page_size, head_dim] indexed by those ids
(two planes for keys and values, one for a mixer that caches a single row per token).  The
reference keeps one tensor [layers, pages, 2, page_size, kv_heads, head_dim] per
model component (mstar/engine/kv_cache_engine.py:132-136); here a page keeps the
tokens of one head contiguous, so a page of one head is one 16-byte-aligned run
that bulk copies can move.

With ``kv_cache_dtype`` "float8_e4m3" the pages hold e4m3 codes, half the bytes of bfloat16, and a
second tensor [pages, planes, kv_heads, page_size] a scale byte for every row
(``mstar_b200.ops.kv8``).

State slots hold per-request state of fixed size for mixers that ask for it; the
architecture served here asks for none, so the pool exists with zero bytes.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from ..parts.base import CacheNeed, LayerCache
from .manager import CacheManager, GroupConfig

KV_CACHE_DTYPES = ("auto", "float8_e4m3")
_STATE_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}


def plan_groups(needs: Sequence[CacheNeed]):
    """Group caches by which keys have to stay: the window of their keys and the number of
    first keys kept beside it.  Returns (windows, group_of): ``windows[g]`` is None, W, or
    (W, keep_first) where first keys are kept; ``group_of[cache]`` the group index or None."""
    windows: list = []
    group_of: list = []
    for need in needs:
        if need is None or need.kv is None:
            group_of.append(None)
            continue
        w = need.kv.window
        if w is not None and need.kv.keep_first:
            w = (w, need.kv.keep_first)
        if w not in windows:
            windows.append(w)
        group_of.append(windows.index(w))
    return windows, group_of


def _kv_shape(kv, pages: int, page_size: int) -> tuple:
    if kv.v_head_dim is not None and kv.v_head_dim != kv.head_dim:
        return (pages, kv.num_kv_heads * page_size * (kv.head_dim + kv.v_head_dim))
    return (pages, kv.planes, kv.num_kv_heads, page_size, kv.head_dim)


def eight_bit_cache(kv_cache_dtype: Optional[str], needs: Sequence[Optional[CacheNeed]]) -> bool:
    """Whether ``kv_cache_dtype`` asks for an 8-bit cache ("auto" or None: pages hold the compute
    type).  Every cache of the model must be able to be one."""
    if kv_cache_dtype is None or kv_cache_dtype == "auto":
        return False
    if kv_cache_dtype not in KV_CACHE_DTYPES:
        raise ValueError(f"kv_cache_dtype {kv_cache_dtype!r} is not known (one of {', '.join(KV_CACHE_DTYPES)})")
    kept = [i for i, n in enumerate(needs) if n is not None and n.kv is not None]
    unable = [i for i in kept if not needs[i].kv.eight_bit]
    if unable or not kept:
        raise ValueError(f"kv_cache_dtype {kv_cache_dtype!r} is for models whose every cache holds plain keys and "
                         "values (rotary or no positions, one head size, no norms, biases or caps on scores); "
                         + (f"caches {unable} of this one do not" if unable else "this one has none"))
    return True


def group_page_sizes(page_size, num_groups: int) -> list:
    """One page size per group from one int for all, or a sequence with one per group."""
    if isinstance(page_size, int):
        sizes = [page_size] * num_groups
    else:
        sizes = [int(p) for p in page_size]
        if len(sizes) != num_groups:
            raise ValueError(f"{num_groups} cache groups but {len(sizes)} page sizes")
    if any(p <= 0 for p in sizes):
        raise ValueError(f"page sizes must be positive, got {sizes}")
    return sizes


def bytes_per_page(needs: Sequence[CacheNeed], group_of, group: int, page_size: int,
                   dtype: torch.dtype, kv_cache_dtype: Optional[str] = None) -> int:
    eight = eight_bit_cache(kv_cache_dtype, needs)
    item = 1 if eight else torch.empty((), dtype=dtype).element_size()
    total = 0
    for need, g in zip(needs, group_of):
        if g == group:
            shape = _kv_shape(need.kv, 1, page_size)
            total += item * int(torch.Size(shape).numel())
            if eight:                           # and a scale byte a row
                total += int(torch.Size(shape[:4]).numel())
    return total


class CacheStorage:
    def __init__(self, needs: Sequence[Optional[CacheNeed]], dtype: torch.dtype,
                 device: torch.device, page_size, num_pages, num_slots: int,
                 kv_cache_dtype: Optional[str] = None):
        """``page_size`` and ``num_pages``: one int for every group, or a list with one per
        group (a group of windowed layers may want smaller pages than one that keeps every
        key: it gives them back sooner).  ``kv_cache_dtype``: None or "auto" keeps pages in
        ``dtype``, "float8_e4m3" in 8 bits a number (``mstar_b200.ops.kv8``)."""
        self.needs = list(needs)
        self.eight_bit = eight_bit_cache(kv_cache_dtype, self.needs)
        self.dtype = dtype
        self.device = device
        self.num_slots = int(num_slots)
        self.windows, self.group_of = plan_groups(self.needs)
        self.page_sizes = group_page_sizes(page_size, len(self.windows))
        if isinstance(num_pages, int):
            num_pages = [num_pages] * len(self.windows)
        if len(num_pages) != len(self.windows):
            raise ValueError(f"{len(self.windows)} cache groups but {len(num_pages)} page counts")
        self.group_configs = [GroupConfig(p, int(n), *(w if isinstance(w, tuple) else (w,)))
                              for p, n, w in zip(self.page_sizes, num_pages, self.windows)]
        self.manager = CacheManager(self.group_configs, self.num_slots)
        self.kv: list = []
        self.kv_scales: list = []
        self.state: list = []
        for need, g in zip(self.needs, self.group_of):
            if g is None:
                self.kv.append(None)
                self.kv_scales.append(None)
            else:
                # one page more than the manager hands out: padding entries of
                # fixed-shape (CUDA graph) batches write their keys there
                n = self.group_configs[g].num_pages + 1
                shape = _kv_shape(need.kv, n, self.page_sizes[g])
                pages = torch.zeros(shape, dtype=torch.uint8 if self.eight_bit else dtype, device=device)
                self.kv.append(pages.view(torch.float8_e4m3fn) if self.eight_bit else pages)
                self.kv_scales.append(torch.zeros(shape[:4], dtype=torch.uint8, device=device)
                                      if self.eight_bit else None)
            if need is not None and need.state is not None:
                self.state.append(torch.zeros((self.num_slots + 1,) + tuple(need.state.shape),
                                              dtype=_STATE_DTYPES[need.state.dtype],
                                              device=device))
            else:
                self.state.append(None)

    def pad_page(self, group: int) -> int:
        """The page of ``group`` that padding entries may scribble on."""
        return self.group_configs[group].num_pages

    @property
    def pad_slot(self) -> int:
        return self.num_slots

    def state_bytes_per_request(self) -> int:
        return sum(0 if s is None else s[0].numel() * s.element_size() for s in self.state)

    @property
    def has_state(self) -> bool:
        return any(s is not None for s in self.state)

    def snapshot_state(self, slots) -> Optional[tuple]:
        """Copies of the state rows of ``slots`` (None when no mixer keeps state).  Mixers
        update their state in place during the forward pass; the step function takes this
        copy before the pass and puts it back if the pass fails, so that state, like the
        lengths, moves only with a step that completed (the reference advances its sequence
        state after the forward pass, mstar/engine/cache_manager.py:811-838)."""
        if not self.has_state:
            return None
        index = torch.as_tensor(list(slots), dtype=torch.long, device=self.device)
        return index, [None if s is None else s.index_select(0, index) for s in self.state]

    def restore_state(self, snapshot) -> None:
        if snapshot is None:
            return
        index, rows = snapshot
        for s, saved in zip(self.state, rows):
            if s is not None:
                s.index_copy_(0, index, saved)

    def reset_slot(self, slot: int) -> None:
        """A request takes the slot: its state starts at zero."""
        for s in self.state:
            if s is not None:
                s[slot].zero_()

    def layer_cache(self, cache_id: int, block_tables: Sequence[torch.Tensor]) -> LayerCache:
        g = self.group_of[cache_id]
        return LayerCache(kv=self.kv[cache_id],
                          page_size=0 if g is None else self.page_sizes[g],
                          block_table=None if g is None else block_tables[g],
                          state=self.state[cache_id], kv_scales=self.kv_scales[cache_id])
