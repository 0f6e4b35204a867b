"""Device memory of the cache: pages per group of layers, fixed-size state per request slot.

Layers whose mixers need the same kind of cache (the same named arrays per token and the same
window) form a group; a group has one pool of pages and one block table per request,
and every layer of the group has its own arrays (attention: K and V) indexed by the same page ids
(the reference has this one implicit group: ``k_base(l)``/``v_base(l)`` share the page id,
include/paged_kv_cache.hpp:38-39; and allocates 2 L separate buffers,
src/paged_kv_cache.cpp:8-14 - here a group is one allocation).  The host bookkeeping
(free lists, block tables, slots) is the native ``CacheManager``.
"""
from __future__ import annotations

from dataclasses import dataclass, replace
from typing import Dict, List, Optional, Sequence

import torch

from ..kernels import ops
from ..kernels.library import host
from ..parts import AttentionLike, CacheNeed


@dataclass
class LayerCache:
    """The pages of one layer: per declared array a tensor ``[num_pages, heads, page_size, width]``."""
    group: int
    arrays: Dict[str, torch.Tensor]
    page_size: int
    window: int
    scales: Optional[Dict[str, torch.Tensor]] = None      # an 8-bit cache: the arrays hold codes, and these ``[num_pages, heads, page_size]`` their scales
    values: Optional["LayerCache"] = None                 # an 8-bit cache: the pages that the codes are read back into (shared by all layers)

    def coded(self, name: str) -> ops.Q8Pages:
        """The codes and scales of an array of an 8-bit cache."""
        return ops.Q8Pages(self.arrays[name], self.scales[name])

    @property
    def k(self) -> torch.Tensor:
        return self.arrays["k"]

    @property
    def v(self) -> torch.Tensor:
        return self.arrays["v"]


@dataclass
class CacheGroup:
    need: CacheNeed
    layers: List[int]
    page_size: int
    num_pages: int
    storage: Optional[torch.Tensor] = None   # one flat allocation: [layer][array][page][head][token][width]
    scale_storage: Optional[torch.Tensor] = None      # of an 8-bit cache: [layer][array][page][head][token]

    def bytes_per_page(self, itemsize: int, coded: bool = False) -> int:
        """Bytes of a page in all layers of the group; ``coded``: a byte an element and 4 a token and head, instead of ``itemsize``."""
        per_token = self.need.elements_per_token()
        per_token = per_token + 4 * sum(a.heads for a in self.need.arrays) if coded else per_token * itemsize
        return len(self.layers) * per_token * self.page_size


def _need_with_readers(model, li: int, need: CacheNeed) -> CacheNeed:
    """A layer's pages stay as long as the layer itself OR a layer that reads its cache can reach them: the
    window that decides when pages go back is the widest of theirs (0, no window, is the widest of all), and the first
    tokens that stay are the most that one of them goes on seeing."""
    readers = [other.mixer for other in model.layers if other.spec.cache_source == li]
    windows = [need.window] + [int(getattr(m, "window", 0)) for m in readers]
    widest = 0 if any(w <= 0 for w in windows) else max(windows)
    keep = max([need.keep_first] + [int(getattr(m, "keep_first", 0)) for m in readers]) if widest else 0
    return need if (widest, keep) == (need.window, need.keep_first) else replace(need, window=widest, keep_first=keep)


def cache_groups_of(model, page_size: int) -> List[CacheGroup]:
    groups: List[CacheGroup] = []
    for li, layer in enumerate(model.layers):
        need = layer.mixer.cache_need()
        if need is None or layer.spec.cache_source is not None:
            continue
        need = _need_with_readers(model, li, need)
        for g in groups:
            if g.need == need:
                g.layers.append(li)
                break
        else:
            groups.append(CacheGroup(need, [li], page_size, 0))
    return groups


CACHE_DTYPES = (None, "int8")


def refuse_coded(model) -> None:
    """Raises if a mixer keeps or reads a cache otherwise than through the step's attention (``StepContext.attention``), which is what
    reads and writes an 8-bit cache."""
    for li, layer in enumerate(model.layers):
        need = layer.mixer.cache_need()
        if need is None and layer.spec.cache_source is None:
            continue
        for m in layer.mixer.cache_users():
            names = set(getattr(m, "kv_arrays", ("k", "v")))
            if not isinstance(m, AttentionLike) or (need is not None and {a.name for a in need.arrays} != names):
                raise ValueError(f"layer {li}: {type(m).__name__} does not keep keys and values that the attention kernels read; "
                                 f"its cache cannot be kept in 8 bits")


class CachePool:
    def __init__(self, model, *, page_size: int = 16, num_pages: Optional[int] = None, max_requests: int = 16,
                 max_tokens: Optional[int] = None, memory_fraction: float = 0.85, device="cuda", cache_dtype: Optional[str] = None):
        """``num_pages`` per group, or ``max_tokens`` (pages = ceil(max_tokens / page_size)), or what
        ``memory_fraction`` of the free device memory holds.  ``cache_dtype`` "int8": keys and values are kept as 8-bit codes
        with a scale per token and head (``kernels.ops.Q8Pages``) instead of in the model's type; beside them the pool
        then holds the pages of one layer in that type, into which codes are read back."""
        if cache_dtype not in CACHE_DTYPES:
            raise ValueError(f"cache_dtype {cache_dtype!r} is not one of {list(CACHE_DTYPES)}")
        self.cache_dtype = cache_dtype
        coded = cache_dtype == "int8"
        if coded:
            refuse_coded(model)
        if page_size <= 0:
            raise ValueError("page_size must be positive")
        self.model, self.page_size, self.max_requests = model, page_size, max_requests
        self.dtype, self.device = model.dtype, torch.device(device)
        self.groups = cache_groups_of(model, page_size)
        itemsize = torch.empty((), dtype=self.dtype).element_size()
        if num_pages is None and max_tokens is not None:
            num_pages = -(-max_tokens // page_size)
        if num_pages is None:
            free, _ = torch.cuda.mem_get_info(self.device)
            per_page = sum(g.bytes_per_page(itemsize, coded) for g in self.groups) or 1
            if coded:
                per_page += max((g.need.elements_per_token() for g in self.groups), default=0) * page_size * itemsize
            num_pages = max(1, int(free * memory_fraction) // per_page)
            # no request can use more than max_requests * max_positions tokens
            num_pages = min(num_pages, max_requests * (-(-model.spec.max_positions // page_size)))
        self.layer_cache: Dict[int, LayerCache] = {}
        specs = []
        align = 256 // (1 if coded else itemsize)    # every array starts on a 256-byte boundary (TMA wants 16)
        for gi, g in enumerate(self.groups):
            g.num_pages = int(num_pages)
            sizes = [(-(-g.num_pages * a.heads * page_size * a.width // align) * align) for a in g.need.arrays]
            g.storage = torch.zeros(len(g.layers) * sum(sizes), dtype=torch.int8 if coded else self.dtype, device=self.device)
            rows = [g.num_pages * a.heads * page_size for a in g.need.arrays]
            if coded:
                g.scale_storage = torch.zeros(len(g.layers) * sum(rows), dtype=torch.float32, device=self.device)
            at = at_scale = 0
            for li in g.layers:
                arrays, scales = {}, {}
                for a, size in zip(g.need.arrays, sizes):
                    n = g.num_pages * a.heads * page_size * a.width
                    arrays[a.name] = g.storage[at:at + n].view(g.num_pages, a.heads, page_size, a.width)
                    at += size
                    if coded:
                        n = g.num_pages * a.heads * page_size
                        scales[a.name] = g.scale_storage[at_scale:at_scale + n].view(g.num_pages, a.heads, page_size)
                        at_scale += n
                self.layer_cache[li] = LayerCache(gi, arrays, page_size, g.need.window, scales if coded else None)
            specs.append(host().GroupSpec(page_size, g.num_pages, g.need.window, g.need.keep_first))
        if coded:
            self._read_back_pages(itemsize)
        if not specs:  # a model without any cache still needs request slots and lengths: pages that are counted only
            specs.append(host().GroupSpec(page_size, int(num_pages), 0))
        for li, layer in enumerate(model.layers):
            src = layer.spec.cache_source
            if src is not None:
                if src not in self.layer_cache:
                    raise ValueError(f"layer {li} reads the cache of layer {src}, which keeps none")
                self.layer_cache[li] = self.layer_cache[src]
        self.manager = host().CacheManager(specs, max_requests)
        # fixed-size per-request state
        self.state: Dict[int, torch.Tensor] = {}
        for li, layer in enumerate(model.layers):
            need = layer.mixer.state_need()
            if need is not None:
                self.state[li] = torch.zeros((max_requests, *need.shape), dtype=need.dtype, device=self.device)

    def _read_back_pages(self, itemsize: int) -> None:
        """One layer's pages in the model's type, page p of which takes what is read back of page p of any layer."""
        align = 256 // itemsize
        sizes = {gi: [(-(-g.num_pages * a.heads * self.page_size * a.width // align) * align) for a in g.need.arrays] for gi, g in enumerate(self.groups)}
        self.read_back = torch.zeros(max((sum(v) for v in sizes.values()), default=0), dtype=self.dtype, device=self.device)
        for gi, g in enumerate(self.groups):
            arrays, at = {}, 0
            for a, size in zip(g.need.arrays, sizes[gi]):
                n = g.num_pages * a.heads * self.page_size * a.width
                arrays[a.name] = self.read_back[at:at + n].view(g.num_pages, a.heads, self.page_size, a.width)
                at += size
            values = LayerCache(gi, arrays, self.page_size, g.need.window)
            for li in g.layers:
                self.layer_cache[li].values = values

    def max_blocks(self, gi: int) -> int:
        return -(-self.model.spec.max_positions // self.page_size)

    def clear_state(self, slot: int) -> None:
        for t in self.state.values():
            t[slot].zero_()

    def bytes_per_token(self) -> int:
        itemsize = torch.empty((), dtype=self.dtype).element_size()
        return sum(g.bytes_per_page(itemsize, self.cache_dtype == "int8") // g.page_size for g in self.groups)

    def poison_pages(self, group: int, pages: Sequence[int]) -> None:
        """Fills the given pages of every array of every layer of ``group`` with NaN (a debugging aid: a
        kernel that reads a page its request no longer holds, or a token slot beyond a request's length
        inside a page that was used before, then shows up as NaN logits)."""
        if not pages or group >= len(self.groups):
            return
        idx = torch.tensor(sorted(set(int(p) for p in pages)), dtype=torch.long, device=self.device)
        for li in self.groups[group].layers:
            lc = self.layer_cache[li]
            for t in (lc.scales or lc.arrays).values():      # codes are always numbers: with a scale of NaN none of them is
                t.index_fill_(0, idx, float("nan"))
