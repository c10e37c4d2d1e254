"""Device memory of the cache: pages per layer group, and the rows of fixed-size per-request
state, laid out from what the model's mixers say they need."""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence

import torch

from ..parts.base import CompositeNeed, KV4Need, KVNeed, PagedNeed, StateNeed
from .manager import CacheManager, KVGroupSpec


@dataclass
class LayerCache:
    """What one execution of a mixer sees of the cache."""
    layer: int
    group: int = -1                     # layer group of a paged layer
    tensors: Dict[str, torch.Tensor] = field(default_factory=dict)   # name -> [page, heads, page_tokens, width]
    state: Optional[torch.Tensor] = None  # [max_requests + 1, *shape] of a stateful mixer
    writes: bool = True
    sub: Dict[str, "LayerCache"] = field(default_factory=dict)   # the parts of a ``CompositeNeed`` by name

    @property
    def k(self) -> Optional[torch.Tensor]:
        return self.tensors.get("k")

    @property
    def v(self) -> Optional[torch.Tensor]:
        return self.tensors.get("v")


class CacheStorage:
    """Groups the model's cache layers by need, creates the manager and the tensors.

    Paged layout per group and named tensor: [layer_in_group, page, heads, page_tokens, width]:
    one page id is valid in every layer and every tensor of the group, and what one (page,
    head) holds is a contiguous [page_tokens, width] tile.  The usual need is a key and a
    value tensor of equal geometry (``KVNeed``); a ``PagedNeed`` lists any other set.  The
    reference keeps one K pool and one V pool per layer, [num_blocks, block_size * kv_heads *
    head_dim] (infMain/source/base/block_allocator.cpp:46-49)."""

    def __init__(self, needs: Sequence[object], page_tokens: int, num_pages, max_requests: int,
                 dtype: torch.dtype, device, lifo: bool = False, poison: bool = False):
        self.page_tokens, self.dtype, self.device = int(page_tokens), dtype, device
        keys: List[tuple] = []
        members: Dict[tuple, List[int]] = {}
        self._layer_group: Dict[int, int] = {}
        self._layer_index: Dict[int, int] = {}
        self.state: Dict[int, torch.Tensor] = {}
        self.max_requests = int(max_requests)
        # a composite need is taken apart: each of its parts gets a cache layer number of its own
        # (beyond the model's), so that equal parts of different layers share pools like whole layers
        self._parts: Dict[int, Dict[str, int]] = {}
        self._next_layer = len(needs)
        for layer, need in enumerate(needs):
            self._place(layer, need, keys, members)
        groups = [KVGroupSpec(tuple(members[k]), k[0][0].heads, k[0][0].width, k[1], tensors=k[0], stride=k[2])
                  for k in keys]
        if isinstance(num_pages, int):
            # a group of one entry per `stride` tokens needs that much fewer pages for the same tokens,
            # and at most one page more per request for its last, partly covered page
            num_pages = [num_pages if g.stride == 1 else -(-num_pages // g.stride) + self.max_requests
                         for g in groups]
        self.manager = CacheManager(groups, page_tokens, num_pages if groups else [], max_requests,
                                    lifo=lifo)
        self.paged: List[Dict[str, torch.Tensor]] = []
        for g, spec in enumerate(groups):
            n = self.manager.pools[g].num_pages
            held = {}
            for t in spec.tensors:
                x = torch.empty((len(spec.layers), n, t.heads, self.page_tokens, t.width), dtype=t.dtype or dtype, device=device)
                if poison:
                    x.fill_(float("nan") if x.is_floating_point() else 0xff)     # the bytes of a NaN too
                held[t.name] = x
            self.paged.append(held)

    def _place(self, layer: int, need, keys, members) -> None:
        if isinstance(need, CompositeNeed):
            self._parts[layer] = {}
            for name, part in need.parts:
                sub_layer = self._next_layer
                self._next_layer += 1
                self._parts[layer][name] = sub_layer
                self._place(sub_layer, part, keys, members)
        elif isinstance(need, (KVNeed, KV4Need, PagedNeed)):
            key = (tuple(need.tensors), need.window, int(getattr(need, "stride", 1) or 1))
            if not key[0]:
                raise TypeError(f"cache layer {layer}: a paged need lists at least one tensor")
            if len({t.name for t in key[0]}) != len(key[0]):
                raise TypeError(f"cache layer {layer}: two cache tensors share a name")
            if key not in members:
                members[key] = []
                keys.append(key)
            self._layer_group[layer] = keys.index(key)
            self._layer_index[layer] = len(members[key])
            members[key].append(layer)
        elif isinstance(need, StateNeed):
            # one row per request slot and one more, which the padding rows of captured
            # decode steps point at
            self.state[layer] = torch.zeros((self.max_requests + 1,) + tuple(need.shape), dtype=need.dtype,
                                            device=self.device)
        elif need is not None:
            raise TypeError(f"cache layer {layer}: unknown need {need!r}")

    @property
    def groups(self):
        return self.manager.groups

    @property
    def state_pad_slot(self) -> int:
        """The row of the state tensors that belongs to no request."""
        return self.max_requests

    def bytes_per_token(self) -> int:
        # a group of one entry per `stride` tokens costs a token that much less
        return sum(-(-len(g.layers) * sum(t.heads * t.width * (t.dtype or self.dtype).itemsize for t in g.tensors)
                     // max(1, g.stride)) for g in self.groups)

    def zero_state(self, slots) -> None:
        """Zeroes the state rows of these request slots in every stateful layer (the step
        function calls it for requests whose first tokens are about to run)."""
        if not self.state or len(slots) == 0:
            return
        idx = torch.as_tensor(list(slots), dtype=torch.long).to(self.device)
        for t in self.state.values():
            t.index_fill_(0, idx, 0)

    def layer(self, cache_layer: int, writes: bool = True) -> LayerCache:
        if cache_layer in self._parts:
            return LayerCache(layer=cache_layer, writes=writes,
                              sub={name: self.layer(l, writes) for name, l in self._parts[cache_layer].items()})
        if cache_layer in self._layer_group:
            g, i = self._layer_group[cache_layer], self._layer_index[cache_layer]
            return LayerCache(layer=cache_layer, group=g, tensors={n: t[i] for n, t in self.paged[g].items()},
                              writes=writes)
        if cache_layer in self.state:
            return LayerCache(layer=cache_layer, state=self.state[cache_layer], writes=writes)
        return LayerCache(layer=cache_layer, writes=writes)
