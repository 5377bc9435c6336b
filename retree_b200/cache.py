"""Preallocated KV cache for tree verification (a ``transformers.Cache``).

Replaces ``DynamicCache``'s per-round ``torch.cat`` of every layer
(transformers/cache_utils.py:102-121) with one HBM slab

    slab[2*layer + {0: K, 1: V}, kv_head, position, head_dim]   (bf16, zeroed)

written in place by the ``rt_kv_append`` kernel.  ``layers[i].keys`` /
``.values`` are views ``[1, kv_heads, length, head_dim]`` of the slab, so code
written against ``DynamicCache`` (the reference's ``compact_dynamic_cache``,
ddtree.py:717-729) keeps working, and the slab as a whole is compacted in ONE
launch by ``retree_b200.ddtree.compact_dynamic_cache``.

Positions past a layer's length are never garbage: the slab starts zeroed and
only ever holds K/V rows, so the attention kernel may read whole 128-key
blocks past the end (they are masked, and finite).

Device-length mode (``use_device_length(True)``): appends land at the offset
held in ``length_dev`` (int64[1] on the device) and ``update`` returns views of
the full capacity, so a verify forward can be captured once in a CUDA graph
and replayed at any prefix length; the attention plugin then reads the prefix
length from the same device word.
"""

from __future__ import annotations

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from . import kernels


class TreeKVLayer(CacheLayerMixin):
    is_sliding = False
    is_compileable = False

    def __init__(self, cache: "TreeKVCache", index: int):
        super().__init__()
        self._cache = cache
        self.index = index
        self.length = 0
        self.is_initialized = True
        self.dtype = cache.dtype
        self.device = cache.device

    # views of the slab -----------------------------------------------------
    def _view(self, kv: int, length: int) -> torch.Tensor:
        return self._cache.slab[2 * self.index + kv, :, :length, :].unsqueeze(0)

    @property
    def keys(self) -> torch.Tensor:  # type: ignore[override]
        return self._view(0, self.length)

    @keys.setter
    def keys(self, value):
        if value is not None:
            raise AttributeError("TreeKVLayer keys are views of the preallocated slab")

    @property
    def values(self) -> torch.Tensor:  # type: ignore[override]
        return self._view(1, self.length)

    @values.setter
    def values(self, value):
        if value is not None:
            raise AttributeError("TreeKVLayer values are views of the preallocated slab")

    # CacheLayerMixin ---------------------------------------------------------
    def lazy_initialization(self, key_states, value_states) -> None:
        return None

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        c = self._cache
        n = key_states.shape[-2]
        kc = c.slab[2 * self.index]
        vc = c.slab[2 * self.index + 1]
        if c.device_length:
            kernels.kv_append(kc, vc, key_states, value_states, offset_dev=c.length_dev)
            self.length = c.capacity
            return self._view(0, c.capacity), self._view(1, c.capacity)
        if self.length + n > c.capacity:
            raise RuntimeError(f"TreeKVCache capacity {c.capacity} exceeded ({self.length} + {n})")
        kernels.kv_append(kc, vc, key_states, value_states, offset=self.length)
        self.length += n
        return self.keys, self.values

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.length + query_length, 0

    def get_seq_length(self) -> int:
        return self.length

    def get_max_cache_shape(self) -> int:
        return self._cache.capacity

    def crop(self, max_length: int) -> None:
        if max_length < 0:
            max_length = self.length - abs(max_length)
        self.length = max(0, min(self.length, max_length))

    def reset(self) -> None:
        self.length = 0

    def offload(self):
        raise NotImplementedError("TreeKVCache stays resident in HBM")

    def prefetch(self):
        return None

    def reorder_cache(self, beam_idx):
        raise NotImplementedError("TreeKVCache holds one sequence")


class TreeKVCache(Cache):
    """One bf16 slab for all layers' K and V, appended and compacted in place."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, capacity: int,
                 dtype=torch.bfloat16, device=None):
        self.num_layers = int(num_layers)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)
        self.capacity = int(capacity)
        self.dtype = dtype
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.type != "cuda":
            raise RuntimeError("TreeKVCache lives on a CUDA device")
        self.slab = self._make_slab()
        self.length_dev = torch.zeros(1, dtype=torch.int64, device=self.device)
        self.device_length = False
        super().__init__(layers=[self.layer_class(self, i) for i in range(self.num_layers)])

    layer_class = TreeKVLayer

    def _make_slab(self) -> torch.Tensor:
        return torch.zeros((2 * self.num_layers, self.num_kv_heads, self.capacity, self.head_dim), dtype=self.dtype,
                           device=self.device)

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, offset: int = 0,
               offset_dev: torch.Tensor | None = None) -> None:
        """Write ``[heads, n, head_dim]`` rows of one layer at ``offset`` (the layer's length is not changed)."""
        kernels.kv_append(self.slab[2 * layer], self.slab[2 * layer + 1], k_new, v_new, offset=offset,
                          offset_dev=offset_dev)

    @classmethod
    def for_model(cls, config, capacity: int, dtype=torch.bfloat16, device=None) -> "TreeKVCache":
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        return cls(config.num_hidden_layers, config.num_key_value_heads, head_dim, capacity, dtype, device)

    # host / device length ----------------------------------------------------
    @property
    def length(self) -> int:
        return self.layers[0].length

    def set_length(self, n: int) -> None:
        for layer in self.layers:
            layer.length = int(n)
        self.length_dev.fill_(int(n))

    def use_device_length(self, enabled: bool) -> None:
        """Append at ``length_dev`` and hand out full-capacity views (for graph capture)."""
        self.device_length = bool(enabled)

    # Cache API ---------------------------------------------------------------
    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self.layers[layer_idx].length

    def get_mask_sizes(self, query_length: int, layer_idx: int = 0) -> tuple[int, int]:
        return self.layers[layer_idx].get_mask_sizes(query_length)

    def get_max_cache_shape(self, layer_idx: int = 0) -> int:
        return self.capacity

    def crop(self, max_length: int) -> None:
        for layer in self.layers:
            layer.crop(max_length)

    def reset(self) -> None:
        self.set_length(0)

    @property
    def is_compileable(self) -> bool:
        return False

    def batch_repeat_interleave(self, repeats: int):
        raise NotImplementedError("TreeKVCache holds one sequence")

    def batch_select_indices(self, indices):
        raise NotImplementedError("TreeKVCache holds one sequence")


class TreeKVLayerQ4(TreeKVLayer):
    """One layer of a ``TreeKVCacheQ4``; ``keys`` / ``values`` are decoded copies."""

    def _view(self, kv: int, length: int) -> torch.Tensor:
        return kernels.kv_read_q4(self._cache.slab[2 * self.index + kv], 0, length).unsqueeze(0)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """Quantise the new rows into the cache; returns what stands for all rows (``Q4Rows``), as keys and values."""
        c = self._cache
        n = key_states.shape[-2]
        before = self.length
        if c.device_length:
            c.append(self.index, key_states, value_states, offset_dev=c.length_dev)
            self.length = c.capacity
            prefix = c.capacity - n
        else:
            if before + n > c.capacity:
                raise RuntimeError(f"TreeKVCache capacity {c.capacity} exceeded ({before} + {n})")
            c.append(self.index, key_states, value_states, offset=before)
            self.length += n
            prefix = before
        rows = Q4Rows(c.slab[2 * self.index], c.slab[2 * self.index + 1], key_states, value_states, prefix,
                      c.device_length)
        return rows, rows


class Q4Rows(torch.Tensor):
    """The keys (and values) a 4-bit cache hands to the attention backend.

    It has the shape that ``TreeKVCache`` would return, but no data: the
    ``retree_tree`` backend reads the cache's rows (``k``, ``v``: uint8 ``[heads,
    capacity, 72]``, of which ``prefix_len`` rows and the new ones are used) or, for a
    prompt over an empty cache, the new rows (``k_new``, ``v_new``), so no bf16 copy of the cached
    rows is made.  Any other use, by another backend, is an error.
    """

    @staticmethod
    def __new__(cls, k, v, k_new, v_new, prefix_len: int, device_length: bool):
        shape = (*k_new.shape[:-2], prefix_len + k_new.shape[-2], k_new.shape[-1])
        self = torch.Tensor._make_wrapper_subclass(cls, shape, dtype=k_new.dtype, device=k_new.device)
        self.k, self.v, self.k_new, self.v_new = k, v, k_new, v_new
        self.prefix_len, self.device_length = prefix_len, device_length
        return self

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError(f"rows of a 4-bit cache are read by the retree_tree attention backend only (asked for "
                           f"{func}); cache.layers[i].keys and .values are decoded copies")

    def data_ptr(self):
        raise RuntimeError("rows of a 4-bit cache have no data of their own")

    def __repr__(self, **kwargs):
        return f"Q4Rows(shape={tuple(self.shape)}, prefix_len={self.prefix_len})"


class TreeKVCacheQ4(TreeKVCache):
    """The same cache with rows of 4 bits: 72 bytes a head and token instead of 256.

    ``slab`` is uint8 ``[2 * layers, kv_heads, capacity, 72]`` (the row's layout is
    in ``include/retree_b200.h``, RT_Q4_ROW_BYTES); the capacity is rounded up to
    an even number.  Appending quantises (``kernels.kv_append_q4``), the
    ``retree_tree`` attention reads the 4-bit rows (``kernels.tree_attention_q4``),
    compaction moves them as they are.  Other attention backends are refused
    (``for_model``, ``Q4Rows``).  A prompt over an empty cache attends to
    its own bf16 keys and values; whatever comes later attends to the cached
    rows, its own among them, so a token's result does not depend on whether its
    ancestors were committed or are still in the tree.
    """

    layer_class = TreeKVLayerQ4

    def _make_slab(self) -> torch.Tensor:
        if self.head_dim != 128 or self.dtype != torch.bfloat16:
            raise RuntimeError("the 4-bit cache holds bf16 rows of head_dim 128")
        self.capacity += self.capacity & 1
        return torch.zeros((2 * self.num_layers, self.num_kv_heads, self.capacity, kernels.Q4_ROW_BYTES),
                           dtype=torch.uint8, device=self.device)

    @classmethod
    def for_model(cls, config, capacity: int, dtype=torch.bfloat16, device=None) -> "TreeKVCacheQ4":
        from .attention import NAME
        from .headsplit import NAME as HEADSPLIT_NAME

        impl = getattr(config, "_attn_implementation", None)
        if impl not in (None, NAME, HEADSPLIT_NAME):
            raise RuntimeError(f"a 4-bit cache needs attn_implementation={NAME!r} (or {HEADSPLIT_NAME!r}), "
                               f"not {impl!r}")
        return super().for_model(config, capacity, dtype, device)

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, offset: int = 0,
               offset_dev: torch.Tensor | None = None) -> None:
        kernels.kv_append_q4(self.slab[2 * layer], self.slab[2 * layer + 1], k_new, v_new, offset=offset,
                             offset_dev=offset_dev)


def make_cache(kv_bits: int, *args, **kwargs) -> TreeKVCache:
    """A ``TreeKVCache`` (16 bits) or a ``TreeKVCacheQ4`` (4 bits)."""
    if kv_bits not in (16, 4):
        raise ValueError("kv_bits must be 16 or 4")
    return (TreeKVCacheQ4 if kv_bits == 4 else TreeKVCache)(*args, **kwargs)
