"""Tree-verify attention as a transformers attention backend.

``register()`` adds ``"retree_tree"`` to ``transformers.AttentionInterface``;
a model loaded with ``attn_implementation="retree_tree"`` then calls
``tree_attention_forward`` from ``Qwen3Attention.forward``
(models/qwen3/modeling_qwen3.py:273-286) with the arguments HF's SDPA backend
receives (integrations/sdpa_attention.py:40-50) and gets the same
``(out [B, n, Hq, D], None)`` back (:102-104).  Every call runs the sm_100a
kernel; there is no repeat_kv and no fallback.

Masks understood (the 4-D mask is passed through untouched by HF,
masking_utils.py:827-829):
  * a ``TreeMask`` from ``retree_b200.ddtree.compile_ddtree_tree``: packed
    ancestor bits of the tree block (and, in device-length mode, the device
    word holding the prefix length);
  * the dense additive mask the reference's ``compile_ddtree_tree`` writes
    (ddtree.py:629-640): its tree block is packed to bits on the device;
  * no mask (prefill / plain decode): causal attention of the new tokens over
    the cache, run as a chain-shaped tree -- unless the caller asks for
    ``is_causal=False`` (the DFlash draft's attention, model/dflash.py:47 and
    its callers' kwargs), which the SDPA backend honours the same way
    (sdpa_attention.py:64-77): then every new token sees every key.

Whole prompts can take their own kernel (``kernels.prompt_attention``: the hidden
half of the scores is not computed and no mask is read): always when the call
carries transformers' packed-sequence offsets (``cu_seq_lens_q`` and
``cu_seq_lens_k``, which a plain causal mask would mix up) or a prompt starts a
4-bit cache, and otherwise inside ``prompt_kernel()``.  Over a 4-bit cache
(``TreeKVCacheQ4``) trees and later tokens read the cached rows
(``kernels.tree_attention_q4``).
"""

from __future__ import annotations

import contextlib
import contextvars

import numpy as np
import torch

from . import kernels
from .cache import Q4Rows

NAME = "retree_tree"

_CAUSAL_BITS: dict = {}

#: when a list, every call appends (start event, end event, prefix_len, n, q heads, kv heads)
PROFILE: list | None = None


#: whether an unmasked causal call runs prompt_attention (set by prompt_kernel())
_PROMPT_KERNEL = contextvars.ContextVar("retree_prompt_kernel", default=False)

#: new tokens over a 4-bit cache above which a causal call reads the cache's values
#: once and runs prompt_attention, instead of a chain-shaped tree over the 4-bit rows.
#: 32 / 8 heads, graph, chain against read and prompt: 128 tokens over 2048 rows 20.5 us and
#: 34.6, over 32768 rows 77 and 120; 256 tokens 33.0 and 34.2, 158 and 171; 512 tokens
#: 57 and 38, 334 and 350; 1024 tokens 65 and 74, 635 and 534.  The bits of a chain also
#: grow with the square of its length.
_Q4_CHAIN_MAX = 256


@contextlib.contextmanager
def prompt_kernel(enabled: bool = True):
    """Inside, calls without a mask (prompts, chunks of prompts) run ``kernels.prompt_attention``."""
    token = _PROMPT_KERNEL.set(bool(enabled))
    try:
        yield
    finally:
        _PROMPT_KERNEL.reset(token)


class TreeMask:
    """Marker carried as attributes on the 4-D mask tensor handed to the model."""

    BITS_ATTR = "_rt_bits"           # int32 [n, W] packed ancestor bits
    PREFIX_DEV_ATTR = "_rt_prefix_dev"  # int64[1] device prefix length (device-length mode) or None


def attach(mask4d: torch.Tensor, bits: torch.Tensor, prefix_dev: torch.Tensor | None = None) -> torch.Tensor:
    setattr(mask4d, TreeMask.BITS_ATTR, bits)
    setattr(mask4d, TreeMask.PREFIX_DEV_ATTR, prefix_dev)
    return mask4d


def causal_bits(n: int, device) -> torch.Tensor:
    """Lower-triangular packed mask: node i sees nodes 0..i (a chain), int32 ``[n, ceil(n/32)]``."""
    key = (torch.device(device).index, n)
    b = _CAUSAL_BITS.get(key)
    if b is None:
        w = (n + 31) // 32
        vis = np.arange(w * 32)[None, :] <= np.arange(n)[:, None]
        words = np.packbits(vis, axis=1, bitorder="little").view("<u4").view(np.int32)
        b = torch.from_numpy(np.ascontiguousarray(words)).to(device)
        _CAUSAL_BITS[key] = b
    return b


def full_bits(n: int, device) -> torch.Tensor:
    """Every node sees every node of the block, int32 ``[n, ceil(n/32)]`` (bits past n are ignored)."""
    key = ("full", torch.device(device).index, n)
    b = _CAUSAL_BITS.get(key)
    if b is None:
        b = torch.full((n, (n + 31) // 32), -1, dtype=torch.int32, device=device)
        _CAUSAL_BITS[key] = b
    return b


def _bits_for(mask, n: int, key_len: int, device, causal: bool = True):
    if mask is None:
        return (causal_bits(n, device) if causal else full_bits(n, device)), None
    bits = getattr(mask, TreeMask.BITS_ATTR, None)
    if bits is not None:
        return bits, getattr(mask, TreeMask.PREFIX_DEV_ATTR, None)
    if mask.dim() != 4:
        raise RuntimeError("retree_tree attention takes a 4-D tree mask")
    if mask.dtype == torch.int32:
        return mask[0, 0, :n], None
    # dense additive mask (0 visible / finfo.min hidden): pack its tree block
    if mask.shape[-1] < key_len:
        raise RuntimeError("dense tree mask narrower than the key length")
    m2 = mask[0, 0, :n, :key_len]
    if m2.stride(-1) != 1:
        m2 = m2.contiguous()
    return kernels.mask_from_dense(m2, key_len - n, n), None


class _Timer:
    """Events around a call's attention kernel, for PROFILE (records nothing when that is None)."""

    def __init__(self):
        self.on = PROFILE is not None
        self.events = [torch.cuda.Event(enable_timing=True) for _ in range(2)] if self.on else None

    def start(self) -> None:
        if self.on:
            self.events[0].record()

    def stop(self, *shape) -> None:
        if self.on:
            self.events[1].record()
            PROFILE.append((*self.events, *shape))


def _q4_forward(query, attention_mask, scaling, causal: bool, rows: Q4Rows, timer) -> torch.Tensor:
    """Attention of new tokens over a 4-bit cache that already holds their rows."""
    n, hq = query.shape[2], query.shape[1]
    if attention_mask is None and not rows.device_length and causal:
        if rows.prefix_len == 0:
            timer.start()
            return kernels.prompt_attention(query, rows.k_new, rows.v_new, scale=scaling)
        if n > _Q4_CHAIN_MAX:
            timer.start()
            k, v = (kernels.kv_read_q4(x, 0, rows.prefix_len + n) for x in (rows.k, rows.v))
            return kernels.prompt_attention(query, k, v, scale=scaling)
    bits, prefix_dev = _bits_for(attention_mask, n, rows.prefix_len + n, query.device, causal=causal)
    if rows.device_length and prefix_dev is None:
        raise RuntimeError("a cache in device-length mode needs a tree mask with its prefix length")
    splits = kernels.default_splits_q4(n, hq, rows.k.shape[0], rows.k.shape[1] - n)
    timer.start()
    return kernels.tree_attention_q4(query, rows.k, rows.v, bits, rows.prefix_len, scale=scaling, num_splits=splits,
                                     prefix_len_dev=prefix_dev)


def _check_key_offsets(cu_q, cu_k, keys: int) -> None:
    """Packed queries over more keys than queries: the keys' offsets have to reach the last key.

    Callers without a cache pass the queries' offsets for both; over a cache those
    are in range, but name its first rows.  (One read of an offset, on this path only.)
    """
    if cu_k is None or cu_k.numel() < 2 or cu_k is cu_q or cu_k.data_ptr() == cu_q.data_ptr():
        raise RuntimeError("packed queries over cached keys need the keys' own offsets")
    if cu_k.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("packed queries over cached keys are not captured: their offsets are checked on the host")
    if int(cu_k[-1]) != keys:
        raise RuntimeError(f"packed queries over cached keys: cu_seq_lens_k ends before the last of the {keys} keys")


def _tree_forward(query, key, value, attention_mask, scaling, causal: bool, timer) -> torch.Tensor:
    """rt_tree_attn over bf16 K/V: the mask's tree, or the new tokens as a chain."""
    n = query.shape[2]
    bits, prefix_dev = _bits_for(attention_mask, n, key.shape[2], query.device, causal=causal)
    timer.start()
    # rows allocated per head: the launch (and its split of the keys) is sized
    # for the cache's capacity, so host-length and device-length rounds over the
    # same cache run the identical launch
    cap = key.shape[2]
    if key.stride(-1) == 1 and key.stride(2) > 0 and key.stride(1) % key.stride(2) == 0:
        cap = max(cap, key.stride(1) // key.stride(2))
    splits = kernels.default_splits(n, query.shape[1], key.shape[1], cap - n)
    if prefix_dev is not None:
        # full-capacity K/V views; the real prefix length lives on the device
        return kernels.tree_attention(query, key, value, bits, prefix_len=cap - n, scale=scaling,
                                      prefix_len_dev=prefix_dev, kv_capacity=cap, num_splits=splits)
    return kernels.tree_attention(query, key, value, bits, prefix_len=key.shape[2] - n, scale=scaling,
                                  kv_capacity=cap, num_splits=splits)


def tree_attention_forward(module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                           attention_mask, dropout: float = 0.0, scaling: float | None = None,
                           sliding_window=None, **kwargs):
    """HF attention backend: ``query [1, Hq, n, D]``, ``key/value [1, Hkv, S, D]``."""
    if dropout and module.training:
        raise RuntimeError("retree_tree attention is inference-only")
    if sliding_window is not None:
        raise RuntimeError("retree_tree attention has no sliding-window mode")
    if query.shape[0] != 1:
        raise RuntimeError("retree_tree attention verifies one sequence (batch 1)")
    n = query.shape[2]
    # the SDPA backend's rule: the call's is_causal, else the module's (default causal)
    causal = kwargs.get("is_causal", None)
    if causal is None:
        causal = getattr(module, "is_causal", True)
    causal = bool(causal)
    rows = key if isinstance(key, Q4Rows) else None
    cu_q, cu_k = kwargs.get("cu_seq_lens_q"), kwargs.get("cu_seq_lens_k")
    prefix = key.shape[2] - n if rows is None else rows.prefix_len
    timer = _Timer()
    if cu_q is not None and attention_mask is None:
        if not causal or (rows is not None and (rows.device_length or rows.prefix_len > 0)):
            raise RuntimeError("packed sequences run causally over keys of their own (no cached prefix)")
        if rows is None and key.shape[2] != n:
            _check_key_offsets(cu_q, cu_k, key.shape[2])
        k, v = (key, value) if rows is None else (rows.k_new, rows.v_new)
        timer.start()
        out = kernels.prompt_attention(query, k, v, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, scale=scaling)
    elif rows is not None:
        out = _q4_forward(query, attention_mask, scaling, causal, rows, timer)
    elif _PROMPT_KERNEL.get() and attention_mask is None and causal:
        timer.start()
        out = kernels.prompt_attention(query, key, value, scale=scaling)
    else:
        out = _tree_forward(query, key, value, attention_mask, scaling, causal, timer)
    timer.stop(prefix, n, query.shape[1], key.shape[1])
    return out.unsqueeze(0), None


def register() -> str:
    """Register the backend with transformers and return its name."""
    from transformers import AttentionInterface

    AttentionInterface.register(NAME, tree_attention_forward)
    return NAME
