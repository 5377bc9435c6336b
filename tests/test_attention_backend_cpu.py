"""Refusals of the attention backend that need no kernel (CPU only)."""

import pytest
import torch

from retree_b200 import attention


class _Module:
    training = False
    is_causal = True


def _call(n, keys, cu_q, cu_k):
    q, kv = torch.zeros((1, 8, n, 128), dtype=torch.bfloat16), torch.zeros((1, 2, keys, 128), dtype=torch.bfloat16)
    off = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32)  # noqa: E731
    cu_q = off(cu_q)
    return attention.tree_attention_forward(_Module(), q, kv, kv, None, scaling=0.1, cu_seq_lens_q=cu_q,
                                            cu_seq_lens_k=cu_q if cu_k == "same" else off(cu_k))


@pytest.mark.parametrize("cu_k", [None, "same", [0, 2, 6], [0, 4, 8], [], [10]])
def test_packed_queries_over_cached_keys_need_offsets_that_reach_the_last_key(cu_k):
    """Offsets of the queries, or of the first rows of a cache, would name other keys than the new ones."""
    with pytest.raises(RuntimeError, match="packed"):
        _call(6, 10, [0, 2, 6], cu_k)


def test_packed_queries_over_keys_of_their_own_reach_the_kernel():
    for cu_k, keys in ((None, 6), ("same", 6), ([0, 4, 10], 10)):
        with pytest.raises(RuntimeError, match="CUDA"):
            _call(6, keys, [0, 2, 6], cu_k)


def _rows():
    from retree_b200.cache import Q4Rows
    k = torch.zeros((1, 2, 3, 128), dtype=torch.bfloat16)
    slab = torch.zeros((2, 16, 72), dtype=torch.uint8)
    return Q4Rows(slab, slab, k, k, prefix_len=7, device_length=False), k


def test_rows_of_a_4bit_cache_are_of_no_use_to_another_backend():
    """They stand for all cached keys, so whatever is asked of them but their shape is refused."""
    from transformers.integrations.sdpa_attention import sdpa_attention_forward
    rows, k = _rows()
    assert rows.shape == (1, 2, 10, 128) and rows.dtype == torch.bfloat16 and rows.device == k.device
    q = torch.zeros((1, 8, 3, 128), dtype=torch.bfloat16)
    for use in (lambda: rows + 1, lambda: rows.clone(), lambda: rows.to(torch.float32), lambda: rows[0],
                lambda: rows.transpose(1, 2), lambda: torch.cat([rows, rows]), lambda: rows.detach(),
                lambda: rows.data_ptr(), lambda: rows.as_subclass(torch.Tensor), lambda: rows.view(2, 10, 128),
                lambda: torch.nn.functional.scaled_dot_product_attention(q, rows, rows, enable_gqa=True),
                lambda: sdpa_attention_forward(_Module(), q[:, :, :1], rows, rows, None)):
        with pytest.raises(RuntimeError, match="4-bit"):
            use()


def test_the_4bit_cache_is_refused_for_a_model_with_another_backend():
    from retree_b200.cache import TreeKVCacheQ4
    from retree_b200.target import qwen3_config
    cfg = qwen3_config("small", num_hidden_layers=1)
    for impl in ("sdpa", "eager", "sdpa_headsplit"):
        cfg._attn_implementation = impl
        with pytest.raises(RuntimeError, match="retree_tree"):
            TreeKVCacheQ4.for_model(cfg, capacity=16, device="cpu")
    for impl in ("retree_tree", "retree_tree_headsplit", None):
        cfg._attn_implementation = impl
        with pytest.raises(RuntimeError, match="CUDA device"):  # (past that check)
            TreeKVCacheQ4.for_model(cfg, capacity=16, device="cpu")
