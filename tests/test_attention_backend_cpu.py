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


@pytest.mark.parametrize("cu_k", [None, "same", [0, 2, 6], [0, 4, 8]])
def test_packed_queries_over_cached_keys_need_offsets_that_reach_the_last_key(cu_k):
    """Offsets of the queries, or of the first rows of a cache, would name other keys than the new ones."""
    with pytest.raises(RuntimeError, match="packed"):
        _call(6, 10, [0, 2, 6], cu_k)


def test_packed_queries_over_keys_of_their_own_reach_the_kernel():
    for cu_k, keys in ((None, 6), ("same", 6), ([0, 4, 10], 10)):
        with pytest.raises(RuntimeError, match="CUDA"):
            _call(6, keys, [0, 2, 6], cu_k)
