"""Torch-tensor wrappers over the C-ABI kernels.

PyTorch supplies device memory and the current stream; every computation is a
call into ``libretree_b200.so``.  Inputs must already be CUDA tensors: there
is no CPU path, and a missing library raises (``retree_b200._lib.load``).
"""

from __future__ import annotations

import ctypes
import functools
import threading

import numpy as np
import torch

from . import _lib

_DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("retree_b200 kernels take CUDA tensors (no CPU path)")


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device=None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class _DeviceState:
    """Per-device scratch and status words (grown on demand, never shrunk)."""

    def __init__(self):
        self.lock = threading.Lock()
        self.bufs: dict = {}

    # Buffers are made outside inference mode: they are updated in place from
    # both inside and outside it (an inference tensor refuses the latter).
    def buffer(self, device, name: str, nbytes: int) -> torch.Tensor:
        key = (torch.device(device).index, name)
        with self.lock:
            b = self.bufs.get(key)
            if b is None or b.numel() < nbytes:
                with torch.inference_mode(False):
                    b = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
                self.bufs[key] = b
            return b

    def status(self, device) -> torch.Tensor:
        key = (torch.device(device).index, "__status__")
        with self.lock:
            s = self.bufs.get(key)
            if s is None:
                with torch.inference_mode(False):
                    s = torch.zeros(1, dtype=torch.int32, device=device)
                self.bufs[key] = s
            return s


_STATE = _DeviceState()

#: number of kernel launches issued through these wrappers (for launch accounting)
LAUNCHES = 0


def _count(n: int = 1) -> None:
    global LAUNCHES
    LAUNCHES += n


def _nccl_group_up() -> bool:
    import torch.distributed as dist
    return dist.is_available() and dist.is_initialized() and dist.get_backend() == "nccl"


def set_pdl(enabled: bool) -> None:
    """Programmatic dependent launch between the verify-forward kernels (rt_set_pdl).

    It is never turned on in a process with an NCCL process group: a 2-process
    run with NCCL collectives between dependent-launched kernels stalled, with
    no cause found, so the two are kept apart (``pdl_guard``).
    """
    if enabled and _nccl_group_up():
        raise RuntimeError("programmatic dependent launch stays off in a process with an NCCL process group")
    _lib.load().rt_set_pdl(int(bool(enabled)))


def pdl_guard() -> None:
    """Turn programmatic dependent launch off if this process has an NCCL process group."""
    if _nccl_group_up():
        _lib.load().rt_set_pdl(0)


def pdl_enabled() -> bool:
    return bool(_lib.load().rt_pdl_enabled())


def status_tensor(device) -> torch.Tensor:
    """The device status word the kernels of this process report into."""
    return _STATE.status(device)


def check_device_status(device, reset: bool = True) -> None:
    """Synchronise on the status word and raise if a kernel reported an error."""
    s = _STATE.status(device)
    code = int(s.item())
    if reset and code:
        s.zero_()
    if code:
        raise RuntimeError(f"retree_b200 kernel reported: {_lib.status_string(code)}")


# ---------------------------------------------------------------------------
# KV cache
# ---------------------------------------------------------------------------
def kv_compact(tensors, past_length: int, keep: torch.Tensor, cur_length: int | None = None,
               n_keep_dev: torch.Tensor | None = None, n_keep: int | None = None,
               past_len_dev: torch.Tensor | None = None) -> None:
    """In-place compaction of appended rows (ddtree.py:666-731 semantics).

    ``tensors``: one ``[..., S, D]`` tensor or a list of them.  All leading
    dims of a tensor are folded into one head axis when their strides allow
    (a whole ``[layers*2, heads, S, D]`` slab then moves in ONE launch).
    ``keep``: int64 CUDA tensor of window-relative indices; ``n_keep_dev``
    (int32[1], optional) supplies the count at run time.
    """
    lib = _lib.load()
    group = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not group:
        return
    _require_cuda(keep, *group)
    if keep.dtype != torch.int64:
        raise RuntimeError("keep_current_indices must have dtype torch.long")
    nk = int(keep.numel()) if n_keep is None else int(n_keep)
    for t in group:
        if t.dim() < 2:
            raise RuntimeError("cache_tensor must have rank >= 2")
        seq = t.shape[-2]
        if past_len_dev is None and (past_length < 0 or past_length > seq):
            raise RuntimeError("past_length exceeds cache sequence length")
        cur = (seq - past_length) if cur_length is None else int(cur_length)
        if cur <= 0:
            continue
        if t.stride(-1) != 1:
            raise RuntimeError("cache rows must be contiguous")
        try:
            v = t.view(-1, seq, t.shape[-1])
        except RuntimeError:
            kv_compact(list(t.unbind(0)), past_length, keep, cur_length, n_keep_dev, n_keep, past_len_dev)
            continue
        es = v.element_size()
        rc = lib.rt_kv_compact(None, v.data_ptr(), 1, 0, v.shape[0], v.stride(0) * es, v.stride(1) * es,
                               v.shape[2] * es, int(past_length), _ptr(past_len_dev), cur, keep.data_ptr(), nk,
                               _ptr(n_keep_dev), _STATE.status(t.device).data_ptr(), _stream(t.device))
        _lib.check(rc, "rt_kv_compact")
        _count()


def kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
              offset: int = 0, offset_dev: torch.Tensor | None = None) -> None:
    """Write ``[heads, n, D]`` new rows at ``offset`` of ``[heads, cap, D]`` caches (views allowed)."""
    lib = _lib.load()
    _require_cuda(k_cache, v_cache, k_new, v_new)
    k_cache, v_cache = _as3(k_cache), _as3(v_cache)
    k_new, v_new = _as3(k_new), _as3(v_new)
    if k_cache.stride() != v_cache.stride():
        raise RuntimeError("K and V caches must share strides")
    if k_new.stride() != v_new.stride():
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    es = k_cache.element_size()
    heads, n, d = k_new.shape
    rc = lib.rt_kv_append(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0) * es, k_cache.stride(1) * es,
                          k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0) * es, k_new.stride(1) * es, heads, n,
                          d * es, k_cache.shape[1], int(offset), _ptr(offset_dev),
                          _STATE.status(k_cache.device).data_ptr(), _stream(k_cache.device))
    _lib.check(rc, "rt_kv_append")
    _count()


def _as3(t: torch.Tensor) -> torch.Tensor:
    if t.dim() == 4:
        if t.shape[0] != 1:
            raise RuntimeError("batch size 1 only")
        t = t[0]
    if t.dim() != 3 or t.stride(-1) != 1:
        raise RuntimeError("expected [heads, seq, head_dim] with contiguous head_dim")
    return t


# ---------------------------------------------------------------------------
# Tree-verify attention
# ---------------------------------------------------------------------------
def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask_bits: torch.Tensor, prefix_len: int,
                   scale: float | None = None, out: torch.Tensor | None = None, num_splits: int = 0,
                   path: int = 0, prefix_len_dev: torch.Tensor | None = None,
                   kv_capacity: int | None = None) -> torch.Tensor:
    """Masked GQA attention of n tree nodes over ``[prefix ; tree block]``.

    q: ``[n, Hq, D]`` or HF's ``[1, Hq, n, D]``; k, v: ``[Hkv, S, D]`` or
    ``[1, Hkv, S, D]`` (rows ``[0, prefix_len + n)`` are used);
    mask_bits: int32 ``[n, W]`` ancestor bits of the tree block.
    Returns ``out`` ``[n, Hq, D]`` bf16 (HF's ``[1, n, Hq, D]`` after unsqueeze).
    """
    lib = _lib.load()
    _require_cuda(q, k, v, mask_bits)
    if q.dim() == 4:
        if q.shape[0] != 1:
            raise RuntimeError("batch size 1 only")
        q = q[0].transpose(0, 1)  # [n, Hq, D] view
    k, v = _as3(k), _as3(v)
    if k.stride() != v.stride():
        raise RuntimeError("K and V must share strides")
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise RuntimeError("tree attention runs on bf16 q/k/v")
    n, hq, d = q.shape
    hkv = k.shape[0]
    if out is None:
        out = torch.empty((n, hq, d), dtype=torch.bfloat16, device=q.device)
    es = 2
    mask_bits = mask_bits if mask_bits.dim() == 2 else mask_bits.reshape(n, -1)
    if mask_bits.stride(-1) != 1:
        mask_bits = mask_bits.contiguous()
    words = mask_bits.stride(0)
    scale = d ** -0.5 if scale is None else float(scale)
    cap = k.shape[1] if kv_capacity is None else int(kv_capacity)
    splits, merged = attn_plan(n, hq, hkv, int(prefix_len), num_splits, path)
    ws_bytes = 0 if merged else lib.rt_tree_attn_workspace_size(n, hq, hkv, d, int(prefix_len), splits)
    ws = _STATE.buffer(q.device, "attn_ws", ws_bytes) if ws_bytes else None
    rc = lib.rt_tree_attn(q.data_ptr(), q.stride(0) * es, q.stride(1) * es, k.data_ptr(), v.data_ptr(),
                          k.stride(0) * es, k.stride(1) * es, cap, out.data_ptr(), out.stride(0) * es,
                          out.stride(1) * es, mask_bits.data_ptr(), words, n, int(prefix_len),
                          _ptr(prefix_len_dev), hq, hkv, d, scale, splits, path, _ptr(ws), ws_bytes,
                          _STATE.status(q.device).data_ptr(), _stream(q.device))
    _lib.check(rc, "rt_tree_attn")
    _count(2 if ws_bytes else 1)  # the combine launch runs only when the partials go through the workspace
    return out


def attn_plan(n: int, num_q_heads: int, num_kv_heads: int, prefix_len: int, num_splits: int = 0,
              path: int = 0) -> tuple[int, bool]:
    """(key splits, merged in the kernel) of an rt_tree_attn launch of this shape (rt_tree_attn_plan)."""
    sp, mg = ctypes.c_int(0), ctypes.c_int(0)
    _lib.check(_lib.load().rt_tree_attn_plan(n, num_q_heads, num_kv_heads, int(prefix_len), int(num_splits), int(path),
                                             ctypes.byref(sp), ctypes.byref(mg), None), "rt_tree_attn_plan")
    return sp.value, bool(mg.value)


def default_splits(n: int, num_q_heads: int, num_kv_heads: int, prefix_len: int) -> int:
    """Key splits rt_tree_attn picks for this shape (one wave of CTAs)."""
    return int(_lib.load().rt_tree_attn_default_splits(n, num_q_heads, num_kv_heads, int(prefix_len)))


def mask_from_dense(dense: torch.Tensor, col0: int, n: int, words: int | None = None) -> torch.Tensor:
    """Packed bits of the tree block of a dense additive mask (0 = visible)."""
    lib = _lib.load()
    _require_cuda(dense)
    d2 = dense.reshape(-1, dense.shape[-1]) if dense.dim() > 2 else dense
    if d2.stride(-1) != 1:
        raise RuntimeError("dense mask rows must be contiguous")
    w = (n + 31) // 32 if words is None else words
    bits = torch.empty((n, w), dtype=torch.int32, device=dense.device)
    rc = lib.rt_mask_from_dense(d2.data_ptr(), _DTYPE_CODE[d2.dtype], d2.stride(0), int(col0), n, bits.data_ptr(),
                                w, _stream(dense.device))
    _lib.check(rc, "rt_mask_from_dense")
    _count()
    return bits


# ---------------------------------------------------------------------------
# Draft top-k and tree construction
# ---------------------------------------------------------------------------
def draft_topk(logits: torch.Tensor, k: int, out=None):
    """``(top_logp f32[R,k], top_ids i64[R,k], log_z f32[R])`` of ``[R, V]`` logits on the device."""
    lib = _lib.load()
    _require_cuda(logits)
    if logits.dim() != 2 or logits.stride(-1) != 1:
        raise RuntimeError("logits must be [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    dev = logits.device
    if out is None:
        out = (torch.empty((rows, k), dtype=torch.float32, device=dev),
               torch.empty((rows, k), dtype=torch.int64, device=dev),
               torch.empty((rows,), dtype=torch.float32, device=dev))
    ws_bytes = lib.rt_draft_topk_workspace_size(rows, vocab, k)
    ws = _STATE.buffer(dev, "topk_ws", ws_bytes)
    rc = lib.rt_draft_topk(logits.data_ptr(), _DTYPE_CODE[logits.dtype], logits.stride(0), rows, vocab, k,
                           out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), ws.data_ptr(), ws_bytes,
                           _stream(dev))
    _lib.check(rc, "rt_draft_topk")
    _count(2)
    return out


STRATEGY_CODE = {"heap": 0, "ngram": 1, "rank_gated_ngram": 2}

_LOG1P_CACHE: dict = {}


def log1p_table(device, n: int) -> torch.Tensor:
    """``np.log1p(c)`` for c = 0..n as binary64 on ``device`` (the reference's bonus base)."""
    key = (torch.device(device).index, n)
    t = _LOG1P_CACHE.get(key)
    if t is None:
        t = torch.from_numpy(np.log1p(np.arange(n + 1, dtype=np.float64))).to(device)
        _LOG1P_CACHE[key] = t
    return t


def tree_build(top_logp: torch.Tensor, top_ids: torch.Tensor, budget: int, strategy: str, params,
               ctx: torch.Tensor | None = None, ctx_len_dev: torch.Tensor | None = None, ctx_len: int | None = None,
               out: dict | None = None, root: int = -1, root_dev=None, start: int = 0, start_dev=None,
               mask_words: int | None = None) -> dict:
    """Best-first expansion on the device; returns a dict of device tensors.

    Keys: tokens i64[budget], depths i64[budget], parents i32[budget+1],
    mask i32[budget+1, W], count i32[1], verify_ids i64[budget+1],
    verify_pos i64[budget+1].  ``params``: oracle-compatible n-gram knobs
    (``max_n, beta, rank_cap, min_count, context_window, use_log_count,
    longer_weight, max_token_bonus``).
    """
    lib = _lib.load()
    _require_cuda(top_logp, top_ids, ctx)
    dev = top_logp.device
    rows, k = top_logp.shape
    code = STRATEGY_CODE[strategy]
    w = (budget + 1 + 31) // 32 if mask_words is None else mask_words
    if out is None:
        out = dict(
            tokens=torch.empty(max(budget, 1), dtype=torch.int64, device=dev),
            depths=torch.empty(max(budget, 1), dtype=torch.int64, device=dev),
            parents=torch.empty(budget + 1, dtype=torch.int32, device=dev),
            mask=torch.empty((budget + 1, w), dtype=torch.int32, device=dev),
            count=torch.empty(1, dtype=torch.int32, device=dev),
            verify_ids=torch.empty(budget + 1, dtype=torch.int64, device=dev),
            verify_pos=torch.empty(budget + 1, dtype=torch.int64, device=dev),
        )
    max_n = int(params.max_n) if code else 2
    ow_vals = [float(params.longer_weight ** max(0, n - 2)) for n in range(2, max_n + 1)]
    ow = (ctypes.c_double * max(len(ow_vals), 1))(*ow_vals)
    window = int(params.context_window)
    if ctx is not None:
        clen = int(ctx.numel()) if ctx_len is None else int(ctx_len)
    else:
        clen = 0
    # one table per window size (not per context length), so it is uploaded once
    table_n = window if window > 0 else max(clen, 1)
    table = log1p_table(dev, max(table_n, 1) + 1)
    rc = lib.rt_tree_build(
        top_logp.data_ptr(), top_ids.data_ptr(), rows, k, int(budget), code, _ptr(ctx), clen, _ptr(ctx_len_dev),
        window, max_n, float(params.beta), int(params.rank_cap), int(params.min_count), int(bool(params.use_log_count)),
        ctypes.addressof(ow), float(params.max_token_bonus), table.data_ptr(), int(table.numel()),
        out["tokens"].data_ptr(), out["depths"].data_ptr(), out["parents"].data_ptr(), out["mask"].data_ptr(), w,
        out["count"].data_ptr(), _ptr(out.get("verify_ids")), _ptr(out.get("verify_pos")), int(root), _ptr(root_dev),
        int(start), _ptr(start_dev), _STATE.status(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "rt_tree_build")
    _count()
    out["_keep_alive"] = (ow, table)
    return out


def tree_walk(parents: torch.Tensor, tokens: torch.Tensor, posterior: torch.Tensor, count: int | None = None,
              count_dev: torch.Tensor | None = None, out: dict | None = None, verify_ids=None, output_ids=None,
              start_dev=None) -> dict:
    """Exact walk on the device; returns ``accepted`` i64[n], ``accepted_len`` i32[1], ``next_token`` i64[1]."""
    lib = _lib.load()
    _require_cuda(parents, tokens, posterior)
    dev = parents.device
    n = parents.numel()
    if out is None:
        out = dict(accepted=torch.empty(n, dtype=torch.int64, device=dev),
                   accepted_len=torch.empty(1, dtype=torch.int32, device=dev),
                   next_token=torch.empty(1, dtype=torch.int64, device=dev))
    cnt = (n - 1) if count is None else int(count)
    post = posterior.reshape(-1)
    if post.dtype != torch.int64:
        post = post.to(torch.int64)
    rc = lib.rt_tree_walk(parents.data_ptr(), tokens.data_ptr(), cnt, _ptr(count_dev), post.data_ptr(),
                          out["accepted"].data_ptr(), out["accepted_len"].data_ptr(), out["next_token"].data_ptr(),
                          _ptr(verify_ids), _ptr(output_ids), 0 if output_ids is None else output_ids.numel(),
                          _ptr(start_dev), _STATE.status(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "rt_tree_walk")
    _count()
    return out


__all__ = ["kv_compact", "kv_append", "tree_attention", "mask_from_dense", "draft_topk", "tree_build",
           "tree_walk", "log1p_table", "status_tensor", "check_device_status", "STRATEGY_CODE"]


# ---------------------------------------------------------------------------
# Elementwise stages of the verify forward (retree_b200.fused)
# ---------------------------------------------------------------------------
def _rows_bf16(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.bfloat16 or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous bf16 tensor")


def embed_rmsnorm(ids: torch.Tensor, table: torch.Tensor, weight: torch.Tensor, eps: float,
                  residual: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """``residual = table[ids]``; ``out = rmsnorm(residual) * weight`` (bf16, rows = ids.numel())."""
    _require_cuda(ids, table, weight, residual, out)
    for t, nm in ((table, "table"), (weight, "weight"), (residual, "residual"), (out, "out")):
        _rows_bf16(t, nm)
    if ids.dtype != torch.int64 or not ids.is_contiguous():
        raise RuntimeError("ids must be contiguous int64")
    rows, hidden = ids.numel(), table.shape[-1]
    _lib.check(_lib.load().rt_embed_rmsnorm(ids.data_ptr(), table.data_ptr(), table.shape[0], residual.data_ptr(),
                                            weight.data_ptr(), out.data_ptr(), rows, hidden, float(eps),
                                            status_tensor(ids.device).data_ptr(), _stream(ids.device)),
               "rt_embed_rmsnorm")
    _count()
    return out


def add_rmsnorm(delta: torch.Tensor | None, residual: torch.Tensor, weight: torch.Tensor, eps: float,
                out: torch.Tensor) -> torch.Tensor:
    """``residual += delta`` (bf16 rounding), ``out = rmsnorm(residual) * weight``; delta may be None."""
    _require_cuda(delta, residual, weight, out)
    for t, nm in ((residual, "residual"), (weight, "weight"), (out, "out")) + (((delta, "delta"),) if delta is not None else ()):
        _rows_bf16(t, nm)
    hidden = residual.shape[-1]
    rows = residual.numel() // hidden
    _lib.check(_lib.load().rt_add_rmsnorm(_ptr(delta), residual.data_ptr(), weight.data_ptr(), out.data_ptr(), rows,
                                          hidden, float(eps), _stream(residual.device)), "rt_add_rmsnorm")
    _count()
    return out


def qk_norm_rope_append(qkv: torch.Tensor, num_q_heads: int, num_kv_heads: int, q_norm_w, k_norm_w, eps: float,
                        cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                        q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, offset: int = 0,
                        offset_dev: torch.Tensor | None = None) -> torch.Tensor:
    """Per-head q/k RMSNorm + rotary embedding; q to ``q_out [n, Hq, 128]``, k/v appended to the cache.

    ``k_cache``/``v_cache`` are ``[Hkv, capacity, 128]`` views with unit inner
    stride; rows land at ``offset`` (+ ``offset_dev[0]`` when given).
    """
    _require_cuda(qkv, cos_table, sin_table, positions, q_out, k_cache, v_cache, q_norm_w, k_norm_w, offset_dev)
    _rows_bf16(qkv, "qkv")
    _rows_bf16(q_out, "q_out")
    n = positions.numel()
    if qkv.numel() != n * (num_q_heads + 2 * num_kv_heads) * 128:
        raise RuntimeError("qkv does not hold n rows of (Hq + 2 Hkv) heads of 128")
    if positions.dtype != torch.int64 or not positions.is_contiguous():
        raise RuntimeError("positions must be contiguous int64")
    if k_cache.stride() != v_cache.stride() or k_cache.stride(-1) != 1 or k_cache.shape[0] != num_kv_heads:
        raise RuntimeError("k_cache/v_cache must be [Hkv, capacity, 128] views with equal strides")
    es = k_cache.element_size()
    _lib.check(_lib.load().rt_qk_norm_rope_append(
        qkv.data_ptr(), n, num_q_heads, num_kv_heads, 128, _ptr(q_norm_w), _ptr(k_norm_w), float(eps),
        cos_table.data_ptr(), sin_table.data_ptr(), cos_table.shape[0], positions.data_ptr(), q_out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0) * es, k_cache.stride(1) * es, k_cache.shape[1],
        int(offset), _ptr(offset_dev), status_tensor(qkv.device).data_ptr(), _stream(qkv.device)),
        "rt_qk_norm_rope_append")
    _count()
    return q_out


def silu_mul(gate_up: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """``out = silu(gate) * up`` over ``gate_up = [gate | up]`` rows (bf16)."""
    _require_cuda(gate_up, out)
    _rows_bf16(gate_up, "gate_up")
    _rows_bf16(out, "out")
    inter = out.shape[-1]
    rows = out.numel() // inter
    if gate_up.numel() != 2 * rows * inter:
        raise RuntimeError("gate_up must hold [rows, 2 * inter]")
    _lib.check(_lib.load().rt_silu_mul(gate_up.data_ptr(), out.data_ptr(), rows, inter, _stream(out.device)),
               "rt_silu_mul")
    _count()
    return out


# ---------------------------------------------------------------------------
# tcgen05 projections with fused epilogues (rt_linear)
# ---------------------------------------------------------------------------
def linear_supported(m: int, n_out: int, k: int, epilogue: int = 0) -> bool:
    """Whether rt_linear takes this projection shape."""
    return _lib.load().rt_linear_check(m, n_out, k, epilogue) == _lib.RT_OK


def linear_plan(m: int, n_out: int, k: int, epilogue: int = 0) -> dict:
    """The launch rt_linear makes for a shape on the current device (K splits, ring stages, smem)."""
    vals = [ctypes.c_int(0) for _ in range(3)]
    _lib.check(_lib.load().rt_linear_plan(m, n_out, k, epilogue, *[ctypes.addressof(v) for v in vals]),
               "rt_linear_plan")
    return dict(splits=vals[0].value, stages=vals[1].value, smem=vals[2].value)


def linear(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None, epilogue: int = 0,
           qkv: dict | None = None) -> torch.Tensor | None:
    """``x [m, k] @ w[n_out, k]^T`` on tcgen05 with an optional fused epilogue (bf16).

    epilogue 0: ``out [m, n_out]``; 1 (w = [gate; up]): ``out [m, n_out/2] =
    silu(gate) * up``; 2 (w = [Wq; Wk; Wv]): head norms + rotary, q to
    ``qkv['q_out']``, k/v into the cache (keys of ``qkv`` as in
    ``qk_norm_rope_append``: num_q_heads, num_kv_heads, q_norm, k_norm, eps,
    cos, sin, positions, q_out, k_cache, v_cache, offset, offset_dev).
    """
    lib = _lib.load()
    _require_cuda(x, w, out)
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(-1) != 1:
        raise RuntimeError("linear takes bf16 x [m, k] with unit inner stride and bf16 w [n_out, k]")
    if not w.is_contiguous():
        raise RuntimeError("linear weights must be contiguous")
    m, k = x.shape
    n_out = w.shape[0]
    if w.shape[1] != k:
        raise RuntimeError("weight / input inner dimensions differ")
    dev = x.device
    if lib.rt_linear_check(m, n_out, k, epilogue) != _lib.RT_OK:
        raise RuntimeError(f"rt_linear does not take m={m}, n_out={n_out}, k={k}")
    epi = None
    keep = []
    if epilogue == _lib.RT_EPI_QKV_ROPE:
        kc, vc = qkv["k_cache"], qkv["v_cache"]
        es = kc.element_size()
        epi = _lib.QkvEpilogue(qkv["num_q_heads"], qkv["num_kv_heads"], _ptr(qkv.get("q_norm")),
                               _ptr(qkv.get("k_norm")), float(qkv["eps"]), qkv["cos"].data_ptr(),
                               qkv["sin"].data_ptr(), qkv["cos"].shape[0], qkv["positions"].data_ptr(),
                               qkv["q_out"].data_ptr(), kc.data_ptr(), vc.data_ptr(), kc.stride(0) * es,
                               kc.stride(1) * es, kc.shape[1], int(qkv.get("offset", 0)),
                               _ptr(qkv.get("offset_dev")))
        keep.append(epi)
        out_ptr, ld = None, 0
    else:
        if out is None:
            width = n_out // 2 if epilogue == _lib.RT_EPI_SILU_MUL else n_out
            out = torch.empty((m, width), dtype=torch.bfloat16, device=dev)
        if out.dtype != torch.bfloat16 or out.stride(-1) != 1:
            raise RuntimeError("linear output must be bf16 with unit inner stride")
        out_ptr, ld = out.data_ptr(), out.stride(0)
    rc = lib.rt_linear(x.data_ptr(), x.stride(0), m, k, w.data_ptr(), n_out, int(epilogue), out_ptr, ld,
                       ctypes.addressof(epi) if epi is not None else None, status_tensor(dev).data_ptr(),
                       _stream(dev))
    _lib.check(rc, "rt_linear")
    _count()
    return out


# ---------------------------------------------------------------------------
# Target-gated sibling-recovery walk (rt_recovery_walk)
# ---------------------------------------------------------------------------
def linear_argmax(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
    """``out [m, n_out] = x @ w^T`` (rt_linear) and ``index [m]`` = each row's argmax (first largest; NaN
    largest) from the same launch (rt_linear_argmax): the temperature-0 posterior without a pass over
    the logits."""
    _require_cuda(x, w, out, index)
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(-1) != 1:
        raise RuntimeError("linear_argmax takes bf16 x [m, k] with unit inner stride")
    if not w.is_contiguous() or out.dtype != torch.bfloat16 or out.stride(-1) != 1:
        raise RuntimeError("linear_argmax: contiguous bf16 weights, bf16 out with unit inner stride")
    if index.dtype != torch.int64 or not index.is_contiguous() or index.numel() < x.shape[0]:
        raise RuntimeError("index must be contiguous int64 [m]")
    m, k = x.shape
    n_out = w.shape[0]
    keys = _STATE.buffer(x.device, "argmax_keys", max(8 * m, 256))
    _lib.check(_lib.load().rt_linear_argmax(x.data_ptr(), x.stride(0), m, k, w.data_ptr(), n_out, out.data_ptr(),
                                            out.stride(0), keys.data_ptr(), index.data_ptr(),
                                            status_tensor(x.device).data_ptr(), _stream(x.device)),
               "rt_linear_argmax")
    _count(2)  # the projection and the index conversion (the key reset is a memset)
    return index


def recovery_walk(parents: torch.Tensor, tokens: torch.Tensor, posterior: torch.Tensor, logits: torch.Tensor,
                  table: tuple, params: dict, count: int | None = None, count_dev: torch.Tensor | None = None,
                  stop_ids: torch.Tensor | None = None, log: tuple | None = None, out: dict | None = None,
                  verify_ids: torch.Tensor | None = None, output_ids: torch.Tensor | None = None,
                  start_dev: torch.Tensor | None = None) -> dict:
    """ReTree's recovery walk on the device.

    ``table`` = (keys int64[cap], prior int32[cap], online int32[cap]) of
    ``recovery_device.RecoveryTable``; ``params`` = gate_threshold,
    freq_threshold, rescue_top_k, record_top_k, online_update; ``log`` =
    (pairs int32[cap, 2], count int32[1]) or None; ``stop_ids`` int64 or None
    (no stop set).  Returns ``out`` with accepted / accepted_len / next_token /
    rescued.
    """
    _require_cuda(parents, tokens, posterior, logits, stop_ids, verify_ids, output_ids, start_dev, *table)
    dev = parents.device
    n_max = parents.numel()
    cnt = n_max - 1 if count is None else int(count)
    if logits.dtype not in (torch.float32, torch.bfloat16) or logits.dim() != 2 or logits.stride(-1) != 1:
        raise RuntimeError("logits must be [nodes, vocab] fp32 or bf16 with contiguous rows")
    if out is None:
        out = dict(accepted=torch.zeros(n_max, dtype=torch.int64, device=dev),
                   accepted_len=torch.zeros(1, dtype=torch.int32, device=dev),
                   next_token=torch.zeros(1, dtype=torch.int64, device=dev),
                   rescued=torch.zeros(1, dtype=torch.int32, device=dev))
    keys, prior, online = table
    log_pairs, log_count = (None, None) if log is None else log
    rc = _lib.load().rt_recovery_walk(
        parents.data_ptr(), _ptr(tokens), cnt, _ptr(count_dev), posterior.data_ptr(), logits.data_ptr(),
        logits.stride(0), 0 if logits.dtype == torch.float32 else 1, logits.shape[1],
        float(params.get("gate_threshold", 0.01)), int(params.get("freq_threshold", 6)),
        int(params.get("rescue_top_k", 8)), int(params.get("record_top_k", 8)),
        int(bool(params.get("online_update", True))), _ptr(stop_ids),
        0 if stop_ids is None else stop_ids.numel(), keys.data_ptr(), prior.data_ptr(), online.data_ptr(),
        keys.numel(), _ptr(log_pairs), _ptr(log_count), 0 if log_pairs is None else log_pairs.shape[0],
        out["accepted"].data_ptr(), out["accepted_len"].data_ptr(), out["next_token"].data_ptr(),
        out["rescued"].data_ptr(), _ptr(verify_ids), _ptr(output_ids),
        0 if output_ids is None else output_ids.numel(), _ptr(start_dev), status_tensor(dev).data_ptr(),
        _stream(dev))
    _lib.check(rc, "rt_recovery_walk")
    _count()
    return out


# ---------------------------------------------------------------------------
# Attention over whole prompts, 4-bit KV cache
#
# A call of these takes a few microseconds on the GPU, so the wrappers test one
# condition on the common layout and look for the reason only when it fails.
# ---------------------------------------------------------------------------
Q4_ROW_BYTES = _lib.RT_Q4_ROW_BYTES


_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch.cuda.current_device
_grad_enabled = torch.is_grad_enabled
_forward_ad = torch.autograd.forward_ad
_BF16, _F16, _U8 = torch.bfloat16, torch.float16, torch.uint8
_STATUS_PTR: dict = {}  # device index -> address of its status word (kept for the process's life)
_SCALE = 128 ** -0.5


def _status_ptr(index: int) -> int:
    ptr = _STATUS_PTR.get(index)
    if ptr is None:
        ptr = _STATUS_PTR[index] = _STATE.status(torch.device("cuda", index)).data_ptr()
    return ptr


@functools.lru_cache(maxsize=1024)
def _prompt_workspace(index, *shape) -> int:
    return _lib.load().rt_prompt_attn_workspace_size(*shape)


@functools.lru_cache(maxsize=1024)
def _tree_q4_workspace(index, *shape) -> int:
    return _lib.load().rt_tree_attn_q4_workspace_size(*shape)


def _refuse(what: str, *conditions) -> None:
    """Raise for the first of ``(ok, reason)`` that does not hold."""
    for ok, reason in conditions:
        if not ok:
            raise RuntimeError(f"{what}: {reason}")
    raise RuntimeError(f"{what}: tensors must be on one device")


def _tangents(*tensors) -> bool:
    """Whether one carries a forward-mode tangent (there are none outside a dual level)."""
    return _forward_ad._current_level >= 0 and any(_forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _needs_grad(*tensors) -> bool:
    return (_grad_enabled() and any(t.requires_grad for t in tensors)) or _tangents(*tensors)


def _workspace(nbytes: int, dev) -> torch.Tensor:
    """Scratch of one call, from the caching allocator: ordered by the call's stream, the graph's own in a capture."""
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def _offsets(t) -> bool:
    return t.dtype is torch.int32 and t.dim() == 1 and t.numel() >= 2 and t.is_contiguous()


def _one_batch(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dim() == 4 and t.shape[0] == 1:
        return t[0]
    if t.dim() != 3:
        raise RuntimeError(f"{what}: expected three dimensions, or four with a batch of 1 (pack sequences along the "
                           "token axis)")
    return t


def _query(q: torch.Tensor, what: str) -> torch.Tensor:
    """``[n, Hq, 128]`` view of a query in that layout or HF's ``[1, Hq, n, 128]``."""
    return q if q.dim() == 3 else _one_batch(q, what).transpose(0, 1)


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """``t`` and the byte strides of its two leading axes (any aligned number for an axis of one).

    A tensor that repeats a row (a zero stride, which a tensor map does not describe) is copied.
    """
    a, b, _ = t.stride()
    if a > 0 and b > 0 and t.shape[0] > 1 and t.shape[1] > 1:
        return t, 2 * a, 2 * b
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        t = t.contiguous()
        a, b, _ = t.stride()
    return t, 2 * a if t.shape[0] > 1 else 256, 2 * b if t.shape[1] > 1 else 256


def _attn_out(out: torch.Tensor | None, q: torch.Tensor, what: str) -> torch.Tensor:
    if out is None:
        return q.new_empty(tuple(q.shape))
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(-1) != 1 or \
            any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise RuntimeError(f"{what}: out must be {q.dtype} {list(q.shape)} on {q.device} with contiguous head_dim and "
                           "rows of its own")
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor | None = None,
                     cu_seqlens_k: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention over whole prompts, several sequences packed along the token axis.

    q: ``[T, Hq, 128]`` or HF's ``[1, Hq, T, 128]``; k, v: ``[Hkv, Tk, 128]`` or
    ``[1, Hkv, Tk, 128]``, any token and head strides of 16 bytes (copied
    where K and V differ in them); bf16 or fp16.  ``cu_seqlens_q`` / ``cu_seqlens_k``: int32 CUDA offsets of the
    sequences' queries and keys (``cu_seqlens_k=None``: the same offsets; both
    None: one sequence).  A sequence's queries are its last tokens: with lq
    queries and lk keys, query i sees keys ``j <= i + lk - lq``, so a chunk of a
    prompt attends to the keys of the chunks before it.  Queries that see no
    key give zero rows; rows outside every sequence are not written.
    Returns ``out`` ``[T, Hq, 128]``.
    """
    what = "prompt_attention"
    if q.dim() != 3:
        q = _query(q, what)
    if k.dim() != 3 or v.dim() != 3:
        k, v = _one_batch(k, what), _one_batch(v, what)
    index = q.get_device()
    t, hq, d = q.shape
    hkv, tk, dk = k_shape = k.shape
    dt = q.dtype
    cq, ck = cu_seqlens_q, cu_seqlens_k
    q0, q1, q2 = q.stride()
    k0, k1, k2 = ks = k.stride()
    vs = v.stride()
    if not (q.is_cuda and k.is_cuda and k.get_device() == index and v.is_cuda and v.get_device() == index
            and (dt is _BF16 or dt is _F16) and k.dtype is dt and v.dtype is dt and d == 128 and dk == 128
            and q2 == 1 and k2 == 1 and vs[2] == 1 and k_shape == v.shape and hq and hkv and hq % hkv == 0
            and (ck is None or (cq is not None and _offsets(ck) and ck.get_device() == index
                                and ck.numel() == cq.numel()))
            and (cq is None or (_offsets(cq) and cq.get_device() == index))
            and not (_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad))
            and not (_forward_ad._current_level >= 0 and _tangents(q, k, v))):
        _refuse(what,
                (q.is_cuda and k.is_cuda and v.is_cuda, "takes CUDA tensors (no CPU path)"),
                (not _needs_grad(q, k, v), "inference-only (no gradient)"),
                (dt in (torch.bfloat16, torch.float16) and k.dtype == dt and v.dtype == dt,
                 "runs on bf16 or fp16 q/k/v of one type"),
                (d == 128 and dk == 128 and q.stride(2) == 1 and k.stride(2) == 1 and v.stride(2) == 1,
                 "head_dim must be 128 and contiguous"),
                (k.shape == v.shape, "K and V must share their shape"),
                (hq and hkv and hq % hkv == 0, "key heads must divide query heads"),
                (cq is not None or ck is None, "cu_seqlens_k needs cu_seqlens_q"),
                (all(x is None or _offsets(x) for x in (cq, ck)),
                 "cu_seqlens must be contiguous int32 tensors of at least two offsets"),
                (ck is None or cq is None or ck.numel() == cq.numel(), "cu_seqlens must name the same number of sequences"))
    if _current_device() != index:
        with torch.cuda.device(index):
            return prompt_attention(q, k, v, cq, ck, scale, out)
    if ks == vs and t > 1 and hq > 1 and tk > 1 and hkv > 1 and q0 and q1 and k0 and k1:
        q0, q1, k0, k1 = 2 * q0, 2 * q1, 2 * k0, 2 * k1
    else:
        q, q0, q1 = _rows(q)
        k, k0, k1 = _rows(k)
        v, v0, v1 = _rows(v)
        if (k0, k1) != (v0, v1):  # (one set of strides for both)
            k, v, k0, k1 = k.contiguous(), v.contiguous(), max(tk, 1) * 256, 256
    if out is None:
        out = q.new_empty((t, hq, 128))
        o0, o1 = hq * 256, 256
    else:
        _, o0, o1 = _rows(_attn_out(out, q, what))
    if t == 0:
        return out
    seqs = 1 if cq is None else cq.numel() - 1
    nbytes = _prompt_workspace(index, t, tk, seqs, hq, hkv)
    ws = _workspace(nbytes, q.device) if nbytes else None
    rc = _lib.load().rt_prompt_attn(q.data_ptr(), q0, q1, k.data_ptr(), v.data_ptr(), k0, k1, out.data_ptr(), o0, o1,
                                    1 if dt is _BF16 else 2, None if cq is None else cq.data_ptr(),
                                    None if ck is None else ck.data_ptr(), seqs, t, tk, hq, hkv, 128,
                                    _SCALE if scale is None else float(scale),
                                    None if ws is None else ws.data_ptr(), nbytes, _status_ptr(index),
                                    _raw_stream(index))
    if rc:
        _lib.check(rc, "rt_prompt_attn")
    _count(2 if nbytes else 1)
    return out


def _q4_rows(t: torch.Tensor) -> bool:
    """Whether ``t`` is a 4-bit cache ``[heads, capacity, 72]`` with contiguous rows."""
    return t.is_cuda and t.dtype is torch.uint8 and t.dim() == 3 and t.shape[2] == 72 and t.stride()[1:] == (72, 1)


def kv_append_q4(k_cache: torch.Tensor, v_cache: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                 offset: int = 0, offset_dev: torch.Tensor | None = None) -> None:
    """Quantise ``[heads, n, 128]`` bf16 rows into rows ``offset..`` of 4-bit caches ``[heads, cap, 72]`` (uint8).

    ``offset_dev`` (int64[1] on the device) supplies the offset at run time;
    rows that do not fit are then left out and reported by the device status.
    Any finite bf16 value can be held and read; ``tree_attention_q4`` needs values below 2^119.
    """
    what = "kv_append_q4"
    if k_new.dim() != 3 or v_new.dim() != 3:
        k_new, v_new = _one_batch(k_new, what), _one_batch(v_new, what)
    index = k_cache.get_device()
    heads, n, d = new_shape = k_new.shape
    c_shape, c_stride = k_cache.shape, k_cache.stride()
    cache_heads, cap, row = c_shape if len(c_shape) == 3 else (-1, 0, 0)
    s0, s1, s2 = ss = k_new.stride()
    sv = v_new.stride()
    if not (k_cache.is_cuda and k_cache.dtype is _U8 and v_cache.dtype is _U8 and row == 72
            and c_stride[1:] == (72, 1) and c_shape == v_cache.shape and c_stride == v_cache.stride()
            and k_new.dtype is _BF16 and v_new.dtype is _BF16
            and new_shape == v_new.shape and heads == cache_heads and d == 128 and s2 == 1 and sv[2] == 1
            and v_cache.is_cuda and v_cache.get_device() == index and k_new.is_cuda and k_new.get_device() == index
            and v_new.is_cuda and v_new.get_device() == index
            and (offset_dev is None or (offset_dev.dtype is torch.int64 and offset_dev.numel() and offset_dev.is_cuda
                                        and offset_dev.get_device() == index))
            and not (_grad_enabled() and (k_new.requires_grad or v_new.requires_grad))
            and not (_forward_ad._current_level >= 0 and _tangents(k_new, v_new))):
        _refuse(what,
                (all(x.is_cuda for x in (k_cache, v_cache, k_new, v_new)), "takes CUDA tensors (no CPU path)"),
                (not _needs_grad(k_new, v_new), "inference-only (no gradient)"),
                (_q4_rows(k_cache) and _q4_rows(v_cache),
                 f"caches must be uint8 [heads, capacity, {Q4_ROW_BYTES}] with contiguous rows"),
                (k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride(),
                 "K and V caches must share shape and strides"),
                (k_new.dtype == _BF16 and v_new.dtype == _BF16, "takes bf16 rows"),
                (k_new.shape == v_new.shape and heads == cache_heads and d == 128 and s2 == 1 and sv[2] == 1,
                 "new rows must be [cache heads, n, 128] with contiguous head_dim, the same for K and V"),
                (offset_dev is None or (offset_dev.dtype == torch.int64 and offset_dev.numel() > 0),
                 "offset_dev must be int64[1]"))
    if _current_device() != index:
        with torch.cuda.device(index):
            return kv_append_q4(k_cache, v_cache, k_new, v_new, offset, offset_dev)
    if ss == sv and heads > 1 and n > 1 and s0 and s1:
        s0, s1 = 2 * s0, 2 * s1
    else:
        k_new, s0, s1 = _rows(k_new)
        v_new, *sv = _rows(v_new)
        if sv != [s0, s1]:
            k_new, v_new, s0, s1 = k_new.contiguous(), v_new.contiguous(), n * 256, 256
    rc = _lib.load().rt_kv_append_q4(k_cache.data_ptr(), v_cache.data_ptr(),
                                     c_stride[0] if heads > 1 else cap * Q4_ROW_BYTES, k_new.data_ptr(),
                                     v_new.data_ptr(), s0, s1, heads, n, d, cap, int(offset),
                                     None if offset_dev is None else offset_dev.data_ptr(),
                                     _status_ptr(index), _raw_stream(index))
    if rc:
        _lib.check(rc, "rt_kv_append_q4")
    _count()


def kv_read_q4(cache: torch.Tensor, start: int, n: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 values ``[..., n, 128]`` of rows ``[start, start + n)`` of a 4-bit cache ``[..., cap, 72]``."""
    what = "kv_read_q4"
    if not cache.is_cuda:
        raise RuntimeError(f"{what}: takes CUDA tensors (no CPU path)")
    size, stride = cache.shape, cache.stride()
    *lead, cap, row = size if len(size) > 1 else (0, 0)
    fold = row == 72 and stride[-2:] == (72, 1) and cache.dtype is _U8
    # the leading axes as one: heads `step` bytes apart
    if len(lead) == 2 and lead[0] > 1 and lead[1] > 1:
        heads, step = lead[0] * lead[1], stride[1]
        fold = fold and stride[0] == lead[1] * step
    else:
        heads, step = 1, cap * 72
        for axis in range(len(lead) - 1, -1, -1):
            if size[axis] > 1:
                if heads == 1:
                    step = stride[axis]
                fold = fold and stride[axis] == heads * step
            heads *= size[axis]
    if not fold:
        raise RuntimeError(f"{what}: the cache must be uint8 [..., capacity, {Q4_ROW_BYTES}] with contiguous rows and "
                           "leading dimensions of one stride")
    start, n = int(start), int(n)
    if start < 0 or n < 0 or start + n > cap:
        raise RuntimeError(f"{what}: rows [{start}, {start + n}) are outside the cache's {cap}")
    shape = (*lead, n, 128)
    if out is None:
        out = cache.new_empty(shape, dtype=_BF16)
    elif out.shape != shape or out.dtype is not torch.bfloat16 or not out.is_contiguous() or out.device != cache.device:
        raise RuntimeError(f"{what}: out must be contiguous bf16 {list(shape)} on {cache.device}")
    if heads == 0 or n == 0:
        return out
    index = cache.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return kv_read_q4(cache, start, n, out)
    rc = _lib.load().rt_kv_read_q4(cache.data_ptr(), step, out.data_ptr(), n * 256, 256, heads, n, 128, cap, start,
                                   _raw_stream(index))
    if rc:
        _lib.check(rc, "rt_kv_read_q4")
    _count()
    return out


def tree_attention_q4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask_bits: torch.Tensor, prefix_len: int,
                      scale: float | None = None, out: torch.Tensor | None = None, num_splits: int = 0,
                      prefix_len_dev: torch.Tensor | None = None) -> torch.Tensor:
    """``tree_attention`` over a 4-bit cache.

    q: bf16 ``[n, Hq, 128]`` or HF's ``[1, Hq, n, 128]``; k, v: uint8 caches
    ``[Hkv, capacity, 72]`` (an even capacity; values below 2^119, whose scales times 192 stay
    finite) of which rows ``[0, prefix_len + n)`` are used;
    mask_bits: int32 ``[n, W]`` ancestor bits of the tree block (one bit, set,
    for a single token).  ``prefix_len_dev`` (int64[1]) supplies the prefix
    length at run time; ``prefix_len`` is then its upper bound.  Returns ``out``
    ``[n, Hq, 128]`` bf16.
    """
    what = "tree_attention_q4"
    if q.dim() != 3:
        q = _query(q, what)
    index = q.get_device()
    n, hq, d = q.shape
    q0, q1, q2 = q.stride()
    k_shape, k_stride, m_shape = k.shape, k.stride(), mask_bits.shape
    hkv, cap, row = k_shape if len(k_shape) == 3 else (0, 0, 0)
    if not (q.is_cuda and q.dtype is _BF16 and d == 128 and q2 == 1 and k.dtype is _U8 and v.dtype is _U8
            and row == 72 and not cap & 1 and k_stride[1:] == (72, 1) and k_shape == v.shape and k_stride == v.stride()
            and k.is_cuda and k.get_device() == index and v.is_cuda and v.get_device() == index
            and mask_bits.is_cuda and mask_bits.get_device() == index and n and hq and hkv and hq % hkv == 0
            and mask_bits.dtype is torch.int32 and len(m_shape) == 2 and m_shape[0] >= n and m_shape[1] * 32 >= n
            and not (_grad_enabled() and q.requires_grad)
            and not (_forward_ad._current_level >= 0 and _tangents(q))
            and (prefix_len_dev is None or (prefix_len_dev.dtype is torch.int64 and prefix_len_dev.numel()
                                        and prefix_len_dev.is_cuda
                                        and prefix_len_dev.get_device() == index))):
        _refuse(what,
                (q.is_cuda and k.is_cuda and v.is_cuda and mask_bits.is_cuda, "takes CUDA tensors (no CPU path)"),
                (not _needs_grad(q), "inference-only (no gradient)"),
                (q.dtype == torch.bfloat16, "runs on bf16 queries"),
                (d == 128 and q.stride(2) == 1, "head_dim must be 128 and contiguous"),
                (_q4_rows(k) and _q4_rows(v),
                 f"caches must be uint8 [heads, capacity, {Q4_ROW_BYTES}] with contiguous rows"),
                (not cap & 1, "the caches' capacity must be even"),
                (k.shape == v.shape and k.stride() == v.stride(), "K and V caches must share shape and strides"),
                (n and hq and hkv and hq % hkv == 0,
                 "at least one node, and key heads that divide the query heads"),
                (mask_bits.dtype == torch.int32 and mask_bits.dim() == 2 and mask_bits.shape[0] >= n
                 and mask_bits.shape[1] * 32 >= n, "mask_bits must be int32 [n, at least ceil(n / 32)]"),
                (prefix_len_dev is None or (prefix_len_dev.dtype == torch.int64 and prefix_len_dev.numel() > 0),
                 "prefix_len_dev must be int64[1]"))
    if _current_device() != index:
        with torch.cuda.device(index):
            return tree_attention_q4(q, k, v, mask_bits, prefix_len, scale, out, num_splits, prefix_len_dev)
    words, unit = mask_bits.stride()
    if unit != 1 or words < m_shape[1]:
        mask_bits = mask_bits.contiguous()
        words = m_shape[1]
    if (q0 or n == 1) and (q1 or hq == 1):
        q0, q1 = 2 * q0 if n > 1 else 256, 2 * q1 if hq > 1 else 256
    else:
        q, q0, q1 = _rows(q)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((n, hq, 128))
        o0, o1 = hq * 256, 256
    else:
        _, o0, o1 = _rows(_attn_out(out, q, what))
    prefix_len, num_splits = int(prefix_len), int(num_splits)
    nbytes = _tree_q4_workspace(index, n, hq, hkv, 128, prefix_len, num_splits)
    ws = _workspace(nbytes, q.device) if nbytes else None
    rc = _lib.load().rt_tree_attn_q4(q.data_ptr(), q0, q1, k.data_ptr(), v.data_ptr(),
                                     k_stride[0] if hkv > 1 else cap * 72, cap, out.data_ptr(), o0, o1,
                                     mask_bits.data_ptr(), words, n, prefix_len,
                                     None if prefix_len_dev is None else prefix_len_dev.data_ptr(), hq, hkv, 128,
                                     _SCALE if scale is None else float(scale), num_splits,
                                     None if ws is None else ws.data_ptr(), nbytes, _status_ptr(index),
                                     _raw_stream(index))
    if rc:
        _lib.check(rc, "rt_tree_attn_q4")
    _count(2 if nbytes else 1)
    return out


def default_splits_q4(n: int, num_q_heads: int, num_kv_heads: int, prefix_len: int) -> int:
    """Key splits ``tree_attention_q4`` picks for this shape."""
    return int(_lib.load().rt_tree_attn_q4_default_splits(n, num_q_heads, num_kv_heads, int(prefix_len)))


__all__ += ["prompt_attention", "kv_append_q4", "kv_read_q4", "tree_attention_q4", "default_splits_q4",
            "Q4_ROW_BYTES"]
