"""The 4-bit row format's definition, and the refusals of the new entry points (CPU only)."""

import ctypes

import pytest
import torch

from oracle import q4
from retree_b200 import _lib, kernels


def _rows(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((*shape, 128), generator=g) * torch.exp(torch.randn((*shape[:-1], 1, 128), generator=g))
    return x.to(torch.bfloat16)


def test_bytes_hold_the_values():
    x = _rows(1, 3, 50)
    x[0, 0] = 0
    x[0, 1] = 1e-39
    x[0, 2, :40] = 0.375          # a flat group, and one that is half flat
    x[0, 3] = 3e38
    x[0, 3, ::2] = -3e38
    rows = q4.pack(x)
    assert rows.shape == (3, 50, q4.ROW_BYTES) and q4.ROW_BYTES == kernels.Q4_ROW_BYTES
    assert torch.equal(q4.unpack(rows), q4.values(x))


def test_values_are_bf16_and_within_half_a_step():
    x = _rows(2, 4, 64)
    val = q4.values(x)
    assert torch.equal(val, val.to(torch.bfloat16).double())
    u, z, s = q4.quantise(x)
    # a code is off its value by half a step; rounding the zero point up or down may cut the range's end by another half
    assert bool(((val - x.double()).abs().unflatten(-1, (4, 32)) <= s).all())
    lo = torch.minimum(x.double().unflatten(-1, (4, 32)).amin(-1, keepdim=True), torch.zeros(()).double())
    hi = torch.maximum(x.double().unflatten(-1, (4, 32)).amax(-1, keepdim=True), torch.zeros(()).double())
    assert bool((s * 15 >= hi - lo).all()) and bool((s * 15 <= (hi - lo) * 1.125).all())


def test_rows_that_are_not_finite_read_as_nan():
    x = _rows(3, 1, 4)
    x[0, 0, 5] = float("nan")
    x[0, 1, 100] = float("-inf")
    val = q4.unpack(q4.pack(x))
    assert bool(val[0, :2].isnan().all()) and bool(val[0, 2:].isfinite().all())


P = 1 << 20  # a pointer that the checks pass over


def test_prompt_attention_host_checks():
    lib = _lib.load()

    def call(q=P, qt=8192, qh=256, k=P, v=P, kh=1 << 16, kr=256, out=P, dtype=1, cu_q=None, cu_k=None, seqs=1, t=4,
             tk=4, hq=32, hkv=8, d=128):
        return lib.rt_prompt_attn(q, qt, qh, k, v, kh, kr, out, 8192, 256, dtype, cu_q, cu_k, seqs, t, tk, hq, hkv, d,
                                  ctypes.c_float(1.0), None, 0, None, None)

    bad, unsup = _lib.RT_ERR_INVALID_ARGUMENT, _lib.RT_ERR_UNSUPPORTED
    assert call(q=None) == bad and call(out=None) == bad and call(k=None) == bad
    assert call(q=P + 8) == bad and call(kr=264) == bad
    assert call(hq=30) == bad and call(hkv=0) == bad and call(t=-1) == bad
    assert call(seqs=2) == bad and call(cu_k=P) == bad
    assert call(dtype=0) == unsup and call(d=64) == unsup
    assert call(hq=129, hkv=1) == unsup and call(t=1 << 31) == unsup
    assert call(t=0) == _lib.RT_OK


def test_q4_host_checks():
    lib = _lib.load()
    bad, unsup, ok = _lib.RT_ERR_INVALID_ARGUMENT, _lib.RT_ERR_UNSUPPORTED, _lib.RT_OK

    def append(k=P, kn=P, hs=72 * 64, nr=256, heads=8, n=4, d=128, cap=64, off=0):
        return lib.rt_kv_append_q4(k, P, hs, kn, P, 1 << 12, nr, heads, n, d, cap, off, None, None, None)

    assert append(k=None) == bad and append(kn=P + 2) == bad and append(k=P + 4) == bad and append(nr=264) == bad
    assert append(off=61) == bad and append(off=-1) == bad and append(n=-1) == bad
    assert append(d=64) == unsup and append(n=0) == ok

    def read(c=P, out=P, n=4, start=0, cap=64, d=128):
        return lib.rt_kv_read_q4(c, 72 * 64, out, 1 << 10, 256, 8, n, d, cap, start, None)

    assert read(c=None) == bad and read(out=P + 8) == bad and read(start=61) == bad and read(start=-1) == bad
    assert read(d=64) == unsup and read(n=0) == ok

    def attn(q=P, k=P, hs=72 * 64, cap=64, mask=P, words=1, n=4, prefix=8, hq=32, hkv=8, d=128, out=P):
        return lib.rt_tree_attn_q4(q, 8192, 256, k, P, hs, cap, out, 8192, 256, mask, words, n, prefix, None, hq, hkv,
                                   d, ctypes.c_float(1.0), 0, None, 0, None, None)

    assert attn(q=None) == bad and attn(mask=None) == bad and attn(out=None) == bad
    assert attn(q=P + 8) == bad and attn(k=P + 8) == bad and attn(hs=72 * 63) == bad
    assert attn(n=0) == bad and attn(prefix=-1) == bad and attn(prefix=61) == bad and attn(hq=30) == bad
    assert attn(n=40, words=1) == bad and attn(cap=63) == bad
    assert attn(d=64) == unsup


def test_lengths_whose_sum_passes_64_bits_are_refused():
    lib = _lib.load()
    bad, far = _lib.RT_ERR_INVALID_ARGUMENT, 2 ** 63 - 1
    assert lib.rt_kv_append_q4(P, P, 72 * 64, P, P, 1 << 12, 256, 8, 4, 128, 64, far, None, None, None) == bad
    assert lib.rt_kv_read_q4(P, 72 * 64, P, 1 << 10, 256, 8, 4, 128, 64, far, None) == bad
    for n in (1, 40):
        assert lib.rt_tree_attn_q4(P, 8192, 256, P, P, 72 * 64, 64, P, 8192, 256, P, 2, n, far, None, 32, 8, 128,
                                   ctypes.c_float(1.0), 0, None, 0, None, None) == bad


def test_wrappers_refuse_cpu_tensors():
    q, kv = torch.zeros(2, 8, 128, dtype=torch.bfloat16), torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    c = torch.zeros(2, 4, 72, dtype=torch.uint8)
    for call in (lambda: kernels.prompt_attention(q, kv, kv), lambda: kernels.kv_append_q4(c, c, kv, kv),
                 lambda: kernels.kv_read_q4(c, 0, 2),
                 lambda: kernels.tree_attention_q4(q, c, c, torch.ones(2, 1, dtype=torch.int32), 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_a_scale_covers_its_range_to_the_last_bit():
    """15 s >= hi - lo in exact arithmetic, for a small end of any size, and the scale below does not."""
    from fractions import Fraction
    for m in range(8, 16):
        for k in (7, 20, 24, 25, 30, 53, 60, 120):
            x = torch.zeros((2, 128), dtype=torch.bfloat16)
            x[0, ::32], x[0, 1::32] = 15 * m / 8, -15 * 2.0 ** -k
            x[1] = -x[0]
            span = Fraction(float(x[0, 0])) - Fraction(float(x[0, 1]))
            for got in q4.quantise(x)[2][:, 0, 0].tolist():
                s = Fraction(got)
                assert 15 * s >= span, (m, k)
                step = Fraction(1, 4) if s > 2 else Fraction(1, 8)
                assert 15 * (s - step if s > 1 else Fraction(15, 16)) < span, (m, k)


def test_tangents_count_as_gradients():
    from torch.autograd import forward_ad
    x = torch.zeros(3)
    assert not kernels._needs_grad(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert kernels._needs_grad(x, dual) and not kernels._needs_grad(x)
        with torch.no_grad():  # (stops gradients of the backward pass only)
            assert kernels._needs_grad(dual)


def test_a_cache_too_small_for_the_tree_is_refused_with_a_device_length_too():
    lib = _lib.load()
    for cap, n in ((0, 1), (0, 40), (4, 6)):
        assert lib.rt_tree_attn_q4(P, 8192, 256, P, P, 72 * 64, cap, P, 8192, 256, P, 2, n, 0, P, 32, 8, 128,
                                   ctypes.c_float(1.0), 0, P, 1 << 30, None, None) == _lib.RT_ERR_INVALID_ARGUMENT
