"""GPU parity of the packed causal prompt attention against its definition in 64 bits.

Tolerance, per element, with eps = half a step of the type (bf16 2^-8, fp16
2^-11) and A = sum_j softmax_j |v_j|: the weights are rounded to the type once
(eps * A), the result once (eps * |o|), and a score's fp32 sum of 128 products
is off by at most delta = 128 * 2^-23 * scale * max_j sum_d |q_d k_jd|, which
moves a weight by a factor exp(+-2 delta) at most (3 * delta * A with room for
the fp32 exponential, whose own error is below 2^-21).
"""

import pytest
import torch

from retree_b200 import kernels
from tests.gpu_util import cuda

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(q, k, v, lens_q, lens_k, scale=128 ** -0.5):
    """float64 ``(out, bound)`` ``[T, Hq, 128]``; hidden rows of k and v are never touched."""
    t, hq, d = q.shape
    grp = hq // k.shape[0]
    eps = EPS[q.dtype]
    out = torch.zeros((t, hq, d), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    a = b = 0
    for lq, lk in zip(lens_q, lens_k):
        for h in range(hq):
            kk, vv = k[h // grp, b:b + lk].double(), v[h // grp, b:b + lk].double()
            qq = q[a:a + lq, h].double()
            see = torch.arange(lk, device=q.device) <= torch.arange(lq, device=q.device)[:, None] + (lk - lq)
            s = torch.where(see, qq @ kk.T * scale, float("-inf"))
            top = s.amax(1, keepdim=True) if lk else torch.full((lq, 1), float("-inf"), device=q.device).double()
            p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
            z = p.sum(1, keepdim=True)
            p = p / torch.where(z == 0, 1.0, z)
            o = p @ vv
            big = p @ vv.abs()
            delta = 128 * 2.0 ** -23 * scale * ((qq.abs() @ kk.abs().T) * see).amax(1, keepdim=True) if lk else 0.0
            out[a:a + lq, h] = o
            bound[a:a + lq, h] = eps * o.abs() + (eps + 2.0 ** -20 + 3 * delta) * big + 1e-30
        a, b = a + lq, b + lk
    return out, bound


def cu(lens, dev):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.cumsum(torch.tensor(lens), 0)
    return t.to(dev)


def make(seed, t, tk, hq, hkv, dtype, dev, layout="tokens"):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(s, device=dev, generator=g).to(dtype)  # noqa: E731
    if layout == "qkv":
        x = r(t, hq + 2 * hkv, 128)
        return x[:, :hq], x[:, hq:hq + hkv].transpose(0, 1), x[:, hq + hkv:].transpose(0, 1)
    if layout == "heads":
        return r(hq, t, 128).transpose(0, 1), r(hkv, tk, 128), r(hkv, tk, 128)
    return r(t, hq, 128), r(tk, hkv, 128).transpose(0, 1), r(tk, hkv, 128).transpose(0, 1)


def check(out, q, k, v, lens_q, lens_k, scale=128 ** -0.5):
    kernels.check_device_status(q.device)
    ref, bound = reference(q, k, v, lens_q, lens_k, scale)
    err = (out.double() - ref).abs()
    over = ~(err <= bound)
    assert not bool(over.any()), (int(over.sum()), float((err / bound).nan_to_num(nan=1e9).max()),
                                  over.nonzero()[0].tolist())


@pytest.mark.parametrize("t", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 1025])
def test_one_sequence(t):
    dev = cuda()
    q, k, v = make(t, t, t, 8, 2, torch.bfloat16, dev, "qkv")
    check(kernels.prompt_attention(q, k, v), q, k, v, [t], [t])


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (6, 2), (7, 1), (10, 2), (12, 1), (16, 2), (33, 3), (64, 1),
                                    (128, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_groups(hq, hkv, dtype):
    dev = cuda()
    lens = [70, 3, 261]
    q, k, v = make(hq, sum(lens), sum(lens), hq, hkv, dtype, dev, "heads")
    check(kernels.prompt_attention(q, k, v, cu(lens, dev)), q, k, v, lens, lens)


@pytest.mark.parametrize("lens,past", [
    ([1], [0]), ([1], [1000]), ([5, 0, 9], [0, 40, 7]), ([64, 64], [64, 128]), ([33, 200, 1, 1], [511, 0, 127, 128]),
    ([0, 0, 130], [0, 0, 0]), ([300], [2500]), ([17], [9000]), ([1, 1, 1, 1, 1], [3000, 0, 1, 129, 64])])
def test_packed_with_earlier_keys(lens, past):
    dev = cuda()
    both = [a + b for a, b in zip(lens, past)]
    q, k, v = make(len(lens) + sum(past), sum(lens), sum(both), 8, 2, torch.bfloat16, dev)
    out = kernels.prompt_attention(q, k, v, cu(lens, dev), cu(both, dev))
    check(out, q, k, v, lens, both)


def test_queries_without_keys_are_zero_rows():
    dev = cuda()
    lens, keys = [10, 5, 200, 40], [4, 0, 130, 40]
    q, k, v = make(5, sum(lens), sum(keys), 4, 2, torch.bfloat16, dev)
    out = kernels.prompt_attention(q, k, v, cu(lens, dev), cu(keys, dev), out=torch.full_like(q, float("nan")))
    check(out, q, k, v, lens, keys)
    assert bool((out[:6] == 0).all()) and bool((out[10:15] == 0).all()) and bool((out[15:85] == 0).all())


def test_rows_outside_the_sequences_stay_and_are_not_read():
    dev = cuda()
    t, lens = 400, [100, 57]
    q, k, v = make(6, t, t, 8, 2, torch.bfloat16, dev)
    for x in (q, k.transpose(0, 1), v.transpose(0, 1)):
        x[157:] = float("nan")
    off = cu(lens, dev)
    out = torch.full_like(q, 7.0)
    kernels.prompt_attention(q, k, v, off, out=out)
    check(out[:157], q[:157], k[:, :157], v[:, :157], lens, lens)
    assert bool((out[157:] == 7).all())
    # and in front of the first sequence
    off2 = off + 157
    q2, k2, v2 = q.roll(157, 0), k.roll(157, 1), v.roll(157, 1)
    out.fill_(7.0)
    kernels.prompt_attention(q2, k2, v2, off2, out=out)
    check(out[157:314], q2[157:314], k2[:, 157:314], v2[:, 157:314], lens, lens)
    assert bool((out[:157] == 7).all()) and bool((out[314:] == 7).all())


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["k", "v"])
def test_hidden_keys_do_not_reach_a_row(what, where):
    """A row of k or v that is not finite changes the rows that see it and no other."""
    dev = cuda()
    lens = [300, 90, 333]
    q, k, v = make(8, sum(lens), sum(lens), 8, 2, torch.bfloat16, dev)
    clean = kernels.prompt_attention(q, k, v, cu(lens, dev))
    x = k if where == "k" else v
    x[0, 250, 3] = what        # head 0, first sequence: rows 250..299 of query heads 0-3 see it
    x[1, 390, :] = what        # head 1, first row of the last sequence: all of its rows see it
    x[1, 722, 100] = what      # the very last row
    out = kernels.prompt_attention(q, k, v, cu(lens, dev))
    kernels.check_device_status(dev)
    touched = torch.zeros((sum(lens), 8), dtype=torch.bool, device=dev)
    touched[250:300, :4] = True
    touched[390:, 4:] = True
    assert torch.equal(out[~touched], clean[~touched])
    if where == "v":
        # a finite weight times the value: the same infinity (or NaN) in its column, the other columns finite
        col = out[250:300, :4, 3].float()
        assert bool(col.isnan().all()) if what != what else bool((col == what).all())
        rest = out[250:300, :4].float()
        rest[..., 3] = 0
        assert bool(rest.isfinite().all())
        assert not bool(out[390:, 4:].isfinite().any())
    elif what != what:
        assert bool(out[touched].isnan().all())


def test_large_scores_and_scale():
    """Scores far apart: the running maximum moves through the whole row."""
    dev = cuda()
    t = 700
    q, k, v = make(9, t, t, 4, 1, torch.bfloat16, dev)
    k *= torch.linspace(0.1, 12, t, device=dev)[None, :, None].to(k.dtype)
    check(kernels.prompt_attention(q, k, v, scale=0.5), q, k, v, [t], [t], 0.5)
    kr = k.flip(1).contiguous()
    vr = v.flip(1).contiguous()
    check(kernels.prompt_attention(q, kr, vr, scale=0.5), q, kr, vr, [t], [t], 0.5)
    check(kernels.prompt_attention(q, k, v, scale=0.0), q, k, v, [t], [t], 0.0)
    for bad in (-0.3, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="invalid argument"):
            kernels.prompt_attention(q, k, v, scale=bad)


def test_hf_layout_strides_and_out_view():
    dev = cuda()
    t = 150
    q, k, v = make(10, t, t, 8, 4, torch.float16, dev, "heads")
    buf = torch.full((t, 3, 8, 128), 5.0, dtype=torch.float16, device=dev)
    out = kernels.prompt_attention(q.transpose(0, 1)[None], k[None], v[None], out=buf[:, 1])
    check(out, q, k, v, [t], [t])
    assert bool((buf[:, 0] == 5).all()) and bool((buf[:, 2] == 5).all())
    # tokens in reverse (a negative stride is a view torch refuses; a step of two rows is not)
    big = torch.randn((8, 2 * t, 128), device=dev).half()
    k2, v2 = big[:4, ::2], big[4:, ::2]
    check(kernels.prompt_attention(q, k2, v2), q, k2, v2, [t], [t])
    # one key row for every token: stride 0
    k3, v3 = (x[:, :1].expand(-1, t, -1) for x in (k, v))
    check(kernels.prompt_attention(q, k3, v3), q, k3, v3, [t], [t])
    q4 = q[:1].expand(t, -1, -1)
    check(kernels.prompt_attention(q4, k, v), q4, k, v, [t], [t])


def test_many_sequences():
    dev = cuda()
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 40, (777,), generator=g).tolist()
    q, k, v = make(11, sum(lens), sum(lens), 4, 2, torch.bfloat16, dev)
    check(kernels.prompt_attention(q, k, v, cu(lens, dev)), q, k, v, lens, lens)


def test_bad_offsets_are_reported_and_skipped():
    dev = cuda()
    q, k, v = make(12, 200, 200, 4, 2, torch.bfloat16, dev)
    for bad in ([0, 300], [0, 100, 50, 200], [-5, 20, 200]):
        off = torch.tensor(bad, dtype=torch.int32, device=dev)
        kernels.prompt_attention(q, k, v, off)
        with pytest.raises(RuntimeError, match="index"):
            kernels.check_device_status(dev)
    # the good sequences of such a call are right
    out = torch.full_like(q, 3.0)
    off = torch.tensor([0, 60, 400, 400], dtype=torch.int32, device=dev)
    kernels.prompt_attention(q, k, v, off, out=out)
    with pytest.raises(RuntimeError, match="index"):
        kernels.check_device_status(dev)
    check(out[:60], q[:60], k[:, :60], v[:, :60], [60], [60])
    assert bool((out[60:] == 3).all())


def test_graph_replay_reads_the_offsets_again_and_streams():
    dev = cuda()
    t = 600
    q, k, v = make(13, t, t, 8, 2, torch.bfloat16, dev)
    off = cu([200, 300, 100], dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graphs = []
    with torch.cuda.stream(side):
        kernels.prompt_attention(q, k, v, off)
        for _ in range(2):
            out = torch.zeros_like(q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                kernels.prompt_attention(q, k, v, off, out=out)
            graphs.append((g, out))
    torch.cuda.current_stream(dev).wait_stream(side)
    for lens in ([200, 300, 100], [1, 598, 1], [0, 0, 600]):
        off.copy_(cu(lens, dev))
        for g, out in graphs:
            out.zero_()
            g.replay()
            check(out, q, k, v, lens, lens)


def test_same_result_twice():
    dev = cuda()
    lens, past = [64, 200], [5000, 0]
    both = [a + b for a, b in zip(lens, past)]
    q, k, v = make(14, sum(lens), sum(both), 8, 2, torch.bfloat16, dev)
    outs = [kernels.prompt_attention(q, k, v, cu(lens, dev), cu(both, dev)) for _ in range(5)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_refusals():
    dev = cuda()
    q, k, v = make(15, 20, 20, 8, 2, torch.bfloat16, dev)
    off = cu([20], dev)
    for args in ((q.float(), k.float(), v.float()), (q, k.half(), v.half()), (q, k, v[:, :10]), (q[:, :7], k, v),
                 (q[..., :64], k, v), (q, k, v, off.long()), (q, k, v, off[:1]), (q, k, v, off, cu([10, 10], dev)),
                 (q, k, v, None, off), (q.unsqueeze(0).expand(2, -1, -1, -1), k, v)):
        with pytest.raises(RuntimeError):
            kernels.prompt_attention(*args)
    with pytest.raises(RuntimeError, match="out"):
        kernels.prompt_attention(q, k, v, out=torch.empty_like(q).float())
    with pytest.raises(RuntimeError, match="gradient"):
        kernels.prompt_attention(q.clone().requires_grad_(), k, v)
    flat = torch.zeros(20 * 8 * 128 + 4, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="invalid argument"):  # not on a 16-byte boundary
        kernels.prompt_attention(flat[4:].view(20, 8, 128), k, v)
    assert kernels.prompt_attention(q[:0], k, v).shape == (0, 8, 128)
    assert kernels.prompt_attention(q, k[:, :0], v[:, :0]).abs().sum() == 0


def test_calls_on_two_streams_at_once():
    """Launches with and without key splits (their workspace) side by side: each as when it runs alone."""
    dev = cuda()
    sets = []
    for t, tk in ((64, 9000), (300, 300), (1500, 2100)):
        args = make(t, t, tk, 8, 2, torch.bfloat16, dev)
        offs = (cu([t], dev), cu([tk], dev))
        sets.append((args, offs, kernels.prompt_attention(*args, *offs)))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize(dev)
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] += [(kernels.prompt_attention(*args, *offs), want) for args, offs, want in sets[::1 - 2 * i]]
    torch.cuda.synchronize(dev)
    kernels.check_device_status(dev)
    assert all(torch.equal(got, want) for o in outs for got, want in o)


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    dev = cuda()
    q, k, v = make(16, 20, 20, 8, 2, torch.bfloat16, dev)
    slab = torch.zeros((2, 2, 32, 72), dtype=torch.uint8, device=dev)
    bits = torch.ones((20, 1), dtype=torch.int32, device=dev)
    with forward_ad.dual_level():
        kernels.prompt_attention(q, k, v)  # (none of these has one)
        for i in range(3):
            args = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate((q, k, v))]
            with pytest.raises(RuntimeError, match="gradient"):
                kernels.prompt_attention(*args)
            if i:
                with pytest.raises(RuntimeError, match="gradient"):
                    kernels.kv_append_q4(slab[0], slab[1], *args[1:])
        with pytest.raises(RuntimeError, match="gradient"):
            kernels.tree_attention_q4(forward_ad.make_dual(q, torch.ones_like(q)), slab[0], slab[1], bits, 4)
    kernels.check_device_status(dev)


def test_keys_and_values_of_different_strides():
    dev = cuda()
    q, k, v = make(17, 90, 90, 8, 2, torch.bfloat16, dev)         # rows of [tokens, heads, 128]
    for k2, v2 in ((k.contiguous(), v), (k, v.contiguous()), (k[:1].expand(2, -1, -1), v)):
        check(kernels.prompt_attention(q, k2, v2), q, k2, v2, [90], [90])


@pytest.mark.parametrize("lens,past", [([300], [2500]), ([17], [9000]), ([1], [4000]), ([64, 200], [5000, 0])])
def test_split_keys_fp16(lens, past):
    dev = cuda()
    both = [a + b for a, b in zip(lens, past)]
    q, k, v = make(len(lens) + sum(past), sum(lens), sum(both), 8, 2, torch.float16, dev, "tokens")
    assert kernels._prompt_workspace(0, sum(lens), sum(both), len(lens), 8, 2) > 0
    out = kernels.prompt_attention(q, k, v, cu(lens, dev), cu(both, dev))
    check(out, q, k, v, lens, both)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_split_keys_and_queries_without_keys(dtype):
    """One sequence's keys are shared out, another has fewer keys than queries, a third none."""
    dev = cuda()
    lens, keys = [40, 60, 5, 300], [9000, 30, 0, 300]
    q, k, v = make(21, sum(lens), sum(keys), 4, 2, dtype, dev)
    assert kernels._prompt_workspace(0, sum(lens), sum(keys), len(lens), 4, 2) > 0
    out = kernels.prompt_attention(q, k, v, cu(lens, dev), cu(keys, dev), out=torch.full_like(q, float("nan")))
    check(out, q, k, v, lens, keys)
    assert bool((out[40:70] == 0).all()) and bool((out[100:105] == 0).all())


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("dtype,past", [(torch.bfloat16, 2500), (torch.float16, 2500), (torch.float16, 0)])
def test_hidden_keys_do_not_reach_a_row_of_a_chunk(dtype, past, where, what):
    """As above with the keys shared out (2500 earlier ones), and in fp16: what a row cannot see does not change it."""
    dev = cuda()
    n, keys = 300, 300 + past
    q, k, v = make(22, n, keys, 8, 2, dtype, dev)
    assert (kernels._prompt_workspace(0, n, keys, 1, 8, 2) > 0) == (past > 0)
    offs = (cu([n], dev), cu([keys], dev))
    clean = kernels.prompt_attention(q, k, v, *offs)
    x = k if where == "k" else v
    x[0, past + 250, 3] = what      # rows 250..299 of query heads 0-3 see it
    x[1, keys - 1, :] = what        # the last row of heads 4-7 alone
    out = kernels.prompt_attention(q, k, v, *offs)
    kernels.check_device_status(dev)
    touched = torch.zeros((n, 8), dtype=torch.bool, device=dev)
    touched[250:, :4] = True
    touched[-1, 4:] = True
    assert torch.equal(out[~touched], clean[~touched])
    if where == "v":
        col = out[250:, :4, 3].float()
        assert bool(col.isnan().all()) if what != what else bool((col == what).all())
        rest = out[250:, :4].float()
        rest[..., 3] = 0
        assert bool(rest.isfinite().all())
        last = out[-1, 4:].float()
        assert bool(last.isnan().all()) if what != what else bool((last == what).all())
    elif what != what:
        assert bool(out[touched].isnan().all())


def test_more_sequences_than_one_launch_takes():
    dev = cuda()
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 4, (5000,), generator=g).tolist()
    q, k, v = make(23, sum(lens), sum(lens), 4, 2, torch.bfloat16, dev)
    out = kernels.prompt_attention(q, k, v, cu(lens, dev), out=torch.full_like(q, float("nan")))
    kernels.check_device_status(dev)
    # every sequence at once: [sequences, 3, ...] padded, the definition of `reference` in 64 bits
    a = cu(lens, "cpu").long()[:-1].to(dev)
    n = torch.tensor(lens, device=dev)
    idx = a[:, None] + torch.arange(3, device=dev)
    live = torch.arange(3, device=dev) < n[:, None]
    idx = torch.where(live, idx, 0)
    qq = q[idx].double()                                                        # [S, 3, 4, 128]
    kk, vv = (x.transpose(0, 1)[idx].double().repeat_interleave(2, 2) for x in (k, v))
    s = torch.einsum("sihd,sjhd->shij", qq, kk) * 128 ** -0.5
    see = live[:, None, None, :] & torch.ones((3, 3), device=dev).tril().bool()
    p = torch.softmax(s.masked_fill(~see, float("-inf")).nan_to_num(neginf=-1e30), -1) * see
    ref, big = (torch.einsum("shij,sjhd->sihd", p, x) for x in (vv, vv.abs()))
    err = (out[idx].double() - ref).abs()[live]
    # weights and result rounded once each; the scores' part with the largest sum_d |q_d k_d| of the call
    delta = 128 * 2.0 ** -23 * 128 ** -0.5 * float(torch.einsum("sihd,sjhd->shij", qq.abs(), kk.abs()).max())
    bound = (2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -20 + 3 * delta) * big)[live]
    assert bool((err <= bound + 1e-30).all())
