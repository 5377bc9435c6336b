"""GPU parity of the 4-bit cache rows and of the tree attention that reads them.

Rows: bytes and values are exact (``oracle.q4``).  Attention, per element, with
A = sum_j softmax_j |v_j| over the cache's values (exact bf16 numbers): weights
rounded to bf16 (2^-8 A), the result rounded to bf16 (2^-8 |o|), scores off by
at most delta = 128 * 2^-23 * scale * max_j sum_d |q_d k_jd| (3 * delta * A),
2^-20 A for the fp32 exponentials and sums.
"""

import numpy as np
import pytest
import torch

from oracle import q4
from oracle import tree as ot
from retree_b200 import kernels
from tests.gpu_util import bits_tensor, cuda, random_tree

pytestmark = pytest.mark.gpu


def rows(seed, dev, *shape):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((*shape, 128), generator=g) * torch.exp(0.7 * torch.randn((*shape[:-1], 1, 128), generator=g))
    return x.to(torch.bfloat16).to(dev)


def caches(seed, dev, hkv, total, extra=30):
    """A cache whose first ``total`` rows are set and whose others hold random bytes."""
    cap = total + extra + ((total + extra) & 1)
    g = torch.Generator(device=dev).manual_seed(seed)
    slab = torch.randint(0, 256, (2, hkv, cap, 72), dtype=torch.uint8, device=dev, generator=g)
    slab[:, :, :total] = q4.pack(rows(seed, dev, 2, hkv, total))
    return slab


def reference(q, slab, prefix, vis, scale=128 ** -0.5):
    n, hq, _ = q.shape
    grp = hq // slab.shape[1]
    see = torch.ones((n, prefix + n), dtype=torch.bool, device=q.device)
    see[:, prefix:] = torch.as_tensor(np.asarray(vis), device=q.device).bool()
    out = torch.empty((n, hq, 128), dtype=torch.float64, device=q.device)
    bound = torch.empty_like(out)
    for h in range(slab.shape[1]):
        k, v = q4.unpack(slab[0, h, :prefix + n]), q4.unpack(slab[1, h, :prefix + n])
        for i in range(h * grp, (h + 1) * grp):
            qq = q[:, i].double()
            s = torch.where(see, qq @ k.T * scale, float("-inf"))
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
            z = p.sum(1, keepdim=True)
            p = p / torch.where(z == 0, 1.0, z)
            p = torch.where(see, p, 0.0)
            vz = torch.where(see.any(0)[:, None], v, 0.0)
            o, big = p @ vz, p @ vz.abs()
            delta = 128 * 2.0 ** -23 * scale * torch.where(see, qq.abs() @ k.abs().T, 0.0).amax(1, keepdim=True)
            out[:, i] = o
            bound[:, i] = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -20 + 3 * delta) * big + 1e-30
    return out, bound


def check(out, q, slab, prefix, vis, scale=128 ** -0.5):
    kernels.check_device_status(q.device)
    ref, bound = reference(q, slab, prefix, vis, scale)
    over = ~((out.double() - ref).abs() <= bound)
    assert not bool(over.any()), (int(over.sum()), float(((out.double() - ref).abs() / bound).nan_to_num(1e9).max()),
                                  over.nonzero()[0].tolist())


# ---------------------------------------------------------------------------- rows
@pytest.mark.parametrize("heads,n,offset", [(1, 1, 0), (8, 17, 2075), (2, 1, 63), (3, 333, 5), (8, 2049, 0)])
def test_append_and_read(heads, n, offset):
    dev = cuda()
    cap = offset + n + 7
    slab = torch.full((2, heads, cap, 72), 171, dtype=torch.uint8, device=dev)
    k, v = rows(n, dev, heads, n), rows(n + 1, dev, heads, n)
    kernels.kv_append_q4(slab[0], slab[1], k, v, offset=offset)
    kernels.check_device_status(dev)
    assert torch.equal(slab[0, :, offset:offset + n], q4.pack(k))
    assert torch.equal(slab[1, :, offset:offset + n], q4.pack(v))
    assert bool((slab[:, :, :offset] == 171).all()) and bool((slab[:, :, offset + n:] == 171).all())
    back = kernels.kv_read_q4(slab, offset, n)
    assert torch.equal(back.double(), torch.stack([q4.values(k), q4.values(v)]))
    assert torch.equal(kernels.kv_read_q4(slab[1], offset, n), back[1])


def test_append_of_edge_rows():
    dev = cuda()
    x = rows(7, dev, 2, 64)
    x[0, 0] = 0
    x[0, 1] = 1e-39
    x[0, 2] = 0.375
    x[0, 3] = -0.375
    x[0, 4] = 3e38
    x[0, 4, ::2] = -3e38
    x[0, 5, 40] = float("nan")
    x[0, 6, 127] = float("inf")
    x[0, 7, 0] = float("-inf")
    x[0, 8] = torch.arange(128, device=dev).to(torch.bfloat16) % 32 * 0.5   # ties of code and zero point
    x[0, 9] = (torch.arange(128, device=dev) % 31 - 15).to(torch.bfloat16)
    x[0, 10] = 2.0 ** -120
    x[0, 11, ::3] = 2.0 ** -126
    slab = torch.zeros((2, 2, 64, 72), dtype=torch.uint8, device=dev)
    kernels.kv_append_q4(slab[0], slab[1], x, -x)
    kernels.check_device_status(dev)
    ref = torch.stack([q4.values(x), q4.values(-x)])
    got = kernels.kv_read_q4(slab, 0, 64).double()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))


def test_append_strided_rows_device_offset_and_overflow():
    dev = cuda()
    qkv = rows(9, dev, 20, 12)                          # [tokens, q | k | v heads]
    k, v = qkv[:, 8:10].transpose(0, 1), qkv[:, 10:].transpose(0, 1)
    slab = torch.zeros((2, 2, 64, 72), dtype=torch.uint8, device=dev)
    off = torch.tensor([30], dtype=torch.int64, device=dev)
    kernels.kv_append_q4(slab[0], slab[1], k[None], v[None], offset_dev=off)
    kernels.check_device_status(dev)
    assert torch.equal(slab[0, :, 30:50], q4.pack(k)) and torch.equal(slab[1, :, 30:50], q4.pack(v))
    before = slab.clone()
    for start, a, b in ((50, 0, 14), (-3, 3, 20)):      # the rows that fit are written, the others reported
        slab.copy_(before)
        off.fill_(start)
        kernels.kv_append_q4(slab[0], slab[1], k, v, offset_dev=off)
        with pytest.raises(RuntimeError, match="capacity"):
            kernels.check_device_status(dev)
        assert torch.equal(slab[0, :, start + a:start + b], q4.pack(k[:, a:b]))


def test_compaction_moves_4bit_rows():
    dev = cuda()
    slab = caches(3, dev, 4, 90).view(4, 2, -1, 72).contiguous()
    keep = torch.tensor([0, 3, 4, 9], dtype=torch.int64, device=dev)
    want = slab.clone()
    want[:, :, 70:74] = slab[:, :, 70 + keep]
    kernels.kv_compact(slab[:, :, :90], 70, keep)
    kernels.check_device_status(dev)
    assert torch.equal(slab, want)


def test_row_refusals():
    dev = cuda()
    slab = torch.zeros((2, 2, 16, 72), dtype=torch.uint8, device=dev)
    x = rows(1, dev, 2, 4)
    for bad in (lambda: kernels.kv_append_q4(slab[0], slab[1], x.half(), x.half()),
                lambda: kernels.kv_append_q4(slab[0], slab[1], x, x[:, :3]),
                lambda: kernels.kv_append_q4(slab[0], slab[1], x[:1], x[:1]),
                lambda: kernels.kv_append_q4(slab[0], slab[1], x, x, offset=13),
                lambda: kernels.kv_append_q4(slab[0, :, ::2], slab[1, :, ::2], x, x),
                lambda: kernels.kv_append_q4(slab[0].view(torch.int8), slab[1].view(torch.int8), x, x),
                lambda: kernels.kv_append_q4(slab[0], slab[1], x, x, offset_dev=torch.zeros(1, device=dev)),
                lambda: kernels.kv_read_q4(slab, 13, 4), lambda: kernels.kv_read_q4(slab, -1, 4),
                lambda: kernels.kv_read_q4(slab, 0, 4, out=torch.empty((2, 2, 4, 128), device=dev)),
                lambda: kernels.kv_read_q4(slab.transpose(0, 1)[:, :, :, :71], 0, 4)):
        with pytest.raises(RuntimeError):
            bad()
    assert kernels.kv_read_q4(slab, 3, 0).shape == (2, 2, 0, 128)


# ---------------------------------------------------------------------------- attention
@pytest.mark.parametrize("n,prefix,splits", [
    (1, 0, 0), (1, 1, 0), (1, 63, 0), (1, 127, 0), (1, 128, 0), (1, 2047, 0), (1, 2048, 3), (1, 20001, 0),
    (2, 130, 0), (3, 700, 1), (4, 129, 2), (5, 300, 0), (9, 1000, 0), (16, 0, 0), (16, 5, 1), (17, 2075, 0), (17, 512, 1),
    (17, 9000, 5), (32, 96, 0), (33, 95, 0), (64, 64, 0), (65, 1023, 0), (100, 5000, 7), (129, 4096, 0), (257, 130, 1),
    (257, 4097, 0), (600, 200, 0)])
def test_tree_attention(n, prefix, splits):
    dev = cuda()
    _, vis = random_tree(1000 + n, n - 1)
    slab = caches(n + prefix, dev, 2, prefix + n)
    q = rows(n, dev, n, 8)
    out = kernels.tree_attention_q4(q, slab[0], slab[1], bits_tensor(vis, dev), prefix, num_splits=splits)
    check(out, q, slab, prefix, vis)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 2), (6, 2), (7, 1), (10, 2), (16, 1), (32, 8), (64, 2), (33, 1)])
@pytest.mark.parametrize("n", [1, 2, 19])
def test_head_groups(hq, hkv, n):
    dev = cuda()
    _, vis = random_tree(hq + n, n - 1)
    slab = caches(hq, dev, hkv, 333 + n)
    q = rows(hkv, dev, n, hq)
    check(kernels.tree_attention_q4(q, slab[0], slab[1], bits_tensor(vis, dev), 333), q, slab, 333, vis)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_equals_bf16_attention_over_the_values(n):
    """The 4-bit cache is a bf16 cache of its values: both kernels stay within the same bound of each other."""
    dev = cuda()
    prefix = 1500
    _, vis = random_tree(n, n - 1)
    slab = caches(17, dev, 8, prefix + n)
    q = rows(18, dev, n, 32)
    bits = bits_tensor(vis, dev)
    kv = kernels.kv_read_q4(slab, 0, prefix + n)
    a = kernels.tree_attention_q4(q, slab[0], slab[1], bits, prefix)
    b = kernels.tree_attention(q, kv[0], kv[1], bits, prefix)
    _, bound = reference(q, slab, prefix, vis)
    assert bool(((a.double() - b.double()).abs() <= 2 * bound).all())


@pytest.mark.parametrize("n,bound_len", [(1, 5000), (17, 5000), (17, 700), (130, 900)])
def test_device_prefix_length(n, bound_len):
    dev = cuda()
    _, vis = random_tree(n, n - 1)
    slab = caches(n, dev, 2, 5000 + n)
    q = rows(n, dev, n, 8)
    plen = torch.zeros(1, dtype=torch.int64, device=dev)
    side = torch.cuda.Stream(dev)
    bits = bits_tensor(vis, dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        kernels.tree_attention_q4(q, slab[0], slab[1], bits, bound_len, prefix_len_dev=plen)
        out = torch.empty_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kernels.tree_attention_q4(q, slab[0], slab[1], bits, bound_len, prefix_len_dev=plen, out=out)
    torch.cuda.current_stream(dev).wait_stream(side)
    for prefix in (0, 1, 640, 700):
        plen.fill_(prefix)
        out.fill_(float("nan"))
        g.replay()
        check(out, q, slab, prefix, vis)
    # outside the cache: reported, not read
    for prefix in (-1, slab.shape[2] - n + 1, 2 ** 40):
        plen.fill_(prefix)
        g.replay()
        with pytest.raises(RuntimeError, match="index"):
            kernels.check_device_status(dev)


def test_rows_that_see_nothing_are_zero():
    dev = cuda()
    for n in (1, 5, 40):
        vis = np.eye(n, dtype=bool)
        vis[n // 2] = False
        slab = caches(n, dev, 2, n)
        q = rows(n, dev, n, 8)
        out = kernels.tree_attention_q4(q, slab[0], slab[1], bits_tensor(vis, dev), 0)
        check(out, q, slab, 0, vis)
        assert bool((out[n // 2] == 0).all())


@pytest.mark.parametrize("n", [1, 3, 20, 150])
@pytest.mark.parametrize("which", [0, 1])
def test_rows_not_finite(n, which):
    """A tree row that reads as NaN reaches the nodes that see it and no other; so do stale rows behind the tree."""
    dev = cuda()
    prefix = 200
    _, vis = random_tree(50 + n, n - 1)
    slab = caches(n, dev, 2, prefix + n)
    q = rows(n, dev, n, 8)
    bits = bits_tensor(vis, dev)
    slab[:, :, prefix + n:, 64:] = 0xFF       # NaN words (and every code) behind the tree
    slab[:, :, prefix + n:, 65::2] = 0x7F
    clean = kernels.tree_attention_q4(q, slab[0], slab[1], bits, prefix)
    check(clean, q, slab, prefix, vis)
    bad = n // 2
    x = rows(1, dev, 1, 1)
    x[..., 9] = float("nan")
    slab[which, 1, prefix + bad] = q4.pack(x)[0, 0]
    out = kernels.tree_attention_q4(q, slab[0], slab[1], bits, prefix)
    sees = torch.as_tensor(np.asarray(vis), device=dev).bool()[:, bad]
    assert torch.equal(out[:, :4], clean[:, :4]) and torch.equal(out[~sees], clean[~sees])
    assert bool(out[sees][:, 4:].isnan().all())
    # and a prefix row of that kind reaches all
    slab[which, 0, 77] = q4.pack(x)[0, 0]
    out = kernels.tree_attention_q4(q, slab[0], slab[1], bits, prefix)
    assert bool(out[:, :4].isnan().all())


def test_large_scores_views_and_scale():
    dev = cuda()
    for n in (1, 33):
        prefix = 900
        _, vis = random_tree(n, n - 1)
        cap = prefix + n + 1 + ((prefix + n + 1) & 1)
        k = (rows(3, dev, 2, prefix + n).float() * torch.linspace(0.1, 6, prefix + n, device=dev)[None, :, None]).bfloat16()
        slab = torch.zeros((2, 2, cap, 72), dtype=torch.uint8, device=dev)
        for flip in (False, True):
            kk = k.flip(1).contiguous() if flip else k
            kernels.kv_append_q4(slab[0], slab[1], kk, rows(4, dev, 2, prefix + n))
            qkv = rows(5, dev, n, 12)
            q = qkv[:, :8]
            buf = torch.full((n, 9, 128), 3.0, dtype=torch.bfloat16, device=dev)
            out = kernels.tree_attention_q4(q.transpose(0, 1)[None], slab[0], slab[1], bits_tensor(vis, dev), prefix,
                                            scale=0.4, out=buf[:, :8])
            check(out, q, slab, prefix, vis, 0.4)
            assert bool((buf[:, 8] == 3).all())


def test_same_result_twice_and_wide_masks():
    dev = cuda()
    for n in (1, 17, 70):
        _, vis = random_tree(n, n - 1)
        slab = caches(n, dev, 8, 3000 + n)
        q = rows(n, dev, n, 32)
        outs = [kernels.tree_attention_q4(q, slab[0], slab[1], bits_tensor(vis, dev, words=w), 3000)
                for w in (None, (n + 31) // 32, 8, 8)]
        assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_attention_refusals():
    dev = cuda()
    slab = caches(1, dev, 2, 60, extra=4)
    q = rows(1, dev, 4, 8)
    bits = bits_tensor(np.tril(np.ones((4, 4), bool)), dev)
    for args in ((q.half(), slab[0], slab[1], bits, 10), (q[:, :7], slab[0], slab[1], bits, 10),
                 (q, slab[0], slab[1][:, :32], bits, 10), (q, slab[0, :, ::2], slab[1, :, ::2], bits, 10),
                 (q, slab[0], slab[1], bits[:3], 10), (q, slab[0], slab[1], bits.long(), 10),
                 (q, slab[0], slab[1], bits, 61), (q, slab[0], slab[1], bits, -1), (q[:0], slab[0], slab[1], bits, 10),
                 (q[..., :64], slab[0], slab[1], bits, 10)):
        with pytest.raises(RuntimeError):
            kernels.tree_attention_q4(*args)
    with pytest.raises(RuntimeError, match="int64"):
        kernels.tree_attention_q4(q, slab[0], slab[1], bits, 10, prefix_len_dev=torch.zeros(1, device=dev))
    with pytest.raises(RuntimeError, match="gradient"):
        kernels.tree_attention_q4(q.clone().requires_grad_(), slab[0], slab[1], bits, 10)
    for scale in (-0.1, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="invalid argument"):
            kernels.tree_attention_q4(q, slab[0], slab[1], bits, 10, scale=scale)


def test_an_odd_capacity_is_refused():
    dev = cuda()
    slab = torch.zeros((2, 1, 41, 72), dtype=torch.uint8, device=dev)
    bits = bits_tensor(np.ones((1, 1), bool), dev)
    with pytest.raises(RuntimeError, match="even"):
        kernels.tree_attention_q4(rows(1, dev, 1, 4), slab[0], slab[1], bits, 10)


@pytest.mark.parametrize("n,prefix", [(1, 3000), (17, 3000), (33, 9000), (65, 4096), (129, 3000), (257, 2075)])
def test_a_given_split_count_splits_like_the_one_picked(n, prefix):
    """One launch sized by its prefix, one given that launch's count and sized for the capacity: the same bits."""
    dev = cuda()
    _, vis = random_tree(n, n - 1)
    slab = caches(n, dev, 8, prefix + n, extra=4000)
    q, bits = rows(n, dev, n, 32), bits_tensor(vis, dev)
    count = kernels.default_splits_q4(n, 32, 8, prefix)
    a = kernels.tree_attention_q4(q, slab[0], slab[1], bits, prefix, num_splits=count)
    b = kernels.tree_attention_q4(q, slab[0], slab[1], bits, slab.shape[2] - n, num_splits=count,
                                  prefix_len_dev=torch.tensor([prefix], device=dev))
    kernels.check_device_status(dev)
    assert torch.equal(a, b)
    check(a, q, slab, prefix, vis)


def test_calls_on_two_streams_at_once():
    """Launches with workspaces, clusters and neither, side by side: each as when it runs alone."""
    dev = cuda()
    sets = []
    for n, prefix in ((1, 3000), (17, 6000), (40, 2000), (129, 5000)):
        _, vis = random_tree(n, n - 1)
        slab = caches(n, dev, 8, prefix + n)
        args = (rows(n, dev, n, 32), slab[0], slab[1], bits_tensor(vis, dev), prefix)
        sets.append((args, kernels.tree_attention_q4(*args)))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize(dev)
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] += [(kernels.tree_attention_q4(*args), want) for args, want in sets[::1 - 2 * i]]
    torch.cuda.synchronize(dev)
    kernels.check_device_status(dev)
    assert all(torch.equal(got, want) for o in outs for got, want in o)


@pytest.mark.parametrize("n", [1, 17, 129])
def test_wild_device_lengths_are_reported(n):
    """Lengths whose sum with the tree passes 64 bits, on the device: nothing is read or written."""
    dev = cuda()
    _, vis = random_tree(n, n - 1)
    slab = caches(n, dev, 2, 2000 + n)
    q = rows(n, dev, n, 8)
    out = torch.full_like(q, 7.0)
    for prefix in (2 ** 63 - 1, 2 ** 63 - n, -2 ** 63):
        plen = torch.tensor([prefix], device=dev)
        kernels.tree_attention_q4(q, slab[0], slab[1], bits_tensor(vis, dev), 2000, prefix_len_dev=plen, out=out)
        with pytest.raises(RuntimeError, match="index"):
            kernels.check_device_status(dev)
    assert bool((out == 7).all())


def test_codes_of_symmetric_ranges_are_clamped():
    """hi = -lo = 7.5 s: both ends round away from zero, and the upper one would be code 16."""
    dev = cuda()
    x = rows(3, dev, 1, 40).clamp(-7.5, 7.5)
    x[:, :, ::32], x[:, :, 1::32] = 7.5, -7.5
    x = torch.where(x.abs() > 7.5, 7.5, x) * (2.0 ** torch.arange(-20, 20, device=dev))[None, :, None].bfloat16()
    slab = torch.zeros((2, 1, 40, 72), dtype=torch.uint8, device=dev)
    kernels.kv_append_q4(slab[0], slab[1], x, -x)
    kernels.check_device_status(dev)
    want = q4.pack(torch.stack([x, -x]))
    assert torch.equal(slab, want)
    top = kernels.kv_read_q4(slab, 0, 40)[0, 0, :, 0].float()
    assert torch.equal(top, 7 * 2.0 ** torch.arange(-20, 20, device=dev))


def _edge_groups(ends):
    """Rows whose four groups have the given (hi, lo), the values in between among them."""
    x = torch.zeros((1, len(ends), 128), dtype=torch.float64)
    for i, (hi, lo) in enumerate(ends):
        x[0, i, 0::32], x[0, i, 1::32], x[0, i, 2::32] = hi, lo, hi / 3
    return x.to(torch.bfloat16)


def test_scales_of_ranges_whose_small_end_is_below_the_large_ones_last_bit():
    """15 times a scale of four bits and a little more takes the next scale, however little it is."""
    dev = cuda()
    ends = [(15 * m / 8 * 2.0 ** e, -15 * 2.0 ** (e - k)) for m in range(8, 16) for e in (-100, -60, -27, 0, 40, 98, 120)
            for k in (7, 20, 23, 24, 25, 30, 53, 60, 90)]
    x = _edge_groups(ends).to(dev)
    slab = torch.zeros((2, 1, len(ends), 72), dtype=torch.uint8, device=dev)
    kernels.kv_append_q4(slab[0], slab[1], x, -x)
    kernels.check_device_status(dev)
    assert torch.equal(slab, q4.pack(torch.stack([x, -x])))


def test_groups_read_as_zero_below_the_smallest_normal_scale():
    dev = cuda()
    ends = [(m / 16 * 2.0 ** -126, 0.0) for m in range(128, 256)] + [(0.0, -m / 16 * 2.0 ** -126) for m in range(200, 256)]
    x = _edge_groups(ends).to(dev)
    slab = torch.zeros((2, 1, len(ends), 72), dtype=torch.uint8, device=dev)
    kernels.kv_append_q4(slab[0], slab[1], x, -x)
    kernels.check_device_status(dev)
    assert torch.equal(slab, q4.pack(torch.stack([x, -x])))


def test_device_words_without_an_entry_are_refused():
    """An empty tensor has no address, which would read as "no device word": the host's number."""
    dev = cuda()
    slab = torch.zeros((2, 2, 16, 72), dtype=torch.uint8, device=dev)
    x = rows(1, dev, 2, 4)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    q = torch.zeros((1, 4, 128), dtype=torch.bfloat16, device=dev)
    bits = torch.ones((1, 1), dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="offset_dev"):
        kernels.kv_append_q4(slab[0], slab[1], x, x, offset_dev=none)
    with pytest.raises(RuntimeError, match="prefix_len_dev"):
        kernels.tree_attention_q4(q, slab[0], slab[1], bits, 8, prefix_len_dev=none)
    assert int(slab.sum()) == 0


@pytest.mark.parametrize("hq,hkv", [(128, 1), (100, 1), (192, 2)])
@pytest.mark.parametrize("n", [1, 2, 3])
def test_groups_of_which_a_tile_holds_one_node(hq, hkv, n):
    """More than 64 query heads a kv head: tiles of one node, with rows to spare."""
    dev = cuda()
    slab = caches(hq, dev, hkv, 400 + n)
    q = rows(hq + 1, dev, n, hq)
    parents, vis = random_tree(n, n - 1)
    check(kernels.tree_attention_q4(q, slab[0], slab[1], bits_tensor(vis, dev), 400), q, slab, 400, vis)
