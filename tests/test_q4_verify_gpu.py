"""The 4-bit target cache and the prompt kernel in the framework's own paths: cache, attention backend,
verifier rounds (module, fused, CUDA graph), decode loop, packed prompts."""

import numpy as np
import pytest
import torch

from oracle import q4
from oracle import tree as ot
from retree_b200 import attention, kernels, synthetic
from retree_b200.cache import TreeKVCache, TreeKVCacheQ4, make_cache
from retree_b200.ddtree import compact_dynamic_cache, ddtree_generate
from retree_b200.target import build_target, qwen3_config
from retree_b200.verify import TreeVerifier
from tests.gpu_util import cuda, random_tree

pytestmark = pytest.mark.gpu

VOCAB = 2000


def _cfg(layers=2):
    return qwen3_config("small", hidden_size=512, intermediate_size=1024, num_hidden_layers=layers,
                        num_attention_heads=8, num_key_value_heads=2, vocab_size=VOCAB, tie_word_embeddings=False)


@pytest.fixture(scope="module")
def model():
    return build_target(_cfg(3), device=cuda(), seed=3)


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _ids(seed, n, dev):
    return torch.randint(0, VOCAB, (1, n), device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def _rows(seed, heads, n, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn((1, heads, n, 128), device=dev, generator=g).to(torch.bfloat16)


def test_make_cache():
    dev = cuda()
    assert type(make_cache(16, 2, 2, 128, 33, device=dev)) is TreeKVCache
    c = make_cache(4, 2, 2, 128, 33, device=dev)
    assert type(c) is TreeKVCacheQ4 and c.capacity == 34 and c.slab.shape == (4, 2, 34, 72)
    with pytest.raises(ValueError):
        make_cache(8, 2, 2, 128, 33, device=dev)
    with pytest.raises(RuntimeError):
        make_cache(4, 2, 2, 64, 32, device=dev)


def test_cache_holds_what_was_appended():
    dev = cuda()
    c = TreeKVCacheQ4(2, 3, 128, 100, device=dev)
    k, v = _rows(1, 3, 40, dev), _rows(2, 3, 40, dev)
    for li in range(2):
        c.update(k, v, li)
        c.update(v[:, :, :17], k[:, :, :17], li)
    assert c.get_seq_length() == 57
    keys = torch.cat([k, v[:, :, :17]], 2)
    for layer in c.layers:
        assert torch.equal(layer.keys.double(), q4.values(keys))
    # compaction of the appended window: bytes move as they are
    before = c.slab.clone()
    compact_dynamic_cache(c, 40, [0, 3, 4, 16])
    kernels.check_device_status(dev)
    assert c.get_seq_length() == 44
    assert torch.equal(c.slab[:, :, :40], before[:, :, :40])
    assert torch.equal(c.slab[:, :, 40:44], before[:, :, [40, 43, 44, 56]])
    with pytest.raises(RuntimeError, match="capacity"):
        c.update(_rows(3, 3, 60, dev), _rows(4, 3, 60, dev), 0)


class _Module:
    training = False
    is_causal = True


@pytest.mark.parametrize("prefix,n", [(0, 200), (0, 1), (300, 1), (300, 60), (300, 300), (77, 17)])
def test_backend_reads_the_4bit_rows(prefix, n):
    """Prompts attend to their own bf16 rows, whatever comes later to the cached values."""
    dev = cuda()
    c = TreeKVCacheQ4(1, 2, 128, 1024, device=dev)
    if prefix:
        c.update(_rows(1, 2, prefix, dev), _rows(2, 2, prefix, dev), 0)
    k, v, q = _rows(3, 2, n, dev), _rows(4, 2, n, dev), _rows(5, 8, n, dev)
    tree = n == 17
    parents, vis = random_tree(7, n - 1)
    mask = None
    if tree:
        bits = torch.from_numpy(ot.pack_bits(vis).view(np.int32)).to(dev)
        mask = attention.attach(bits.view(1, 1, n, -1), bits)
    key, value = c.update(k, v, 0)
    out, _ = attention.tree_attention_forward(_Module(), q, key, value, mask, scaling=128 ** -0.5)
    kernels.check_device_status(dev)
    kk, vv = (k, v) if prefix == 0 else (c.layers[0].keys, c.layers[0].values)
    see = torch.ones((n, prefix + n), dtype=torch.bool, device=dev)
    see[:, prefix:] = torch.from_numpy(np.asarray(vis)).to(dev) if tree else torch.ones((n, n), device=dev).tril().bool()
    s = (q[0].double() @ kk[0].double().repeat_interleave(4, 0).transpose(1, 2)) * 128 ** -0.5
    p = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
    ref = (p @ vv[0].double().repeat_interleave(4, 0)).transpose(0, 1)
    # weights and result each rounded once to bf16 (half a step 2^-8 each), values of order one
    assert float((out[0].double() - ref).abs().max()) < 2 * 2.0 ** -8 * float(vv.abs().max())
    assert _rel(out[0], ref) < 2.0 ** -8


def test_device_length_needs_a_tree_mask():
    dev = cuda()
    c = TreeKVCacheQ4(1, 2, 128, 64, device=dev)
    c.use_device_length(True)
    key, value = c.update(_rows(1, 2, 4, dev), _rows(2, 2, 4, dev), 0)
    with pytest.raises(RuntimeError, match="device-length"):
        attention.tree_attention_forward(_Module(), _rows(3, 8, 4, dev), key, value, None)


@torch.inference_mode()
def test_prompt_kernel_and_packed_prompts_through_the_model(model):
    dev = cuda()
    lens = [130, 7, 250]
    ids = _ids(0, sum(lens), dev)
    pos = torch.cat([torch.arange(n, device=dev) for n in lens])[None]
    plain, ends = [], torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32)
    for a, n in zip(ends.tolist(), lens):
        one = ids[:, a:a + n]
        c = TreeKVCache.for_model(model.config, capacity=512, device=dev)
        plain.append(model(one, position_ids=torch.arange(n, device=dev)[None], past_key_values=c, use_cache=True).logits)
        with attention.prompt_kernel():
            c2 = TreeKVCache.for_model(model.config, capacity=512, device=dev)
            half = n // 2
            p = torch.arange(n, device=dev)[None]
            a1 = model(one[:, :half], position_ids=p[:, :half], past_key_values=c2, use_cache=True).logits
            a2 = model(one[:, half:], position_ids=p[:, half:], past_key_values=c2, use_cache=True).logits
        assert _rel(torch.cat([a1, a2], 1), plain[-1]) < 2e-2
    cu = ends.to(dev)
    out = model(ids, position_ids=pos, use_cache=False, cu_seq_lens_q=cu, cu_seq_lens_k=cu,
                max_length_q=max(lens), max_length_k=max(lens)).logits
    kernels.check_device_status(dev)
    assert _rel(out, torch.cat(plain, 1)) < 2e-2


@pytest.mark.parametrize("fused", [False, True])
@torch.inference_mode()
def test_rounds_over_a_4bit_cache(model, monkeypatch, fused):
    """Stage by stage: what a round commits and moves, and CUDA-graph rounds equal to eager ones."""
    monkeypatch.setenv("DDTREE_TREE_STRATEGY", "rank_gated_ngram")
    dev = cuda()
    prompt = torch.from_numpy(synthetic.context_ids(8, 150, VOCAB, alphabet=40))[None].to(dev)
    drafts = [torch.from_numpy(synthetic.draft_logits(300 + r, 15, VOCAB, amp=6.0)).to(dev).to(torch.bfloat16)
              for r in range(5)]
    mk = lambda: TreeVerifier(model, tree_budget=24, max_length=500, draft_horizon=15, fused=fused, kv_bits=4)  # noqa
    eager, graph = mk(), mk()
    eager.debug = True
    for v in (eager, graph):
        v.prefill(prompt)
    graph.enable_graph(True)
    for d in drafts:
        start = eager.start
        acc = eager.round(d)
        n = 25
        tree_ids = eager.tree["verify_ids"][:n].tolist()
        kept, nxt = ot.follow_tree(ot.child_maps(eager.tree["parents"][:n].tolist(), np.array(tree_ids[1:])),
                                   eager.last_posterior[0].cpu().numpy())
        assert acc == len(kept)
        assert eager.output_ids[start:start + acc + 1].tolist() == [tree_ids[i] for i in kept] + [int(nxt)]
        moved = eager.last_slab[:, :, start:][:, :, kept]
        assert torch.equal(eager.cache.slab[:, :, start:start + acc], moved)
        assert torch.equal(eager.cache.slab[:, :, :start], eager.last_slab[:, :, :start])
        assert graph.round(d) == acc and graph.start == eager.start
    s = eager.start
    kernels.check_device_status(dev)
    assert torch.equal(eager.output_ids[: s + 1], graph.output_ids[: s + 1])
    assert torch.equal(eager.cache.slab[:, :, :s], graph.cache.slab[:, :, :s])


@torch.inference_mode()
def test_fused_forward_equals_the_module_over_a_4bit_cache(model):
    dev = cuda()
    n, L = 33, 200
    outs = []
    for fused in (False, True):
        v = TreeVerifier(model, tree_budget=n - 1, max_length=400, fused=fused, kv_bits=4, gemm="cublas")
        v.prefill(_ids(1, L, dev))
        parents, vis = random_tree(3, n - 1)
        bits = torch.from_numpy(ot.pack_bits(vis).view(np.int32)).to(dev)
        pos = torch.from_numpy(L + synthetic.depths_from_parents(parents)).to(dev)
        tok = _ids(2, n, dev)
        if fused:
            outs.append(v.fused.forward(tok[0], pos, bits, offset=L).clone())
        else:
            mask = attention.attach(bits.view(1, 1, n, -1), bits)
            outs.append(v.target(tok, position_ids=pos[None], attention_mask=mask, past_key_values=v.cache,
                                 use_cache=True).logits[0])
    kernels.check_device_status(dev)
    # the two forwards round in different places (see the bf16 comparison of the same
    # forwards); a code of the cache may then differ by one step of 4 bits
    assert _rel(outs[1], outs[0]) < 5e-2


@torch.inference_mode()
def test_tree_decoding_equals_greedy_decoding_over_a_4bit_cache(monkeypatch):
    monkeypatch.setenv("DDTREE_TREE_STRATEGY", "rank_gated_ngram")
    dev = cuda()
    m = build_target(_cfg(2), device=dev, seed=9)
    m.lm_head.weight.mul_(8.0)  # wide logit margins: argmax immune to bf16 reordering
    prompt = torch.from_numpy(synthetic.context_ids(4, 64, VOCAB, alphabet=30))[None].to(dev)
    new = 40
    cache = TreeKVCacheQ4.for_model(m.config, capacity=256, device=dev)
    out = m(prompt, position_ids=torch.arange(64, device=dev)[None], past_key_values=cache, use_cache=True)
    greedy, margins = [int(out.logits[0, -1].argmax())], [1.0]
    for i in range(new - 1):
        t = torch.tensor([[greedy[-1]]], device=dev)
        out = m(t, position_ids=torch.tensor([[64 + i]], device=dev), past_key_values=cache, use_cache=True)
        top2 = out.logits[0, -1].float().topk(2).values
        margins.append(float(top2[0] - top2[1]) / max(float(top2[0].abs()), 1.0))
        greedy.append(int(out.logits[0, -1].argmax()))

    def draft_fn(output_ids, start, r):
        g = torch.Generator(device=dev).manual_seed(r)
        return torch.randn((15, VOCAB), device=dev, generator=g)

    res = ddtree_generate(None, m, prompt, mask_token_id=VOCAB - 1, max_new_tokens=new, block_size=16,
                          stop_token_ids=None, tree_budget=24, draft_fn=draft_fn, kv_bits=4, fused=False)
    got = res.output_ids[0, 64:].tolist()
    assert res.num_output_tokens >= new
    # as over the bf16 cache: the runs may part only at a near tie of the greedy run's top two logits
    if got[: len(greedy)] != greedy[: len(got)]:
        first = next(i for i, (a, b) in enumerate(zip(got, greedy)) if a != b)
        assert margins[first] < 2e-2, (first, margins[first])


@torch.inference_mode()
def test_prefill_random_fills_a_4bit_cache(model):
    dev = cuda()
    v = TreeVerifier(model, tree_budget=16, max_length=300, kv_bits=4)
    v.prefill_random(200, seed=1)
    keys = v.cache.layers[1].keys
    assert keys.shape == (1, 2, 200, 128) and 0.9 < float(keys.float().std()) < 1.1
    v.round(torch.from_numpy(synthetic.draft_logits(1, 15, VOCAB, amp=6.0)).to(dev).to(torch.bfloat16))
    kernels.check_device_status(dev)


def test_packed_queries_over_earlier_keys_need_their_offsets():
    """Without the keys' own offsets the queries' would point at the first keys of the cache."""
    dev = cuda()
    c = TreeKVCache(1, 2, 128, 64, device=dev)
    c.update(_rows(1, 2, 4, dev), _rows(2, 2, 4, dev), 0)
    key, value = c.update(_rows(3, 2, 6, dev), _rows(4, 2, 6, dev), 0)
    cu = torch.tensor([0, 6], dtype=torch.int32, device=dev)
    q = _rows(5, 8, 6, dev)
    with pytest.raises(RuntimeError, match="packed"):
        attention.tree_attention_forward(_Module(), q, key, value, None, scaling=0.1, cu_seq_lens_q=cu)
    cu_k = torch.tensor([0, 10], dtype=torch.int32, device=dev)
    out, _ = attention.tree_attention_forward(_Module(), q, key, value, None, scaling=0.1, cu_seq_lens_q=cu,
                                              cu_seq_lens_k=cu_k)
    with attention.prompt_kernel():
        one, _ = attention.tree_attention_forward(_Module(), q, key, value, None, scaling=0.1)
    kernels.check_device_status(dev)
    assert torch.equal(out, one)


@torch.inference_mode()
def test_another_backend_over_a_4bit_cache_is_an_error():
    """A prompt and a single token after it: neither runs on a part of the keys."""
    dev = cuda()
    m = build_target(_cfg(1), device=dev, seed=4, attn_implementation="sdpa")
    cache = TreeKVCacheQ4(1, 2, 128, 64, device=dev)
    for n in (5, 1):
        with pytest.raises(RuntimeError, match="4-bit"):
            m(_ids(n, n, dev), past_key_values=cache, use_cache=True)
    with pytest.raises(RuntimeError, match="retree_tree"):
        TreeKVCacheQ4.for_model(m.config, capacity=64, device=dev)


@torch.inference_mode()
def test_a_target_split_by_kv_head_over_a_4bit_cache(model, monkeypatch):
    """Each rank's heads over its own 4-bit cache (the gather left out) are the whole cache's heads."""
    from retree_b200 import headsplit
    dev = cuda()
    monkeypatch.setattr(headsplit, "gather_heads", lambda out, group, world: out)
    backend = headsplit.headsplit_backend(attention.tree_attention_forward)
    L, n = 300, 17
    k, v, q = (_rows(s, h, L + n, dev) for s, h in ((1, 2), (2, 2), (3, 8)))
    _, vis = random_tree(7, n - 1)
    bits = torch.from_numpy(ot.pack_bits(vis).view(np.int32)).to(dev)
    mask = attention.attach(bits.view(1, 1, n, -1), bits)
    outs = []
    for heads, split in ((slice(0, 2), None), (slice(0, 1), (None, 2, 0)), (slice(1, 2), (None, 2, 1))):
        c = make_cache(4, 1, heads.stop - heads.start, 128, 512, device=dev)
        mod = _Module()
        mod._rt_head_split = split
        qh = q[:, 4 * heads.start:4 * heads.stop]
        kh, vh = k[:, heads], v[:, heads]
        rows = c.update(kh[:, :, :L], vh[:, :, :L], 0)
        a, _ = backend(mod, qh[:, :, :L], *rows, None, scaling=128 ** -0.5)
        rows = c.update(kh[:, :, L:], vh[:, :, L:], 0)
        b, _ = backend(mod, qh[:, :, L:], *rows, mask, scaling=128 ** -0.5)
        outs.append(torch.cat([a, b], 1))
    kernels.check_device_status(dev)
    split = torch.cat(outs[1:], 2)
    # (the heads' work is shared out differently: two roundings of weights and of results, values of order one)
    assert float((split.float() - outs[0].float()).abs().max()) < 4 * 2.0 ** -8 * float(v.abs().max())
    assert _rel(split, outs[0]) < 2.0 ** -7
