"""The attention and cache operators of the verify path over a 4-bit cache, as measured.

Three operators: causal attention over whole prompts (packed sequences, grouped
heads), append into / read from a cache whose rows are held in 4 bits, and the
tree-verify attention over such a cache.  ``own`` picks between the plain form
(elementary torch operations in 32 bits) and the framework's kernels.

A 4-bit row (one head, one token, 128 values) is 72 bytes: 64 bytes of 4-bit
codes u and four 16-bit words, one per 32 consecutive values.  Bits 4-14 of a
word are the exponent and the top three mantissa bits of the scale s, bits 0-3
the zero point z; a value is (u - z) * s, which bf16 holds exactly.  Of the
32-bit word i of the codes, bits 4j..4j+3 belong to value 8i + ORDER[j].
"""

import torch

own = False

D = 128              # head size
ROW = 72             # bytes of a 4-bit row
GROUP = 32           # values that share a scale
ORDER = (0, 2, 4, 6, 1, 3, 5, 7)
LOG2E = 1.4426950408889634


# ----------------------------------------------------------------------------- cases
def listed():
    """The cases; each says what it stands for."""
    def prompt(name, lens, past=None, hq=32, hkv=8, dtype="bf16", layout="qkv"):
        past = past or [0] * len(lens)
        return dict(name=name, op="prompt", lens=",".join(map(str, lens)), past=",".join(map(str, past)), hq=hq,
                    hkv=hkv, dtype=dtype, layout=layout)

    def append(name, rows, offset, hkv=8):
        return dict(name=name, op="append", rows=rows, offset=offset, hkv=hkv)

    def verify(name, nodes, prefix, hq=32, hkv=8):
        return dict(name=name, op="verify", nodes=nodes, prefix=prefix, hq=hq, hkv=hkv)

    return [
        # a short chat turn: one small prompt, where the launch's latency counts
        prompt("prompt-64", [64]),
        # the prompt of the verify benchmark, read straight from the packed q|k|v projection
        prompt("prompt-2048", [2048]),
        # a long document, the largest call
        prompt("prompt-7122", [7122]),
        # a batch of requests of very different lengths, odd ones among them
        prompt("prompt-ragged", [1, 17, 4095, 129, 600, 2047, 5, 1301]),
        # no grouping, fp16, head-major tensors as the transformers modules hand them over
        prompt("prompt-fp16-mha", [1531, 2500], hq=16, hkv=16, dtype="fp16", layout="heads"),
        # the next chunk of a long prompt over the keys of the chunks before it, beside a fresh request
        prompt("prompt-chunk", [512, 77], past=[8192, 0]),
        # one round's tree goes into the cache
        append("append-17", 17, 2075),
        # a whole prompt goes into the cache
        append("append-8191", 8191, 0),
        # plain decoding: one token over a short and over a very long cache
        verify("verify-1-2048", 1, 2048),
        verify("verify-1-131072", 1, 131071),
        # a round of the default budget over a long cache
        verify("verify-17-32768", 17, 32768),
        # a wide tree over a long cache
        verify("verify-257-32768", 257, 32768),
    ]


HEADS = [(32, 8), (32, 8), (16, 16), (28, 4), (8, 1), (12, 4), (16, 8)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["prompt", "prompt", "append", "verify", "verify"])
    hq, hkv = rng.choice(HEADS)
    if op == "append":
        rows = _log(rng, 1, 8191)
        return dict(op=op, rows=rows, offset=rng.randrange(0, 5000), hkv=hkv)
    if op == "verify":
        nodes = rng.choice([1, 1, 2, 3, _log(rng, 1, 257), _log(rng, 1, 257)])
        prefix = _log(rng, 1, 131071 if nodes <= 4 else 32768) - rng.choice([0, 1])
        return dict(op=op, nodes=nodes, prefix=prefix, hq=hq, hkv=hkv)
    count = rng.choice([1, 1, 2, 3, 5, 8, 13])
    total = _log(rng, 1, 6000)
    lens = [max(1, int(total * rng.random() ** 2) // count) for _ in range(count)]
    lens[rng.randrange(count)] += rng.randrange(0, 900)
    past = [0] * count
    if rng.random() < 0.4:
        past[rng.randrange(count)] = _log(rng, 1, 8192 if total < 1000 else 2000)
    return dict(op=op, lens=",".join(map(str, lens)), past=",".join(map(str, past)), hq=hq, hkv=hkv,
                dtype=rng.choice(["bf16", "bf16", "fp16"]), layout=rng.choice(["qkv", "heads", "tokens"]))


def _lens(case):
    return [int(x) for x in case["lens"].split(",")], [int(x) for x in case["past"].split(",")]


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)


def _randn(g, shape, dtype):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _kv_rows(g, shape):
    """K/V rows as a cache meets them: a few channels of a head are much larger than the rest."""
    x = torch.randn(shape, device="cuda", generator=g)
    gain = torch.exp(0.7 * torch.randn((shape[0], 1, shape[2]), device="cuda", generator=g))
    return (x * gain).to(torch.bfloat16)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "prompt":
        lens, past = _lens(case)
        hq, hkv = case["hq"], case["hkv"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
        t, tk = sum(lens), sum(lens) + sum(past)
        if case["layout"] == "qkv" and t == tk:
            # views of the packed projection's rows [q heads | k heads | v heads]
            x = _randn(g, (t, hq + 2 * hkv, D), dtype)
            q, k, v = x[:, :hq], x[:, hq:hq + hkv].transpose(0, 1), x[:, hq + hkv:].transpose(0, 1)
        elif case["layout"] == "tokens" or case["layout"] == "qkv":
            q = _randn(g, (t, hq, D), dtype)
            k, v = (_randn(g, (tk, hkv, D), dtype).transpose(0, 1) for _ in range(2))
        else:
            q = _randn(g, (hq, t, D), dtype).transpose(0, 1)
            k, v = (_randn(g, (hkv, tk, D), dtype) for _ in range(2))
        cu_q = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        both = [a + b for a, b in zip(lens, past)]
        cu_k = torch.tensor([sum(both[:i]) for i in range(len(both) + 1)], dtype=torch.int32, device="cuda")
        return dict(case=case, q=q, k=k, v=v, cu_q=cu_q, cu_k=cu_k if t != tk else None, lens=lens, both=both)
    if case["op"] == "append":
        hkv, rows = case["hkv"], case["rows"]
        cap = case["offset"] + rows + 129
        cap += cap & 1
        slab = torch.zeros((2, hkv, cap, ROW), dtype=torch.uint8, device="cuda")
        k = _kv_rows(g, (hkv, rows, D))
        v = _kv_rows(g, (hkv, rows, D))
        return dict(case=case, slab=slab, k=k, v=v)
    hq, hkv, n = case["hq"], case["hkv"], case["nodes"]
    total = case["prefix"] + n
    cap = total + 130
    cap += cap & 1
    # rows behind the tree hold what earlier rounds left there
    slab = torch.randint(0, 256, (2, hkv, cap, ROW), dtype=torch.uint8, device="cuda", generator=g)
    for i in range(2):
        for h in range(hkv):
            slab[i, h, :total] = _pack(_kv_rows(g, (1, total, D)))[0]
    q = _randn(g, (n, hq, D), torch.bfloat16)
    # a random tree: parents come before children, each node sees itself and its ancestors
    parent = (torch.rand(n, device="cuda", generator=g) * torch.arange(n, device="cuda")).long().tolist()
    see = []
    for i in range(n):
        see.append((see[parent[i]] if i else 0) | (1 << i))
    words = (n + 31) // 32
    bits = torch.tensor([[(s >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for s in see], dtype=torch.int64)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32).cuda()
    return dict(case=case, slab=slab, q=q, bits=bits)


# ----------------------------------------------------------------------------- plain form
def _quant(x):
    """Codes [.., 4, 32], zero points and scales [.., 4, 1] of rows [.., 128], in 32 bits."""
    y = x.float().unflatten(-1, (D // GROUP, GROUP))
    lo = y.amin(-1, keepdim=True).clamp(max=0.0)
    hi = y.amax(-1, keepdim=True).clamp(min=0.0)
    # in 64 bits: a quotient of 4 significant bits must come out as itself, not a step above
    s = ((hi - lo).double() / 15.0).float()
    # up to 4 significant bits, 0 below the smallest normal number
    s = ((s.view(torch.int32) + 0xFFFFF) & ~0xFFFFF).view(torch.float32)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    d = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.where(s > 0, torch.round(-lo / d), torch.zeros_like(s))
    u = torch.where(s > 0, (torch.round(y / d) + z).clamp(0, 15), torch.zeros_like(y))
    return u, z, s


def _pack(x):
    """4-bit rows [.., 72] of rows [.., 128]."""
    u, z, s = _quant(x)
    c = u.to(torch.uint8).flatten(-2).unflatten(-1, (D // 8, 8))[..., list(ORDER)]
    codes = c[..., 0::2] | (c[..., 1::2] << 4)
    word = (((s.view(torch.int32) >> 16) & 0x7FF0) | z.to(torch.int32)).squeeze(-1)
    meta = torch.stack([word & 0xFF, word >> 8], dim=-1).to(torch.uint8)
    return torch.cat([codes.flatten(-2), meta.flatten(-2)], dim=-1)


def _unpack(rows):
    """Values [.., 128] in 32 bits of 4-bit rows [.., 72]."""
    codes = rows[..., :64].unflatten(-1, (16, 4))
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    u = torch.empty_like(c)
    u[..., list(ORDER)] = c
    u = u.flatten(-2).unflatten(-1, (D // GROUP, GROUP)).float()
    m = rows[..., 64:].unflatten(-1, (4, 2)).to(torch.int32)
    word = m[..., 0] | (m[..., 1] << 8)
    s = ((word & 0x7FF0) << 16).view(torch.float32).unsqueeze(-1)
    z = (word & 15).float().unsqueeze(-1)
    return ((u - z) * s).flatten(-2)


def _attend(q, k, v, see, scale):
    """softmax(q k^T scale) v over the visible keys; rows without one are zero.  [.., n, D] x [.., m, D]."""
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    if see is not None:
        s = s.masked_fill(~see, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp2((s - top) * LOG2E)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_prompt(st):
    q, k, v = st["q"], st["k"], st["v"]
    hq, hkv = q.shape[1], k.shape[0]
    out = torch.empty((q.shape[0], hq, D), dtype=q.dtype, device=q.device)
    a = b = 0
    for lq, lk in zip(st["lens"], st["both"]):
        see = torch.arange(lk, device=q.device)[None, :] <= torch.arange(lq, device=q.device)[:, None] + (lk - lq)
        for h in range(hkv):
            grp = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            o = _attend(q[a:a + lq, grp].transpose(0, 1).float(), k[h, b:b + lk].float(), v[h, b:b + lk].float(), see,
                        D ** -0.5)
            out[a:a + lq, grp] = o.transpose(0, 1).to(q.dtype)
        a += lq
        b += lk
    return out


def _plain_append(st):
    c, slab = st["case"], st["slab"]
    for i, x in enumerate((st["k"], st["v"])):
        slab[i, :, c["offset"]:c["offset"] + c["rows"]] = _pack(x)
    return _unpack(slab[:, :, c["offset"]:c["offset"] + c["rows"]]).to(torch.bfloat16)


def _plain_verify(st):
    c, q, slab = st["case"], st["q"], st["slab"]
    n, hq = q.shape[:2]
    hkv = slab.shape[1]
    grp, total = hq // hkv, c["prefix"] + n
    j = torch.arange(n, device=q.device)
    tree = ((st["bits"][:, j // 32] >> (j % 32)) & 1).bool()
    see = torch.cat([torch.ones((n, c["prefix"]), dtype=torch.bool, device=q.device), tree], 1)
    out = torch.empty((n, hq, D), dtype=torch.bfloat16, device=q.device)
    for h in range(hkv):
        k, v = _unpack(slab[0, h, :total]), _unpack(slab[1, h, :total])
        o = _attend(q[:, h * grp:(h + 1) * grp].transpose(0, 1).float(), k, v, see, D ** -0.5)
        out[:, h * grp:(h + 1) * grp] = o.transpose(0, 1).to(torch.bfloat16)
    return out


# ----------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append, "verify": _plain_verify}[op](state)
    from retree_b200 import kernels
    if op == "prompt":
        return kernels.prompt_attention(state["q"], state["k"], state["v"], cu_seqlens_q=state["cu_q"],
                                        cu_seqlens_k=state["cu_k"])
    slab, case = state["slab"], state["case"]
    if op == "append":
        kernels.kv_append_q4(slab[0], slab[1], state["k"], state["v"], offset=case["offset"])
        return kernels.kv_read_q4(slab, case["offset"], case["rows"])
    return kernels.tree_attention_q4(state["q"], slab[0], slab[1], state["bits"], case["prefix"])


# ----------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["op"] == "prompt":
        lens, past = _lens(case)
        t, tk = sum(lens), sum(lens) + sum(past)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, past))
        return {"bytes": 2 * D * (2 * t * case["hq"] + 2 * tk * case["hkv"]), "flops": 4 * D * case["hq"] * pairs}
    if case["op"] == "append":
        rows = 2 * case["rows"] * case["hkv"]
        return {"bytes": rows * (2 * D + ROW) + rows * (ROW + 2 * D), "flops": rows * D * 8}
    n, keys = case["nodes"], case["prefix"] + case["nodes"]
    return {"bytes": 2 * keys * case["hkv"] * ROW + 4 * D * n * case["hq"] + 4 * n * ((n + 31) // 32),
            "flops": 4 * D * case["hq"] * n * (case["prefix"] + 1)}


# ----------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_softmax_rows(q, k, v, visible):
    """Row by row of a block of queries [r, D]: sum over visible keys, float64."""
    s = (q @ k.T) / D ** 0.5
    w = torch.exp(s - torch.where(visible, s, -torch.inf).max(1, keepdim=True).values.nan_to_num(neginf=0.0))
    w = w * visible
    z = w.sum(1, keepdim=True)
    return (w @ v) / torch.where(z == 0, 1.0, z)


def _exact_values(rows):
    """float64 values of 4-bit rows, code by code from the layout's definition."""
    r = rows.to(torch.int64)
    out = torch.empty(r.shape[:-1] + (D,), dtype=torch.float64, device=r.device)
    for d in range(D):
        j = ORDER.index(d % 8)
        byte = r[..., 4 * (d // 8) + j // 2]
        word = r[..., 64 + 2 * (d // GROUP)] + 256 * r[..., 65 + 2 * (d // GROUP)]
        scale = (1 + ((word >> 4) & 7).double() / 8) * torch.pow(2.0, ((word >> 7) & 255).double() - 127)
        scale = torch.where(((word >> 7) & 255) == 0, 0.0, scale)
        out[..., d] = (((byte >> (4 * (j % 2))) & 15) - (word & 15)).double() * scale
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "prompt":
        q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
        hq, hkv = case["hq"], case["hkv"]
        out = torch.zeros((q.shape[0], hq, D), dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for lq, lk in zip(st["lens"], st["both"]):
            for i0 in range(0, lq, 2048):
                i1 = min(lq, i0 + 2048)
                last = torch.arange(i0, i1, device="cuda") + (lk - lq)
                visible = torch.arange(lk, device="cuda")[None] <= last[:, None]
                for h in range(hq):
                    g = h // (hq // hkv)
                    out[q0 + i0:q0 + i1, h] = _exact_softmax_rows(q[q0 + i0:q0 + i1, h], k[g, k0:k0 + lk],
                                                                  v[g, k0:k0 + lk], visible)
            q0, k0 = q0 + lq, k0 + lk
        return out
    if case["op"] == "append":
        x = torch.stack([st["k"], st["v"]]).double()
        out = torch.empty_like(x)
        for g0 in range(0, D, GROUP):
            part = x[..., g0:g0 + GROUP]
            low = torch.minimum(part.min(-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device="cuda"))
            high = torch.maximum(part.max(-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device="cuda"))
            step = (high - low) / 15
            mant, expo = torch.frexp(step)
            step = torch.ldexp(torch.ceil(mant * 16) / 16, expo)
            step = torch.where(step < 2.0 ** -126, 0.0, step)
            safe = torch.where(step == 0, 1.0, step)
            zero = torch.round(-low / safe)
            code = torch.clamp(torch.round(part / safe) + zero, 0, 15)
            out[..., g0:g0 + GROUP] = (code - zero) * step
        return out
    n, hq, hkv, total = case["nodes"], case["hq"], case["hkv"], case["prefix"] + case["nodes"]
    bits = st["bits"].to(torch.int64) & 0xFFFFFFFF
    visible = torch.ones((n, total), dtype=torch.bool, device="cuda")
    for t in range(n):
        visible[:, case["prefix"] + t] = ((bits[:, t // 32] >> (t % 32)) & 1) == 1
    out = torch.empty((n, hq, D), dtype=torch.float64, device="cuda")
    for g in range(hkv):
        k, v = _exact_values(st["slab"][0, g, :total]), _exact_values(st["slab"][1, g, :total])
        for h in range(g * (hq // hkv), (g + 1) * (hq // hkv)):
            out[:, h] = _exact_softmax_rows(st["q"][:, h].double(), k, v, visible)
    return out
