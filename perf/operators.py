"""The decoder operators of ``siliconed_b200.lm_abi`` as measurable cases: inputs, the calls, plain forms, exact values.

A text encoder or prompt writer that decodes on 8-bit weights runs, per layer: the residual addition, RMS norm and
quantization to e4m3 in blocks of 128 ("norm"); the product of such codes with a weight quantized in blocks of 128 x 128
("linear"); the QK-norm, position rotation and append to the paged key-value cache ("append"); and the attention of one
new token over that cache ("attention").  ``own`` chooses between the framework's calls and the plain torch forms.
"""
import math

import torch

own = False

BLOCK = 128          # values under one quantization scale
E4M3_MAX = 448.0
FLOOR = 1e-30        # smallest scale of a block
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # One new token of one request, a small encoder's width: latency alone.
        {"name": "norm-1x2560", "op": "norm", "rows": 1, "d": 2560, "stream": "bf16", "delta": "bf16"},
        # A decode batch with an odd count of requests, fp32 residual stream as the DiT blocks keep it.
        {"name": "norm-37x4096", "op": "norm", "rows": 37, "d": 4096, "stream": "f32", "delta": "bf16"},
        # A long prompt of config 3's token count and width.
        {"name": "norm-4608x3840", "op": "norm", "rows": 4608, "d": 3840, "stream": "f32", "delta": "f32"},
        # Sixteen requests, one new token each, grouped heads, small pages.
        {"name": "append-decode16", "op": "append", "seqs": 16, "per_seq": 1, "max_pos": 2048, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "kv": "bf16", "pairs": "halves", "norm": True},
        # Prompts of several requests, appended in one call to an 8-bit cache.
        {"name": "append-prompt", "op": "append", "seqs": 9, "per_seq": 517, "max_pos": 1024, "heads": 30, "kv_heads": 6,
         "head_dim": 128, "page": 64, "kv": "e4m3", "pairs": "adjacent", "norm": True},
        # One request, a short context: the smallest decode step's attention.
        {"name": "attention-1x513", "op": "attention", "batch": 1, "max_len": 513, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "kv": "bf16", "ragged": False},
        # A serving batch of ragged contexts, one request still empty.
        {"name": "attention-33-ragged", "op": "attention", "batch": 33, "max_len": 4400, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "kv": "bf16", "ragged": True},
        # One request with a very long context.
        {"name": "attention-1x131072", "op": "attention", "batch": 1, "max_len": 131072, "heads": 32, "kv_heads": 4,
         "head_dim": 128, "page": 64, "kv": "bf16", "ragged": False},
        # A large batch over an 8-bit cache.
        {"name": "attention-64-e4m3", "op": "attention", "batch": 64, "max_len": 8192, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "kv": "e4m3", "ragged": True},
        # Config 4's decode weight at one and at sixteen rows.
        {"name": "linear-1x12288x4096", "op": "linear", "m": 1, "n": 12288, "k": 4096, "bias": False},
        # The text encoder's prefill product, a row count that fills no tile.
        {"name": "linear-131x9728x2560", "op": "linear", "m": 131, "n": 9728, "k": 2560, "bias": True},
        # Config 2's shape: compute-bound.
        {"name": "linear-4096x10240x3840", "op": "linear", "m": 4096, "n": 10240, "k": 3840, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "append", "attention", "linear"])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 4608), "d": 16 * _log(rng, 8, 240), "stream": rng.choice(["bf16", "f32"]),
                "delta": rng.choice(["bf16", "f32", "none"])}
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
    if op == "append":
        decode = rng.random() < 0.5
        return {"op": op, "seqs": _log(rng, 1, 64) if decode else rng.randint(1, 8), "per_seq": 1 if decode else _log(rng, 2, 500),
                "max_pos": rng.randint(500, 1500), "heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128]),
                "page": rng.choice([8, 16, 24, 64]), "kv": rng.choice(["bf16", "e4m3"]), "pairs": rng.choice(["adjacent", "halves"]),
                "norm": rng.random() < 0.7}
    if op == "attention":
        batch = _log(rng, 1, 64)
        return {"op": op, "batch": batch, "max_len": _log(rng, 1, min(131072, 262144 // batch)), "heads": heads,
                "kv_heads": kv_heads, "head_dim": rng.choice([64, 128]), "page": rng.choice([8, 16, 24, 64]),
                "kv": rng.choice(["bf16", "e4m3"]), "ragged": rng.random() < 0.7}
    while True:
        m, n, k = _log(rng, 1, 4096), _log(rng, 200, 12288), 16 * _log(rng, 8, 768)
        if m * n * k <= 4096 * 10240 * 3840:
            return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5}


def _spread(i, n, top):
    """The i-th of n whole numbers spread over [0, top] (golden-ratio steps, the first one the top)."""
    return top if i == 0 else int(top * ((i * 0.6180339887498949) % 1.0))


def _lengths(case):
    """Context lengths of an attention case: all the longest, or ragged with one empty request among four or more."""
    b = case["batch"]
    if not case["ragged"]:
        return [case["max_len"]] * b
    lens = [max(1, _spread(i, b, case["max_len"])) for i in range(b)]
    if b >= 4:
        lens[b // 2] = 0
    return lens


def _spans(case):
    """(first position, token count) of each sequence of an append case."""
    out = []
    for i in range(case["seqs"]):
        if case["per_seq"] == 1:
            out.append((_spread(i, case["seqs"], case["max_pos"] - 1), 1))
        else:
            n = max(1, _spread(i, case["seqs"], case["per_seq"]))
            out.append((_spread(i + 1, case["seqs"], case["max_pos"] - n), n))
    return out


def work(case):
    op = case["op"]
    if op == "norm":
        rows, d = case["rows"], case["d"]
        size = {"bf16": 2, "f32": 4, "none": 0}
        moved = size[case["stream"]] * (2 if case["delta"] != "none" else 1) + size[case["delta"]] + 1
        blocks = -(-d // BLOCK)
        return {"bytes": rows * d * moved + 4 * d + 4 * rows * blocks, "flops": 6 * rows * d}
    if op == "append":
        t = sum(n for _, n in _spans(case))
        h, hk, dim = case["heads"], case["kv_heads"], case["head_dim"]
        kv = 2 if case["kv"] == "bf16" else 1
        scales = 0 if case["kv"] == "bf16" else 8 * t * hk
        return {"bytes": t * dim * (2 * (h + 2 * hk) + 2 * h + 2 * kv * hk) + scales + t * dim * 4 + 8 * t,
                "flops": t * dim * (h + hk) * (6 if case["norm"] else 3)}
    if op == "attention":
        total, b = sum(_lengths(case)), case["batch"]
        h, hk, dim = case["heads"], case["kv_heads"], case["head_dim"]
        per = 4 * dim if case["kv"] == "bf16" else 2 * dim + 8
        return {"bytes": total * hk * per + 4 * (total // case["page"] + b) + b * h * (4 * dim + 4), "flops": 4 * total * h * dim}
    m, n, k = case["m"], case["n"], case["k"]
    kb, nb = -(-k // BLOCK), -(-n // BLOCK)
    return {"bytes": m * k + n * k + 4 * (m * kb + nb * kb) + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _pages(g, seqs, max_pos, page):
    """(page table [seqs, width] int32, page count): every sequence's pages at random places of the pool."""
    width = -(-max_pos // page)
    count = seqs * width + 3
    return torch.randperm(count, generator=g, device="cuda")[: seqs * width].to(torch.int32).view(seqs, width).contiguous(), count


def _cache(g, case, count):
    """k and v caches [pages, kv_heads, page, head_dim], with scales [pages, kv_heads, page] where they are e4m3."""
    shape = (count, case["kv_heads"], case["page"], case["head_dim"])
    if case["kv"] == "bf16":
        return {"k_cache": _randn(g, *shape, dtype=torch.bfloat16), "v_cache": _randn(g, *shape, dtype=torch.bfloat16),
                "k_scale": None, "v_scale": None}
    out = {}
    for name in ("k", "v"):
        x = torch.randn(*shape, generator=g, device="cuda")
        s = (x.abs().amax(-1) / E4M3_MAX).clamp_min(FLOOR)
        out[name + "_cache"], out[name + "_scale"] = _e4m3(x / s.unsqueeze(-1)), s
    return out


def prepare(case, seed):
    g = _gen(seed)
    types = {"bf16": torch.bfloat16, "f32": torch.float32}
    op = case["op"]
    st = {"op": op}
    if op == "norm":
        rows, d = case["rows"], case["d"]
        # a residual stream with a few massive channels, as trained decoders have them
        gain = torch.where(torch.rand(d, generator=g, device="cuda") < 0.004, 30.0, 1.0)
        st["x"] = (torch.randn(rows, d, generator=g, device="cuda") * gain).to(types[case["stream"]])
        st["delta"] = None if case["delta"] == "none" else _randn(g, rows, d, dtype=types[case["delta"]], scale=0.5)
        st["weight"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        st["x_out"] = torch.empty_like(st["x"])
        st["codes"] = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device="cuda")
        st["scales"] = torch.empty(rows, -(-d // BLOCK), device="cuda")
        return st
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        x = torch.randn(m, kb * BLOCK, generator=g, device="cuda")
        x[:, k:] = 0
        s = (x.view(m, kb, BLOCK).abs().amax(-1) / E4M3_MAX).clamp_min(FLOOR)
        st["codes"] = _e4m3(x.view(m, kb, BLOCK) / s.unsqueeze(-1)).view(torch.uint8).view(m, kb * BLOCK)[:, :k].contiguous() \
            .view(torch.float8_e4m3fn)
        st["scales"] = s
        w = torch.randn(nb * BLOCK, kb * BLOCK, generator=g, device="cuda") * 0.02
        w[n:] = 0
        w[:, k:] = 0
        w = w.view(nb, BLOCK, kb, BLOCK)
        ws = (w.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(FLOOR)
        st["weight"] = _e4m3(w / ws[:, None, :, None]).view(torch.uint8).view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous() \
            .view(torch.float8_e4m3fn)
        st["weight_scales"] = ws
        st["bias"] = _randn(g, n, dtype=torch.bfloat16, scale=0.1) if case["bias"] else None
        st["out"] = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        return st
    dim, heads, kv_heads = case["head_dim"], case["heads"], case["kv_heads"]
    if op == "append":
        spans = _spans(case)
        st["table"], count = _pages(g, case["seqs"], case["max_pos"], case["page"])
        st |= _cache(g, case, count)
        seq = [i for i, (_, n) in enumerate(spans) for _ in range(n)]
        pos = [p + j for p, n in spans for j in range(n)]
        st["seq"] = torch.tensor(seq, dtype=torch.int32, device="cuda")
        st["positions"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
        st["qkv"] = _randn(g, len(seq), (heads + 2 * kv_heads) * dim, dtype=torch.bfloat16)
        inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        ang = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * inv
        st["freqs"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        st["norm_q"] = 1.0 + 0.1 * torch.randn(dim, generator=g, device="cuda") if case["norm"] else None
        st["norm_k"] = 1.0 + 0.1 * torch.randn(dim, generator=g, device="cuda") if case["norm"] else None
        st["q"] = torch.empty(len(seq), heads, dim, dtype=torch.bfloat16, device="cuda")
        st["heads"], st["kv_heads"], st["pairs"] = heads, kv_heads, case["pairs"]
        return st
    st["table"], count = _pages(g, case["batch"], case["max_len"], case["page"])
    st |= _cache(g, case, count)
    st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    st["q"] = _randn(g, case["batch"], heads, dim, dtype=torch.bfloat16, scale=2.0)
    st["scale"] = 1.0 / math.sqrt(dim)
    st["out"] = torch.empty_like(st["q"])
    st["lse"] = torch.empty(case["batch"], heads, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _own_norm(st):
    from siliconed_b200 import lm_abi
    out = st["x"] if st["delta"] is None else st["x_out"]
    lm_abi.rms_norm_quantize(st["x"], st["delta"], st["weight"], EPS, out, st["codes"], st["scales"])
    return {"x": out, "codes": st["codes"], "scales": st["scales"]}


def _own_append(st):
    from siliconed_b200 import lm_abi
    lm_abi.append_paged(st["qkv"], st["heads"], st["kv_heads"], st["norm_q"], st["norm_k"], EPS, st["freqs"], st["pairs"],
                        st["seq"], st["positions"], st["table"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"],
                        st["q"])
    return _appended(st, st["q"])


def _own_attention(st):
    from siliconed_b200 import lm_abi
    lm_abi.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["table"], st["lengths"],
                           st["scale"], st["out"], st["lse"])
    return {"out": st["out"], "lse": st["lse"]}


def _own_linear(st):
    from siliconed_b200 import lm_abi
    return lm_abi.linear_block_fp8(st["codes"], st["scales"], st["weight"], st["weight_scales"], st["bias"], st["out"])


_own = {"norm": _own_norm, "append": _own_append, "attention": _own_attention, "linear": _own_linear}


def _appended(st, q):
    out = {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if st["k_scale"] is not None:
        out |= {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    return out


def _quantize(y):
    """(codes, scales) of fp32 rows [..., d] in blocks of 128 along the last axis."""
    d = y.shape[-1]
    padded = torch.nn.functional.pad(y, (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))
    s = (padded.abs().amax(-1) / E4M3_MAX).clamp_min(FLOOR)
    return _e4m3(padded / s.unsqueeze(-1)).view(torch.uint8).flatten(-2)[..., :d].contiguous().view(torch.float8_e4m3fn), s


def _plain_norm(st):
    x = st["x"].float()
    if st["delta"] is not None:
        x = x + st["delta"].float()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * st["weight"]
    codes, scales = _quantize(y)
    return {"x": x.to(st["x"].dtype), "codes": codes, "scales": scales}


def _rotate(x, cs, pairs):
    """x [tokens, heads, dim] rotated by cs [tokens, dim / 2, 2], on adjacent pairs or on the two halves."""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if pairs == "adjacent":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_append(st):
    t, h, hk = st["qkv"].shape[0], st["heads"], st["kv_heads"]
    rows = st["qkv"].float().view(t, h + 2 * hk, -1)
    q, k, v = rows.split([h, hk, hk], 1)
    if st["norm_q"] is not None:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * st["norm_q"]
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * st["norm_k"]
    pos = st["positions"].long()
    cs = st["freqs"][pos]
    q, k = _rotate(q, cs, st["pairs"]), _rotate(k, cs, st["pairs"])
    size = st["k_cache"].shape[2]
    page, slot = st["table"].long()[st["seq"].long(), pos // size], pos % size
    if st["k_scale"] is None:
        st["k_cache"][page, :, slot] = k.to(torch.bfloat16)
        st["v_cache"][page, :, slot] = v.to(torch.bfloat16)
    else:
        ks = (k.abs().amax(-1) / E4M3_MAX).clamp_min(FLOOR)
        vs = (v.abs().amax(-1) / E4M3_MAX).clamp_min(FLOOR)
        st["k_cache"].view(torch.uint8)[page, :, slot] = _e4m3(k / ks.unsqueeze(-1)).view(torch.uint8)
        st["v_cache"].view(torch.uint8)[page, :, slot] = _e4m3(v / vs.unsqueeze(-1)).view(torch.uint8)
        st["k_scale"][page, :, slot] = ks
        st["v_scale"][page, :, slot] = vs
    return _appended(st, q.to(torch.bfloat16))


def _plain_attention(st):
    table = st["table"].long()
    b, h, dim = st["q"].shape
    hk = st["k_cache"].shape[1]

    def rows(cache, scale):
        """[batch, kv_heads, width * page, dim] in fp32."""
        x = cache.view(torch.uint8)[table].view(cache.dtype).float() if scale is not None else cache[table].float()
        if scale is not None:
            x = x * scale[table].unsqueeze(-1)
        return x.transpose(1, 2).flatten(2, 3)

    k = rows(st["k_cache"], st["k_scale"])
    valid = torch.arange(k.shape[2], device="cuda") < st["lengths"].long()[:, None]
    scores = torch.matmul(st["q"].float().view(b, hk, h // hk, dim), k.transpose(-1, -2)) * st["scale"]
    scores = scores.masked_fill(~valid[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    del k, scores
    total = p.sum(-1, keepdim=True)
    v = rows(st["v_cache"], st["v_scale"]) * valid[:, None, :, None]
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = top.squeeze(-1) + torch.log(total.squeeze(-1))
    lse = torch.where(total.squeeze(-1) == 0, -math.inf, lse)
    return {"out": out.reshape(b, h, dim).to(torch.bfloat16), "lse": lse.reshape(b, h)}


def _plain_linear(st):
    m, k = st["codes"].shape
    n = st["weight"].shape[0]
    a = st["codes"].float() * st["scales"].repeat_interleave(BLOCK, 1)[:, :k]
    ws = st["weight_scales"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = torch.matmul(a, (st["weight"].float() * ws).t())
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(torch.bfloat16)


_plain = {"norm": _plain_norm, "append": _plain_append, "attention": _plain_attention, "linear": _plain_linear}


# ------------------------------------------------------------------------------------------------ exact values

def exact(case, seed):
    """The definitions in 64 bits.  Values held in 8 bits are given before their rounding to 8 bits."""
    st = prepare(case, seed)
    return _exact[case["op"]](st)


def _block_scale(y):
    return torch.clamp(torch.amax(torch.abs(y), dim=-1) / E4M3_MAX, min=FLOOR)


def _exact_norm(st):
    x = st["x"].double()
    if st["delta"] is not None:
        x = x + st["delta"].double()
    rms = torch.rsqrt(x.square().sum(1) / x.shape[1] + EPS)
    y = x * rms[:, None] * st["weight"].double()
    scales = torch.stack([_block_scale(part) for part in y.split(BLOCK, 1)], 1)
    codes = torch.cat([part / scales[:, i, None] for i, part in enumerate(y.split(BLOCK, 1))], 1)
    return {"x": x, "codes": codes, "scales": scales}


def _exact_append(st):
    h, hk = st["heads"], st["kv_heads"]
    dim = st["k_cache"].shape[3]
    tokens = st["qkv"].shape[0]
    rows = st["qkv"].double().reshape(tokens, h + 2 * hk, dim)
    angle = st["freqs"].double()[st["positions"].long()]
    turn = torch.complex(angle[..., 0], angle[..., 1])[:, None, :]

    def turned(x, norm):
        if norm is not None:
            x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / dim + EPS) * norm.double()
        if st["pairs"] == "adjacent":
            return torch.view_as_real(torch.view_as_complex(x.reshape(tokens, -1, dim // 2, 2).contiguous()) * turn).reshape(x.shape)
        z = torch.complex(x[..., : dim // 2].contiguous(), x[..., dim // 2:].contiguous()) * turn
        return torch.cat((z.real, z.imag), dim=2)

    q, k, v = turned(rows[:, :h], st["norm_q"]), turned(rows[:, h:h + hk], st["norm_k"]), rows[:, h + hk:]
    size = st["k_cache"].shape[2]
    where, pos = st["table"][st["seq"].long(), (st["positions"] // size).long()].long(), (st["positions"] % size).long()
    out = {"q": q, "k_cache": st["k_cache"].double(), "v_cache": st["v_cache"].double()}
    if st["k_scale"] is not None:
        out["k_scale"], out["v_scale"] = st["k_scale"].double(), st["v_scale"].double()
    for name, x in (("k", k), ("v", v)):
        if st["k_scale"] is not None:
            s = _block_scale(x)
            out[name + "_scale"][where, :, pos] = s
            x = x / s[..., None]
        out[name + "_cache"][where, :, pos] = x
    return out


def _exact_attention(st):
    b, h, dim = st["q"].shape
    hk, size = st["k_cache"].shape[1], st["k_cache"].shape[2]
    out = torch.zeros(b, h, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device="cuda")
    for i, length in enumerate(st["lengths"].tolist()):
        if length == 0:
            continue
        t = torch.arange(length, device="cuda")
        page, slot = st["table"][i].long()[t // size], t % size
        for j in range(hk):
            k, v = (st[c + "_cache"].view(torch.uint8 if st["k_scale"] is not None else torch.bfloat16)[page, j, slot]
                    .view(st[c + "_cache"].dtype).double() for c in "kv")
            if st["k_scale"] is not None:
                k, v = k * st["k_scale"][page, j, slot].double()[:, None], v * st["v_scale"][page, j, slot].double()[:, None]
            group = slice(j * (h // hk), (j + 1) * (h // hk))
            s = st["q"][i, group].double() @ k.t() * st["scale"]
            out[i, group] = torch.softmax(s, -1) @ v
            lse[i, group] = torch.logsumexp(s, -1)
    return {"out": out, "lse": lse}


def _exact_linear(st):
    m, k = st["codes"].shape
    n = st["weight"].shape[0]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for i, at in enumerate(range(0, k, BLOCK)):
        part = st["codes"][:, at:at + BLOCK].double() @ st["weight"][:, at:at + BLOCK].double().t()
        spread = st["weight_scales"][:, i].double().repeat_interleave(BLOCK)[:n]
        y += part * st["scales"][:, i, None].double() * spread
    return y if st["bias"] is None else y + st["bias"].double()


_exact = {"norm": _exact_norm, "append": _exact_append, "attention": _exact_attention, "linear": _exact_linear}
