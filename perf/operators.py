"""Cases of three families of operators: attention over packed documents, embedding rows with their gradient, and AdamW over
many tensors at once.  `run` computes them with elementary torch operations, or (`own`) through this package's entry points."""
import math
import random

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SMALLEST_NORMAL = 2.0 ** -126
BLOCK = 256                      # elements that share a scale in the 8-bit states


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    docs = dict(op="docs", causal=False, prefix=False, cap=0.0, bias=False, train=False, queries="self", kv_heads=8, heads=8, dim=96)
    embed = dict(op="embed", rows=16384, width=768, scale=1.0, train=True)
    adam = dict(op="adamw", bits=8, clip=1.0, grad16=False)
    return [
        # one prompt and the empty one of classifier-free guidance, one layer of the text encoder: latency alone
        dict(docs, name="docs_prompt", docs=2, shortest=2, longest=17, mix=1),
        # a training batch of captions without padding rows: a few dozen tokens each, at most 77
        dict(docs, name="docs_captions_train", docs=1920, shortest=3, longest=77, mix=2, train=True),
        # long documents with a prefix that sees itself whole, capped scores, a distance bias, shared key heads
        dict(docs, name="docs_long_prefix_train", docs=4, shortest=4001, longest=8191, mix=3, train=True, causal=True, prefix=True,
             cap=30.0, bias=True, kv_heads=2, dim=64),
        # image tokens of one denoiser level over each image's own caption
        dict(docs, name="docs_image_text_train", docs=8, shortest=5, longest=77, mix=4, train=True, queries="image", per_doc=4096, dim=40),
        # one query for each document over everything that the document holds
        dict(docs, name="docs_single_query", docs=48, shortest=900, longest=16000, mix=5, queries="single", causal=True, bias=True,
             kv_heads=2, dim=96),
        # the lookup of one prompt
        dict(embed, name="embed_prompt", tokens=77, train=False),
        # rows and the table's gradient for a small training batch of captions
        dict(embed, name="embed_batch_train", tokens=1601),
        # the same for a large one; a few ids make up most of it
        dict(embed, name="embed_large_train", tokens=262143, scale=768 ** 0.5),
        # low-rank adapters of every attention projection: many small tensors
        dict(adam, name="adamw8_adapters", params="adapters", width=320, layers=16),
        # the whole text encoder, states in 8 bits
        dict(adam, name="adamw8_encoder", params="encoder", width=768, layers=8),
        # the same with states in 32 bits, no clipping
        dict(adam, name="adamw32_encoder", params="encoder", width=768, layers=8, bits=32, clip=0.0),
        # convolution and projection weights of a denoiser, gradients as the all-reduce leaves them
        dict(adam, name="adamw8_denoiser", params="denoiser", width=320, layers=2, grad16=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    largest = {c["op"]: max(_cost(x) for x in listed() if x["op"] == c["op"]) for c in listed()}
    op = rng.choice(("docs", "docs", "docs", "embed", "adamw"))
    while True:
        if op == "docs":
            queries = rng.choice(("self", "self", "image", "single"))
            kv = rng.choice((1, 2, 4, 8))
            c = dict(op=op, queries=queries, heads=kv * rng.choice((1, 1, 2, 3, 4)), kv_heads=kv, dim=8 * rng.randint(3, 16), mix=rng.randint(0, 1 << 20),
                     causal=queries != "image" and rng.random() < 0.5, cap=rng.choice((0.0, 0.0, 15.0, 50.0)), bias=rng.random() < 0.4,
                     train=queries != "single" and rng.random() < 0.6)
            c["prefix"] = c["causal"] and rng.random() < 0.5
            c["longest"] = _log(rng, 2, 16000 if queries == "single" else 77 if queries == "image" else 8191)
            c["shortest"] = rng.randint(0, c["longest"])
            c["docs"] = _log(rng, 1, 2000 if c["longest"] < 100 else 48)
            if queries == "image":
                c["per_doc"] = _log(rng, 16, 4096)
            fits = c["docs"] * c["longest"] * (c["longest"] if queries == "self" else c.get("per_doc", 1)) * c["heads"] <= 4 * 8 * 8191 ** 2
        elif op == "embed":
            c = dict(op=op, rows=_log(rng, 300, 130000), width=rng.choice((8 * rng.randint(4, 160), rng.randint(33, 1280))), tokens=_log(rng, 1, 262143),
                     scale=rng.choice((1.0, 27.7, 0.125)), train=rng.random() < 0.75)
            fits = c["rows"] * c["width"] <= 1 << 26
        else:
            c = dict(op=op, params=rng.choice(("adapters", "encoder", "denoiser", "odd")), width=8 * rng.randint(16, 96), layers=rng.randint(1, 8),
                     bits=rng.choice((8, 8, 32)), clip=rng.choice((0.0, 1.0, 0.05)), grad16=rng.random() < 0.4)
            fits = True
        if fits and _cost(c) <= largest[op]:
            return c


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


# ------------------------------------------------------------------------------------------------------------------
# attention over packed documents.  Row i of document n sits at position c = i - q_end + k_end (its last row over its last
# key) and sees the keys j of the same document with j <= c or j < k_begin + prefix[n] (causal), or all of them:
#   s = scale q k;  s = cap tanh(s / cap);  s -= slope[head] |c - j|;  out = softmax(s) v;  a row that sees nothing: 0
# ------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(queries, keys, prefix) of each document: many short ones, few long ones."""
    r = random.Random(case["mix"])
    lo, hi, n = case["shortest"], case["longest"], case["docs"]
    keys = [lo + int((hi - lo) * r.random() ** 1.7 + 0.5) for _ in range(n)]
    keys[0], keys[-1] = hi, (lo if n > 1 else hi)
    queries = {"self": keys, "image": [case.get("per_doc", 0)] * n, "single": [1] * n}[case["queries"]]
    return queries, keys, [int(k * r.random() * 0.5) for k in keys]


def _pairs(case):
    total = 0
    for lq, lk, pre in zip(*_lengths(case)):
        if not case["causal"]:
            total += lq * lk
        elif lq:
            lq = min(lq, lk) if not (case["prefix"] and pre) else lq
            first = lk - lq + 1                              # keys that the first row sees, then one more each
            total += lq * first + lq * (lq - 1) // 2
            if case["prefix"]:
                short = max(0, min(lq, pre - first))         # rows that see less than the prefix
                total += short * (pre - first) - short * (short - 1) // 2
    return total * case["heads"]


def _docs_prepare(case, g):
    queries, keys, pre = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    tq, tk = sum(queries), sum(keys)
    offsets = lambda n: torch.tensor([0] + list(_running(n)), dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": case, "k_off": offsets(keys), "max_q": max(1, max(queries)), "max_k": max(1, max(keys)), "scale": d ** -0.5}
    if case["queries"] == "self":                            # one projection's output, as the encoder has it
        qkv = torch.randn(tk, (hq + 2 * hk) * d, generator=g, device="cuda").to(BF16)
        s["q"], s["k"], s["v"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        s["q_off"] = s["k_off"]
    else:
        kv = torch.randn(tk, 2 * hk * d, generator=g, device="cuda").to(BF16)
        s["q"] = torch.randn(tq, hq * d, generator=g, device="cuda").to(BF16)
        s["k"], s["v"], s["q_off"] = kv[:, :hk * d], kv[:, hk * d:], offsets(queries)
    s["prefix"] = torch.tensor(pre, dtype=torch.int32, device="cuda") if case["prefix"] else None
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=F32, device="cuda") if case["bias"] else None
    s["do"] = torch.randn(tq, hq * d, generator=g, device="cuda").to(BF16) if case["train"] else None
    return s


def _running(n):
    t = 0
    for x in n:
        t += x
        yield t


def _docs_own(s):
    from image_generator_amd import ops
    c = s["case"]
    how = dict(heads=c["heads"], kv_heads=c["kv_heads"], q_offsets=s["q_off"], k_offsets=s["k_off"], causal=c["causal"], prefix=s["prefix"],
               slopes=s["slopes"], cap=c["cap"], scale=s["scale"])
    out, lse = ops.doc_attention_fwd(s["q"], s["k"], s["v"], **how)
    if not c["train"]:
        return out
    dq, dk, dv = ops.doc_attention_bwd(s["do"], s["q"], s["k"], s["v"], out, lse, **how)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _docs_plain(s):
    c = s["case"]
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    grp, mq, mk, n = hq // hk, s["max_q"], s["max_k"], c["docs"]
    tq, tk = s["q"].shape[0], s["k"].shape[0]
    q_off, k_off = s["q_off"].long(), s["k_off"].long()
    iq = q_off[:-1, None] + torch.arange(mq, device="cuda")
    ik = k_off[:-1, None] + torch.arange(mk, device="cuda")
    okq, okk = iq < q_off[1:, None], ik < k_off[1:, None]

    def spread(x, at, ok, heads):                            # [rows, heads * d] -> [n, kv head, group * rows of the longest, d]
        x = torch.cat((x.float(), x.new_zeros(1, x.shape[1], dtype=F32)))[torch.where(ok, at, x.shape[0])]
        return x.view(n, at.shape[1], hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)

    def gather(x, at, ok, rows, heads):                      # back, rows of no document left zero
        x = x.view(n, hk, heads // hk, at.shape[1], d).permute(0, 3, 1, 2, 4).reshape(n, at.shape[1], heads * d)
        out = torch.zeros(rows + 1, heads * d, dtype=F32, device="cuda")
        out[torch.where(ok, at, rows)] = x
        return out[:rows].to(BF16)

    q, k, v = spread(s["q"], iq, okq, hq), spread(s["k"], ik, okk, hk), spread(s["v"], ik, okk, hk)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(n, hk, grp, mq, mk)
    if c["cap"]:
        bent = torch.tanh(score / c["cap"])
        score = bent * c["cap"]
    centre = (iq - q_off[1:, None] + k_off[1:, None])[:, :, None]
    key = ik[:, None, :]
    sees = okq[:, :, None] & okk[:, None, :]
    if c["causal"]:
        near = key <= centre
        if s["prefix"] is not None:
            near = near | (key < (k_off[:-1] + s["prefix"])[:, None, None])
        sees = sees & near
    if s["slopes"] is not None:
        score = score - s["slopes"].view(hk, grp, 1, 1) * (centre - key).abs().float()[:, None, None]
    score = score.masked_fill(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del score
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, torch.ones_like(total), total)).view(n, hk, grp * mq, mk)
    out = gather(torch.matmul(p, v), iq, okq, tq, hq)
    if not c["train"]:
        return out
    do = spread(s["do"], iq, okq, hq)
    dv = gather(torch.matmul(p.transpose(2, 3), do), ik, okk, tk, hk)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    del p, dp
    if c["cap"]:
        ds = ds * (1 - bent * bent).view(ds.shape)
    ds = ds * s["scale"]
    return {"out": out, "dq": gather(torch.matmul(ds, k), iq, okq, tq, hq), "dk": gather(torch.matmul(ds.transpose(2, 3), q), ik, okk, tk, hk), "dv": dv}


def _docs_exact(s):
    """Document by document and query head by query head, in 64 bits."""
    c = s["case"]
    hq, hk, d = c["heads"], c["kv_heads"], c["dim"]
    queries, keys, pre = _lengths(c)
    q, k, v = (s[x].double() for x in "qkv")
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    do = s["do"].double() if c["train"] else None
    q0 = k0 = 0
    for lq, lk, npre in zip(queries, keys, pre):
        if lq and lk:
            gap = torch.arange(lk - lq, lk, device="cuda")[:, None] - torch.arange(lk, device="cuda")
            hidden = (gap < 0) & (torch.arange(lk, device="cuda") >= (npre if c["prefix"] else 0)) if c["causal"] else torch.zeros_like(gap, dtype=torch.bool)
            for part in range(0, hq, hq if lq * lk < 1 << 20 else 1):
                hs = range(part, hq if lq * lk < 1 << 20 else part + 1)
                rows = lambda x, t0, t, of: torch.stack([x[t0:t0 + t, of(h) * d:(of(h) + 1) * d] for h in hs])  # noqa: E731
                mine, shared = (lambda h: h), (lambda h: h * hk // hq)
                Q, K, V = rows(q, q0, lq, mine), rows(k, k0, lk, shared), rows(v, k0, lk, shared)
                x = torch.einsum("hid,hjd->hij", Q, K) * s["scale"]
                slope = c["cap"] and 1 - torch.tanh(x / c["cap"]) ** 2
                x = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
                if c["bias"]:
                    x = x - s["slopes"].double()[list(hs)][:, None, None] * gap.abs()
                x = x.masked_fill(hidden, -math.inf)
                P = torch.softmax(x, -1).nan_to_num(0.0)
                O = torch.einsum("hij,hjd->hid", P, V)
                if c["train"]:
                    G = rows(do, q0, lq, mine)
                    dS = P * (torch.einsum("hid,hjd->hij", G, V) - (G * O).sum(-1, keepdim=True)) * s["scale"]
                    dS = dS * slope if c["cap"] else dS
                for e, h in enumerate(hs):
                    a, b = slice(h * d, h * d + d), slice(shared(h) * d, shared(h) * d + d)
                    out[q0:q0 + lq, a] = O[e]
                    if c["train"]:
                        dq[q0:q0 + lq, a] = dS[e] @ K[e]
                        dk[k0:k0 + lk, b] += dS[e].T @ Q[e]
                        dv[k0:k0 + lk, b] += P[e].T @ G[e]
        q0, k0 = q0 + lq, k0 + lk
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if c["train"] else out


# ------------------------------------------------------------------------------------------------------------------
# embedding rows: out = scale table[id], rounded to bf16; the table's gradient: scale times the sum of the rows dy of an id
# ------------------------------------------------------------------------------------------------------------------
def _embed_prepare(case, g):
    n, rows, w = case["tokens"], case["rows"], case["width"]
    u = torch.rand(n, generator=g, device="cuda", dtype=F64)
    s = {"case": case, "ids": (torch.exp(u * math.log(rows)) - 1).long().clamp_(0, rows - 1), "table": torch.randn(rows, w, generator=g, device="cuda") * 0.02}
    if case["train"]:
        s["dy"] = (torch.randn(n, w, generator=g, device="cuda") * 1e-3).to(BF16)
    return s


def _embed_own(s):
    from image_generator_amd import ops
    c = s["case"]
    out = ops.embedding_fwd(s["ids"], s["table"], scale=c["scale"])
    return {"out": out, "dtable": ops.embedding_bwd(s["ids"], s["dy"], c["rows"], scale=c["scale"])} if c["train"] else out


def _embed_plain(s):
    c = s["case"]
    out = (s["table"][s["ids"]] * c["scale"]).to(BF16)
    if not c["train"]:
        return out
    total = torch.zeros(c["rows"], c["width"], dtype=F64, device="cuda")        # up to tens of thousands of rows of one id
    total.index_add_(0, s["ids"], s["dy"].double())
    return {"out": out, "dtable": (total * c["scale"]).float()}


def _embed_exact(s):
    c = s["case"]
    out = s["table"].double()[s["ids"]] * c["scale"]
    if not c["train"]:
        return out
    order = torch.sort(s["ids"], stable=True)
    ends = torch.bincount(s["ids"], minlength=c["rows"]).cumsum(0)
    upto = torch.cat((torch.zeros(1, c["width"], dtype=F64, device="cuda"), s["dy"].double()[order.indices].cumsum(0)))
    starts = torch.cat((ends.new_zeros(1), ends[:-1]))
    return {"out": out, "dtable": (upto[ends] - upto[starts]) * c["scale"]}


# ------------------------------------------------------------------------------------------------------------------
# AdamW over many tensors, global norm clipped.  States in 32 bits, or in 8: each 256 elements of a tensor share a scale s (the
# largest magnitude, in 32 bits), and a value x >= 0 is held as the whole number nearest to n sqrt(x / s), n = 127 with a sign for the
# first moment, n = 255 for the ROOT of the second, where anything above zero stays above zero.
# ------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    w, n = case["width"], case["layers"]
    if case["params"] == "adapters":
        return [x for i in range(n) for m in ((1, 2, 4)[i % 3] * w,) for _ in range(8) for x in ((4, m), (m, 4))]
    if case["params"] == "encoder":
        layer = [(3 * w, w), (3 * w,), (w, w), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,), (w,), (w,), (w,), (w,)]
        return [(16384, w)] + layer * n + [(w,), (w,), (w, w), (w,)]
    if case["params"] == "odd":
        r = random.Random(w * 10 + n)
        return [(1,), (3,), (w + 1, 2 * w + 3)] + [(r.randint(1, 2 * w), r.randint(1, 2 * w)) for _ in range(8 * n)]
    return [x for i in range(n) for m in (w, 2 * w, 4 * w, 4 * w) for x in ((m, 3, 3, m), (m,), (m, 3, 3, m), (m,), (m, 2 * m), (8 * m, m), (8 * m,), (m, 4 * m))] + [(w, 3, 3, 4)]


def _sizes(case):
    return [math.prod(x) for x in _shapes(case)]


def _up(n):
    return -(-n // BLOCK) * BLOCK


def _adamw_prepare(case, g):
    shapes, sizes = _shapes(case), _sizes(case)
    starts = [0] + list(_running([_up(n) for n in sizes]))
    total, blocks = starts[-1], starts[-1] // BLOCK
    views = lambda flat: [flat[o:o + n].view(x) for o, n, x in zip(starts, sizes, shapes)]  # noqa: E731
    held = torch.zeros(total, dtype=torch.bool, device="cuda")
    for x in views(held):
        x.fill_(True)
    flat = lambda: torch.randn(total, generator=g, device="cuda").mul_(held)  # noqa: E731
    s = {"case": case, "p": flat().mul_(0.02), "t": 10}
    size = torch.exp(torch.randn(blocks, 1, generator=g, device="cuda") * 0.5) * 1e-4     # gradients differ by row,
    s["g"] = (flat() * torch.exp(flat() * 0.7)).view(blocks, BLOCK).mul_(size).view(-1)    # and have heavy tails
    s["g"] = s["g"].to(BF16) if case["grad16"] else s["g"]
    s["p16"] = s["p"].to(BF16)
    # moments after some steps: as 8-bit codes and scales, or as the values
    s["ms"], s["us"] = (size * 0.5).view(-1), (size * 2).view(-1)
    s["mq"] = (flat() * 50).round_().clamp_(-127, 127).to(torch.int8)
    s["uq"] = (flat().abs_() * 60 + 1).round_().clamp_(1, 255).mul_(held).to(torch.uint8)
    s["hyper"] = dict(lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
    if case["bits"] == 32:
        s["m"], s["v"] = _first(s["mq"], s["ms"]).float(), _second(s["uq"], s["us"]).float()
    if own:
        from image_generator_amd.optim import TensorAdamW
        s["grads"] = views(s["g"])
        s["opt"] = TensorAdamW(views(s["p"]), copies=views(s["p16"]), state_bits=case["bits"], max_grad_norm=case["clip"], **s["hyper"])
        s["opt"].t = s["t"]
        for mine, theirs in zip(("m", "v") if case["bits"] == 32 else ("m_codes", "m_scales", "u_codes", "u_scales"), ("m", "v") if case["bits"] == 32 else ("mq", "ms", "uq", "us")):
            getattr(s["opt"], mine).copy_(s.pop(theirs))
    return s


def _first(q, scale):
    """First moment from its codes, in 64 bits: scale sign(q) (q / 127)^2."""
    q = q.view(-1, BLOCK).double()
    return (q * q.abs() * (1 / 16129) * scale[:, None]).view(-1)


def _second(q, scale):
    """Second moment from the codes of its root scale (q / 255)^2, in 64 bits."""
    q = q.view(-1, BLOCK).double()
    return (q * q * (1 / 65025) * scale[:, None]).square().view(-1)


def _adamw_own(s):
    opt = s["opt"]
    opt.step(s["grads"])
    m, v = opt.moments()
    return {"p": s["p"], "p16": s["p16"], "m": m, "v": v}


def _adamw_plain(s):
    """States of 32 bits are stepped in 32 bits.  Those of 8 bits are stepped in 64: a code is a whole number, and a value next to
    the border of two codes has to fall on the same side wherever the step is computed.  So is the norm, a long sum."""
    c, h = s["case"], s["hyper"]
    b1, b2 = h["betas"]
    s["t"] += 1
    step, rbc2 = h["lr"] / (1 - b1 ** s["t"]), 1 / math.sqrt(1 - b2 ** s["t"])
    norm = s["g"].double().square().sum().sqrt()
    fine = torch.isfinite(norm)
    factor = torch.clamp(c["clip"] / (norm + 1e-6), max=1.0) if c["clip"] else torch.ones_like(norm)
    if c["bits"] == 32:
        g, m, v = s["g"].float() * factor.float(), s["m"], s["v"]
    else:
        g, m, v = s["g"].double() * factor, _first(s["mq"], s["ms"]), _second(s["uq"], s["us"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    u = v.sqrt()
    p = s["p"] * (1 - h["lr"] * h["weight_decay"]) - (m / (u * rbc2 + h["eps"])) * step
    s["p"].copy_(torch.where(fine, p, s["p"]))
    s["p16"].copy_(s["p"])
    if c["bits"] == 32:
        s["m"].copy_(torch.where(fine, m, s["m"]))
        s["v"].copy_(torch.where(fine, v, s["v"]))
        return {"p": s["p"], "p16": s["p16"], "m": s["m"], "v": s["v"]}
    mq, ms = _codes(m.abs(), 127)
    uq, us = _codes(u, 255)
    uq = torch.where((u.view(-1, BLOCK) > 0) & (us[:, None] > 0), uq.clamp(min=1), uq)
    s["mq"].copy_(torch.where(fine, (mq * torch.sign(m).view(-1, BLOCK)).view(-1).to(torch.int8), s["mq"]))
    s["uq"].copy_(torch.where(fine, uq.view(-1).to(torch.uint8), s["uq"]))
    s["ms"].copy_(torch.where(fine, ms, s["ms"]))
    s["us"].copy_(torch.where(fine, us, s["us"]))
    return {"p": s["p"], "p16": s["p16"], "m": _first(s["mq"], s["ms"]).float(), "v": _second(s["uq"], s["us"]).float()}


def _codes(x, n):
    """Magnitudes x >= 0 as the whole numbers nearest to n sqrt(x / scale), the scale the largest of 256, rounded to 32 bits (zero
    if below their normal range)."""
    x = x.view(-1, BLOCK)
    scale = x.amax(1).float()
    scale = torch.where(scale >= SMALLEST_NORMAL, scale, torch.zeros_like(scale))
    inverse = torch.where(scale > 0, 1 / scale.double(), torch.zeros_like(x[:, 0]))
    return ((x * inverse[:, None]).sqrt() * n).round().clamp(max=n), scale


def _adamw_exact(s):
    c, h = s["case"], s["hyper"]
    b1, b2 = h["betas"]
    t = s["t"] + 1
    g = s["g"].double()
    if c["clip"]:
        g = g * min(1.0, c["clip"] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    if c["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        at = lambda q, sc, n: sc.double().repeat_interleave(BLOCK) * (q.double() / n).square()  # noqa: E731
        m, v = at(s["mq"], s["ms"], 127) * torch.sign(s["mq"].double()), at(s["uq"], s["us"], 255).square()
    m, v = torch.lerp(g, m, b1), torch.lerp(g.square(), v, b2)
    p = s["p"].double() * (1 - h["lr"] * h["weight_decay"]) - h["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + h["eps"])
    if c["bits"] == 32:
        return {"p": p, "p16": p, "m": m, "v": v}

    def held(x, n, least):                                    # what the nearest code stands for
        x = x.view(-1, BLOCK)
        top = x.amax(1, keepdim=True).float().double()
        q = torch.round(n * torch.sqrt(x / top.clamp(min=SMALLEST_NORMAL)))
        q = torch.where(x > 0, q.clamp(min=least), q).clamp(max=n)
        return (top * (q / n).square()).view(-1)
    return {"p": p, "p16": p, "m": held(m.abs(), 127, 0) * torch.sign(m), "v": held(v.sqrt(), 255, 1).square()}


# ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"docs": _docs_prepare, "embed": _embed_prepare, "adamw": _adamw_prepare}[case["op"]](case, g)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"docs": _docs_own, "embed": _embed_own, "adamw": _adamw_own}[op](state)
    return {"docs": _docs_plain, "embed": _embed_plain, "adamw": _adamw_plain}[op](state)


def exact(case, seed):
    return {"docs": _docs_exact, "embed": _embed_exact, "adamw": _adamw_exact}[case["op"]](prepare(case, seed))


def work(case):
    if case["op"] == "docs":
        queries, keys, _ = _lengths(case)
        q, kv = sum(queries) * case["heads"] * case["dim"] * 2, sum(keys) * case["kv_heads"] * case["dim"] * 2
        # forward: q, k, v in, out out; backward: out, its gradient in, three gradients out (q, k, v are in hand already)
        return {"bytes": 2 * q + 2 * kv + ((2 * q + 2 * kv) if case["train"] else 0), "flops": _pairs(case) * case["dim"] * (4 + (10 if case["train"] else 0))}
    if case["op"] == "embed":
        n, w, rows = case["tokens"], case["width"], case["rows"]
        looked = min(n, rows) * w * 4 + n * (8 + 2 * w)
        return {"bytes": looked + ((2 * n * w + 4 * rows * w) if case["train"] else 0), "flops": n * w * (2 if case["train"] else 1)}
    n = sum(_sizes(case))
    # parameters in and out, their bf16 copy out, gradients in; moments in and out as held; 8 bits: the values handed out too
    return {"bytes": n * (8 + 2 + (2 if case["grad16"] else 4) + (16 if case["bits"] == 32 else 4 + 8 + 16 / BLOCK)), "flops": n * (16 if case["bits"] == 32 else 30)}
