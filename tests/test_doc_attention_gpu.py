"""Attention over packed documents against a dense fp64 evaluation of its definition, entry by entry bounds.

Bounds (first order, per entry; u = 2^-24).  A score is a dot product of D bf16 products in fp32, a scaling and, with a cap, a
tanh whose argument passes through exp2 and a reciprocal: e_ij = (D + 4) u scale sum |q k| + 2^-20 cap' + 4 u |t_ij - bias_ij|
(cap' = cap if there is one).  A probability is then off by the relative r_ij = e_ij + sum_j P_ij e_ij + 2^-20 (exp2, sum, division).
  out: P rounded to bf16 for the matrix product, and the result:  2^-8 |out| + sum_j (2^-8 + r_ij) P_ij |v_j|
  dv:  the same over i:                                           2^-8 |dv| + sum_i (2^-8 + r_ij) P_ij |do_i|
  dS = P (dP - delta) bend:  delta is summed from the rounded out: |d delta| <= sum |do| tol_out; dP has D products: D u sum |do v|;
       bend = 1 - tanh^2 is off by 2^-19;  dS is rounded to bf16:
       tol_dS = P (|d delta| + D u sum |do v| + 2^-19 |dP - delta|) + (2^-8 + r) |dS|
  dq: 2^-8 |dq| + scale sum_j tol_dS |k_j|,   dk likewise over i.
The products of two bounds are covered by a factor of 1.05."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24


def offsets(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def visible(qo, ko, Tq, Tk, causal, prefix, align):
    """(mask [Tq, Tk], centre [Tq]) from the definition."""
    mask, centre = torch.zeros(Tq, Tk, dtype=torch.bool), torch.zeros(Tq, dtype=torch.int64)
    for n in range(len(qo) - 1):
        qb, qe, kb, ke = (int(x) for x in (qo[n], qo[n + 1], ko[n], ko[n + 1]))
        for i in range(qb, qe):
            c = i - qe + ke if align == "end" else i - qb + kb
            centre[i] = c
            j = torch.arange(kb, ke)
            ok = torch.ones(ke - kb, dtype=torch.bool)
            if causal:
                ok = j <= c
                if prefix is not None:
                    ok |= j < kb + int(prefix[n])
            mask[i, kb:ke] = ok
    return mask, centre


def reference(q, k, v, do, heads, kv_heads, qo, ko, causal=False, prefix=None, slopes=None, cap=0.0, scale=None, align="end", keep=None, drop=0.0):
    """fp64 results and bounds: {name: (value, tolerance)}."""
    Tq, Tk, d = q.shape[0], k.shape[0], q.shape[1] // heads
    scale = d ** -0.5 if scale is None else scale
    mask, centre = visible(qo, ko, Tq, Tk, causal, prefix, align)
    names = ("out", "dq", "dk", "dv")
    val = {n: torch.zeros_like(t, dtype=F64) for n, t in zip(names, (q, q, k, v))}
    tol = {n: torch.zeros_like(t, dtype=F64) for n, t in zip(names, (q, q, k, v))}
    lse = torch.full((heads, Tq), -math.inf, dtype=F64)
    for h in range(heads):
        hk = h * kv_heads // heads
        a, b = slice(h * d, h * d + d), slice(hk * d, hk * d + d)
        Q, K, V, G = q[:, a].double(), k[:, b].double(), v[:, b].double(), do[:, a].double()
        t = Q @ K.T * scale
        e = (d + 4) * U * scale * (Q.abs() @ K.abs().T) + 2.0 ** -20 * cap
        bend = torch.ones_like(t)
        if cap:
            th = torch.tanh(t / cap)
            t, bend = cap * th, 1 - th * th
        if slopes is not None:
            t = t - float(slopes[h]) * (centre[:, None] - torch.arange(Tk)).abs()
        e = e + 4 * U * t.abs()
        t = t.masked_fill(~mask, -math.inf)
        lse[h] = torch.logsumexp(t, 1) / math.log(2)
        P = torch.softmax(t, 1).nan_to_num(0.0)
        r = torch.where(mask, e + (P * e).sum(1, keepdim=True) + 2.0 ** -20, torch.zeros_like(e))
        w = torch.ones_like(P) if keep is None else keep[h].double() / (1 - drop)
        Pd = P * w
        out = Pd @ V
        tout = 2.0 ** -8 * out.abs() + ((2.0 ** -8 + r) * Pd) @ V.abs()
        dP = (G @ V.T) * w
        delta = (G * out).sum(1, keepdim=True)
        dS = P * (dP - delta) * bend
        tdS = P * ((G.abs() * tout).sum(1, keepdim=True) + d * U * (G.abs() @ V.abs().T) * w + 2.0 ** -19 * (dP - delta).abs()) + (2.0 ** -8 + r) * dS.abs()
        val["out"][:, a], tol["out"][:, a] = out, tout
        val["dq"][:, a] = dS @ K * scale
        tol["dq"][:, a] = scale * tdS @ K.abs()
        val["dk"][:, b] += dS.T @ Q * scale
        tol["dk"][:, b] += scale * tdS.T @ Q.abs()
        val["dv"][:, b] += Pd.T @ G
        tol["dv"][:, b] += ((2.0 ** -8 + r) * Pd).T @ G.abs()
    for n in ("dq", "dk", "dv"):
        tol[n] += 2.0 ** -8 * val[n].abs()
    return {n: (val[n], 1.05 * tol[n] + 1e-30) for n in names}, lse


def inputs(Tq, Tk, heads, kv_heads, d, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, do = ((torch.randn(Tq, heads * d, generator=g) * scale).to(BF) for _ in range(2))
    k, v = ((torch.randn(Tk, kv_heads * d, generator=g) * scale).to(BF) for _ in range(2))
    return q, k, v, do


def run(q, k, v, do, **how):
    from image_generator_amd import ops
    how = {n: x.cuda() if torch.is_tensor(x) else x for n, x in how.items()}
    q, k, v, do = (t if t.is_cuda else t.cuda() for t in (q, k, v, do))
    out, lse = ops.doc_attention_fwd(q, k, v, **how)
    return {"out": out, "lse": lse, **dict(zip(("dq", "dk", "dv"), ops.doc_attention_bwd(do, q, k, v, out, lse, **how)))}


def check(got, ref, rows=None):
    want, lse = ref
    for n, (val, tol) in want.items():
        x = got[n].cpu().double()
        bad = ~((x - val).abs() <= tol)
        if rows is not None and n in rows:
            bad = bad[rows[n]]
        assert not bad.any(), (n, int(bad.sum()), bad.numel(), float(((x - val).abs() - tol).nan_to_num(9e9).max()), float(val.abs().max()))
    return want


LENS = {
    "one": [1], "single_tokens": [1] * 37, "tile": [64, 64, 128], "odd": [3, 0, 65, 17, 0, 0, 1, 130, 31, 63, 2], "captions": [5, 77, 12, 30, 9, 44, 77, 3, 21, 60, 8],
    "long": [700], "two": [257, 391],
}


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (8, 8, 96), (6, 2, 40)])
def test_self_attention_of_documents(lens, heads, kv_heads, d):
    off = offsets(LENS[lens])
    T = int(off[-1])
    x = inputs(T, T, heads, kv_heads, d, 1)
    got = run(*x, heads=heads, kv_heads=kv_heads, q_offsets=off)
    ref = reference(*x, heads, kv_heads, off, off)
    check(got, ref)
    # 2^-8 of a unit in log2 covers the score bounds of these inputs many times over
    assert (got["lse"].cpu().double() - ref[1]).abs().max() < 2.0 ** -8


@pytest.mark.parametrize("d", [8, 16, 24, 32, 48, 56, 64, 72, 80, 88, 104, 112, 120, 128])
def test_head_widths(d):
    off = offsets([50, 3, 140])
    x = inputs(193, 193, 2, 1, d, 2)
    check(run(*x, heads=2, kv_heads=1, q_offsets=off, causal=True), reference(*x, 2, 1, off, off, causal=True))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (3, 1), (10, 2), (7, 7), (16, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_key_heads(heads, kv_heads, causal):
    off = offsets([33, 100, 1, 66])
    x = inputs(200, 200, heads, kv_heads, 32, 3)
    check(run(*x, heads=heads, kv_heads=kv_heads, q_offsets=off, causal=causal), reference(*x, heads, kv_heads, off, off, causal=causal))


@pytest.mark.parametrize("causal,prefix", [(False, None), (True, None), (True, [0, 5, 200, 7, 0, 70])])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("lens", [[9, 40, 130, 0, 1, 71]])
def test_scores_and_masks(causal, prefix, cap, bias, lens):
    off = offsets(lens)
    T = int(off[-1])
    x = inputs(T, T, 4, 2, 64, 4, 1.5)
    how = dict(causal=causal, prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32), cap=cap,
               slopes=torch.tensor([0.5, 0.1, 0.0, 0.02]) if bias else None)
    check(run(*x, heads=4, kv_heads=2, q_offsets=off, **how), reference(*x, 4, 2, off, off, **how))


@pytest.mark.parametrize("ql,kl", [([1, 1, 1, 1], [70, 0, 1, 300]), ([200, 64, 3], [5, 77, 12]), ([5, 9, 130], [3, 0, 260]), ([0, 4, 0], [10, 10, 10]), ([1], [1000])])
@pytest.mark.parametrize("align", ["end", "start"])
@pytest.mark.parametrize("causal", [False, True])
def test_queries_and_keys_of_different_lengths(ql, kl, align, causal):
    """Appended queries, single queries, images over captions; with more queries than keys the first rows see nothing."""
    qo, ko = offsets(ql), offsets(kl)
    x = inputs(int(qo[-1]), int(ko[-1]), 4, 2, 48, 5)
    how = dict(causal=causal, align=align, slopes=torch.tensor([0.3, 0.0, 0.05, 0.01]))
    got = run(*x, heads=4, kv_heads=2, q_offsets=qo, k_offsets=ko, **how)
    ref = reference(*x, 4, 2, qo, ko, **how)
    check(got, ref)
    mask, _ = visible(qo, ko, x[0].shape[0], x[1].shape[0], causal, None, align)
    empty = ~mask.any(1)
    assert (got["out"].cpu()[empty] == 0).all() and (got["dq"].cpu()[empty] == 0).all() and (got["lse"].cpu()[:, empty] == -math.inf).all()


def test_rows_and_keys_of_no_document():
    """Tokens before the first and behind the last document: zeros, whatever they hold."""
    qo, ko = offsets([40, 30], 7), offsets([50, 20], 3)
    q, k, v, do = inputs(90, 90, 2, 2, 64, 6)
    for t, o in ((q, qo), (do, qo), (k, ko), (v, ko)):
        t[:int(o[0])] = float("nan")
        t[int(o[-1]):] = float("inf")
    got = run(q, k, v, do, heads=2, q_offsets=qo, k_offsets=ko)
    clean = [torch.nan_to_num(t.float(), 0, 0, 0).to(BF) for t in (q, k, v, do)]
    check(got, reference(*clean, 2, 2, qo, ko))
    for n, o in (("out", qo), ("dq", qo), ("dk", ko), ("dv", ko)):
        assert (got[n][:int(o[0])] == 0).all() and (got[n][int(o[-1]):] == 0).all()


@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("which", ["k", "v", "q", "do"])
def test_what_is_not_finite_stays_in_its_document(value, which):
    off = offsets([20, 30, 25, 80])
    x = dict(zip(("q", "k", "v", "do"), inputs(155, 155, 4, 2, 64, 7)))
    clean = {n: t.clone() for n, t in x.items()}
    x[which][22, 3] = value                                # document 1
    x[which][140, 70] = value                              # document 3, the second head's columns
    how = dict(heads=4, kv_heads=2, q_offsets=off)
    got = run(*x.values(), **how)
    ref = reference(*clean.values(), 4, 2, off, off)
    fine = torch.cat((torch.arange(0, 20), torch.arange(50, 75)))
    check(got, ref, {n: fine for n in ("out", "dq", "dk", "dv")})
    assert not torch.isfinite(torch.cat([got[n].float()[20:50].flatten() for n in ("out", "dq", "dk", "dv")])).all()


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_what_is_not_finite_behind_a_causal_row(value):
    off = offsets([150])
    q, k, v, do = inputs(150, 150, 2, 2, 40, 8)
    clean = [t.clone() for t in (q, k, v, do)]
    k[100, 1] = value
    v[100, 2] = value
    got = run(q, k, v, do, heads=2, q_offsets=off, causal=True)
    ref = reference(*clean, 2, 2, off, off, causal=True)
    check({n: got[n] for n in ("out", "dq")} | {n: torch.zeros_like(got[n]) for n in ("dk", "dv")},
          ({n: x for n, x in ref[0].items() if n in ("out", "dq")}, ref[1]), {"out": torch.arange(100), "dq": torch.arange(100)})
    assert torch.isnan(got["out"][100:, 2]).all() or torch.isinf(got["out"][100:, 2]).any()
    # a value without a probability's weight: rows that see it become not finite in its column alone
    _, k, _, _ = clean
    got = run(q, k, v, do, heads=2, q_offsets=off, causal=True)
    x = got["out"].float().cpu()
    assert not torch.isfinite(x[100:, 2]).any() and torch.isfinite(x[100:, :2]).all() and torch.isfinite(x[100:, 3:]).all()


def test_large_scores():
    """Scores of some thousands: the running maximum carries them; equal largest scores share the row."""
    off = offsets([70, 130])
    q, k, v, do = inputs(200, 200, 2, 2, 64, 9)
    q, k = q * 24, k * 24
    check(run(q, k, v, do, heads=2, q_offsets=off), reference(q, k, v, do, 2, 2, off, off))
    k[:70] = k[0]
    check(run(q, k, v, do, heads=2, q_offsets=off), reference(q, k, v, do, 2, 2, off, off))


def test_strided_operands_and_gradients_in_one_buffer():
    from image_generator_amd import ops
    off = offsets([33, 60, 41]).cuda()
    qkv = inputs(134, 134, 12, 1, 64, 10)[0].cuda()         # [q 6 heads | k 3 | v 3]
    q, k, v = qkv[:, :384], qkv[:, 384:576], qkv[:, 576:]
    do = torch.randn(134, 400, device="cuda").to(BF)[:, 8:392]
    how = dict(heads=6, kv_heads=3, q_offsets=off)
    whole = run(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), **how)
    got = run(q, k, v, do, **how)
    assert all(torch.equal(got[n], whole[n]) for n in whole)
    d = torch.full((134, 800), 7.0, device="cuda", dtype=BF)
    ops.doc_attention_bwd(do, q, k, v, got["out"], got["lse"], dq=d[:, 8:392], dk=d[:, 392:584], dv=d[:, 584:776], **how)
    assert torch.equal(d[:, 8:776], torch.cat([whole[n] for n in ("dq", "dk", "dv")], 1)) and (d[:, :8] == 7).all() and (d[:, 776:] == 7).all()


def test_equal_calls_return_equal_bits_on_any_stream():
    off = offsets([300, 5, 211])
    x = [t.cuda() for t in inputs(516, 516, 8, 2, 64, 11)]
    a = run(*x, heads=8, kv_heads=2, q_offsets=off, causal=True, cap=20.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = run(*x, heads=8, kv_heads=2, q_offsets=off, causal=True, cap=20.0)
    s.synchronize()
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_gradients_against_differences():
    """Directional derivative of sum(out * do), fp64 differences of the reference's forward along a bf16 direction."""
    off = offsets([20, 37])
    x = inputs(57, 57, 4, 2, 32, 12)
    how = dict(causal=True, cap=3.0, slopes=torch.tensor([0.2, 0.1, 0.05, 0.0]))
    got = run(*x, heads=4, kv_heads=2, q_offsets=off, **how)
    q, k, v, do = x
    g = torch.Generator().manual_seed(13)
    for n, t in (("dq", 0), ("dk", 1), ("dv", 2)):
        way = torch.randn(x[t].shape, generator=g, dtype=F64)
        f = lambda s: (reference(*[y.double() + (s * way if m == t else 0) for m, y in enumerate((q, k, v))], do, 4, 2, off, off, **how)[0]["out"][0] * do.double()).sum()  # noqa: E731
        slope = float((f(1e-4) - f(-1e-4)) / 2e-4)
        val, tol = reference(*x, 4, 2, off, off, **how)[0][n]
        # the directional derivative of the bounds, and 1e-6 for the difference quotient
        assert abs(float((got[n].cpu().double() * way).sum()) - slope) <= float((tol * way.abs()).sum()) + 1e-6 * (1 + abs(slope))


def test_autograd_layouts():
    from image_generator_amd import ops
    off = offsets([30, 50]).cuda()
    q, k, v, do = (t.cuda() for t in inputs(80, 80, 4, 2, 64, 14))
    want = run(q, k, v, do, heads=4, kv_heads=2, q_offsets=off, causal=True)
    how = dict(heads=4, kv_heads=2, q_offsets=off, causal=True)
    for parts in ((torch.cat((q, k, v), 1),), (q, torch.cat((k, v), 1)), (q, k, v)):
        leaves = [t.clone().requires_grad_(True) for t in parts]
        out = ops.doc_attention(*leaves, **how)
        assert torch.equal(out, want["out"])
        out.backward(do)
        assert torch.equal(torch.cat([t.grad for t in leaves], 1), torch.cat([want[n] for n in ("dq", "dk", "dv")], 1))


def keep_mask(heads, Tq, Tk, p, seed):
    """The hash that decides which probabilities are dropped, in whole numbers."""
    M = 0xFFFFFFFF
    i, j = torch.arange(Tq)[:, None], torch.arange(Tk)[None]
    out = []
    for h in range(heads):
        x = (i * 0x9E3779B1 + h * 0x85EBCA6B + seed) & M
        x = x ^ (x >> 15)
        x = (x * 0x2C1B3C6D) & M
        x = x ^ (x >> 12)
        x = (x + j * 0xC2B2AE35) & M
        x = x ^ (x >> 16)
        x = (x * 0x7FEB352D) & M
        x = x ^ (x >> 15)
        x = (x * 0x846CA68B) & M
        x = x ^ (x >> 16)
        out.append(x >= int(p * 4294967296.0))
    return out


@pytest.mark.parametrize("p", [0.25, 0.9])
def test_dropout(p):
    off = offsets([40, 1, 90])
    x = inputs(131, 131, 4, 2, 64, 15)
    keep = keep_mask(4, 131, 131, p, 1234)
    rate = float(torch.stack(keep).double().mean())
    assert abs(rate - (1 - p)) < 0.01
    check(run(*x, heads=4, kv_heads=2, q_offsets=off, causal=True, drop_p=p, seed=1234), reference(*x, 4, 2, off, off, causal=True, keep=keep, drop=p))


def test_captured_and_replayed():
    from image_generator_amd import ops
    off = offsets([50, 70, 9]).cuda()
    x = [t.cuda() for t in inputs(129, 129, 4, 4, 64, 16)]
    how = dict(heads=4, q_offsets=off, causal=True)
    run(*x, **how)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.doc_attention_fwd(*x[:3], **how)
        grads = ops.doc_attention_bwd(x[3], *x[:3], out, lse, **how)
    for k in range(4):
        for t in x:
            t.normal_()
        off.copy_(offsets([20 + k, 100, 9 - k]))
        graph.replay()
        torch.cuda.synchronize()
        want = run(*x, **how)
        assert torch.equal(out, want["out"]) and torch.equal(lse, want["lse"])
        assert all(torch.equal(a, want[n]) for a, n in zip(grads, ("dq", "dk", "dv")))


def test_no_tokens():
    from image_generator_amd import ops
    off = offsets([0, 0]).cuda()
    none = torch.empty(0, 64, device="cuda", dtype=BF)
    out, lse = ops.doc_attention_fwd(none, none, none, heads=2, q_offsets=off)
    assert out.shape == (0, 64) and lse.shape == (2, 0)
    q = torch.randn(5, 64, device="cuda").to(BF)
    out, lse = ops.doc_attention_fwd(q, none, none, heads=2, q_offsets=offsets([5, 0]).cuda(), k_offsets=off)
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = ops.doc_attention_bwd(q, q, none, none, out, lse, heads=2, q_offsets=offsets([5, 0]).cuda(), k_offsets=off)
    assert (dq == 0).all() and dk.shape == (0, 64)


@pytest.mark.parametrize("docs", [1, 40])
def test_wrong_offsets_stay_in_bounds(docs):
    """Offsets past the tensors or out of order: the kernels clamp them; tokens inside well-formed documents are right."""
    off = offsets([60] * docs)
    T = 60 * docs
    x = inputs(T, T, 2, 2, 64, 17)
    bad = off.clone()
    bad[-1] = T + 1000
    got = run(*x, heads=2, q_offsets=bad)
    check(got, reference(*x, 2, 2, off, off))
    if docs > 1:
        bad = off.clone()
        bad[20], bad[21] = T, -5
        got = run(*x, heads=2, q_offsets=bad)
        assert all(t.shape[0] in (T, 2) for t in got.values())


SPLIT = {                                                  # (queries, keys) whose forward pass, or key gradients, run in pieces
    "few_rows": ([1, 1, 1, 2, 1], [700, 0, 901, 33, 64]), "one_row": ([1], [2500]), "rows_at_the_end": ([3, 30], [1100, 1500]),
    "few_keys": ([1500, 0, 900], [40, 3, 5]), "one_key": ([3000], [1]), "both": ([600, 1], [7, 1200]),
}


@pytest.mark.parametrize("case", list(SPLIT))
@pytest.mark.parametrize("how", ["plain", "bent", "dropped"])
def test_split_work(case, how):
    ql, kl = SPLIT[case]
    qo, ko = offsets(ql), offsets(kl)
    x = inputs(int(qo[-1]), int(ko[-1]), 4, 2, 72, 20)
    kw = {} if how == "plain" else dict(causal=True, cap=8.0, slopes=torch.tensor([0.01, 0.0, 0.1, 0.003]))
    drop = dict(drop_p=0.3, seed=99) if how == "dropped" else {}
    keep = keep_mask(4, x[0].shape[0], x[1].shape[0], 0.3, 99) if drop else None
    got = run(*x, heads=4, kv_heads=2, q_offsets=qo, k_offsets=ko, **kw, **drop)
    check(got, reference(*x, 4, 2, qo, ko, keep=keep, drop=0.3, **kw))
    again = run(*x, heads=4, kv_heads=2, q_offsets=qo, k_offsets=ko, **kw, **drop)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("case", ["few_rows", "few_keys", "both"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["k", "v", "q", "do"])
def test_split_work_with_what_is_not_finite(case, value, which):
    ql, kl = SPLIT[case]
    qo, ko = offsets(ql), offsets(kl)
    x = dict(zip(("q", "k", "v", "do"), inputs(int(qo[-1]), int(ko[-1]), 4, 2, 72, 21)))
    clean = [t.clone() for t in x.values()]
    x[which][0, 5] = value                                 # document 0
    got = run(*x.values(), heads=4, kv_heads=2, q_offsets=qo, k_offsets=ko)
    rows, keys = torch.arange(int(qo[1]), int(qo[-1])), torch.arange(int(ko[1]), int(ko[-1]))
    check(got, reference(*clean, 4, 2, qo, ko), {"out": rows, "dq": rows, "dk": keys, "dv": keys})
    assert not torch.isfinite(torch.cat([got[n][:1].float().flatten() for n in ("out", "dq", "dk", "dv")])).all()


def test_one_row_of_any_stride():
    """The stride of a matrix of one row is whatever made it: 1 here."""
    off = offsets([1])
    x = [t.cuda() for t in inputs(1, 1, 4, 2, 64, 30)]
    want = run(*x, heads=4, kv_heads=2, q_offsets=off)
    odd = [t.as_strided(t.shape, (1, 1)) for t in x]
    assert all(t.stride(0) == 1 for t in odd)
    got = run(*odd, heads=4, kv_heads=2, q_offsets=off)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_gradient_that_is_a_piece_of_another():
    """cat's backward hands out views of one buffer, 3 elements in here."""
    from image_generator_amd import ops
    off = offsets([30, 50]).cuda()
    q, k, v, do = (t.cuda() for t in inputs(80, 80, 4, 2, 64, 31))
    want = run(q, k, v, do, heads=4, kv_heads=2, q_offsets=off)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = ops.doc_attention(*leaves, heads=4, kv_heads=2, q_offsets=off)
    torch.cat((torch.zeros(3, device="cuda", dtype=BF), out.flatten())).backward(torch.cat((torch.zeros(3, device="cuda", dtype=BF), do.flatten())))
    assert all(torch.equal(t.grad, want[n]) for t, n in zip(leaves, ("dq", "dk", "dv")))


def test_small_values_under_low_scores():
    """Scores around -48 and values around 2^-70: neither alone leaves fp32's range, their product would."""
    off = offsets([90, 40])
    q, k, v, do = inputs(130, 130, 2, 2, 64, 32)
    q, k, v = (q.float() * 0.1 + 2).to(BF), (k.float() * 0.1 - 3).to(BF), (v.float() * 2.0 ** -70).to(BF)
    check(run(q, k, v, do, heads=2, q_offsets=off), reference(q, k, v, do, 2, 2, off, off))


def test_places_that_are_refused():
    from image_generator_amd import ops
    off = offsets([8]).cuda()
    q, k, v, do = (t.cuda() for t in inputs(8, 8, 2, 2, 64, 33))
    out, lse = ops.doc_attention_fwd(q, k, v, 2, off)
    for bad in (dict(dq=q), dict(dk=k), dict(dv=do), dict(dk=out), dict(dk=torch.empty_like(k), dv=None)):
        if "dv" in bad and bad["dv"] is None:
            bad["dv"] = bad["dk"]
        with pytest.raises(ValueError, match="in the place"):
            ops.doc_attention_bwd(do, q, k, v, out, lse, 2, off, **bad)
    with pytest.raises(ValueError, match="operands"):
        ops.doc_attention(q, None, v, heads=2, q_offsets=off)
    for n, t in zip(("dq", "dk", "dv"), ops.doc_attention_bwd(out, q, q, q, out, lse, 2, off)):       # one tensor in several places is read only
        assert torch.isfinite(t).all(), n


@pytest.mark.parametrize("lens", [[2, 3, 1, 32, 7, 16, 2], [2, 300, 2, 1], [1] * 9])
@pytest.mark.parametrize("d,cap", [(64, 0.0), (40, 5.0), (128, 0.0)])
def test_gradients_of_few_keys_do_not_carry_the_rounding_of_the_result(lens, d, cap):
    """Values that differ by little beside their size: delta = sum dO o of the bf16 result would be off by 2^-8 sum |dO| |o|, far more
    than dP - delta.  Rows of at most 32 keys sum P dP instead:  |d delta| <= sum_j P (D u sum |dO v| + r |dP|)  and, as above,
    tol_dS = P (|d delta| + D u sum |dO v| + 2^-19 |dP - delta|) + (2^-8 + r) |dS|."""
    off = offsets(lens)
    T = int(off[-1])
    q, k, v, do = inputs(T, T, 1, 1, d, 34)
    v = (v.float() * 0.25 + 100).to(BF)
    got = run(q, k, v, do, heads=1, q_offsets=off, cap=cap)
    for n, size in enumerate(lens):
        if size > 32:
            continue
        rows = slice(int(off[n]), int(off[n + 1]))
        Q, K, V, G = (t[rows].double() for t in (q, k, v, do))
        scale = d ** -0.5
        t = Q @ K.T * scale
        e = (d + 4) * U * scale * (Q.abs() @ K.abs().T) + 2.0 ** -20 * cap + 4 * U * t.abs()
        bend = torch.ones_like(t)
        if cap:
            bend = 1 - torch.tanh(t / cap) ** 2
            t = cap * torch.tanh(t / cap)
        P = torch.softmax(t, 1)
        r = e + (P * e).sum(1, keepdim=True) + 2.0 ** -20
        dP = G @ V.T
        rough = d * U * (G.abs() @ V.abs().T)
        delta = (P * dP).sum(1, keepdim=True)
        ddelta = (P * (rough + r * dP.abs())).sum(1, keepdim=True)
        dS = P * (dP - delta) * bend
        tol = P * (ddelta + rough + 2.0 ** -19 * (dP - delta).abs()) + (2.0 ** -8 + r) * dS.abs()
        for name, want, bound in (("dq", scale * dS @ K, scale * tol @ K.abs()), ("dk", scale * dS.T @ Q, scale * tol.T @ Q.abs())):
            x = got[name][rows].cpu().double()
            assert ((x - want).abs() <= 1.05 * (bound + 2.0 ** -8 * want.abs()) + 1e-30).all(), (name, n, float((x - want).abs().max()), float(want.abs().max()))


@pytest.mark.parametrize("lens", [[2500, 40], [1, 2600], [1900]])
@pytest.mark.parametrize("how", [dict(), dict(causal=True), dict(causal=True, cap=5.0, bias=True), dict(bias=True), dict(causal=True, drop_p=0.3, seed=7), dict(cap=3.0, prefix=True, causal=True)],
                         ids=["plain", "causal", "bent", "bias", "dropped", "prefix"])
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 1, 64), (1, 1, 96), (2, 2, 128)])
def test_few_tiles_over_many_keys(lens, how, heads, kv_heads, d):
    """Few heads, few long documents: the keys of a tile of rows are dealt out in runs, in both directions."""
    from image_generator_amd._lib import lib
    off = offsets(lens)
    T = int(off[-1])
    assert lib.mi355_doc_attention_fwd_workspace_bytes(T, T, heads, kv_heads, d, len(lens)) > 0            # in runs
    how = dict(how)
    if how.pop("bias", False):
        how["slopes"] = torch.tensor([0.5, 0.01][:heads])            # far runs that weigh nothing, and some that do
    if how.pop("prefix", False):
        how["prefix"] = torch.tensor([n // 3 for n in lens], dtype=torch.int32)
    x = inputs(T, T, heads, kv_heads, d, 35)
    got = run(*x, heads=heads, kv_heads=kv_heads, q_offsets=off, **how)
    p, seed = how.pop("drop_p", 0.0), how.pop("seed", 0)
    ref = reference(*x, heads, kv_heads, off, off, keep=keep_mask(heads, T, T, p, seed) if p else None, drop=p, **how)
    check(got, ref)
    assert (got["lse"].cpu().double() - ref[1]).abs().max() < 2.0 ** -8
    again = run(*x, heads=heads, kv_heads=kv_heads, q_offsets=off, **how, drop_p=p, seed=seed)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_what_is_not_finite_in_one_run(value):
    """A key that only the last rows see, and one of the other document: nobody else is touched by either."""
    off = offsets([2000, 500])
    q, k, v, do = inputs(2500, 2500, 1, 1, 64, 36)
    clean = [t.clone() for t in (q, k, v, do)]
    for at in (1950, 2300):
        k[at, 3] = value
        v[at, 5] = value
    got = run(q, k, v, do, heads=1, q_offsets=off, causal=True)
    ref = reference(*clean, 1, 1, off, off, causal=True)
    fine = torch.cat((torch.arange(0, 1950), torch.arange(2000, 2300)))
    for n in ("out", "dq"):
        val, tol = ref[0][n]
        assert ((got[n].cpu().double() - val).abs() <= tol)[fine].all(), n
    assert not torch.isfinite(got["out"][1950:2000]).all() and not torch.isfinite(got["dq"][2300:]).all()


def test_queries_behind_many_keys_in_runs():
    """Appended queries over a long past, fewer keys than queries in one document, and tokens of none."""
    qo, ko = offsets([300, 200, 0], 5), offsets([3000, 100, 900], 2)
    x = inputs(520, 4010, 2, 1, 48, 37)
    how = dict(causal=True, slopes=torch.tensor([0.02, 0.0]))
    got = run(*x, heads=2, kv_heads=1, q_offsets=qo, k_offsets=ko, **how)
    check(got, reference(*x, 2, 1, qo, ko, **how))
    assert (got["out"][:5] == 0).all() and (got["dq"][505:] == 0).all() and (got["dk"][-8:] == 0).all()


@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 40), (3, 1, 64), (4, 2, 96), (8, 1, 128)])
@pytest.mark.parametrize("ql", [[1] * 6, [3, 1, 0, 2, 1, 5]])
def test_single_queries_over_long_pasts(heads, kv_heads, d, ql):
    """Waves that take runs of keys by themselves, with as few rows each as it takes to fill the chip."""
    qo, ko = offsets(ql), offsets([9000, 5000, 0, 1, 7000, 300])
    x = inputs(int(qo[-1]), int(ko[-1]), heads, kv_heads, d, 38)
    how = dict(causal=True, slopes=torch.tensor([0.5, 0.01, 0.0, 0.001, 0.1, 0.2, 0.003, 0.02][:heads]))
    check(run(*x, heads=heads, kv_heads=kv_heads, q_offsets=qo, k_offsets=ko, **how), reference(*x, heads, kv_heads, qo, ko, **how))


@pytest.mark.parametrize("ql,kl,train", [([2500, 40], None, True), ([1] * 4, [3000, 100, 4000, 50], False)], ids=["tiles", "waves"])
def test_runs_captured_and_replayed_in_two_graphs(ql, kl, train):
    """Partial results live in workspaces of the capture: two graphs, replayed in turn with eager calls between, do not meet in them."""
    from image_generator_amd import ops
    qo = offsets(ql).cuda()
    ko = qo if kl is None else offsets(kl).cuda()
    xs = [[t.cuda() for t in inputs(int(qo[-1]), int(ko[-1]), 2, 1, 64, 40 + i)] for i in range(2)]
    how = dict(heads=2, kv_heads=1, q_offsets=qo, k_offsets=ko, causal=True)

    def call(x):
        out, lse = ops.doc_attention_fwd(*x[:3], **how)
        return (out, lse, *(ops.doc_attention_bwd(x[3], *x[:3], out, lse, **how) if train else ()))

    call(xs[0])
    torch.cuda.synchronize()
    graphs, got = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(call(x))
    for _ in range(3):
        for x in xs:
            for t in x:
                t.normal_()
        for g in graphs:
            g.replay()
        want = [call(x) for x in xs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
