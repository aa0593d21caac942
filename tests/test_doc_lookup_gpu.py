"""Which document a token belongs to, where the offsets are many and uneven: hundreds of documents, runs of empty ones, more starts
under one wave than its window holds, tokens in front of the first document and behind the last.

Forward and backward against the dense fp64 reference and its bounds (test_doc_attention_gpu).  The layouts are laid against the
estimate that the lookup starts from (documents of equal length, 64 offsets around that place)."""
import pytest
import torch

from test_doc_attention_gpu import check, inputs, offsets, reference, run

pytestmark = pytest.mark.gpu


def mixed(seed, docs, top):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, top + 1, (docs,), generator=g).tolist()


LAYOUTS = {  # document lengths; tokens in front of the first and behind the last document
    "long_at_the_end": ([1] * 200 + [700], 0, 0),
    "long_in_front": ([700] + [1] * 200, 0, 0),
    "long_in_the_middle": ([1] * 150 + [400] + [2] * 150, 0, 0),
    "empty_in_front": ([0] * 300 + [5, 90, 33] * 4, 0, 0),
    "empty_behind": ([5, 90, 33] * 4 + [0] * 300, 0, 0),
    "empty_in_the_middle": ([40, 7] * 6 + [0] * 300 + [7, 40] * 6, 0, 0),
    "all_but_one_empty": ([0] * 500 + [300] + [0] * 500, 0, 0),
    "tiny": (mixed(1, 700, 2), 0, 0),
    "tiny_and_long": (mixed(2, 300, 2) + [300] + mixed(3, 300, 1), 0, 0),
    "single_tokens": ([1] * 500, 0, 0),
    "one_in_four": ([1, 0, 0, 0] * 160, 0, 0),                  # 128 starts under a wave's 32 rows
    "loose_tokens": ([3] * 90, 130, 200),
    "loose_in_front_of_empty": ([0] * 200 + [1] * 100, 90, 0),
    "loose_behind_empty": ([1] * 100 + [0] * 200, 0, 90),
    "captions": (mixed(4, 40, 77), 5, 5),
}


def packed(layout):
    lens, front, behind = LAYOUTS[layout]
    off = offsets(lens, front)
    return off, int(off[-1]) + behind


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("kind", ["plain", "causal"])
def test_one_list(layout, kind):
    off, T = packed(layout)
    heads, kv_heads = (2, 2) if kind == "plain" else (4, 2)
    x = inputs(T, T, heads, kv_heads, 32, 31)
    how = {} if kind == "plain" else dict(causal=True, slopes=torch.linspace(0.5, 0.0, heads))
    check(run(*x, heads=heads, kv_heads=kv_heads, q_offsets=off, **how), reference(*x, heads, kv_heads, off, off, **how))


@pytest.mark.parametrize("queries,keys", [("long_at_the_end", "long_in_front"), ("tiny", "tiny_reversed"), ("empty_in_front", "empty_behind"),
                                          ("single_tokens", "one_list_500"), ("all_but_one_empty", "spread_1001"), ("long_in_front", "long_at_the_end")])
@pytest.mark.parametrize("align", ["end", "start"])
def test_two_lists(queries, keys, align):
    """Queries and keys whose documents lie at quite different places; the keys' own lookup in the backward pass."""
    qo, Tq = packed(queries)
    n = qo.numel() - 1
    if keys == "tiny_reversed":
        ko, Tk = offsets(LAYOUTS[queries][0][::-1]), int(qo[-1])
    elif keys == "one_list_500":
        ko = offsets([0] * 250 + [2] * 250)
        Tk = int(ko[-1])
    elif keys == "spread_1001":
        ko = offsets([1] * 1001, 40)
        Tk = int(ko[-1]) + 40
    else:
        ko, Tk = packed(keys)
    assert ko.numel() - 1 == n
    x = inputs(Tq, Tk, 2, 1, 40, 32)
    how = dict(causal=True, prefix=torch.randint(0, 3, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(5)), align=align)
    got = run(*x, heads=2, kv_heads=1, q_offsets=qo, k_offsets=ko, **how)
    check(got, reference(*x, 2, 1, qo, ko, **how))


@pytest.mark.parametrize("docs,rows", [(1920, "training"), (4000, "single")])
def test_a_batch_of_real_size_against_its_documents(docs, rows):
    """Captions of 3 .. 77 tokens, and one query for each: every document by itself gives the same (same kernels, other places)."""
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(3, 78, (docs,), generator=g).tolist()
    ko = offsets(lens)
    T = int(ko[-1])
    qo = ko if rows == "training" else torch.arange(docs + 1, dtype=torch.int32)
    heads, d = 1, 16
    q, k, v, do = inputs(int(qo[-1]), T, heads, heads, d, 33)
    align = "end" if rows == "training" else "start"
    got = run(q, k, v, do, heads=heads, q_offsets=qo, k_offsets=ko, align=align)
    got = {n: t.cpu() for n, t in got.items()}
    for lo in range(0, docs, 100):                           # a hundred documents at a time in the dense reference
        hi = min(lo + 100, docs)
        a, b, c, e = int(qo[lo]), int(qo[hi]), int(ko[lo]), int(ko[hi])
        ref = reference(q[a:b], k[c:e], v[c:e], do[a:b], heads, heads, qo[lo:hi + 1] - a, ko[lo:hi + 1] - c, align=align)
        check({"out": got["out"][a:b], "dq": got["dq"][a:b], "dk": got["dk"][c:e], "dv": got["dv"][c:e]}, ref)


def guarded(rows, width, seed):
    """(matrix inside a larger buffer, the buffer, a copy of what it holds): 3 rows in front and behind, 8 columns at the sides."""
    g = torch.Generator().manual_seed(seed)
    whole = torch.randn(rows + 6, width + 16, generator=g).to(torch.bfloat16).cuda()
    return whole[3:3 + rows, 8:8 + width], whole, whole.clone()


@pytest.mark.parametrize("name", ["swapped", "negative", "far", "descending", "huge", "constant"])
@pytest.mark.parametrize("kind", ["plain", "causal"])
def test_damaged_offsets(name, kind):
    """Offsets out of order: every gradient element is written, nothing beside them, the same bits twice, and the documents that a
    search over the damaged list still finds - all, for a damage behind the last of them - are right."""
    from image_generator_amd import ops
    docs, each = 40, 60
    T = docs * each
    good = offsets([each] * docs)
    bad = good.clone()
    if name == "swapped":
        bad[20], bad[21] = good[21], good[20]
    elif name == "negative":
        bad[20], bad[21] = T, -5
    elif name == "far":
        bad[30] = T + 100000
    elif name == "descending":
        bad = good.flip(0).contiguous()
    elif name == "huge":
        bad[-1] = 2 ** 31 - 1
    else:
        bad[:] = 7
    heads, d = 2, 32
    q, k, v, do = (t.cuda() for t in inputs(T, T, heads, heads, d, 34))
    how = dict(heads=heads, q_offsets=bad.cuda(), causal=kind == "causal")
    results = []
    for _ in range(2):
        out, lse = ops.doc_attention_fwd(q, k, v, **how)
        held = [guarded(T, heads * d, 40 + i) for i in range(3)]
        for m, whole, copy in held:
            m.fill_(float("nan"))
            copy[3:3 + T, 8:8 + heads * d] = float("nan")
        ops.doc_attention_bwd(do, q, k, v, out, lse, dq=held[0][0], dk=held[1][0], dv=held[2][0], **how)
        torch.cuda.synchronize()
        for m, whole, copy in held:
            assert bool(torch.isfinite(m).all())                            # every element written
            whole[3:3 + T, 8:8 + heads * d] = float("nan")
            assert torch.equal(whole.nan_to_num(0.0), copy.nan_to_num(0.0))      # and none beside them
        results.append((out, lse))
        assert bool(torch.isfinite(out).all())
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    if name in ("far", "huge") and kind == "plain":
        # up to the damage the list ascends: documents well in front of it are found by any search
        keep = torch.arange(0, 28 * each)
        x = tuple(t.cpu() for t in (q, k, v, do))
        got = run(*x, heads=heads, q_offsets=bad)
        check(got, reference(*x, heads, heads, good, good), {n: keep for n in ("out", "dq", "dk", "dv")})
