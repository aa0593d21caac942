"""Embedding rows and their table's gradient against fp64 sums of the same inputs.

Tolerances.  A row is one fp32 product rounded once: half a step of the output's type (bf16 2^-8, fp32 2^-24) plus the product's
own 2^-24.  A gradient element is a sum of c terms in fp32: each of at most c + 1 roundings (c additions, the scaling) is off by
2^-24 of a partial sum, and no partial sum exceeds S = sum |terms|, so |error| <= (c + 1) 2^-24 S |scale|, plus the output's
half step when it is bf16."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _ids(kind, n, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, rows, (n,), generator=g)
    if kind == "one":
        return torch.full((n,), rows - 1)
    if kind == "skewed":
        return (rows ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, rows - 1)
    if kind == "runs":                                   # the same id many times in a row, and every id in descending order
        return torch.arange(n).div(97, rounding_mode="floor").neg().remainder(rows)
    raise ValueError(kind)


def _grad_ref(ids, dy, rows, scale):
    ok = (ids >= 0) & (ids < rows)
    ref = torch.zeros(rows, dy.shape[1], dtype=torch.float64).index_add_(0, ids[ok], dy[ok].double()) * scale
    mag = torch.zeros(rows, dy.shape[1], dtype=torch.float64).index_add_(0, ids[ok], dy[ok].double().abs()) * abs(scale)
    return ref, mag, torch.bincount(ids[ok], minlength=rows)[:, None].double()


@pytest.mark.parametrize("n,rows,width,table,out,id32", [
    (1, 1, 8, F32, BF, False), (77, 16384, 768, F32, BF, False), (5, 3, 1, F32, F32, True), (130, 301, 33, BF, BF, False),
    (64, 50, 1000, BF, F32, True), (1023, 97, 260, F32, F32, False)])
def test_rows(n, rows, width, table, out, id32):
    from image_generator_amd import ops
    g = torch.Generator().manual_seed(1)
    w = torch.randn(rows, width, generator=g).to(table)
    ids = _ids("uniform", n, rows).to(torch.int32 if id32 else torch.int64)
    scale = 27.7
    got = ops.embedding_fwd(ids.cuda(), w.cuda(), scale, out).cpu()
    assert got.shape == (n, width) and got.dtype == out
    ref = w.double()[ids.long()] * float(torch.tensor(scale, dtype=F32))
    half = 2.0 ** -8 if out == BF else 2.0 ** -24
    assert ((got.double() - ref).abs() <= (half + 2.0 ** -23) * ref.abs()).all()


def test_rows_equal_the_lookup_followed_by_the_cast():
    """Scale 1 and a bf16 result: the same bits as gathering fp32 rows and rounding them."""
    from image_generator_amd import ops
    w = torch.randn(500, 96, device="cuda")
    ids = torch.randint(0, 500, (3, 41), device="cuda")
    assert torch.equal(ops.embedding_fwd(ids, w), ops.cast_bf16(torch.nn.functional.embedding(ids, w)))


def test_ids_out_of_range_and_special_values():
    from image_generator_amd import ops
    w = torch.randn(10, 8, device="cuda")
    w[3] = float("inf")
    ids = torch.tensor([0, -1, 10, 3, 2 ** 40, 9], device="cuda")
    out = ops.embedding_fwd(ids, w, 2.0, F32)
    assert torch.isnan(out[[1, 2, 4]]).all() and torch.isinf(out[3]).all()
    assert torch.equal(out[[0, 5]], w[[0, 9]] * 2)
    dy = torch.ones(6, 8, device="cuda")
    dy[1] = float("nan")                                  # an id out of range adds to nothing, whatever its gradient is
    dw = ops.embedding_bwd(ids, dy, 10)
    assert torch.equal(dw.sum(1).cpu(), torch.tensor([8., 0, 0, 8, 0, 0, 0, 0, 0, 8]))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 129, 1601, 4096, 8191, 8192, 8193, 12345])
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed", "runs"])
def test_table_gradient_over_lengths(n, kind):
    from image_generator_amd import ops
    rows, width, scale = 1009, 36, 0.75
    ids = _ids(kind, n, rows)
    dy = torch.randn(n, width, generator=torch.Generator().manual_seed(2)).to(BF)
    got = ops.embedding_bwd(ids.cuda(), dy.cuda(), rows, scale).cpu()
    ref, mag, count = _grad_ref(ids, dy, rows, scale)
    assert ((got.double() - ref).abs() <= (count + 1) * 2.0 ** -24 * mag).all()
    assert (got[count[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("rows,width,dtype,out,n", [
    (1, 4, BF, F32, 300), (2, 768, F32, F32, 40), (16384, 768, BF, F32, 5000), (300, 33, F32, F32, 9000), (70001, 20, BF, BF, 20000),
    (7, 1300, BF, F32, 30000), (130000, 8, F32, BF, 8193), (255, 257, BF, F32, 10000), (256, 256, BF, F32, 10000)])
def test_table_gradient_over_shapes(rows, width, dtype, out, n):
    from image_generator_amd import ops
    ids = _ids("skewed", n, rows, 3).to(torch.int32 if rows % 2 else torch.int64)
    dy = torch.randn(n, width, generator=torch.Generator().manual_seed(4)).to(dtype)
    got = ops.embedding_bwd(ids.cuda(), dy.cuda(), rows, 1.0, out).cpu()
    ref, mag, count = _grad_ref(ids.long(), dy, rows, 1.0)
    tol = (count + 1) * 2.0 ** -24 * mag
    if out == BF:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs()
    assert ((got.double() - ref).abs() <= tol).all()


def test_gradient_repeats_its_bits_and_takes_views():
    from image_generator_amd import ops
    ids = _ids("skewed", 20001, 500).cuda()
    dy = torch.randn(20001, 64, device="cuda", dtype=F32)
    a = ops.embedding_bwd(ids, dy, 500)
    for _ in range(3):
        assert torch.equal(a, ops.embedding_bwd(ids, dy, 500))
    wide = torch.empty(20001, 130, device="cuda")
    wide[:, 1:65] = dy                                    # not contiguous, rows not aligned to 16 bytes
    assert torch.equal(a, ops.embedding_bwd(ids, wide[:, 1:65], 500))
    flat = torch.empty(20001 * 64 + 1, device="cuda")
    flat[1:] = dy.view(-1)                                # contiguous at an odd address: the one-element path, the same sums
    assert torch.equal(a, ops.embedding_bwd(ids, flat[1:].view(20001, 64), 500))
    pairs = torch.stack((ids, ids + 1), 1)
    assert torch.equal(a, ops.embedding_bwd(pairs[:, 0], dy, 500))


def test_autograd_against_torch_and_differences():
    from image_generator_amd import ops
    g = torch.Generator().manual_seed(5)
    w = torch.randn(50, 24, generator=g).cuda().requires_grad_(True)
    ids = torch.randint(0, 50, (4, 9), generator=g).cuda()
    t = torch.randn(4, 9, 24, generator=g).cuda()
    (ops.embedding(ids, w, 3.0, F32) * t).sum().backward()
    ref = torch.zeros(50, 24, dtype=torch.float64).index_add_(0, ids.flatten().cpu(), t.cpu().double().view(-1, 24)) * 3.0
    assert (w.grad.cpu().double() - ref).abs().max() <= 37 * 2.0 ** -24 * ref.abs().max() * 3
    # the loss is linear in the table: a difference over a step of 1 is the gradient itself, up to the sum's rounding
    v, f = int(ids[0, 0]), lambda x: float((ops.embedding(ids, x, 3.0, F32) * t).double().sum())
    up = w.detach().clone()
    up[v, 7] += 1
    assert abs(f(up) - f(w.detach()) - float(w.grad[v, 7])) <= 1e-5 * (1 + abs(float(w.grad[v, 7])))


def test_empty_and_captured():
    from image_generator_amd import ops
    w = torch.randn(12, 8, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert ops.embedding_fwd(none, w).shape == (0, 8)
    assert (ops.embedding_bwd(none, torch.empty(0, 8, device="cuda"), 12) == 0).all()
    ids, dy = torch.randint(0, 12, (9000,), device="cuda"), torch.randn(9000, 8, device="cuda")
    ops.embedding_bwd(ids, dy, 12)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = ops.embedding_fwd(ids, w), ops.embedding_bwd(ids, dy, 12)
    for k in range(4):
        ids.copy_(torch.randint(0, 12, (9000,), device="cuda"))
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.embedding_fwd(ids, w)) and torch.equal(dw, ops.embedding_bwd(ids, dy, 12))


def test_another_stream():
    from image_generator_amd import ops
    ids, dy = torch.randint(0, 100, (9001,), device="cuda"), torch.randn(9001, 40, device="cuda")
    ref = ops.embedding_bwd(ids, dy, 100)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.embedding_bwd(ids, dy, 100)
    s.synchronize()
    assert torch.equal(got, ref)
