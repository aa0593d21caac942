"""Sizes at which the loops of the text operators take their later turns, against plain torch operations on the same device."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def test_embedding_of_nearly_2_32_elements():
    """The largest call of an odd width: elements beyond 2^31, bytes beyond 2^32, exact (a factor of 1 rounds nothing)."""
    from image_generator_amd import ops
    n, width = 65537, 65533
    g = torch.Generator(device=D).manual_seed(1)
    table = torch.randn(5, width, generator=g, device=D).to(BF)
    ids = torch.randint(0, 5, (n,), generator=g, device=D, dtype=torch.int32)
    ids[-1], ids[7] = 5, -1                                   # outside
    out = ops.embedding_fwd(ids, table)
    for a in range(0, n, 8192):
        part = ids[a:a + 8192]
        ok = (part >= 0) & (part < 5)
        want = table[part.clamp(0, 4).long()]
        got = out[a:a + 8192]
        assert bool((got[ok] == want[ok]).all()) and bool(torch.isnan(got[~ok]).all()), a
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_norm_over_many_runs(bits):
    """25 million elements, three to six runs for every wave of the norm, ragged ends, bf16 and fp32 gradients, one that is None.

    The norm is an fp64 sum: one rounding to fp32, 2^-24.  A first moment is (1 - b1) c g and a second (1 - b2) (c g)^2, with c, 1 - b
    and up to three products rounded in 32-bit states: 8 steps of 2^-24; a scale of 8-bit states is the fp64 value rounded."""
    from image_generator_amd.optim import BLOCK, TensorAdamW
    g = torch.Generator(device=D).manual_seed(3)
    shapes = [(9000001,), (4096, 2048), (7,), (5000003,), (257, 1009), (2300000,), (3,)]
    bf16, none = {1, 5}, 4
    ps = [torch.randn(s, generator=g, device=D) * 0.05 for s in shapes]
    # the later a tensor, the larger its gradients: a run that is counted twice or not at all shows
    gs = [torch.randn(s, generator=g, device=D) * 2.0 ** i for i, s in enumerate(shapes)]
    gs = [None if i == none else x.to(BF) if i in bf16 else x for i, x in enumerate(gs)]
    before = [p.clone() for p in ps]
    opt = TensorAdamW(ps, lr=1e-3, weight_decay=0.0, max_grad_norm=1.0, state_bits=bits)
    opt.step(gs)
    norm = sum(float(x.double().square().sum()) for x in gs if x is not None) ** 0.5
    assert abs(opt.grad_norm() - norm) <= 2.0 ** -23 * norm
    c = 1.0 / (norm + 1e-6)
    for i, (p, x) in enumerate(zip(ps, gs)):
        a, b = opt.starts[i], opt.starts[i + 1]
        if x is None:
            assert torch.equal(p, before[i])
            continue
        m = 0.1 * c * x.double().flatten()
        v = 0.001 * (c * x.double().flatten()).square()
        if bits == 32:
            for held, want in ((opt.m, m), (opt.v, v)):
                held = held[a * BLOCK:a * BLOCK + x.numel()].double()
                assert bool(((held - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()), i
        else:
            pad = torch.zeros((b - a) * BLOCK, dtype=F64, device=D)
            for held, want in ((opt.m_scales, m.abs()), (opt.u_scales, v.sqrt())):
                pad.zero_()
                pad[:x.numel()] = want
                top = pad.view(-1, BLOCK).amax(1)
                assert bool(((held[a:b].double() - top).abs() <= 2 * 2.0 ** -24 * top).all()), i
        # one step of Adam is lr by the sign, but for eps beside sqrt(v / (1 - b2)) = |c g| and some sixteen roundings
        size = c * x.double().flatten().abs()
        moved = (before[i].double() - p.double()).flatten()
        bound = 1e-3 * (16 * 2.0 ** -24 + 1e-8 / size.clamp(min=1e-30)) + 2.0 ** -24 * before[i].double().abs().flatten()
        assert bool(((moved - 1e-3 * x.double().flatten().sign()).abs() <= bound)[size > 1e-12].all()), i


@pytest.mark.parametrize("kind", ["uniform", "one", "skewed"])
def test_table_gradient_of_many_tiles(kind):
    """200 001 ids: 98 tiles, so the prefix sums of a bin carry over from its first 64; bounds of test_embedding_gpu."""
    from test_embedding_gpu import _grad_ref, _ids
    from image_generator_amd import ops
    n, rows, width, scale = 200001, 5003, 20, 0.5
    ids = _ids(kind, n, rows)
    ids[::1000] = -1
    dy = torch.randn(n, width, generator=torch.Generator().manual_seed(4)).to(BF)
    got = ops.embedding_bwd(ids.to(D), dy.to(D), rows, scale)
    ref, mag, count = _grad_ref(ids, dy, rows, scale)
    assert bool(((got.cpu().double() - ref).abs() <= (count + 1) * 2.0 ** -24 * mag).all())
    assert torch.equal(got, ops.embedding_bwd(ids.to(D), dy.to(D), rows, scale))


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("over", [False, True])
def test_rows_on_either_side_of_half_the_cache(out, over):
    """An output of 128 MB and one a row larger, which is stored past the caches: gathering and rounding gives the same bits."""
    from image_generator_amd import ops
    width = 1024
    n = (128 << 20) // (width * (2 if out == BF else 4)) + (1 if over else 0)
    g = torch.Generator(device=D).manual_seed(5)
    table = torch.randn(3001, width, generator=g, device=D)
    ids = torch.randint(0, 3001, (n,), generator=g, device=D)
    ids[n // 2] = 3001
    got = ops.embedding_fwd(ids, table, 1.0, out)
    want = table[ids.clamp(max=3000)].to(out)
    ok = ids < 3001
    assert torch.equal(got[ok], want[ok]) and bool(torch.isnan(got[~ok]).all())
    again = ops.embedding_fwd(ids, table, 1.0, out)
    assert torch.equal(again[ok], got[ok])
