"""Weight gradients of a launch of their own (`ops.wgrad`): pixel splits added in their order, so equal calls return equal bits.

Reference: the same sums in fp64.  A product of two bf16 values is exact in fp32, so what an fp32 result is off by is its
additions' roundings, at most one half step each: (terms + splits) 2^-24 sum |dy x|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = "cuda:0"
BF = torch.bfloat16


def _operands(M, cin, cout, ksize, B, H, W, stride, seed):
    g = torch.Generator().manual_seed(seed)
    Ho, Wo = (H + stride - 1) // stride, (W + stride - 1) // stride
    rows = M if ksize == 1 and B is None else B * Ho * Wo
    x = torch.randn(M if B is None else B * H * W, cin, generator=g).to(BF)
    dy = torch.randn(rows, cout, generator=g).to(BF)
    return x, dy, (None if B is None else (B, H, W, Ho, Wo))


def _columns(x, ksize, geom, stride):
    if geom is None:
        return x.double()[:, None, :]
    B, H, W, Ho, Wo = geom
    img = x.double().view(B, H, W, -1).permute(0, 3, 1, 2)
    col = torch.nn.functional.unfold(img, ksize, padding=ksize // 2, stride=stride)            # [B][C k k][Ho Wo]
    return col.view(B, img.shape[1], ksize * ksize, Ho * Wo).permute(0, 3, 2, 1).reshape(B * Ho * Wo, ksize * ksize, -1)


CASES = [  # rows, in, out, kernel, B, H, W, stride
    (0, 8, 64, 3, 4, 8, 8, 1), (0, 64, 8, 3, 4, 8, 8, 1), (0, 16, 24, 3, 3, 10, 6, 1), (0, 32, 32, 3, 2, 16, 16, 2),
    (4096, 128, 128, 1, None, 0, 0, 1), (1601, 200, 168, 1, None, 0, 0, 1), (31, 8, 8, 1, None, 0, 0, 1), (130, 8, 328, 1, None, 0, 0, 1),
]


@pytest.mark.parametrize("case", CASES)
def test_equal_calls_return_equal_bits_and_the_sums(case):
    from image_generator_amd import ops
    from image_generator_amd._lib import lib
    M, cin, cout, ksize, B, H, W, stride = case
    x, dy, geom = _operands(M, cin, cout, ksize, B, H, W, stride, seed=5)
    col = _columns(x, ksize, geom, stride)
    want = torch.einsum("mo,mtc->otc", dy.double(), col)
    size = torch.einsum("mo,mtc->otc", dy.double().abs(), col.abs())
    xd, dyd = x.to(D), dy.to(D)
    args = (dy.shape[0], 1, 1, cin, cout, ksize, stride, 0, 1, 1) if geom is None else (*geom[:3], cin, cout, ksize, stride, 0, *geom[3:])
    split = lib.mi355_wgrad_ordered_bytes(*args) > 0
    assert split == (dy.shape[0] >= 128)                   # (what the cases are for)
    runs = []
    for _ in range(12):
        db = torch.full((cout,), float("nan"), device=D)
        out = torch.full((cout, ksize * ksize, cin), float("nan"), device=D)
        ops.wgrad(dyd, xd, cin, cout, ksize, stride, geom=geom, out=out, dbias=db)
        runs.append((out, db))
    torch.cuda.synchronize()
    for out, db in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(db, runs[0][1])
    out, db = (t.cpu().double() for t in runs[0])
    terms = dy.shape[0] + 64
    assert bool(((out - want).abs() <= terms * 2.0 ** -24 * size).all())
    assert bool(((db - dy.double().sum(0)).abs() <= terms * 2.0 ** -24 * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("shift", [0, 1])
def test_into_a_buffer_that_the_caller_zeroed(shift):
    """accumulate=2: the weights are written, the bias added to what another launch left; gradients at any 4-byte address."""
    from image_generator_amd import ops
    x, dy, geom = _operands(0, 8, 64, 3, 4, 8, 8, 1, seed=6)
    xd, dyd = x.to(D), dy.to(D)
    plain_db = torch.empty(64, device=D)
    plain = ops.wgrad(dyd, xd, 8, 64, 3, geom=geom, dbias=plain_db)
    flat = torch.zeros(64 * 72 + 64 + 8, device=D)
    out, db = flat[shift:shift + 64 * 72].view(64, 9, 8), flat[shift + 64 * 72:shift + 64 * 73]
    db.fill_(3.0)
    ops.wgrad(dyd, xd, 8, 64, 3, geom=geom, out=out, accumulate=2, dbias=db)
    assert torch.equal(out, plain) and torch.equal(db, plain_db + 3.0)
    assert bool((flat[:shift] == 0).all()) and bool((flat[shift + 64 * 73:] == 0).all())


def test_captured_and_replayed():
    from image_generator_amd import ops
    x, dy, geom = _operands(0, 8, 64, 3, 4, 8, 8, 1, seed=7)
    xd, dyd = x.to(D), dy.to(D)
    db, out = torch.empty(64, device=D), torch.empty(64, 9, 8, device=D)
    ops.wgrad(dyd, xd, 8, 64, 3, geom=geom, out=out, dbias=db)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.wgrad(dyd, xd, 8, 64, 3, geom=geom, out=out, dbias=db)
    g = torch.Generator().manual_seed(8)
    for _ in range(4):
        dyd.copy_(torch.randn(dy.shape, generator=g).to(BF))
        out.fill_(float("nan"))
        db.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want_db = torch.empty(64, device=D)
        want = ops.wgrad(dyd, xd, 8, 64, 3, geom=geom, dbias=want_db)
        assert torch.equal(out, want) and torch.equal(db, want_db)


def test_equal_training_steps_leave_equal_weights():
    """Small denoiser, gradients of padded convolutions among them: ten runs of three steps, the same bits."""
    from image_generator_amd.trainer import DenoiserTrainer
    from image_generator_amd.unet import UNet2DConditionModel, DenoiserConfig
    g = torch.Generator().manual_seed(29)
    lat, noise = torch.randn(4, 4, 8, 8, generator=g).to(D), torch.randn(4, 4, 8, 8, generator=g).to(D)
    ts, ctx = torch.randint(0, 1000, (4,), generator=g).to(D), torch.randn(4, 16, 64, generator=g).to(D).to(BF)
    first = None
    for _ in range(10):
        torch.manual_seed(0)
        unet = UNet2DConditionModel(DenoiserConfig.small()).to(D)
        tr = DenoiserTrainer(unet, lr=1e-3, max_grad_norm=0.0)       # (the clip factor of a single process is a sum in any order)
        grads = []
        for _ in range(3):
            tr.train_step(lat, noise, ts, ctx)
            grads.append(tr.full_grad())
        if first is None:
            first = grads
        for a, b in zip(first, grads):
            assert torch.equal(a, b)


def test_the_register_staged_kernel_too():
    """The kernel for operands of 2 GB and more, taken by an environment switch that a process reads once: a process of its own."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
import test_weight_gradient_gpu as t
from image_generator_amd import ops
from image_generator_amd._lib import lib
for case in t.CASES:
    M, cin, cout, ksize, B, H, W, stride = case
    x, dy, geom = t._operands(M, cin, cout, ksize, B, H, W, stride, seed=9)
    col = t._columns(x, ksize, geom, stride)
    want, size = torch.einsum("mo,mtc->otc", dy.double(), col), torch.einsum("mo,mtc->otc", dy.double().abs(), col.abs())
    xd, dyd = x.to(t.D), dy.to(t.D)
    runs = []
    for _ in range(8):
        db = torch.empty(cout, device=t.D)
        runs.append((ops.wgrad(dyd, xd, cin, cout, ksize, stride, geom=geom, dbias=db), db))
    assert all(torch.equal(a, runs[0][0]) and torch.equal(b, runs[0][1]) for a, b in runs), case
    out, db = (v.cpu().double() for v in runs[0])
    terms = dy.shape[0] + 64
    assert bool(((out - want).abs() <= terms * 2.0 ** -24 * size).all()), case
    assert bool(((db - dy.double().sum(0)).abs() <= terms * 2.0 ** -24 * dy.double().abs().sum(0)).all()), case
assert lib.mi355_wgrad_ordered_bytes(4096, 1, 1, 128, 128, 1, 1, 0, 1, 1) > 0
print("done")
""" % (root, os.path.join(root, "tests"))
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "MI355_WGRAD_V1": "1"}, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), (r.returncode, r.stdout[-500:], r.stderr[-2000:])
