"""AdamW over a list of tensors against fp64 steps of the same states.

Tolerances.  States of 32 bits: a moment is a product, a product and a sum (up to four fp32 roundings of terms no larger than
|b1 m| + |(1 - b1) g|, and the weights' own): 8 x 2^-24 of those magnitudes for m and of v for v.  The quotient m / denom then
adds half of v's error, the rounding of 1 - b2^t (0.007 at the tested step: 2^-25 / 0.007 = 72 x 2^-24, half of it in the root)
and six roundings of its own: 50 x 2^-24; p is off by that much of the update and 3 x 2^-24 of p.
States of 8 bits are compared as whole numbers: the kernel steps them in fp64, as the reference here does, and they are equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 2.0 ** -24
BLK = 256
SETS = {
    "one": [(1,)],
    "small": [(1,), (3,), (255,), (256,), (257,), (4, 320), (2049,)],
    "mixed": [(768, 96), (768,), (96,), (33, 65), (5000,), (2048,), (4, 3, 3, 8), (1,)],
}


def _make(name, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    shapes = SETS[name]
    ps = [torch.randn(s, generator=g) * 0.05 for s in shapes]
    gs = [torch.randn(s, generator=g) * 10.0 ** (-1 - i % 4) for i, s in enumerate(shapes)]
    if offset:                                            # views at addresses that are no multiple of 16 bytes
        def put(x):
            flat = torch.zeros(x.numel() + offset, dtype=x.dtype)
            flat[offset:] = x.flatten()
            return flat.cuda()[offset:].view(x.shape)
        return [put(p) for p in ps], gs, put
    return [p.cuda() for p in ps], gs, lambda x: x.cuda()


def _codes(x, n):
    """(codes, scale) of the magnitudes of one tensor, fp64."""
    pad = torch.zeros(-(-x.numel() // BLK) * BLK, dtype=F64)
    pad[:x.numel()] = x.flatten()
    b = pad.view(-1, BLK)
    s = b.amax(1).float()
    s = torch.where(s >= 2.0 ** -126, s, torch.zeros_like(s))
    inv = torch.where(s > 0, 1 / s.double(), torch.zeros(len(s), dtype=F64))
    # the nearest whole number, the lower one of a tie
    return (b * inv[:, None]).sqrt().mul(n).add(0.5 - 2.0 ** -30).floor().clamp(max=n), s, b


class Ref8:
    def __init__(self, ps):
        self.p = [p.cpu().double() for p in ps]
        nb = [-(-p.numel() // BLK) for p in ps]
        self.mq = [torch.zeros(n, BLK, dtype=F64) for n in nb]
        self.uq = [torch.zeros(n, BLK, dtype=F64) for n in nb]
        self.ms = [torch.zeros(n) for n in nb]
        self.us = [torch.zeros(n) for n in nb]

    def step(self, grads, t, lr, b1, b2, eps, wd, clip):
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads if g is not None))
        c = min(1.0, clip / (norm + 1e-6)) if clip else 1.0
        for i, g in enumerate(grads):
            if g is None:
                continue
            n = g.numel()
            g = g.double().flatten() * c
            m0 = (self.mq[i] * self.mq[i].abs() / 16129 * self.ms[i].double()[:, None]).view(-1)[:n]
            u0 = (self.uq[i].square() / 65025 * self.us[i].double()[:, None]).view(-1)[:n]
            m = b1 * m0 + (1 - b1) * g
            u = (b2 * u0.square() + (1 - b2) * g.square()).sqrt()
            upd = lr / (1 - b1 ** t) * m / (u / math.sqrt(1 - b2 ** t) + eps)
            self.p[i] = (self.p[i].flatten() * (1 - lr * wd) - upd).view(self.p[i].shape).float().double()
            q, self.ms[i], _ = _codes(m.abs(), 127)
            sign = torch.zeros(q.numel(), dtype=F64)
            sign[:n] = torch.sign(m)
            self.mq[i] = q * sign.view(q.shape)
            q, self.us[i], b = _codes(u, 255)
            self.uq[i] = torch.where((b > 0) & (self.us[i][:, None] > 0), q.clamp(min=1), q)


HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("clip", [0.0, 0.3])
@pytest.mark.parametrize("offset,g16", [(0, False), (0, True), (1, False), (3, True)])
def test_8_bit_states(name, clip, offset, g16):
    from image_generator_amd.optim import TensorAdamW
    ps, _, put = _make(name, 1, offset)
    copies = [put(torch.zeros(p.shape, dtype=BF)) for p in ps]
    opt = TensorAdamW(ps, state_bits=8, max_grad_norm=clip, copies=copies, **HYPER)
    ref = Ref8(ps)
    for t in range(1, 5):
        gs = _make(name, 10 + t)[1]
        gs = [g.to(BF) if g16 else g for g in gs]
        if t == 3 and len(gs) > 2:
            gs[1] = None                                  # left alone
            gs[2] = torch.zeros_like(gs[2])
        opt.step([None if g is None else put(g) for g in gs])
        ref.step(gs, t, HYPER["lr"], 0.9, 0.999, 1e-8, 0.05, clip)
        for i, p in enumerate(ps):
            a, b = opt.starts[i], opt.starts[i + 1]
            assert torch.equal(opt.m_codes[a * BLK:b * BLK].cpu().double(), ref.mq[i].view(-1)), (t, i)
            assert torch.equal(opt.u_codes[a * BLK:b * BLK].cpu().double(), ref.uq[i].view(-1)), (t, i)
            # a scale is the fp32 rounding of an fp64 value, which may sit at a border of its own
            for mine, theirs in ((opt.m_scales, ref.ms), (opt.u_scales, ref.us)):
                assert ((mine[a:b].cpu() - theirs[i]).abs() <= 2 * EPS * theirs[i]).all()
            # lr / sqrt(1 - b2^t) m / u bounds an update by lr * (1 - b1) / sqrt(1 - b2) < 4 lr; its quotient has five fp32 roundings
            assert ((p.cpu().double() - ref.p[i]).abs() <= 3 * EPS * ref.p[i].abs() * t + 8 * EPS * 4 * HYPER["lr"] * t).all(), (t, i)
            assert torch.equal(copies[i], p.to(BF)) or (t == 3 and i == 1)


def test_moments_are_what_the_codes_stand_for():
    from image_generator_amd.optim import TensorAdamW
    ps, gs, put = _make("mixed")
    opt = TensorAdamW(ps, state_bits=8)
    opt.step([put(g) for g in gs])
    m, v = (x.cpu().double() for x in opt.moments())
    mq, uq = opt.m_codes.cpu().double(), opt.u_codes.cpu().double()
    ms, us = (s.cpu().double().repeat_interleave(BLK) for s in (opt.m_scales, opt.u_scales))
    assert ((m - mq * mq.abs() / 16129 * ms).abs() <= 2 * EPS * m.abs()).all()
    assert ((v - (uq.square() / 65025 * us).square()).abs() <= 2 * EPS * v).all()
    for (a, p) in zip(opt.split(opt.moments()[0]), ps):
        assert a.shape == p.shape
    # the codes hold the first step's moments to within half a step of the code: (q + 1/2)^2 / q^2 - 1 relative to the value
    for i, g in enumerate(gs):
        want = 0.1 * g.double().flatten()
        a = opt.starts[i] * BLK
        err, step = (m[a:a + g.numel()] - want).abs(), ms[a:a + g.numel()] * (mq[a:a + g.numel()].abs() + 0.5) / 16129
        assert (err <= step * (1 + 1e-5)).all()


@pytest.mark.parametrize("name", list(SETS))
@pytest.mark.parametrize("clip,offset,g16", [(0.0, 0, False), (0.3, 0, True), (0.3, 1, False)])
def test_32_bit_states(name, clip, offset, g16):
    from image_generator_amd.optim import TensorAdamW
    ps, gs, put = _make(name, 2, offset)
    gs = [g.to(BF) if g16 else g for g in gs]
    opt = TensorAdamW(ps, max_grad_norm=clip, **HYPER)
    opt.m.normal_(generator=torch.Generator("cuda").manual_seed(3)).mul_(1e-2)
    opt.v.uniform_(1e-6, 1e-3, generator=torch.Generator("cuda").manual_seed(4))
    opt.t = 6
    m0, v0, p0 = ([x.cpu().double() for x in opt.split(opt.m)], [x.cpu().double() for x in opt.split(opt.v)], [p.cpu().double() for p in ps])
    opt.step([put(g) for g in gs])
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(opt.grad_norm() - norm) <= 2 * EPS * norm
    c = min(1.0, clip / (norm + 1e-6)) if clip else 1.0
    lr, wd, t = HYPER["lr"], HYPER["weight_decay"], 7
    for i, g in enumerate(gs):
        g = g.double() * c
        m, v = 0.9 * m0[i] + 0.1 * g, 0.999 * v0[i] + 1e-3 * g * g
        mag = (0.9 * m0[i]).abs() + (0.1 * g).abs()
        tm, tv = 8 * EPS * mag, 8 * EPS * v
        den = v.sqrt() / math.sqrt(1 - 0.999 ** t) + 1e-8
        upd = lr / (1 - 0.9 ** t) * m / den
        tu = lr / (1 - 0.9 ** t) * tm / den + upd.abs() * 50 * EPS
        p = p0[i] * (1 - lr * wd) - upd
        assert ((opt.split(opt.m)[i].cpu().double() - m).abs() <= tm).all()
        assert ((opt.split(opt.v)[i].cpu().double() - v).abs() <= tv).all()
        assert ((ps[i].cpu().double() - p).abs() <= tu + 3 * EPS * p0[i].abs()).all()


def test_32_bit_states_equal_the_per_tensor_update():
    """Without clipping, with its weights 1 - beta: the bits of `mi355_adamw_step` on each tensor."""
    from image_generator_amd._lib import lib, check
    from image_generator_amd.ops import _stream
    from image_generator_amd.optim import TensorAdamW
    shapes = [(768, 96), (96,), (4, 320), (5000,)]
    g = torch.Generator().manual_seed(7)
    mine = [torch.randn(s, generator=g).cuda() for s in shapes]
    theirs = [p.clone() for p in mine]
    c_mine, c_theirs = ([torch.zeros(s, dtype=BF, device="cuda") for s in shapes] for _ in range(2))
    ms, vs = ([torch.zeros(s, device="cuda") for s in shapes] for _ in range(2))
    opt = TensorAdamW(mine, copies=c_mine, fp32_betas=True, **HYPER)
    hyper, state = torch.zeros(9), torch.zeros(2, device="cuda")
    for t in range(1, 6):
        gs = [(torch.randn(s, generator=g) * 0.1).cuda() for s in shapes]
        opt.step(gs)
        for k, x in enumerate((HYPER["lr"], 0.9, 0.999, 1e-8, 0.05, 1 - 0.9 ** t, 1 - 0.999 ** t, 0.0, 1.0)):
            hyper[k] = x
        h = hyper.cuda()
        for p, q, m, v, c in zip(theirs, gs, ms, vs, c_theirs):
            check(lib.mi355_adamw_step(p.data_ptr(), q.data_ptr(), m.data_ptr(), v.data_ptr(), c.data_ptr(), h.data_ptr(), state.data_ptr(),
                                       p.numel(), _stream()))
    for a, b in zip(mine + c_mine + opt.split(opt.m) + opt.split(opt.v), theirs + c_theirs + ms + vs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_step_with_a_gradient_that_is_not_finite_changes_nothing(bits, bad):
    from image_generator_amd.optim import TensorAdamW
    ps, gs, put = _make("mixed")
    opt = TensorAdamW(ps, state_bits=bits, max_grad_norm=1.0)
    opt.step([put(g) for g in gs])
    before = [p.clone() for p in ps] + [x.clone() for x in opt.moments()]
    gs[3][2, 1] = bad
    opt.step([put(g) for g in gs])
    assert all(torch.equal(a, b) for a, b in zip(before, ps + list(opt.moments()))) and opt.skipped_steps() == 1
    gs[3][2, 1] = 0
    opt.step([put(g) for g in gs])
    assert opt.skipped_steps() == 1 and not torch.equal(before[0], ps[0])


def test_zero_gradients_and_tiny_ones():
    """Zero moments stay zero codes (no division by their scale); gradients whose squares leave fp32 are still stepped."""
    from image_generator_amd.optim import TensorAdamW
    p = torch.ones(600, device="cuda")
    opt = TensorAdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8)
    opt.step([torch.zeros(600, device="cuda")])
    assert (p == 1).all() and (opt.u_codes == 0).all() and (opt.u_scales == 0).all()
    g = torch.full((600,), 1e-30, device="cuda")
    opt.step([g])
    m, v = opt.moments()
    assert torch.isfinite(p).all() and (opt.u_codes[:600] == 255).all() and (opt.u_scales > 0).all()
    opt.step([torch.full((600,), 1e-44, device="cuda")])
    assert torch.isfinite(p).all() and torch.isfinite(opt.moments()[0]).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_step_replays_like_eager(bits):
    from image_generator_amd.optim import TensorAdamW
    ps, gs, put = _make("mixed")
    qs = [p.clone() for p in ps]
    grads = [put(g) for g in gs]
    a, b = TensorAdamW(ps, state_bits=bits, max_grad_norm=0.5), TensorAdamW(qs, state_bits=bits, max_grad_norm=0.5)
    a.step(grads)
    b.step(grads)
    a.bind(grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.apply()
        with pytest.raises(RuntimeError, match="capture"):
            a.bind(grads)
    for k in range(4):
        if k:
            a.bind(grads)
        for g in grads:
            g.normal_(std=0.1)
        graph.replay()
        b.step(grads)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(ps + list(a.moments()), qs + list(b.moments()))), k


def test_state_dict_resumes_with_the_same_bits():
    from image_generator_amd.optim import TensorAdamW
    for bits in (8, 32):
        ps, gs, put = _make("mixed")
        a = TensorAdamW(ps, state_bits=bits)
        for _ in range(2):
            a.step([put(g) for g in gs])
        qs = [p.clone() for p in ps]
        b = TensorAdamW(qs, state_bits=bits)
        b.load_state_dict(a.state_dict())
        for o in (a, b):
            o.step([put(g) for g in gs])
        assert all(torch.equal(x, y) for x, y in zip(ps, qs))
        with pytest.raises(ValueError):
            TensorAdamW(qs[:2], state_bits=bits).load_state_dict(a.state_dict())


def test_many_steps_follow_the_32_bit_run():
    """200 steps on a noisy quadratic: parameters of 8-bit states stay near those of 32-bit ones (a smoke test of the held format:
    the distance is measured against the distance travelled)."""
    from image_generator_amd.optim import TensorAdamW
    target = torch.randn(4096, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    ends = []
    for bits in (8, 32):
        p = torch.zeros(4096, device="cuda")
        opt = TensorAdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
        g = torch.Generator("cuda").manual_seed(2)
        for _ in range(200):
            opt.step([p - target + 0.1 * torch.randn(4096, device="cuda", generator=g)])
        ends.append(p.clone())
    assert float((ends[0] - ends[1]).norm() / ends[1].norm()) < 0.1


def test_parameter_versions_move():
    from image_generator_amd.optim import TensorAdamW
    p = torch.ones(8, device="cuda", requires_grad=True)
    p.grad = torch.ones(8, device="cuda")
    v = p._version
    TensorAdamW([p]).step()
    assert p._version > v


def test_refusals():
    from image_generator_amd.optim import TensorAdamW
    p, q = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    for bad, kw in (([], {}), ([p, p], {}), ([p, p[4:]], {}), ([p.half()], {}), ([torch.zeros(4, 4, device="cuda").t()[:3]], {}),
                    ([p], dict(state_bits=16)), ([p, q], dict(copies=[None])), ([p], dict(copies=[torch.zeros(8, device="cuda")])),
                    ([p], dict(copies=[torch.zeros(7, device="cuda", dtype=BF)]))):
        with pytest.raises(ValueError):
            TensorAdamW(bad, **kw)
    opt = TensorAdamW([p, q])
    for grads in ([p.clone()], [p.clone(), torch.zeros(9, device="cuda")], [p.clone().double(), None], [torch.zeros(8), None]):
        with pytest.raises(ValueError):
            opt.step(grads)
    with pytest.raises(RuntimeError):
        opt.apply()


def test_parameter_that_moved_is_refused():
    """The addresses of parameters and copies live on the device: a step after one of them moved would write to its old place."""
    from image_generator_amd.optim import TensorAdamW
    p, c = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda", dtype=BF)
    opt = TensorAdamW([p], copies=[c], lr=0.5, weight_decay=0.0)
    old, p.data = p.data, torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="moved"):
        opt.step([torch.ones(8, device="cuda")])
    opt.set_copies([c])
    opt.step([torch.ones(8, device="cuda")])
    assert (old == 0).all() and opt.t == 1 and torch.allclose(p, torch.full_like(p, 0.5)) and torch.equal(c, p.to(BF))
    p.data = torch.ones(9, device="cuda")
    with pytest.raises(ValueError, match="become"):
        opt.set_copies([c])


@pytest.mark.parametrize("kw", [dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(eps=0.0), dict(eps=1e-40), dict(eps=float("nan"))])
def test_refused_hyperparameters(kw):
    from image_generator_amd.optim import TensorAdamW
    with pytest.raises(ValueError, match="betas"):
        TensorAdamW([torch.zeros(8, device="cuda")], **kw)
