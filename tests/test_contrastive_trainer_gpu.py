"""What `ContrastiveTrainer` takes: parameters whose storage is replaced between steps, and the calls around it."""
import pytest
import torch

from test_packed_encoder_gpu import D, fixture

pytestmark = pytest.mark.gpu


def trainer(dropout=0.0, temperature=True, **kw):
    """temperature=False: held fixed, for steps that are compared bit by bit (its gradient is a sum in any order)."""
    from image_generator_amd.encoder_trainer import ContrastiveTrainer
    from image_generator_amd.loss import ContrastiveLoss
    z, enc, ids, off, padded, mask = fixture(dropout)
    crit = ContrastiveLoss(0.07).to(D)
    crit.requires_grad_(temperature)
    tr = ContrastiveTrainer(enc, crit, lr=1e-3, **kw)
    return tr, enc, (padded, mask, torch.from_numpy(z["img"]).to(D)), (ids, off, torch.from_numpy(z["img"]).to(D))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_may_move_between_steps(bits):
    """`p.data = x` for every parameter (the embedding and the norms have no bf16 copy): the same steps as without."""
    a, enc_a, _, step = trainer(state_bits=bits, temperature=False)
    b, enc_b, _, _ = trainer(state_bits=bits, temperature=False)
    a.train_step_packed(*step)
    b.train_step_packed(*step)
    old = [p.data for p in enc_b.parameters()]
    kept = [x.clone() for x in old]
    for p in enc_b.parameters():
        p.data = p.data.clone()
    for _ in range(2):
        a.train_step_packed(*step)
        b.train_step_packed(*step)
    assert a.t == b.t == 3
    for (n, p), q in zip(enc_a.named_parameters(), enc_b.parameters()):
        assert torch.equal(p, q), n
    assert all(torch.equal(x, y) for x, y in zip(old, kept))              # nothing was written to the old places
    named = dict(enc_b.named_parameters())
    for n, pk in enc_b._train_packs().items():
        assert torch.equal(pk.w16, named[n].detach().to(torch.bfloat16)), n


def test_a_step_that_raises_is_not_counted(monkeypatch):
    tr, enc, _, step = trainer()
    tr.train_step_packed(*step)

    def refuse(*a, **kw):
        raise ValueError("no")
    monkeypatch.setattr(tr.opt, "bind", refuse)
    with pytest.raises(ValueError, match="no"):
        tr.train_step_packed(*step)
    assert tr.t == 1 and tr.step_count == 1
    monkeypatch.undo()
    tr.train_step_packed(*step)
    assert tr.t == tr.opt.t == 2 and tr.step_count == 2


def test_eps_zero():
    """eps = 0, as before the optimizer over many tensors: a first step of every element with a gradient is lr, by its sign.

    The first step moves by lr sqrt(1 - b2) (1 - b1') / ((1 - b1) sqrt(1 - b2')), betas rounded to fp32 on one side: 2^-25 / 0.001 / 2 =
    1.5e-5 and 2^-25 / 0.1 = 3e-7 of it, and some ten roundings of 2^-24; the parameter's product with 1 - lr wd and the difference
    another 2^-23 of it."""
    tr, enc, _, step = trainer(eps=0.0)
    before = [p.detach().double() for p in enc.parameters()]
    tr.train_step_packed(*step)
    for (n, p), old in zip(enc.named_parameters(), before):
        seen = p.grad.abs() > 1e-12                      # (its square is a normal fp32 number)
        want = old * (1 - tr.lr * tr.wd) - tr.lr * p.grad.double().sign()
        off = (p.detach().double() - want).abs()
        assert bool((off <= tr.lr * 2.0 ** -15 + 2.0 ** -23 * old.abs())[seen].all()), n
    with pytest.raises(ValueError, match="eps"):
        trainer(eps=-1e-8)
    with pytest.raises(ValueError, match="eps"):
        trainer(eps=0.0, state_bits=8)                   # roots that are held as 0 divide by eps alone


def test_frozen_encoder():
    """Nothing of the encoder trains (the image tower's turn): the temperature moves, the image gradients come back."""
    from image_generator_amd.encoder_trainer import ContrastiveTrainer
    from image_generator_amd.loss import ContrastiveLoss
    for bits in (32, 8):
        z, enc, ids, off, padded, mask = fixture()
        enc.requires_grad_(False)
        img = torch.from_numpy(z["img"]).to(D)
        before = [p.detach().clone() for p in enc.parameters()]
        crit = ContrastiveLoss(0.07).to(D)
        temp = crit.log_temp.detach().clone()
        tr = ContrastiveTrainer(enc, crit, lr=1e-3, state_bits=bits)
        for step in (lambda x: tr.train_step(padded, mask, x), lambda x: tr.train_step_packed(ids, off, x)):
            loss, d_img = step(img)
            assert torch.isfinite(loss) and float(d_img.norm()) > 0
        assert not torch.equal(crit.log_temp.detach(), temp) and tr.skipped_steps() == 0
        assert tr.opt.grad_norm() == pytest.approx(abs(float(crit.log_temp.grad)), rel=1e-6)
        temp = crit.log_temp.detach().clone()
        bad = img.clone()
        bad[0, 0] = float("nan")
        tr.train_step(padded, mask, bad)
        assert tr.skipped_steps() == 1 and torch.equal(crit.log_temp.detach(), temp)
        assert all(torch.equal(x, p) for x, p in zip(before, enc.parameters()))
        crit.requires_grad_(False)
        loss, d_img = ContrastiveTrainer(enc, crit, lr=1e-3, state_bits=bits).train_step(padded, mask, img)
        assert torch.isfinite(loss) and float(d_img.norm()) > 0


def test_moments_put_back_by_hand():
    """`trainer.m` / `.v` are lists of the parameters' moments: entries or lists that a program puts in their place are stepped on."""
    a, enc_a, _, step = trainer(temperature=False)
    for _ in range(2):
        a.train_step_packed(*step)
    saved = [p.detach().clone() for p in enc_a.parameters()], [m.clone() for m in a.m], [v.cpu() for v in a.v]
    a.train_step_packed(*step)
    for whole in (True, False):
        b, enc_b, _, _ = trainer(temperature=False)
        with torch.no_grad():
            for p, x in zip(enc_b.parameters(), saved[0]):
                p.copy_(x)
        if whole:
            b.m, b.v = tuple(saved[1]), list(saved[2])
        else:
            for i, (m, v) in enumerate(zip(saved[1], saved[2])):
                b.m[i], b.v[i] = m, v
        b.t = 2
        b.train_step_packed(*step)
        for (n, p), q, m, k in zip(enc_a.named_parameters(), enc_b.parameters(), a.m, b.m):
            assert torch.equal(p, q) and torch.equal(m, k), n
    b.m = b.m[:-1]
    with pytest.raises(ValueError, match="moments"):
        b.train_step_packed(*step)


def test_optimizer_refuses_a_parameter_cut_short_where_it_lies():
    from image_generator_amd.optim import TensorAdamW
    p = torch.ones(4096, device=D)
    opt = TensorAdamW([p], lr=0.5, weight_decay=0.0)
    whole, p.data = p.data, p.data[:100]
    with pytest.raises(ValueError, match="has become 100 elements"):
        opt.step([torch.ones(100, device=D)])
    assert opt.t == 0 and bool((whole == 1).all())
    opt.step([None])
    p.data = whole
    opt.step([torch.ones(4096, device=D)])
    # the second step (one without a gradient counts), the first gradient: m = 0.1, v = 0.001
    assert torch.allclose(p, torch.full_like(p, 1 - 0.5 * (0.1 / (1 - 0.9 ** 2)) / (0.001 / (1 - 0.999 ** 2)) ** 0.5))
