"""Score cap and distance bias of the text encoder: the same function on every path, kept by its state dict.

Two paths of one function agree as test_packed_encoder_gpu's padded and packed paths do: bf16 activations, 2e-2 relative L2 of states
and 0.1 of gradients; a path that leaves the options out is off by more than three times that."""
import io

import pytest
import torch

from test_packed_encoder_gpu import D, fixture, rel

pytestmark = pytest.mark.gpu


def set_options(enc, cap, bias):
    enc.score_cap = cap
    enc.distance_slopes = torch.tensor([1.0, 0.5, 0.25, 0.0], device=D) if bias else None


@pytest.mark.parametrize("cap,bias", [(0.05, False), (0.0, True), (0.5, True)])
def test_padded_paths_are_the_packed_one(cap, bias):
    _, enc, ids, off, padded, mask = fixture()
    enc.eval()
    with torch.no_grad():
        plain = enc(padded, mask, return_pooled=False)[mask], enc(padded, mask)
        set_options(enc, cap, bias)
        want = enc.forward_packed(ids, off, return_pooled=False), enc.forward_packed(ids, off)
        got = enc(padded, mask, return_pooled=False)[mask], enc(padded, mask)
        for a, b, c in zip(got, want, plain):
            assert rel(a, b) <= 2e-2
            if bias:
                assert rel(c, b) > 6e-2
        # no mask: every caption as long as the batch
        B, T = padded.shape
        whole = torch.arange(0, (B + 1) * T, T, dtype=torch.int32, device=D)
        assert rel(enc(padded, None, return_pooled=False).view(B * T, -1), enc.forward_packed(padded.view(-1), whole, return_pooled=False)) <= 2e-2


def test_padded_gradients_are_the_packed_ones():
    from image_generator_amd.loss import ContrastiveLoss
    z, enc, ids, off, padded, mask = fixture()
    enc.train()
    set_options(enc, 0.5, True)
    crit, img = ContrastiveLoss(0.07).to(D), torch.from_numpy(z["img"]).to(D)
    grads = []
    for run in (lambda: enc.forward_packed(ids, off), lambda: enc(padded, mask)):
        for p in enc.parameters():
            p.grad = None
        crit(run(), img).backward()
        grads.append({n: p.grad.clone() for n, p in enc.named_parameters()})
    for n, want in grads[0].items():
        if float(want.norm()) > 1e-6:
            assert rel(grads[1][n], want) <= 0.1, n


def test_a_mask_that_is_not_right_padded_is_still_marked():
    _, enc, _, _, padded, mask = fixture()
    enc.eval()
    set_options(enc, 0.5, True)
    holes = mask.clone()
    holes[1, 0] = False
    with torch.no_grad():
        got, want = enc(padded, holes), enc(padded, mask)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0])


def test_state_dict_keeps_them():
    from image_generator_amd.text_encoder import TextEncoder
    make = lambda: TextEncoder(vocab_size=300, embed_dim=96, num_layers=2, n_head=4, projection_dim=64, dropout=0.0)  # noqa: E731
    _, enc, ids, off, padded, mask = fixture()
    enc.eval()
    plain = enc.state_dict()
    assert not any("slopes" in k or "cap" in k for k in plain)
    set_options(enc, 0.5, True)
    f = io.BytesIO()
    torch.save(enc.state_dict(), f)
    f.seek(0)
    again = make()
    again.load_state_dict(torch.load(f, weights_only=True))
    again = again.to(D).eval()                              # the slopes move with the module
    with torch.no_grad():
        assert torch.equal(again(padded, mask), enc(padded, mask)) and torch.equal(again.forward_packed(ids, off), enc.forward_packed(ids, off))
    again.load_state_dict(plain)                            # the reference's keys: the options stay
    assert again.score_cap == 0.5 and torch.equal(again.distance_slopes, enc.distance_slopes)
    holder = torch.nn.ModuleDict({"text": make()})          # ... under a prefix too
    holder.load_state_dict({"text." + k: v for k, v in enc.state_dict().items()})
    assert holder["text"].score_cap == 0.5 and torch.equal(holder["text"].distance_slopes.cpu(), enc.distance_slopes.cpu())
    with pytest.raises(RuntimeError, match="nonsense"):
        make().load_state_dict({**plain, "nonsense": torch.zeros(1)})


def test_a_batch_without_tokens_is_refused():
    _, enc, ids, off, _, _ = fixture()
    with pytest.raises(ValueError, match="no tokens"):
        enc.forward_packed(ids[:0], torch.zeros_like(off))
