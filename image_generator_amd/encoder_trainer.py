"""Contrastive pre-training step of the text encoder: the build's counterpart of the hot loop in
/root/reference/encoder/train_encoder.py:83-110.

Step order kept from the reference: tokenised captions -> `TextEncoder` in training mode (pooled, L2-normalised) ->
`ContrastiveLoss` against the image embeddings -> backward -> AdamW (train_encoder.py:42-49: lr for the encoder, 0.1 lr
for the loss's log-temperature, torch's default weight decay 1e-2, no gradient clipping).

What is different on purpose:
  * the image tower (`encoder/image_encoder.py`: a pretrained CLIP ViT fetched by name) is not part of this package; the
    step takes its output, the image embeddings, as an input and returns their gradient for whoever owns that tower;
  * bf16 compute with fp32 masters instead of fp16 autocast + GradScaler (train_encoder.py:51,103-109).  What the
    GradScaler also does - leave every parameter untouched when a gradient is not finite - is kept: the optimizer's norm
    covers all gradients (the temperature's included), its update skips on a non-finite one and counts the skip, and the
    temperature's own update is gated by the same device value.  No host synchronisation;
  * every matrix product, the attention (mask and dropout inside the flash kernels), the normalisations, the loss and
    the parameter update run in libmi355_denoiser.so; the update is `optim.TensorAdamW`, two launches for all tensors,
    which also write the bf16 operand copies the next forward pass multiplies with.  `state_bits=8` holds its moments in
    8 bits;
  * `train_step_packed` takes captions without padding (tokens one behind another, documents by offsets) through
    `TextEncoder.forward_packed`.
"""
from __future__ import annotations

import torch

from ._lib import lib, check
from .ops import F32, _stream
from .optim import TensorAdamW


class ContrastiveTrainer:
    def __init__(self, text_encoder, criterion, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        self.enc, self.crit = text_encoder, criterion
        self.lr, self.betas, self.eps, self.wd = lr, betas, eps, weight_decay
        self.t = 0
        dev = next(text_encoder.parameters()).device
        if dev.type != "cuda":
            raise RuntimeError("ContrastiveTrainer: parameters must live on the HIP device (no CPU path)")
        named = [(n, p) for n, p in text_encoder.named_parameters() if p.requires_grad]
        self.names, self.params = [n for n, _ in named], [p for _, p in named]
        # the loss's single scalar: AdamW in a few one-element tensor ops, lr 0.1 x the encoder's (train_encoder.py:42-49),
        # gated by the optimizer's norm, in which its gradient counts
        self.temp = [p for p in criterion.parameters() if p.requires_grad]
        self.temp_m = [torch.zeros_like(p) for p in self.temp]
        self.temp_v = [torch.zeros_like(p) for p in self.temp]
        self.opt = TensorAdamW(self.params, lr, betas, eps, weight_decay, state_bits=state_bits, watched=[p.numel() for p in self.temp],
                               fp32_betas=state_bits == 32, device=dev)
        self.state = self.opt.state            # [0] = norm of the step's gradients (no clipping: only its finiteness is used)
        if state_bits == 32:
            self._moments = self.opt.split(self.opt.m), self.opt.split(self.opt.v)
            self.m, self.v = (list(views) for views in self._moments)
        self.step_count = 0

    def train_step(self, input_ids, attention_mask, image_embeds):
        """Returns (loss, gradient of the loss with respect to image_embeds)."""
        return self._train_step(lambda: self.enc(input_ids, attention_mask, return_pooled=True), image_embeds)

    def train_step_packed(self, input_ids, offsets, image_embeds):
        """`train_step` on captions without padding: input_ids [tokens], offsets int32 [captions + 1]."""
        return self._train_step(lambda: self.enc.forward_packed(input_ids, offsets, return_pooled=True), image_embeds)

    def _train_step(self, encode, image_embeds):
        self.enc.train()
        img = image_embeds.detach().to(F32).requires_grad_(True)
        for p in self.params:
            p.grad = None
        for p in self.temp:
            p.grad = None
        loss = self.crit(encode(), img)
        loss.backward()
        packs = self.enc._train_packs()
        copies = [packs[n].w16 if n in packs else None for n in self.names]
        if self.opt.moved() or [c is not None and c.data_ptr() for c in copies] != [c is not None and c.data_ptr() for c in self.opt.copies]:
            self.opt.set_copies(copies)
        tgrads = [None if p.grad is None else p.grad.to(F32).contiguous() for p in self.temp]
        o = self.opt
        if o.bits == 32:
            self._take_moments()
        o.betas, o.eps, o.wd, o.t = self.betas, self.eps, self.wd, self.t
        o.step([None if p.grad is None else p.grad.to(F32) for p in self.params], lr=self.lr, watched=tgrads)
        self.t = o.t
        s = _stream()
        for pk in packs.values():        # the data-gradient operands of the next step
            check(lib.mi355_transpose_bf16(pk.w16.data_ptr(), pk.w16_t.data_ptr(), 1, pk.n, pk.k, s), "transpose")
        self.enc.operands_current()
        self._temperature_step(tgrads)
        self.step_count += 1
        return loss.detach(), img.grad

    def _take_moments(self):
        """Moments that a program put into `m` and `v` (a checkpoint's, say) go where the optimizer holds them."""
        for name, views in zip("mv", self._moments):
            held = getattr(self, name)
            if len(held) != len(views):
                raise ValueError(f"ContrastiveTrainer: {len(held)} moments of {len(views)} parameters")
            if any(x is not y for x, y in zip(held, views)):
                for x, y in zip(held, views):
                    if x is not y:
                        y.copy_(x.reshape(y.shape))
                setattr(self, name, list(views))

    def _temperature_step(self, tgrads):
        b1, b2 = self.betas
        lr = self.lr * 0.1
        bc1, bc2 = 1 - b1 ** self.t, 1 - b2 ** self.t
        ok = torch.isfinite(self.state[0])                      # device value: nothing moves on a non-finite step
        with torch.no_grad():
            for p, g, m, v in zip(self.temp, tgrads, self.temp_m, self.temp_v):
                if g is None:
                    continue
                g = torch.where(ok, g, torch.zeros_like(g))
                m_new = b1 * m + (1 - b1) * g
                v_new = b2 * v + (1 - b2) * g * g
                p_new = p * (1 - lr * self.wd) - lr * (m_new / bc1) / ((v_new / bc2).sqrt() + self.eps)
                m.copy_(torch.where(ok, m_new, m))
                v.copy_(torch.where(ok, v_new, v))
                p.copy_(torch.where(ok, p_new, p))

    def skipped_steps(self) -> int:
        """Steps whose gradients were not finite and that therefore changed nothing (host synchronisation)."""
        return self.opt.skipped_steps()
