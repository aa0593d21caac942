"""AdamW over a list of tensors: the whole step is two launches, whatever their number and sizes.

The counterpart of `torch.optim.AdamW` in /root/reference/encoder/train_encoder.py:42-49 for parameters that are tensors of
their own (the denoiser's, one flat buffer, have `trainer.FusedAdamW`).  Moments are fp32, or 8 bits each with an fp32 scale
for every 256 elements of a tensor: 2.03 instead of 8 bytes of state for a parameter, and as many fewer to move each step.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from ._lib import lib, check, host
from .ops import BF16, F32, PinnedRing, _stream

BLOCK = 256            # elements that share a scale
_WG_BLOCKS = 8         # blocks per workgroup of the update
_HYPER = 16            # doubles in front of the gradient addresses in the step's upload


class TensorAdamW:
    """params: fp32 contiguous tensors on one HIP device.  copies: bf16 tensors (or None) that receive each updated parameter.
    max_grad_norm: global norm to clip to (0: none).  A step whose gradients are not finite changes nothing and is counted
    (`skipped_steps`), as in `trainer.FusedAdamW`; like there, its number still advances the bias correction.

    watched: sizes of further gradients, stepped by someone else, that count in the norm (and in the test for finite values); they
    follow as `bind(..., watched=[...])`.  device: where they are, if there is no parameter.

    fp32_betas: a new gradient's weights are 1 - beta of betas rounded to fp32, as `trainer.FusedAdamW` forms them (1 - 0.999 is
    7e-6 off then), instead of 1 - beta rounded itself, and any eps >= 0 is taken, as there (with eps = 0, an element that never had a
    gradient becomes NaN); an option of 32-bit states.

    `step(grads)` uploads what changes (addresses, bias corrections) and launches.  For a captured graph: `bind(grads)` before
    the capture and before every replay, `apply()` inside it; the gradients stay the caller's to keep."""

    def __init__(self, params, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_grad_norm=0.0, state_bits=32, copies=None,
                 watched=(), fp32_betas=False, device=None):
        self.params = list(params)
        if not self.params and device is None:
            raise ValueError("TensorAdamW: no parameters")
        # (0 / 0 behind a smaller eps: untouched rows have m = v = 0)
        if not all(0 <= b < 1 for b in betas) or not eps >= (0.0 if fp32_betas and state_bits == 32 else 2.0 ** -126):
            raise ValueError(f"TensorAdamW: betas {tuple(betas)} not below 1, or eps {eps} not a normal fp32 number above 0")
        if state_bits not in (8, 32):
            raise ValueError(f"TensorAdamW: states of 8 or 32 bits, not {state_bits}")
        dev = self.params[0].device if self.params else torch.device(device)
        if dev.type != "cuda" or dev.index is None:
            raise RuntimeError("TensorAdamW: parameters must live on the HIP device (no CPU path)")
        for p in self.params:
            if p.device != dev:
                raise ValueError(f"TensorAdamW: parameters on {dev} and {p.device}")
            if p.dtype != F32 or not p.is_contiguous():
                raise ValueError("TensorAdamW: parameters must be contiguous fp32 tensors")
        _disjoint(self.params, "parameters")
        self._shapes = [p.shape for p in self.params]
        self._sizes = np.array([p.numel() for p in self.params], dtype=np.int64)
        self.lr, self.betas, self.eps, self.wd, self.max_norm = lr, tuple(betas), eps, weight_decay, max_grad_norm
        self.bits, self.device, self.t = state_bits, dev, 0
        self.fp32_betas = fp32_betas
        self.watched = list(watched)
        blocks = [-(-p.numel() // BLOCK) for p in self.params]
        self.starts = [0]
        for b in blocks:
            self.starts.append(self.starts[-1] + b)
        total = self.starts[-1]
        room = max(total, 1)                          # (an address for the launch, also where only watched gradients count)
        if state_bits == 32:
            self.m, self.v = (torch.zeros(room * BLOCK, dtype=F32, device=dev) for _ in range(2))
        else:
            self.m_codes = torch.zeros(room * BLOCK, dtype=torch.int8, device=dev)
            self.u_codes = torch.zeros(room * BLOCK, dtype=torch.uint8, device=dev)
            self.m_scales, self.u_scales = (torch.zeros(room, dtype=F32, device=dev) for _ in range(2))
        wgs = np.array([-(-b // _WG_BLOCKS) for b in blocks + [-(-n // BLOCK) for n in self.watched]], dtype=np.int64)
        places = np.empty((int(wgs.sum()), 2), dtype=np.int32)           # (tensor, first block within it) of each workgroup
        places[:, 0] = np.repeat(np.arange(len(wgs)), wgs)
        places[:, 1] = (np.arange(len(places)) - np.repeat(np.cumsum(wgs) - wgs, wgs)) * _WG_BLOCKS
        self._map = torch.from_numpy(places).to(dev)
        self._elements = float(sum(p.numel() for p in self.params))
        self._partial = torch.zeros(int(lib.mi355_multi_adamw_parts()), dtype=torch.float64, device=dev)
        self.state = torch.zeros(2, dtype=F32, device=dev)          # norm of the last step, skipped steps
        n = len(self.params) + len(self.watched)
        self._upload = torch.zeros(_HYPER + n, dtype=torch.int64, device=dev)
        self._ring = PinnedRing(lambda: torch.zeros(_HYPER + n, dtype=torch.int64).pin_memory(), 8)
        self._kept, self._bound = [], False
        self.set_copies(copies)

    def set_copies(self, copies=None):
        """The bf16 tensors that receive the updated parameters (one for each parameter, or None in its place)."""
        for p, shape in zip(self.params, self._shapes):
            if p.device != self.device or p.dtype != F32 or p.shape != shape or not p.is_contiguous():
                raise ValueError(f"TensorAdamW: a parameter has become {p.dtype} {tuple(p.shape)} on {p.device}")
        copies = [None] * len(self.params) if copies is None else list(copies)
        if len(copies) != len(self.params):
            raise ValueError(f"TensorAdamW: {len(copies)} copies of {len(self.params)} parameters")
        for p, c in zip(self.params, copies):
            if c is not None and (c.dtype != BF16 or c.device != self.device or c.numel() != p.numel() or not c.is_contiguous()):
                raise ValueError("TensorAdamW: a copy must be a contiguous bf16 tensor of its parameter's size on its device")
        _disjoint([c for c in copies if c is not None], "copies")
        self.copies = copies
        self._written = [t for t in self.params + copies if t is not None]
        self._places = np.empty(len(self._written), dtype=np.int64)
        host().places(self._written, self._places.ctypes.data, True)
        self._places_at = self._places.ctypes.data
        rows = np.zeros((len(self.params) + len(self.watched), 4), dtype=np.int64)
        rows[:len(copies), 0] = self._places[:len(copies)]               # (the parameters come first in `_written`)
        rows[:len(copies), 1] = [0 if c is None else c.data_ptr() for c in copies]
        rows[:len(copies), 2] = self._sizes
        rows[:len(copies), 3] = self.starts[:-1]
        rows[len(copies):, 2] = self.watched
        self._recs = torch.from_numpy(rows).to(self.device)

    def moved(self):
        """Whether a parameter or copy lies elsewhere than `set_copies` found it."""
        return host().places(self._written, self._places_at, False)

    def bind(self, grads=None, lr=None, watched=None):
        """Begin a step: gradients (default: the parameters' own `.grad`; None leaves a parameter alone) and learning rate.
        Addresses and scalars go to the device in one asynchronous copy on the current stream."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("TensorAdamW: bind() before the capture (and before every replay); only apply() can be captured")
        self._on_device()
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"TensorAdamW: {len(grads)} gradients of {len(self.params)} parameters")
        if self.moved():
            raise RuntimeError("TensorAdamW: a parameter or copy has moved to other memory (set_copies(copies) takes the new places)")
        watched = [None] * len(self.watched) if watched is None else list(watched)
        if len(watched) != len(self.watched):
            raise ValueError(f"TensorAdamW: {len(watched)} watched gradients, {len(self.watched)} announced")
        for n, g in zip(self.watched, watched):
            if g is not None and (g.numel() != n or g.device != self.device or g.dtype not in (F32, BF16) or not g.is_contiguous()):
                raise ValueError("TensorAdamW: a watched gradient must be a contiguous fp32 or bf16 tensor of the announced size")
        slot, kept = self._ring.acquire(), []
        words = (self.params, self.device.index, slot.data_ptr() + 8 * _HYPER, self._sizes.ctypes.data)
        if host().gradient_words(grads, *words) >= 0:
            grads, kept = self._contiguous(grads)
            host().gradient_words(grads, *words)
        if lr is not None:
            self.lr = lr
        self.t += 1
        b1, b2 = self.betas
        c1, c2 = 1 - b1 ** self.t, 1 - b2 ** self.t
        hyper = (self.lr, b1, b2, self.eps, self.wd, c1, c2, self.max_norm or 0.0, 1 - self.lr * self.wd, self.lr / c1, 1 / math.sqrt(c2),
                 *(1 - float(np.float32(b)) if self.fp32_betas else 1 - b for b in self.betas))
        h = slot.numpy()
        h[:len(hyper)].view("float64")[:] = hyper
        for i, g in enumerate(watched, _HYPER + len(grads)):
            h[i] = 0 if g is None else g.data_ptr() | (g.dtype == BF16)
        self._upload.copy_(slot, non_blocking=True)
        self._ring.copied()
        self._ring.release()
        self._kept, self._bound = kept, True

    def _contiguous(self, grads):
        """(gradients with contiguous copies of those that are not, the copies); refuses what is no gradient of its parameter."""
        out, kept = [], []
        for i, (p, g) in enumerate(zip(self.params, grads)):
            if g is not None:
                if g.shape != p.shape or g.device != self.device:
                    raise ValueError(f"TensorAdamW: gradient {i} is {tuple(g.shape)} on {g.device}, its parameter {tuple(p.shape)} on {self.device}")
                if g.dtype not in (F32, BF16):
                    raise ValueError(f"TensorAdamW: gradient {i} is {g.dtype}, neither fp32 nor bf16")
                if not g.is_contiguous():
                    g = g.contiguous()
                    kept.append(g)
            out.append(g)
        return out, kept

    def apply(self):
        """The launches of the step that `bind` began (capturable)."""
        capturing = torch.cuda.is_current_stream_capturing()
        if not self._bound:
            raise RuntimeError("TensorAdamW: apply() without bind()")
        self._bound = capturing                     # a captured step is bound again by the host before each replay
        self._on_device()
        m, ms, v, us = (self.m, None, self.v, None) if self.bits == 32 else (self.m_codes, self.m_scales, self.u_codes, self.u_scales)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        check(lib.mi355_multi_adamw_step(self._recs.data_ptr(), self._upload.data_ptr() + 8 * _HYPER, self._map.data_ptr(),
                                         self._map.shape[0], self.bits, m.data_ptr(), ptr(ms), v.data_ptr(), ptr(us),
                                         self._partial.data_ptr(), self._upload.data_ptr(), self.state.data_ptr(), self._elements,
                                         _stream()), "multi_adamw")
        host().bump(self._written)

    def step(self, grads=None, lr=None, watched=None):
        self.bind(grads, lr, watched)
        self.apply()

    def _on_device(self):
        current = torch._C._cuda_getDevice()
        if current != self.device.index:
            raise RuntimeError(f"TensorAdamW: parameters on {self.device}, the current device is {current}")

    def moments(self):
        """(first, second) moments as flat fp32 tensors, each parameter padded to a multiple of 256 elements: the states
        themselves (32 bits), or what their codes stand for (8 bits, newly written).  `split` cuts them up."""
        if self.bits == 32:
            return self.m, self.v
        self._on_device()
        m, v = (torch.empty(self.starts[-1] * BLOCK, dtype=F32, device=self.device) for _ in range(2))
        check(lib.mi355_adamw_moments(self.m_codes.data_ptr(), self.m_scales.data_ptr(), self.u_codes.data_ptr(), self.u_scales.data_ptr(),
                                      self.starts[-1], m.data_ptr(), v.data_ptr(), _stream()), "adamw_moments")
        return m, v

    def split(self, flat):
        """Views of a flat moment tensor in the parameters' shapes."""
        return [flat[s * BLOCK:s * BLOCK + p.numel()].view(p.shape) for s, p in zip(self.starts, self.params)]

    _BUFFERS = {32: ("m", "v"), 8: ("m_codes", "m_scales", "u_codes", "u_scales")}

    def state_dict(self):
        out = {"step": self.t, "state_bits": self.bits, "sizes": [p.numel() for p in self.params]}
        out.update((n, getattr(self, n).detach().cpu()) for n in self._BUFFERS[self.bits])
        return out

    def load_state_dict(self, sd):
        if sd["state_bits"] != self.bits or list(sd["sizes"]) != [p.numel() for p in self.params]:
            raise ValueError("TensorAdamW: the state is of other parameters or another number of bits")
        for n in self._BUFFERS[self.bits]:
            getattr(self, n).copy_(sd[n])
        self.t = int(sd["step"])

    def grad_norm(self):
        """Norm of the last step's gradients before clipping (host synchronisation)."""
        return float(self.state[0])

    def skipped_steps(self):
        """Steps that changed nothing because a gradient was not finite (host synchronisation)."""
        return int(self.state[1])


def _disjoint(tensors, what):
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError(f"TensorAdamW: {what} share memory")
