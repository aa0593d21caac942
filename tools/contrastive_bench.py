"""Times the fused ContrastiveLoss (loss.py:16-28: forward + every gradient in one library call) at the reference's
encoder batch (train_encoder.py:180: 512 x 768) and the text encoder's pre-training step (run on the GPU box)."""
import sys, os, time
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from image_generator_amd.loss import ContrastiveLoss
from image_generator_amd.text_encoder import TextEncoder
from image_generator_amd.encoder_trainer import ContrastiveTrainer

d = "cuda:0"


def timeit(fn, iters=20):
    for _ in range(3):
        fn()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(iters):
        fn()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) / iters


for B in (64, 512):
    t, i = torch.randn(B, 768, device=d, requires_grad=True), torch.randn(B, 768, device=d, requires_grad=True)
    crit = ContrastiveLoss().to(d)
    dt = timeit(lambda: crit(t, i))          # the call computes the loss and all three gradients
    print(f"ContrastiveLoss B={B} D=768: {dt*1e6:8.1f} us per call ({6.0*B*B*768/dt/1e12:6.2f} TFLOP/s fp32, 5 launches)")

torch.manual_seed(0)
enc = TextEncoder().to(d)                     # the reference's default: 16384 x 768, 8 layers, 8 heads of 96
crit = ContrastiveLoss().to(d)
tr = ContrastiveTrainer(enc, crit)
B, T = 512, 64
ids = torch.randint(4, 16384, (B, T), device=d)
lens = torch.randint(8, T + 1, (B,), device=d)
mask = (torch.arange(T, device=d)[None, :] < lens[:, None]).long()
img = torch.nn.functional.normalize(torch.randn(B, 768, device=d), dim=-1)
dt = timeit(lambda: tr.train_step(ids, mask, img), iters=10)
flops = 3 * 8 * (2 * B * T * 768 * (3 * 768 + 768 + 2 * 3072) + 4 * B * T * T * 768)
print(f"encoder pre-training step B={B} T={T} (8 layers, dropout 0.2): {dt*1e3:7.2f} ms, {B/dt:8.0f} captions/s, "
      f"{flops/dt/1e12:6.1f} TFLOP/s bf16")
# the same captions without their padding rows
off = torch.cat((torch.zeros(1, dtype=torch.int64, device=d), lens.cumsum(0))).to(torch.int32)
packed = ids[mask.bool()]
dt = timeit(lambda: tr.train_step_packed(packed, off, img), iters=10)
print(f"the same without padding ({packed.numel()} of {B * T} rows): {dt*1e3:7.2f} ms, {B/dt:8.0f} captions/s")
