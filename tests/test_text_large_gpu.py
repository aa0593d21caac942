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
