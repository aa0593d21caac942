"""CPU: what the embedding, optimizer and document-attention entry points refuse before anything reaches a GPU."""
import pytest
import torch


def test_embedding_refusals():
    from image_generator_amd import ops
    from image_generator_amd._lib import lib
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.embedding_fwd(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.embedding_bwd(torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8), 4)
    err = lambda: lib.mi355_last_error().decode()  # noqa: E731
    assert lib.mi355_embedding_fwd(None, 1, 3, None, 0, 4, 8, 1.0, None, 1, None) == -1 and "null" in err()
    assert lib.mi355_embedding_fwd(16, 1, 3, 16, 0, 0, 8, 1.0, 16, 1, None) == -1 and "empty" in err()
    assert lib.mi355_embedding_fwd(16, 1, 1 << 22, 16, 0, 4, 1024, 1.0, 16, 1, None) == -1 and "2^32" in err()
    assert lib.mi355_embedding_fwd(16, 1, 0, 16, 0, 4, 8, 1.0, 16, 1, None) == 0
    need = lib.mi355_embedding_bwd_workspace_bytes(100, 50, 8)
    assert need > 0 and lib.mi355_embedding_bwd_workspace_bytes(-1, 50, 8) == 0
    assert lib.mi355_embedding_bwd(16, 1, 100, 16, 1, 50, 8, 1.0, 16, 0, 16, need - 1, None) == -1 and "workspace" in err()
    assert lib.mi355_embedding_bwd(16, 1, 100, 16, 1, 50, 8, 1.0, 16, 0, 24, need, None) == -1 and "aligned" in err()
    assert lib.mi355_embedding_bwd(16, 1, 100, 16, 1, 50, 8, 1.0, None, 0, 16, need, None) == -1 and "null" in err()


def test_optimizer_refusals():
    from image_generator_amd.optim import TensorAdamW
    from image_generator_amd._lib import lib
    with pytest.raises(RuntimeError, match="no CPU path"):
        TensorAdamW([torch.zeros(4)])
    with pytest.raises(ValueError):
        TensorAdamW([])
    err = lambda: lib.mi355_last_error().decode()  # noqa: E731
    step = lambda bits, n, m, ms, partial=16: lib.mi355_multi_adamw_step(16, 16, 16, n, bits, m, ms, 16, ms, partial, 16, 16, 0.0, None)  # noqa: E731
    assert step(16, 1, 16, 16) == -1 and "8 or 32" in err()
    assert step(8, 1, 16, None) == -1 and "null" in err()
    assert step(32, 1, None, None) == -1 and step(32, 1, 16, None, None) == -1 and step(32, -1, 16, None) == -1
    assert step(32, 1, 8, None) == -1 and "aligned" in err()
    assert step(32, 0, 16, None) == 0
    assert lib.mi355_adamw_moments(16, 16, 16, 16, -1, 16, 16, None) == -1
    assert lib.mi355_adamw_moments(16, 16, 16, 16, 4, 8, 16, None) == -1 and lib.mi355_adamw_moments(None, 16, 16, 16, 4, 16, 16, None) == -1
