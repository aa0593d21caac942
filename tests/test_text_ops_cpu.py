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
    assert lib.mi355_embedding_bwd(16, 1, 100, 16, 1, (1 << 26) + 1, 8, 1.0, 16, 0, 16, 1 << 40, None) == -1 and "2^26" in err()


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


def test_doc_attention_refusals():
    from image_generator_amd import ops
    from image_generator_amd._lib import lib
    q, off = torch.zeros(4, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.doc_attention_fwd(q, q, q, heads=2, q_offsets=off)
    with pytest.raises(RuntimeError, match="slopes"):
        ops.doc_attention(q, q, q, heads=2, q_offsets=off, slopes=torch.ones(2, requires_grad=True))
    err = lambda: lib.mi355_last_error().decode()  # noqa: E731

    def fwd(docs=1, prefix=None, cap=0.0, causal=0, Tq=4, Tk=4, Hq=2, Hkv=2, D=32, ld=64, ldo=64, drop=0.0, ptr=16, ws=16, ws_bytes=1 << 30, off=16):
        return lib.mi355_doc_attention_fwd(ptr, ptr, ptr, ptr, 16, off, off, docs, prefix, None, cap, causal, 0, Tq, Tk, Hq, Hkv, D, ld, ld, ld, ldo,
                                           1.0, drop, 0, ws, ws_bytes, None)

    for kw, why in ((dict(docs=0), "document"), (dict(Tq=-1), "document"), (dict(Hq=3), "multiple"), (dict(D=36), "multiple of 8"),
                    (dict(D=136), "128"), (dict(prefix=16), "prefix"), (dict(cap=-1.0), "cap"), (dict(cap=2000.0), "cap"), (dict(ld=(1 << 23) + 8), "strides"), (dict(cap=float("nan")), "cap"),
                    (dict(drop=1.0), "dropout"), (dict(ld=60), "strides"), (dict(ldo=32), "strides"), (dict(ptr=8), "aligned"),
                    (dict(ptr=None), "null"), (dict(off=None), "null"), (dict(ws=None, Tk=5000), "workspace"), (dict(ws_bytes=0, Tk=5000), "workspace"),
                    (dict(Tq=1 << 29), "2^30"), (dict(docs=2 ** 31 - 1), "document"), (dict(ld=-64), "strides")):
        assert fwd(**kw) == -1 and why in err(), (kw, err())
    assert fwd(Tq=0) == 0

    def bwd(ld=64, ldd=64, ptr=16, ws=16, ws_bytes=1 << 30, prefix=None):
        return lib.mi355_doc_attention_bwd(ptr, ptr, ptr, ptr, ptr, 16, ptr, ptr, ptr, 16, 16, 1, prefix, None, 0.0, 0, 0, 4, 4, 2, 2, 32, ld, ld,
                                           ld, ld, ld, ldd, ldd, ldd, 1.0, 0.0, 0, ws, ws_bytes, None)

    for kw, why in ((dict(ld=4), "strides"), (dict(ldd=32), "overlap"), (dict(ptr=24), "aligned"), (dict(ptr=None), "null"),
                    (dict(ws_bytes=8), "workspace"), (dict(prefix=16), "prefix")):
        assert bwd(**kw) == -1 and why in err(), (kw, err())
    assert lib.mi355_doc_attention_bwd_workspace_bytes(-1, 4, 2, 2, 32, 1, 0) == 0 and lib.mi355_doc_attention_fwd_workspace_bytes(4, 4, 3, 2, 32, 1) == 0


def test_host_extension_refusals():
    """The native checks turn every bad call into a Python error."""
    import numpy as np
    from image_generator_amd._lib import host
    h = host()
    for fn in (h.doc_attention_fwd, h.doc_attention_bwd, h.embedding_fwd, h.embedding_bwd, h.gradient_words, h.places, h.bump, h.bind):
        with pytest.raises(TypeError):
            fn()
    with pytest.raises(TypeError, match="tensor"):
        h.embedding_fwd(3, 4, 1.0, True, -1, 0)
    with pytest.raises(KeyError):
        h.bind({}, print)
    with pytest.raises(TypeError, match="list"):
        h.places((), 0, True)
    ts = [torch.zeros(3), torch.zeros(0), torch.ones(2)]
    at = np.empty(3, dtype=np.int64)
    assert h.places(ts, at.ctypes.data, True) is False and at.tolist() == [t.data_ptr() for t in ts]
    assert h.places(ts, at.ctypes.data, False) is False
    ts[2].data = torch.ones(2)
    assert h.places(ts, at.ctypes.data, False) is True
    assert h.gradient_words([None, None], ts[:2], 0, at.ctypes.data) == -1 and at.tolist()[:2] == [0, 0]
    assert h.gradient_words([None, ts[1]], ts[:2], 0, at.ctypes.data) == 1          # on no device
    with pytest.raises(ValueError, match="gradients"):
        h.gradient_words([None], ts, 0, at.ctypes.data)
    with pytest.raises(TypeError, match="tensor"):
        h.gradient_words([3], ts[:1], 0, at.ctypes.data)
    before = ts[0]._version
    h.bump(ts)
    assert ts[0]._version == before + 1
    with torch.inference_mode():
        h.bump([torch.zeros(2)])


def test_host_extension_argument_errors():
    from image_generator_amd import ops
    q, off = torch.zeros(4, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.doc_attention_fwd(q, q, q, heads="2", q_offsets=off)
    with pytest.raises(TypeError):
        ops.doc_attention_fwd(q, None, q, heads=2, q_offsets=off)
    with pytest.raises(RuntimeError, match="not"):
        ops.embedding_fwd(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), out_dtype=torch.float16)
