"""CPU: the largest sizes that the embedding and document-attention entries take, one step past them, and what lies in between."""


def err():
    from image_generator_amd._lib import lib
    return lib.mi355_last_error().decode()


def test_documents_up_to_2_30():
    """The lookup estimates where a token's document is in fp32: 2^31 documents times (nearly) 1 would pass the largest int."""
    from image_generator_amd._lib import lib

    def fwd(docs):
        return lib.mi355_doc_attention_fwd(16, 16, 16, 16, 16, 16, 16, docs, None, None, 0.0, 0, 0, 4, 4, 2, 2, 32, 64, 64, 64, 64, 1.0, 0.0, 0, None, 0, None)

    def bwd(docs):
        return lib.mi355_doc_attention_bwd(*[16] * 9, 16, 16, docs, None, None, 0.0, 0, 0, 4, 4, 2, 2, 32, *[64] * 8, 1.0, 0.0, 0, None, 0, None)
    for docs in ((1 << 30) + 1, 2 ** 31 - 2):
        assert fwd(docs) == -1 and "document" in err()
        assert bwd(docs) == -1 and "document" in err()
        assert lib.mi355_doc_attention_bwd_workspace_bytes(4, 4, 2, 2, 32, docs, 0) == 0
    assert lib.mi355_doc_attention_bwd_workspace_bytes(4, 4, 2, 2, 32, 1 << 30, 0) > 0


def test_embedding_rows_element_by_element():
    """Odd widths take a thread for each element, and a launch has fewer than 2^32 threads in whole workgroups of 256."""
    from image_generator_amd._lib import lib
    rows = lambda n, width, out=16: lib.mi355_embedding_fwd(16, 1, n, 16, 0, 4, width, 1.0, out, 1, None)  # noqa: E731
    grad = lambda n, width: lib.mi355_embedding_bwd(16, 1, n, 16, 1, 4, width, 1.0, 16, 0, 16, 0, None)  # noqa: E731
    n, width = 65537, 65535                                  # 2^32 - 1 elements
    assert n * width == 2 ** 32 - 1
    assert rows(n, width) == -1 and "2^32" in err()
    assert lib.mi355_embedding_bwd_workspace_bytes(n, 4, width) == 0
    assert grad(n, width) == -1 and "2^32" in err()
    assert grad(n - 1, width) == -1 and "workspace" in err()      # the largest below


def test_caps_whose_reciprocal_is_no_number():
    """Below 2^-126, 1 / cap is infinite and a score of 0 would be 0 times it."""
    from image_generator_amd._lib import lib
    for cap in (1e-45, 2.0 ** -127, 1e-39):
        assert lib.mi355_doc_attention_fwd(16, 16, 16, 16, 16, 16, 16, 1, None, None, cap, 0, 0, 4, 4, 2, 2, 32, 64, 64, 64, 64, 1.0, 0.0, 0, None, 0,
                                           None) == -1 and "cap" in err()
        assert lib.mi355_doc_attention_bwd(*[16] * 9, 16, 16, 1, None, None, cap, 0, 0, 4, 4, 2, 2, 32, *[64] * 8, 1.0, 0.0, 0, None, 0, None) == -1 and "cap" in err()
    assert lib.mi355_doc_attention_fwd(None, 16, 16, None, None, 16, 16, 1, None, None, 2.0 ** -126, 0, 0, 0, 4, 2, 2, 32, 64, 64, 64, 64, 1.0, 0.0, 0, None, 0,
                                       None) == 0


def test_a_parameter_of_another_size_is_refused():
    """A gradient has its parameter's shape; a parameter cut short where it lies would have the step read past that gradient."""
    import numpy as np
    import pytest
    import torch
    from image_generator_amd._lib import host
    p, other = torch.zeros(8), torch.zeros(3)
    to, sizes = np.empty(2, dtype=np.int64), np.array([3, 8], dtype=np.int64)
    words = lambda g: host().gradient_words([None, g], [other, p], 0, to.ctypes.data, sizes.ctypes.data)  # noqa: E731
    assert words(torch.zeros(8)) == 1                        # (on no device)
    p.data = p.data[:5]
    with pytest.raises(ValueError, match="parameter 1 has become 5 elements"):
        words(torch.zeros(5))
    assert words(None) == -1
