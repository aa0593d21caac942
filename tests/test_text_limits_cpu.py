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
