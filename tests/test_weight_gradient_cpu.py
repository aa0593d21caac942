"""CPU: sizes and refusals of the weight gradient whose partial sums are added in order."""


def test_workspace_and_refusals():
    from image_generator_amd._lib import lib
    err = lambda: lib.mi355_last_error().decode()  # noqa: E731
    dense = lambda M, k, n: (M, 1, 1, k, n, 1, 1, 0, 1, 1)  # noqa: E731
    assert lib.mi355_wgrad_ordered_bytes(*dense(31, 8, 16)) == 0                      # one tile of rows: nothing to split
    need = lib.mi355_wgrad_ordered_bytes(*dense(4096, 128, 256))
    each = 4 * (128 * 256 + 256)
    assert need > each and need % each == 0
    assert lib.mi355_wgrad_ordered_bytes(*dense(64, 7, 16)) == -1 and lib.mi355_wgrad_ordered_bytes(4, 8, 8, 8, 8, 5, 1, 0, 8, 8) == -1
    call = lambda dy=16, dw=16, db=None, shape=dense(4096, 128, 256), ws=16, size=need: lib.mi355_wgrad_bf16_ordered(  # noqa: E731
        dy, 16, dw, db, *shape, 0, ws, size, None)
    assert call(dy=None) == -1 and "null" in err()
    assert call(dw=None) == -1 and "null" in err()
    assert call(shape=dense(4096, 12, 256)) == -1 and "multiples of 8" in err()
    assert call(size=need - 1) == -1 and "workspace" in err()
    assert call(ws=None) == -1 and "workspace" in err()
    assert call(ws=24) == -1 and "aligned" in err()
