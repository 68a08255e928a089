"""CPU checks of what an attention call over packed sequences or the paged cache runs, by its sizes (the query function that the GPU
tests use to make sure that a case takes the kernel it is meant for)."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from iggt_official_amd import _C, build_ext

    build_ext.build(verbose=False)
    return _C.load()


def plan(lib, paged, requests, rows, keys, hq, hkv, dim):
    """(rows of a work item, key ranges), or the error code."""
    item, ranges = ctypes.c_int(), ctypes.c_int()
    rc = lib.iggt_seq_attn_plan(int(paged), requests, rows, keys, hq, hkv, dim, item, ranges)
    return rc or (item.value, ranges.value)


def test_plan_names_the_kernel_and_fits_the_scratch(lib):
    assert plan(lib, True, 1, 1, 1374, 16, 16, 64) == (16, 1)
    assert plan(lib, True, 2, 1374, 1374, 16, 16, 128)[0] == 256
    assert plan(lib, False, 40, 300, 300, 16, 16, 64) == (256, 1) and plan(lib, False, 1, 1374, 1374, 16, 16, 128)[0] == 128
    for paged in (False, True):
        size = lib.iggt_paged_attn_ws_bytes if paged else lib.iggt_packed_attn_ws_bytes
        for requests, rows, keys, hq, hkv, dim in ((1, 1, 100000, 16, 16, 64), (3, 40, 9000, 8, 2, 128), (1, 1374, 1374, 16, 16, 64), (2, 200, 20000, 1, 1, 128)):
            ranges = plan(lib, paged, requests, rows, keys, hq, hkv, dim)[1]
            assert size(requests, rows, keys, hq, hkv, dim) == (ranges * requests * rows * hq * (dim + 2) * 4 if ranges > 1 else 0)
        assert [plan(lib, paged, *a) for a in ((0, 1, 1, 1, 1, 64), (1, 0, 1, 1, 1, 64), (1, 1, -1, 1, 1, 64), (1, 1, 1, 3, 2, 64), (1, 1, 1, 1, 1, 96))] == [-1] * 5


def test_one_key_has_no_row_stride(lib):
    """The limit of the row strides holds from two keys on (B = 0: nothing is launched)."""
    call = lambda tk, rs: lib.iggt_packed_attn_f16(16, 64, 64, 16, rs, 64, 16, rs, 64, 16, 64, 64, 16, 16, 0, 4, tk, 4, 4, 1, 1, 64, 1.0, 1, 0, 0, 0)  # noqa: E731
    assert call(1, 1 << 24) == 0 and call(2, 1 << 24) == -2 and call(2, (1 << 24) - 8) == 0 and call(1, (1 << 24) + 4) == -2


def test_tokens_of_a_write_stay_below_2_to_the_30(lib):
    """More would not be a grid; no pages: nothing is launched."""
    call = lambda tokens: lib.iggt_append_pages_bf16(16, 64, 64, 16, 64, 64, 16, tokens, 16, 16, 16, 16, 0, 64, 1, 64, 0)  # noqa: E731
    assert call(1 << 30) == -1 and call((1 << 30) - 1) == 0
