"""Refusals of the C entries for log probabilities and a router's experts, which come before anything is asked of a device; and the size of a plan."""
import ctypes

import pytest


def call(name, *args):
    """The error message of an entry point called with integers and addresses."""
    from comet_b200 import _lib
    lib = _lib.load()
    status = getattr(lib, name)(*args)
    message = lib.comet_b200_last_error()
    assert status != 0 and message
    return message.decode()


@pytest.fixture(scope="module")
def room():
    """16-byte aligned host memory that no refused call reads."""
    a = (ctypes.c_char * 4096)()
    at = ctypes.addressof(a)
    yield at + (-at) % 16
    del a


@pytest.mark.parametrize("nnz,ncols", [(0, 1), (1, 1), (8, 64), (63, 64), (2040, 10), (65536, 64), (65537, 1023), (1 << 30, 1024)])
def test_size_of_a_plan(nnz, ncols):
    """As device.group_entries allocates it: a header, counts and first tiles of the columns, tiles, and two numbers for each of 128 slots a tile."""
    from comet_b200 import _lib
    tiles = nnz // 128 + min(nnz, ncols) + 1
    size = _lib.load().comet_b200_dev_group_entries_size(nnz, ncols)
    assert size == 16 + (ncols + 3) // 4 * 4 + (ncols + 4) // 4 * 4 + (tiles + 3) // 4 * 4 + 256 * tiles
    # each column's entries in tiles of their own fit, whatever the columns are
    assert tiles >= nnz // 128 + min(nnz, ncols)


@pytest.mark.parametrize("nrows,ncols,nnz", [(-1, 4, 0), (4, 0, 0), (4, 1025, 0), (4, 4, -1), (1 << 31, 4, 8), (4, 4, 0x70000001)])
def test_group_entries(nrows, ncols, nnz, room):
    assert "group_entries" in call("comet_b200_dev_group_entries_i64", nrows, ncols, nnz, room, room, room, 0)


BAD_SIZES = [(-1, 4, 8, 64, 32), (4, 0, 8, 64, 32), (4, 1025, 8, 64, 32), (4, 4, -1, 64, 32), (4, 4, 8, 0, 32), (4, 4, 8, 60, 32), (4, 4, 8, 64, 36), (4, 4, 8, 64, 4),
             (4, 4, 8, (1 << 20) + 8, 32), (4, 4, 8, 64, (1 << 20) + 8), (1 << 31, 4, 8, 64, 32), (4, 4, 0x70000001, 64, 32)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", BAD_SIZES)
def test_sizes_of_experts(sizes, kind, room):
    p = room
    assert "gated_experts:" in call("comet_b200_dev_gated_experts_%s_i64" % kind, *sizes, 0, p, p, 64, p, p, 0)
    assert "gated_experts_grad:" in call("comet_b200_dev_gated_experts_grad_%s_i64" % kind, *sizes, 0, p, p, p, 64, p, p, p, p, p, p, 0)
    assert "combine_experts:" in call("comet_b200_dev_combine_experts_%s_i64" % kind, *sizes, p, p, p, p, p, p, p, p, 0)
    assert "combine_experts_grad:" in call("comet_b200_dev_combine_experts_grad_%s_i64" % kind, *sizes, p, p, p, p, p, 64, p, p, p, p, p, 0)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_strides_and_addresses_of_experts(kind, room):
    sizes, p, odd = (4, 4, 8, 64, 32), room, room + 2
    for ld in (56, 68):
        assert "stride" in call("comet_b200_dev_gated_experts_%s_i64" % kind, *sizes, 0, p, p, ld, p, p, 0)
        assert "stride" in call("comet_b200_dev_gated_experts_grad_%s_i64" % kind, *sizes, 0, p, p, p, ld, p, p, p, p, p, p, 0)
        assert "stride" in call("comet_b200_dev_combine_experts_grad_%s_i64" % kind, *sizes, p, p, p, p, p, ld, p, p, p, p, p, 0)
    gated, combine = [p, 64, p, p], [p, p, p, p]
    for i in (0, 2, 3):
        args = list(gated)
        args[i] = odd
        assert "16 bytes" in call("comet_b200_dev_gated_experts_%s_i64" % kind, *sizes, 0, p, *args, 0)
    for i, name in enumerate(("h", "v", "sums", "y")):
        args = list(combine)
        args[i] = odd
        h, v, sums, y = args
        assert "16 bytes" in call("comet_b200_dev_combine_experts_%s_i64" % kind, *sizes, p, p, p, h, p, v, sums, y, 0), name
    for i in range(6):
        args = [p, p, p, p, p, p]
        args[i] = odd
        w, dh, dz, sums, dx, dw = args
        assert "16 bytes" in call("comet_b200_dev_gated_experts_grad_%s_i64" % kind, *sizes, 0, p, p, p, 64, w, dh, dz, sums, dx, dw, 0)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_log_probs(kind, room):
    p, one, size = room, (ctypes.c_double * 1)(1.0), 4 if kind == "f32" else 2
    t = ctypes.addressof(one)
    forward, back = "comet_b200_dev_log_probs_%s_i64" % kind, "comet_b200_dev_log_probs_grad_%s_i64" % kind
    for nrows, ncols, ld in [(-1, 8, 8), (4, 0, 8), (4, 1 << 30, 1 << 30), (4, 8, 7), (1 << 29, 8, 8)]:
        assert "log_probs:" in call(forward, nrows, ncols, p, p, p, ld, t, p, p, 0, 0, 0, 0, 0, 0)
        assert "log_probs_grad:" in call(back, nrows, ncols, p, p, p, ld, t, p, p, 0, 0, p, 8, 0)
    for k in (-1, 9):
        assert "alternatives" in call(forward, 4, 8, p, p, p, 8, t, p, p, 0, k, p, p, p, 0)
    assert "alternatives" in call(forward, 4, 2000, p, p, p, 2000, t, p, p, 0, 1025, p, p, p, 0)
    assert "element's size" in call(forward, 4, 8, p, p, p + size // 2, 8, t, p, p, 0, 0, 0, 0, 0, 0)
    assert "element's size" in call(back, 4, 8, p, p, p, 8, t, p, p, 0, 0, p + size // 2, 8, 0)
    assert "leading dimension" in call(back, 4, 8, p, p, p, 8, t, p, p, 0, 0, p, 7, 0)
    assert "need the entropies" in call(back, 4, 8, p, p, p, 8, t, p, p, 0, p, p, 8, 0)
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-39, 1e31):
        one[0] = bad
        assert "temperature" in call(forward, 4, 8, p, p, p, 8, t, p, p, 0, 0, 0, 0, 0, 0)
        assert "temperature" in call(back, 4, 8, p, p, p, 8, t, p, p, 0, 0, p, 8, 0)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("k", [0, 2])
def test_address_of_sums(kind, k, room):
    """Both numbers of a row are read and written at once."""
    p, one = room, (ctypes.c_double * 1)(1.0)
    t = ctypes.addressof(one)
    for ncols in (8, 5000):
        assert "8 bytes" in call("comet_b200_dev_log_probs_%s_i64" % kind, 4, ncols, p, p, p, ncols, t, p, p + 4, 0, k, p, p, p, 0)
        assert "8 bytes" in call("comet_b200_dev_log_probs_grad_%s_i64" % kind, 4, ncols, p, p, p, ncols, t, p + 4, p, 0, 0, p, ncols, 0)
