"""Newton-Schulz's choice of tiles, asked of the library without a GPU."""

from sr_states.cuda import _native


def tile(*shapes, y_format=1):
    table = (_native.SrsMuonClass * max(1, len(shapes)))()
    for entry, (count, m, n) in zip(table, shapes):
        entry.count, entry.m, entry.n = count, m, n
    return _native.load_library().srs_newton_tile(table, len(shapes), y_format)


def test_tile_sides():
    for shape in ((1, 1, 1), (1, 128, 512), (12, 768, 768), (1, 2048, 2048), (1, 1001, 333)):
        assert tile(shape) == 128, shape
    for shape in ((1, 3500, 3500), (1, 2500, 4100), (1, 4100, 2500), (24, 768, 768)):
        assert tile(shape) == 256, shape
        assert tile(shape, y_format=0) == 256, shape
    assert tile((1, 64, 64), (2, 4096, 4096)) == 256
    assert tile((1, 1 << 25, 4)) == _native.SRS_ERR_INVALID_ARGUMENT
    assert tile((-1, 4, 4)) == _native.SRS_ERR_INVALID_ARGUMENT
    lib = _native.load_library()
    assert lib.srs_newton_tile(None, 1, 1) == _native.SRS_ERR_INVALID_ARGUMENT
    assert lib.srs_newton_tile(None, 17, 1) == _native.SRS_ERR_INVALID_ARGUMENT
