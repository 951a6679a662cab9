"""The tiled products that a cross entropy gradient is made of, from the host's arithmetic
alone: what every workgroup takes is there, and together they take all of it, once."""

import ctypes as C
import random

import pytest

from emeans_amd import _lib

CUS = 256
LOGITS, DX, DW = range(3)
SLAB = 64


def products(n, d, k, kind, workspace=0):
    lib, count = _lib.lib(), C.c_uint64()
    _lib.check(lib.emh_host_xent_products(n, d, k, kind, CUS, workspace, None, 0, C.byref(count)))
    out = (_lib.XentProduct * max(1, count.value))()
    _lib.check(lib.emh_host_xent_products(n, d, k, kind, CUS, workspace, out, count.value,
                                          C.byref(count)))
    return list(out)[:count.value]


def check(n, d, k, kind, workspace=0):
    got = products(n, d, k, kind, workspace)
    area = {LOGITS: 0, DX: 0, DW: 0}
    planes = 4 if kind == _lib.EMH_F32 else 1
    most = max((workspace or 1 << 30) * 17 // 16, 256 * 768 * 2 * planes)
    for p in got:
        where = (n, d, k, kind, workspace, p.what, p.row0, p.rows, p.class0, p.classes)
        assert p.rows > 0 and p.classes > 0, where
        assert p.row0 + p.rows <= n and p.class0 + p.classes <= k, where
        rows, cols, deep = {LOGITS: (p.rows, p.classes, d), DX: (p.rows, d, p.classes),
                            DW: (p.classes, d, p.rows)}[p.what]
        # Tiles that cover the result, none of them outside of it.
        assert (p.row_tiles - 1) * p.tile_rows < rows <= p.row_tiles * p.tile_rows, where
        assert (p.col_tiles - 1) * p.tile_cols < cols <= p.col_tiles * p.tile_cols, where
        assert p.slabs == -(-deep // SLAB), where
        # Every workgroup has a step: an empty split's loads would come from nowhere.
        assert 1 <= p.splits <= p.slabs * p.passes, where
        assert p.passes == 1 or (p.passes == 3 and kind == _lib.EMH_F32), where
        # The softmax in memory holds the product, in the workspace.
        assert p.rows * p.classes * 2 * planes <= p.softmax_bytes <= most, where
        if p.what == DX and p.rows < n:  # (the sums of dx are of all rows)
            assert p.splits == 1, where
        area[p.what] += p.rows * p.classes
    assert all(a == n * k for a in area.values()), (n, d, k, kind, workspace)


# The last of the pieces of the classes is much smaller than the others.
SHORT = [(80_000, 100, 179_753), (70_000, 300, 222_778), (100_000, 40, 107_554),
         (32_768, 200, 1_032_193), (100_000, 40, 107_521), (80_000, 100, 179_713),
         (40_960, 250, 678_913)]


@pytest.mark.parametrize("kind", [_lib.EMH_F32, _lib.EMH_F16, _lib.EMH_BF16])
@pytest.mark.parametrize("n,d,k", SHORT)
def test_a_short_last_piece(n, d, k, kind):
    check(n, d, k, kind)


@pytest.mark.parametrize("kind", [_lib.EMH_F32, _lib.EMH_BF16])
@pytest.mark.parametrize("last", [1, 63, 64, 65, 257, 700])
def test_short_pieces_of_a_small_workspace(last, kind):
    for n, d in ((300, 40), (1000, 200), (65, 500)):
        check(n, d, 3 * 768 + last, kind, workspace=1)


def test_any_sizes():
    r = random.Random(5)
    size = lambda lo, hi: int(round(lo * (hi / lo) ** r.random()))  # noqa: E731
    for _ in range(3000):
        n, d, k = size(1, 1_000_000), size(1, 4096), size(1, 3_000_000)
        workspace = r.choice([0, 0, 1, 1 << 20, 1 << 26, 1 << 32])
        if n * k > 200 * max(1 << 17, (workspace or 1 << 30) >> 4):  # (a few hundred parts)
            continue
        check(n, d, k, r.choice([_lib.EMH_F32, _lib.EMH_BF16]), workspace)


@pytest.mark.parametrize("kind", [_lib.EMH_F32, _lib.EMH_BF16])
def test_many_rows_in_the_default_workspace(kind):
    for n in (170_000, 200_000, 700_000, 1_000_000, 10_000_001):
        for d, k in ((768, 1024), (40, 10), (64, 5000)):
            check(n, d, k, kind)


def test_a_launch_holds_the_tiles():
    """Fewer than 2^32 threads of at most 512 a tile, at sizes whose matrices fit a device."""
    for n, d, k in ((1 << 30, 1, 2), (1 << 30, 64, 1), (100, 1, 1 << 30), (1 << 24, 1024, 5)):
        for kind in (_lib.EMH_F32, _lib.EMH_BF16):
            for p in products(n, d, k, kind):
                assert p.row_tiles * p.col_tiles * p.splits < 1 << 23, (n, d, k, kind, p.what)


def test_refusals():
    lib, count = _lib.lib(), C.c_uint64()
    for bad in ((1, 0, 1, 0, CUS), (1, 1, 0, 0, CUS), (1, 1, 1, _lib.EMH_U32, CUS), (1, 1, 1, 0, 0),
                (1 << 31, 1, 1, 0, CUS)):
        with pytest.raises(_lib.EmeansHipInvalid):
            _lib.check(lib.emh_host_xent_products(*bad, 0, None, 0, C.byref(count)))
    with pytest.raises(_lib.EmeansHipInvalid):
        _lib.check(lib.emh_host_xent_products(1, 1, 1, 0, CUS, 0, None, 1, C.byref(count)))
    assert products(0, 4, 3, 0) == []
