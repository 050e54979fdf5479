"""What zklm_compile_b200.serving turns down before it reaches the library: sizes, strides and arrays, without a GPU."""
import pytest

from zklm_compile_b200 import serving as zs


class Device:
    device = 0


class Array:
    """As much of a tensor on the GPU as the package looks at."""

    def __init__(self, n, size=4, device=0, dense=True, at=0x1000):
        self.n, self.itemsize, self.device, self.dense, self.at = n, size, device, dense, at
        self.nbytes = n * size

    def data_ptr(self): return self.at
    def element_size(self): return self.itemsize
    def numel(self): return self.n
    def get_device(self): return self.device
    def is_contiguous(self): return self.dense


def test_arrays():
    ctx = Device()
    assert zs._addr(ctx, Array(10), 10, "x") == 0x1000
    assert zs._addr(ctx, Array(10, size=2), 10, "x", 2) == 0x1000
    for bad in (Array(9), Array(10, size=2), Array(10, size=8), Array(10, device=1), Array(10, device=-1), Array(10, dense=False)):
        with pytest.raises(ValueError, match="x"):
            zs._addr(ctx, bad, 10, "x")
    for bad in (None, [1, 2], 5):
        with pytest.raises(TypeError, match="x"):
            zs._addr(ctx, bad, 0, "x")


def test_rows():
    assert zs._rows(3, 8, 0) == 24 and zs._rows(3, 8, 10) == 28 and zs._rows(0, 8, 10) == 0 and zs._rows(1, 8, 100) == 8
    with pytest.raises(ValueError):
        zs._rows(3, 8, 7)


def test_sizes():
    zs._counts(a=0, b=0xffffffff)
    for bad in (-1, 1 << 32):
        with pytest.raises(ValueError, match="tokens"):
            zs._counts(tokens=bad)


def test_caches():
    ctx = Device()
    c = zs.KvCache(ctx, 8, 2, 16, 4, False, Array(4 * 256), Array(4 * 256))
    assert (c._c.page_size, c._c.num_kv_heads, c._c.d_head, c._c.num_pages, c._c.elem, c._c.page_stride) == (8, 2, 16, 4, 0, 0)
    zs.KvCache(ctx, 8, 2, 16, 4, True, Array(4 * 256, 2), Array(4 * 256, 2))
    zs.KvCache(ctx, 8, 2, 16, 4, False, Array(3 * 300 + 256), Array(3 * 300 + 256), page_stride=300)
    for args in ((8, 2, 16, 4, False, Array(4 * 256), None), (8, 2, 16, 4, False, Array(4 * 256 - 1), Array(4 * 256)), (8, 2, 16, 4, True, Array(4 * 256), Array(4 * 256)),
                 (8, 2, 16, 0, False, Array(8), Array(8)), (8, 0, 16, 4, False, Array(8), Array(8)), (0, 2, 16, 4, False, Array(8), Array(8))):
        with pytest.raises(ValueError):
            zs.KvCache(ctx, *args)
    with pytest.raises(ValueError, match="stride"):
        zs.KvCache(ctx, 8, 2, 16, 4, False, Array(4 * 256), Array(4 * 256), page_stride=255)


def test_both_or_neither():
    ctx = Device()
    cache = zs.KvCache(ctx, 8, 2, 16, 4, False, Array(4 * 256), Array(4 * 256))
    with pytest.raises(ValueError, match="q and q_out"):
        zs.kv_append(cache, Array(64), Array(64), 2, Array(2), 1, 2, Array(2), Array(1), Array(1), q=Array(64), num_heads=2)
    with pytest.raises(ValueError, match="adapters"):
        zs.adapter_linear(ctx, Array(32), Array(128), 2, 8, 16, Array(16), adapter_of=Array(2))


def test_rotation_is_checked_at_the_size_that_is_sent():
    ctx = Device()
    cache = zs.KvCache(ctx, 8, 2, 16, 4, False, Array(4 * 256), Array(4 * 256))
    rot = zs.Rotation(Array(8 * 16 - 1), 8, 16)
    rot.positions = 1                          # the library's own copy still says 8
    with pytest.raises(ValueError, match="rotation's table"):
        zs.kv_append(cache, Array(64), Array(64), 2, Array(2), 1, 2, Array(2), Array(1), Array(1), rotation=rot)
    for bad in ((-1, 16), (8, -2), (8, 16, 1 << 32)):
        with pytest.raises(ValueError):
            zs.Rotation(Array(8), *bad)
