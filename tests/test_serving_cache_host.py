"""What a KvCache is made with stays what its calls are checked against and what the library is given.  Without a GPU."""
import numpy as np
import pytest

from tests.test_serving_host import Array, Device
from zklm_compile_b200 import DeviceBuffer, serving as zs


@pytest.mark.parametrize("name,value", [("d_head", 4), ("num_kv_heads", 1), ("page_size", 4), ("num_pages", 100), ("page_stride", 512), ("small", True), ("k_pages", Array(8)), ("v_pages", None),
                                        ("ctx", None)])
def test_a_cache_is_fixed(name, value):
    """A smaller head would let smaller arrays through the checks than the kernels read, other pages would not be the ones that are read."""
    ctx = Device()
    ctx.h = None
    cache = zs.KvCache(ctx, 8, 2, 16, 4, False, Array(4 * 256), Array(4 * 256))
    before = getattr(cache, name)
    with pytest.raises(AttributeError):
        setattr(cache, name, value)
    assert getattr(cache, name) is before or getattr(cache, name) == before
    with pytest.raises(ValueError, match="k: 31 elements"):
        zs.kv_append(cache, Array(31), Array(32), 1, Array(2), 1, 2, Array(2), Array(1), Array(1))


def test_sizes_that_32_bits_do_not_hold():
    """They would reach the library as other sizes."""
    class Vast(Array):
        def __init__(self):
            super().__init__(1 << 60)
    for change in (dict(page_size=(1 << 32) + 8), dict(num_pages=(1 << 32) + 4), dict(d_head=(1 << 32) + 16), dict(num_kv_heads=(1 << 32) + 2), dict(page_size=-8, num_kv_heads=-2)):
        with pytest.raises(ValueError, match="2\\^32"):
            zs.KvCache(Device(), **{**dict(page_size=8, num_kv_heads=2, d_head=16, num_pages=4, k_pages=Vast(), v_pages=Vast()), **change})


def test_buffers_that_are_freed():
    """An address of nothing is no array of the right size; for a bias or a workspace it would mean that there is none."""
    ctx = Device()
    ctx.h = None
    gone = DeviceBuffer.wrap(ctx, 0x1000, 64)
    assert zs._addr(ctx, gone, 64, "bias") == 0x1000
    gone.free()
    for least in (0, 64):
        with pytest.raises(ValueError, match="bias has been freed"):
            zs._addr(ctx, gone, least, "bias")
    with pytest.raises(ValueError, match="freed"):
        zs.adapter_linear(ctx, Array(32), Array(128), 2, 8, 16, Array(16), bias=gone)
    with pytest.raises(ValueError, match="freed"):
        zs.adapter_linear(ctx, Array(32), Array(128), 2, 8, 16, Array(16), workspace=gone)


def test_workspaces_that_are_no_arrays_of_the_gpu():
    ctx = Device()
    for bad in (np.zeros(64, np.uint8), [0], 0x1000):
        with pytest.raises(TypeError, match="workspace"):
            zs.adapter_linear(ctx, Array(32), Array(128), 2, 8, 16, Array(16), workspace=bad)
    for size in (1, 2, 4, 8):
        assert zs._workspace(ctx, Array(64, size)) == (0x1000, 64 * size)
    with pytest.raises(ValueError, match="another device"):
        zs._workspace(ctx, Array(64, 1, device=-1))
