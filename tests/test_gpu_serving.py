"""Paged cache, attention over it and projections with adapters on the GPU against their definition in 64-bit integers.  Everything is a
whole number, so results are equal or wrong: no tolerance."""
import numpy as np
import pytest

import zklm_compile_b200 as zk
from tests import serving_ref as R
from zklm_compile_b200 import attention, protocols, serving as zs, tables

pytestmark = pytest.mark.gpu
P = R.P


@pytest.fixture(scope="module")
def ctx():
    c = zk.Context(0)
    yield c
    c.close()


def field(rng, *shape):
    return rng.integers(0, P, shape, dtype=np.int64).astype(np.uint32)


def embed(x):
    return np.mod(x, P).astype(np.uint32)


def small(rng, most, *shape):
    return embed(rng.integers(-most, most + 1, shape, dtype=np.int64))


def words(a):
    """int16 and int32 arrays as the u32 words that a DeviceBuffer holds."""
    a = np.ascontiguousarray(a)
    if a.dtype.itemsize * a.size % 4:
        a = np.concatenate([a.reshape(-1), np.zeros(1, a.dtype)])
    return np.frombuffer(a.tobytes(), np.uint32)


class Paged:
    """A cache on the GPU with the same pages in numpy, and a block table that scatters the sequences' pages."""

    def __init__(self, ctx, rng, after, kv, d, page, is_small, most_k=127, spare=2, stride=0):
        self.ctx, self.small = ctx, is_small
        blocks = [-(-n // page) for n in after]
        pages = sum(blocks) + spare
        self.table = np.full((len(after), max(1, max(blocks))), -1, np.int32)
        order, at = rng.permutation(pages), 0
        for s, n in enumerate(blocks):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape, dense = (pages, kv, page, d), kv * page * d
        self.stride = stride or dense
        self.k, self.v = (self._values(rng, most, *shape) for most in (most_k, 0))
        self.cache = zs.KvCache(ctx, page, kv, d, pages, is_small, *(self._upload(x) for x in (self.k, self.v)), page_stride=stride)
        self.table_dev, self.max_blocks = ctx.upload(words(self.table)), self.table.shape[1]

    def _values(self, rng, most, *shape):
        if self.small:
            return rng.integers(-(most or 32768), (most or 32767) + 1, shape).astype(np.int16)
        return small(rng, most, *shape) if most else field(rng, *shape)

    def _upload(self, x):
        flat = np.full((len(x), self.stride), 0x5a5a if self.small else 0x5a5a5a5a, x.dtype)
        flat[:, :x[0].size] = x.reshape(len(x), -1)
        return self.ctx.upload(words(flat))

    def fetch(self):
        out = []
        for buf in (self.cache.k_pages, self.cache.v_pages):
            raw = np.frombuffer(buf.download().tobytes(), self.k.dtype)
            raw = raw[:len(self.k) * self.stride].reshape(len(self.k), self.stride)
            assert (raw[:, self.k[0].size:] == self.k.dtype.type(0x5a5a if self.small else 0x5a5a5a5a)).all()
            out.append(raw[:, :self.k[0].size].reshape(self.k.shape))
        return out


def shift_for(d, most=127):
    s = 0
    while (d * most * most >> s) > 32766:
        s += 1
    return s


# ---- attention ---------------------------------------------------------------------------------------
def check_attend(ctx, paged, q, lens, table, shift, fill=7):
    b, h, d = q.shape
    out, status = ctx.upload(np.full(b * h * d, fill, np.uint32)), ctx.upload(np.zeros(b, np.uint32))
    zs.paged_attention(paged.cache, ctx.upload(q), paged.table_dev, b, paged.max_blocks, ctx.upload(words(np.asarray(lens, np.int32))), h, ctx.upload(table), out, status,
                       score_shift=shift, n_table=len(table))
    want, want_status = R.attend(paged.k, paged.v, q, paged.table, lens, table, shift)
    assert status.download().tolist() == want_status.tolist()
    assert np.array_equal(out.download().reshape(b, h, d), want)
    return want_status


@pytest.mark.parametrize("is_small", [False, True])
@pytest.mark.parametrize("h,kv,d,page,lens", [
    (1, 1, 1, 1, [1]), (2, 1, 3, 2, [5, 0, 1]), (4, 4, 8, 16, [16, 17, 15]), (12, 12, 64, 16, [77]), (32, 8, 128, 16, [33, 0, 300, 1, 64]),
    (8, 1, 128, 64, [129, 1000]), (16, 1, 128, 32, [77, 5]), (5, 1, 80, 32, [100, 31]), (14, 2, 256, 8, [51, 600]), (3, 3, 256, 128, [128, 127]),
    (6, 2, 20, 4, [9, 70]), (2, 2, 200, 16, [40]), (9, 3, 33, 16, [50, 20]), (24, 2, 40, 8, [1, 0, 0, 65]), (84, 12, 64, 16, [6]),
])
def test_attention_over_pages(ctx, is_small, h, kv, d, page, lens):
    rng = np.random.default_rng(h * 1000 + d)
    paged = Paged(ctx, rng, lens, kv, d, page, is_small)
    check_attend(ctx, paged, small(rng, 127, len(lens), h, d), lens, tables.build_exp_table(1000), shift_for(d))


@pytest.mark.parametrize("is_small", [False, True])
def test_attention_of_whole_field_values(ctx, is_small):
    """q and the table hold any field element, K is chosen so that scores are small all the same: K of one non-zero element a row, q a small
    multiple of its inverse there, or plain small values where q is large nowhere else."""
    rng = np.random.default_rng(9)
    h, kv, d, lens = 4, 2, 24, [90, 200]
    paged = Paged(ctx, rng, lens, kv, d, 16, is_small)
    unit = 12345 if is_small else 1234567890
    paged.k[...] = 0
    paged.k[..., 7] = unit
    if is_small:
        paged.k[..., 9] = rng.integers(-32768, 32768, paged.k.shape[:3])
    else:
        paged.k[..., 9] = field(rng, *paged.k.shape[:3])
    paged.cache = zs.KvCache(ctx, 16, kv, d, len(paged.k), is_small, paged._upload(paged.k), paged._upload(paged.v))
    q = field(rng, 2, h, d)
    inverse = pow(unit, P - 2, P)
    for s in range(2):
        for i in range(h):
            q[s, i, 7] = int(rng.integers(-500, 500)) % P * inverse % P
            q[s, i, 9] = 0
    check_attend(ctx, paged, q, lens, field(rng, 65536), 0)
    check_attend(ctx, paged, q, lens, field(rng, 65536), 3)


def test_attention_long_rows_split_and_join(ctx):
    rng = np.random.default_rng(3)
    lens = [9000, 3, 0, 20011, 1]
    paged = Paged(ctx, rng, lens, 1, 64, 64, True)
    check_attend(ctx, paged, small(rng, 127, len(lens), 4, 64), lens, tables.build_exp_table(1000), shift_for(64))


@pytest.mark.parametrize("is_small", [False, True])
def test_attention_many_rows(ctx, is_small):
    """More sequences than fill the GPU once, most of them empty or short."""
    rng = np.random.default_rng(4)
    lens = rng.choice([0, 0, 1, 2, 17, 40], 700).tolist()
    paged = Paged(ctx, rng, lens, 2, 16, 8, is_small)
    check_attend(ctx, paged, small(rng, 127, len(lens), 4, 16), lens, tables.build_exp_table(1000), shift_for(16))


def test_attention_every_value_at_its_largest(ctx):
    """Digits of all ones everywhere: the largest sums that the kernel's partial products can meet."""
    rng = np.random.default_rng(5)
    lens = [17000]
    paged = Paged(ctx, rng, lens, 1, 128, 128, False)
    paged.k[...] = P - 1
    paged.v[...] = P - 1
    paged.cache = zs.KvCache(ctx, 128, 1, 128, len(paged.k), False, paged._upload(paged.k), paged._upload(paged.v))
    q = np.full((1, 8, 128), P - 1, np.uint32)         # every score is 128
    table = np.full(65536, P - 1, np.uint32)
    check_attend(ctx, paged, q, lens, table, 0)
    q[0, 3] = (1 << 30)                                # and sums of large positive products
    paged.k[...] = 2
    paged.cache = zs.KvCache(ctx, 128, 1, 128, len(paged.k), False, paged._upload(paged.k), paged._upload(paged.v))
    check_attend(ctx, paged, q, lens, table, 0)


def test_attention_small_cache_at_its_limits(ctx):
    rng = np.random.default_rng(6)
    lens = [16500]
    paged = Paged(ctx, rng, lens, 1, 128, 64, True)
    paged.k[...] = -32768
    paged.v[...] = np.where(rng.integers(0, 2, paged.v.shape), 32767, -32768)
    paged.cache = zs.KvCache(ctx, 64, 1, 128, len(paged.k), True, paged._upload(paged.k), paged._upload(paged.v))
    q = np.zeros((1, 8, 128), np.uint32)
    for h in range(8):
        q[0, h, 11 * h] = 1 if h % 2 else P - 1          # scores of -32768 and 32768, halved below
    check_attend(ctx, paged, q, lens, field(rng, 65536), 1)


def test_attention_strided_pages_and_queries(ctx):
    """K and V pages of one pool in turn, q inside rows of a fused projection."""
    rng = np.random.default_rng(7)
    h, kv, d, page, lens = 8, 2, 64, 16, [40, 77, 3]
    dense = kv * page * d
    paged = Paged(ctx, rng, lens, kv, d, page, False, stride=dense + 64)
    q = small(rng, 127, 3, h, d)
    row = h * d + 2 * kv * d
    wide = field(rng, 3, row)
    wide[:, :h * d] = q.reshape(3, -1)
    out, status = ctx.upload(np.zeros(3 * h * d, np.uint32)), ctx.upload(np.zeros(3, np.uint32))
    table = tables.build_exp_table(1000)
    zs.paged_attention(paged.cache, ctx.upload(wide), paged.table_dev, 3, paged.max_blocks, ctx.upload(words(np.array(lens, np.int32))), h, ctx.upload(table), out, status,
                       score_shift=shift_for(d), q_stride=row)
    want, _ = R.attend(paged.k, paged.v, q, paged.table, lens, table, shift_for(d))
    assert np.array_equal(out.download().reshape(3, h, d), want) and not status.download().any()


def test_attention_pages_that_start_on_no_16_byte_boundary(ctx):
    rng = np.random.default_rng(8)
    for is_small in (False, True):
        lens = [50, 21]
        paged = Paged(ctx, rng, lens, 2, 64, 16, is_small)
        moved = []
        for x in (paged.k, paged.v):
            raw = np.concatenate([np.zeros(1, np.uint32), words(x)])
            buf = ctx.upload(raw)
            moved.append((buf, zk.DeviceBuffer.wrap(ctx, buf_address(buf) + 4, raw.size - 1)))
        paged.cache = zs.KvCache(ctx, 16, 2, 64, len(paged.k), is_small, moved[0][1], moved[1][1])
        check_attend(ctx, paged, small(rng, 127, 2, 6, 64), lens, tables.build_exp_table(1000), shift_for(64))


def buf_address(buf):
    import ctypes
    return ctypes.cast(buf.ptr, ctypes.c_void_p).value


@pytest.mark.parametrize("h,kv,s,d", [(4, 4, 37, 64), (8, 2, 128, 64), (6, 2, 5, 7)])
def test_attention_is_the_row_of_the_whole_sequence(ctx, h, kv, s, d):
    """The rows that row_attention_forward computes (and prove_row_attention proves) come out of the cache one by one."""
    rng = np.random.default_rng(11)
    table = tables.build_exp_table(100)
    q, k, v = small(rng, 1, h, s, d), small(rng, 1, kv, s, d), field(rng, kv, s, d)
    whole = attention.row_attention_forward(ctx, q.reshape(-1), k.reshape(-1), v.reshape(-1), h, s, d, table, num_kv_heads=kv).reshape(h, s, d)
    paged = Paged(ctx, rng, [s] * s, kv, d, 16, False)
    status = ctx.upload(np.zeros(s, np.uint32))
    rows = np.arange(0, s * s + 1, s, dtype=np.int32)        # one copy of the sequence for each of its rows
    tile = lambda x: np.tile(x.transpose(1, 0, 2), (s, 1, 1))
    zs.kv_append(paged.cache, ctx.upload(tile(k)), ctx.upload(tile(v)), s * s, paged.table_dev, s, paged.max_blocks, ctx.upload(words(rows)), ctx.upload(np.zeros(s, np.uint32)), status)
    out = ctx.upload(np.zeros(s * h * d, np.uint32))
    zs.paged_attention(paged.cache, ctx.upload(q.transpose(1, 0, 2)), paged.table_dev, s, paged.max_blocks, ctx.upload(np.full(s, s, np.uint32)), h, ctx.upload(table), out, status)
    zs.check_status(ctx, status)
    assert np.array_equal(out.download().reshape(s, h, d).transpose(1, 0, 2), whole)


def test_attention_refuses_what_only_the_device_sees(ctx):
    """Lengths and pages outside the cache, scores outside the table, weights that add up to zero: the sequence's status, zeros in its rows, and
    the other sequences as they were."""
    rng = np.random.default_rng(12)
    h, kv, d, page = 4, 2, 32, 8
    lens = [20, 20, 20, 20, 20, -1, 100000, 0]
    paged = Paged(ctx, rng, [max(0, min(n, 24)) for n in lens], kv, d, page, False)
    paged.table[1, 1] = len(paged.k)                      # one past the pool
    paged.table[2, 2] = -5
    paged.table[7, :] = 1 << 30                           # never looked at
    paged.table_dev = ctx.upload(words(paged.table))
    q = small(rng, 127, len(lens), h, d)
    q[3, 2] = field(rng, d)                               # scores anywhere in the field
    q[4] = 0                                              # every score is 0, and the table's entry there too
    table = tables.build_exp_table(1000).copy()
    table[0] = 0
    got = check_attend(ctx, paged, q, lens, table, shift_for(d))
    assert got.tolist() == [0, 1, 1, 4, 5, 1, 1, 0]


def test_attention_256_entry_table(ctx):
    rng = np.random.default_rng(13)
    paged = Paged(ctx, rng, [60], 1, 16, 16, False, most_k=2)
    check_attend(ctx, paged, small(rng, 2, 1, 3, 16), [60], field(rng, 256), 0)
    q = small(rng, 2, 1, 3, 16)
    q[0, 1, 0] = 100
    assert check_attend(ctx, paged, q, [60], field(rng, 256), 0)[0] == 4


# ---- the cache -----------------------------------------------------------------------------------------
def check_append(ctx, rng, new, start, h, kv, d, page, rot, pairs, is_small, shift=14, pad=3, cs=None, stride=0, values=None, in_place=False):
    after = [a + b for a, b in zip(start, new)]
    paged = Paged(ctx, rng, after, kv, d, page, is_small, stride=stride)
    t = sum(new) + pad
    k = small(rng, 127, t, kv, d) if values is None else values(t, kv, d)
    v = small(rng, 32767, t, kv, d) if is_small else field(rng, t, kv, d)
    q = field(rng, t, h, d)
    if cs is None:
        cs = np.round(np.stack([np.cos(a := rng.uniform(0, 6.3, (max(after) + 1, rot // 2))), np.sin(a)], -1) * (1 << min(shift, 24))).astype(np.int32)
    row_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    before = field(rng, t, h, d)
    q_dev = ctx.upload(q)
    q_out = q_dev if in_place else ctx.upload(before)
    status = ctx.upload(np.zeros(len(new), np.uint32))
    rotation = zs.Rotation(ctx.upload(words(cs)) if cs.size else None, len(cs), rot, shift, pairs) if rot else None
    zs.kv_append(paged.cache, ctx.upload(k), ctx.upload(v), t, paged.table_dev, len(new), paged.max_blocks, ctx.upload(words(row_start)),
                 ctx.upload(words(np.array(start, np.int32))), status, rotation=rotation, q=q_dev, q_out=q_out, num_heads=h)
    want_q = (q if in_place else before).astype(np.int64)
    want_status = R.append(paged.k, paged.v, k, v, paged.table, row_start, start, cs if rot else None, shift, pairs, q, want_q, is_small)
    got_k, got_v = paged.fetch()
    assert np.array_equal(got_k, paged.k) and np.array_equal(got_v, paged.v)
    assert np.array_equal(q_out.download().reshape(t, h, d), want_q)
    assert status.download().tolist() == want_status.tolist()
    return want_status


@pytest.mark.parametrize("is_small", [False, True])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("new,start,h,kv,d,page,rot", [
    ([1], [0], 1, 1, 1, 1, 0), ([1, 1, 1], [0, 15, 16], 4, 2, 64, 16, 64), ([5, 0, 31], [3, 9, 0], 6, 2, 32, 8, 16), ([2, 1], [7, 0], 3, 1, 7, 4, 6),
    ([40], [100], 2, 2, 128, 16, 128), ([1] * 70, list(range(70)), 2, 1, 24, 32, 8), ([3, 4], [0, 1], 5, 1, 256, 16, 250), ([9], [2], 2, 1, 20, 8, 12),
    ([1] * 300, [i % 9 for i in range(300)], 1, 1, 8, 2, 2),
])
def test_append(ctx, is_small, pairs, new, start, h, kv, d, page, rot):
    check_append(ctx, np.random.default_rng(d + len(new)), new, start, h, kv, d, page, rot, pairs, is_small)


@pytest.mark.parametrize("shift", [0, 1, 30])
@pytest.mark.parametrize("pairs", [False, True])
def test_append_rounding_and_extremes(ctx, shift, pairs):
    """Whole field elements through tables of any 32-bit integers, the most negative among them; halves in both directions."""
    rng = np.random.default_rng(shift)
    cs = rng.integers(-(1 << 31), 1 << 31, (40, 16, 2)).astype(np.int32)
    cs[::3] = rng.choice([-(1 << 31), (1 << 31) - 1, 1, -1, 0], (14, 16, 2)).astype(np.int32)
    edge = np.array([0, 1, P - 1, P // 2, P // 2 + 1, 3, P - 3], np.uint32)
    check_append(ctx, rng, [13, 20], [0, 5], 3, 2, 48, 8, 32, pairs, False, shift, cs=cs, values=lambda *s: rng.choice(np.concatenate([edge, field(rng, 7)]), s).astype(np.uint32))


def test_append_in_place_queries_and_strided_pages(ctx):
    for pairs in (False, True):
        check_append(ctx, np.random.default_rng(1), [3, 8], [30, 0], 8, 2, 64, 16, 64, pairs, False, stride=2 * 16 * 64 + 12, in_place=True)
        check_append(ctx, np.random.default_rng(2), [3, 8], [30, 0], 8, 2, 63, 16, 62, pairs, True, stride=2 * 16 * 63 + 3, in_place=True)


def test_append_refuses_what_only_the_device_sees(ctx):
    rng = np.random.default_rng(3)
    kv, d, page = 2, 16, 8
    new, start = [2, 2, 2, 2, 2], [0, 7, 0, -1, 1 << 30]
    paged = Paged(ctx, rng, [16] * 5, kv, d, page, True)
    paged.table[1, 1] = len(paged.k)
    paged.table_dev = ctx.upload(words(paged.table))
    k, v = small(rng, 100, 10, kv, d), small(rng, 100, 10, kv, d)
    v[4, 0, 3] = 32768
    cs = np.zeros((3, d // 2, 2), np.int32)
    cs[..., 0] = 1 << 14
    row_start = np.arange(0, 11, 2).astype(np.int32)
    status = ctx.upload(np.zeros(5, np.uint32))
    args = (paged.table_dev, 5, paged.max_blocks, ctx.upload(words(row_start)), ctx.upload(words(np.array(start, np.int32))), status)
    zs.kv_append(paged.cache, ctx.upload(k), ctx.upload(v), 10, *args, rotation=zs.Rotation(ctx.upload(words(cs)), 3, d, 14))
    want = R.append(paged.k, paged.v, k, v, paged.table, row_start, start, cs, 14, False, small=True)
    assert want.tolist() == [0, 2, 3, 1, 1]
    assert status.download().tolist() == want.tolist()
    got_k, got_v = paged.fetch()
    assert np.array_equal(got_k, paged.k) and np.array_equal(got_v, paged.v)
    with pytest.raises(zk.ZkbError, match="sequence 1: a position"):
        zs.check_status(ctx, status)
    zs.kv_append(paged.cache, ctx.upload(k), ctx.upload(v), 0, *args)          # codes stay until the caller clears them
    assert status.download().tolist() == want.tolist()


# ---- projections -----------------------------------------------------------------------------------------
def check_linear(ctx, x, w, bias=None, a=None, b=None, of=None, x_pad=0, y_pad=0, workspace=False):
    t, n = x.shape
    m = len(w)
    wide = np.full((t, n + x_pad), 0x7a7a7a7a, np.uint32)
    wide[:, :n] = x
    out = ctx.upload(np.full((t, m + y_pad), 0x5a5a5a5a, np.uint32))
    adapters = zs.Adapters(ctx.upload(a), ctx.upload(b), len(a), a.shape[1]) if a is not None else None
    ws = ctx.alloc(max(1, zs.adapter_linear_workspace(ctx, t, m, n, len(a) if a is not None else 0, a.shape[1] if a is not None else 0) // 4)) if workspace else None
    zs.adapter_linear(ctx, ctx.upload(wide), ctx.upload(w), t, m, n, out, bias=ctx.upload(bias) if bias is not None else None, adapters=adapters,
                      adapter_of=ctx.upload(words(np.asarray(of, np.int32))) if of is not None else None, x_stride=n + x_pad if x_pad else 0, out_stride=m + y_pad if y_pad else 0,
                      workspace=ws)
    got = out.download().reshape(t, m + y_pad)
    assert np.array_equal(got[:, :m], R.linear(x, w, bias, a, b, of))
    assert (got[:, m:] == 0x5a5a5a5a).all()


@pytest.mark.parametrize("t", [1, 2, 3, 5, 8, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("m,n", [(1, 1), (3, 5), (128, 128), (130, 260), (257, 1023), (1000, 64), (77, 4100)])
def test_linear(ctx, t, m, n):
    rng = np.random.default_rng(t * 7 + m)
    check_linear(ctx, field(rng, t, n), field(rng, m, n), field(rng, m) if (t + m) % 2 else None)


@pytest.mark.parametrize("t,m,n,count,rank", [(1, 64, 64, 1, 1), (1, 200, 300, 3, 8), (7, 130, 132, 2, 5), (48, 256, 512, 12, 16), (100, 129, 77, 4, 33), (260, 140, 256, 40, 7), (64, 96, 2052, 3, 64)])
def test_linear_with_adapters(ctx, t, m, n, count, rank):
    rng = np.random.default_rng(t + rank)
    of = rng.integers(-1, count, t)
    of[rng.integers(0, t)] = count + 3                       # nobody's adapter
    check_linear(ctx, field(rng, t, n), field(rng, m, n), field(rng, m), field(rng, count, rank, n), field(rng, count, m, rank), of, workspace=t % 2 == 0)


@pytest.mark.parametrize("t", [1, 6, 40, 200])
def test_linear_every_value_at_its_largest(ctx, t):
    for n in (8192, 16388):
        x, w = np.full((t, n), P - 1, np.uint32), np.full((130, n), P - 1, np.uint32)
        check_linear(ctx, x, w, np.full(130, P - 1, np.uint32), np.full((1, 3, n), P - 1, np.uint32), np.full((1, 130, 3), P - 1, np.uint32), np.zeros(t, np.int64))
        # digits of all ones: (p + 1) / 2 - 1 and its rotations are the words with the most of them
        x[...] = 0x7fffff7f
        w[...] = 0x7ffffffe
        check_linear(ctx, x, w)


@pytest.mark.parametrize("t,m,n,count,rank", [(300, 5000, 40, 2, 130), (300, 5000, 33, 3, 66), (9, 70, 64, 2, 300), (5, 130, 36, 30, 65), (700, 3300, 36, 5, 20), (400, 4100, 20, 1, 64)])
def test_linear_with_adapters_of_many_ranks_and_rows(ctx, t, m, n, count, rank):
    """Ranks beyond one pass of the join, and joins whose CTAs take several blocks of rows."""
    rng = np.random.default_rng(rank)
    of = np.sort(rng.integers(-1, count, t)) if t > 50 else rng.integers(-1, count, t)
    check_linear(ctx, field(rng, t, n), field(rng, m, n), field(rng, m), field(rng, count, rank, n), field(rng, count, m, rank), of)


@pytest.mark.parametrize("count,rank", [(2, 4), (600, 3)])
def test_linear_more_tokens_than_one_pass_takes(ctx, count, rank):
    rng = np.random.default_rng(rank)
    t, m, n = 2100, 24, 36
    check_linear(ctx, field(rng, t, n), field(rng, m, n), field(rng, m), field(rng, count, rank, n), field(rng, count, m, rank), rng.integers(-1, count, t), x_pad=4, y_pad=4)


@pytest.mark.parametrize("t", [1, 12, 30, 36, 48, 61, 64, 100])
@pytest.mark.parametrize("m,n", [(6000, 2048), (5000, 2051), (300, 20000)])
def test_linear_many_steps(ctx, t, m, n):
    """Matrices of many more steps than a ring has stages, whose stretches end inside tiles; called again and again without waiting in between."""
    rng = np.random.default_rng(t)
    x, w = field(rng, t, n), field(rng, m, n)
    x_dev, w_dev, outs = ctx.upload(x), ctx.upload(w), [ctx.upload(np.zeros(t * m, np.uint32)) for _ in range(4)]
    for out in outs:
        zs.adapter_linear(ctx, x_dev, w_dev, t, m, n, out)
    want = R.linear_wide(x, w)
    for out in outs:
        assert np.array_equal(out.download().reshape(t, m), want)
    ctx.sync()                                              # raises if a wait inside a kernel ran out


@pytest.mark.parametrize("t", [1, 20, 150])
def test_linear_strided_rows(ctx, t):
    rng = np.random.default_rng(t)
    for x_pad, y_pad in ((4, 4), (3, 1)):
        check_linear(ctx, field(rng, t, 256), field(rng, 160, 256), None, x_pad=x_pad, y_pad=y_pad)


def test_linear_matrix_on_no_16_byte_boundary(ctx):
    rng = np.random.default_rng(2)
    for t in (1, 9, 70):
        x, w = field(rng, t, 128), field(rng, 96, 128)
        raw = ctx.upload(np.concatenate([np.zeros(1, np.uint32), w.reshape(-1)]))
        out = ctx.upload(np.zeros(t * 96, np.uint32))
        zs.adapter_linear(ctx, ctx.upload(x), zk.DeviceBuffer.wrap(ctx, buf_address(raw) + 4, w.size), t, 96, 128, out)
        assert np.array_equal(out.download().reshape(t, 96), R.linear(x, w))


@pytest.mark.parametrize("t,n,m", [(1, 128, 96), (5, 127, 95), (70, 256, 130), (2100, 64, 36)])
def test_linear_rows_of_x_and_of_the_result_in_one_array(ctx, t, n, m):
    """The result's words lie between the rows of x: neither is read or written as the other."""
    rng = np.random.default_rng(t)
    x, w, a, b, of = field(rng, t, n), field(rng, m, n), field(rng, 2, 3, n), field(rng, 2, m, 3), rng.integers(-1, 2, t)
    both = np.full((t, n + m), 0x5a5a5a5a, np.uint32)
    both[:, :n] = x
    raw = ctx.upload(both)
    zs.adapter_linear(ctx, raw, ctx.upload(w), t, m, n, zk.DeviceBuffer.wrap(ctx, buf_address(raw) + 4 * n, raw.n - n), adapters=zs.Adapters(ctx.upload(a), ctx.upload(b), 2, 3),
                      adapter_of=ctx.upload(words(of.astype(np.int32))), x_stride=n + m, out_stride=n + m)
    got = raw.download().reshape(t, n + m)
    assert np.array_equal(got[:, :n], x)
    assert np.array_equal(got[:, n:], R.linear(x, w, None, a, b, of))


def test_linear_is_the_product_with_the_merged_matrix(ctx):
    """One row equals the framework's matrix-vector product, and an adapter the matrix W + B A, whose product the framework proves."""
    rng = np.random.default_rng(5)
    m, n, r = 96, 160, 4
    x, w, a, b = field(rng, 1, n), field(rng, m, n), field(rng, 1, r, n), field(rng, 1, m, r)
    out = ctx.upload(np.zeros(m, np.uint32))
    zs.adapter_linear(ctx, ctx.upload(x), ctx.upload(w), 1, m, n, out)
    assert np.array_equal(out.download(), protocols.matmul_forward(ctx, w.reshape(-1), x.reshape(-1), m, n))
    merged = w.astype(np.int64).copy()
    for i in range(r):
        merged = (merged + b[0, :, i, None].astype(np.int64) * a[0, i].astype(np.int64) % P) % P
    merged = merged.astype(np.uint32)
    zs.adapter_linear(ctx, ctx.upload(x), ctx.upload(w), 1, m, n, out, adapters=zs.Adapters(ctx.upload(a), ctx.upload(b), 1, r), adapter_of=ctx.upload(np.zeros(1, np.uint32)))
    assert np.array_equal(out.download(), protocols.matmul_forward(ctx, merged.reshape(-1), x.reshape(-1), m, n))


# ---- refusals ------------------------------------------------------------------------------------------------
def test_refused_arguments(ctx):
    """Everything here is turned down on the host, before anything is launched."""
    z = lambda n: ctx.upload(np.zeros(n, np.uint32))
    cache = zs.KvCache(ctx, 8, 2, 16, 4, False)
    before = ctx.launches
    ok = dict(q=z(64), block_table=z(2), num_seqs=1, max_blocks=2, lens=z(1), num_heads=4, exp_table=z(65536), out=z(64), status=z(1))
    for change in (dict(num_heads=3), dict(num_heads=0), dict(score_shift=31), dict(q_stride=8), dict(max_blocks=0), dict(exp_table=z(300), n_table=300), dict(q=z(63)), dict(out=z(63)),
                   dict(block_table=z(1)), dict(status=z(1), lens=np.zeros(1, np.int32)), dict(num_seqs=-1), dict(workspace=z(1))):
        with pytest.raises((zk.ZkbError, ValueError, TypeError)):
            zs.paged_attention(cache, **{**ok, **change})
    for bad in (dict(page_size=7), dict(page_size=0), dict(d_head=257), dict(num_pages=0), dict(num_kv_heads=0), dict(page_stride=100)):
        with pytest.raises((zk.ZkbError, ValueError)):
            c = zs.KvCache(ctx, **{**dict(page_size=8, num_kv_heads=2, d_head=16, num_pages=4), **bad})
            zs.paged_attention(c, **{**ok, "q": z(4 * 257)})
    ok = dict(k=z(64), v=z(64), num_tokens=2, block_table=z(2), num_seqs=1, max_blocks=2, row_start=z(2), start=z(1), status=z(1))
    for change in (dict(q=z(128)), dict(q=z(128), q_out=z(128)), dict(q=z(128), q_out=z(127), num_heads=4), dict(k_stride=31), dict(rotation=zs.Rotation(z(64), 4, 15)),
                   dict(rotation=zs.Rotation(z(64), 4, 18)), dict(rotation=zs.Rotation(z(64), 4, 16, shift=31)), dict(rotation=zs.Rotation(z(63), 4, 16)), dict(row_start=z(1)),
                   dict(max_blocks=0, block_table=z(1))):
        with pytest.raises((zk.ZkbError, ValueError)):
            zs.kv_append(cache, **{**ok, **change})
    ok = dict(x=z(32), w=z(128), tokens=2, m=8, n=16, out=z(16))
    for change in (dict(m=0), dict(n=0), dict(x=z(31)), dict(w=z(127)), dict(out=z(15)), dict(x_stride=15), dict(out_stride=7), dict(bias=z(7)), dict(adapters=zs.Adapters(z(16), z(8), 1, 1)),
                   dict(adapters=zs.Adapters(z(16), z(8), 1, 0), adapter_of=z(2)), dict(adapters=zs.Adapters(z(15), z(8), 1, 1), adapter_of=z(2)),
                   dict(adapters=zs.Adapters(z(16), z(8), 1, 1), adapter_of=z(1))):
        with pytest.raises((zk.ZkbError, ValueError)):
            zs.adapter_linear(ctx, **{**ok, **change})
    assert ctx.launches == before


def test_results_in_place_of_their_inputs_are_refused(ctx):
    z = lambda n: ctx.upload(np.zeros(n, np.uint32))
    cache, rows = zs.KvCache(ctx, 8, 2, 16, 4, False), z(64)
    before = ctx.launches
    with pytest.raises(zk.ZkbError, match="out is not q"):
        zs.paged_attention(cache, rows, z(2), 1, 2, z(1), 4, z(65536), rows, z(1))
    with pytest.raises(zk.ZkbError, match="y is not x"):
        zs.adapter_linear(ctx, rows, z(256), 4, 16, 16, rows)
    assert ctx.launches == before


def test_nothing_to_do(ctx):
    z = lambda n: ctx.upload(np.zeros(n, np.uint32))
    cache, before = zs.KvCache(ctx, 8, 2, 16, 4, True), ctx.launches
    zs.paged_attention(cache, z(1), z(1), 0, 1, z(1), 4, z(65536), z(1), z(1))
    zs.kv_append(cache, z(1), z(1), 0, z(1), 1, 1, z(2), z(1), z(1))
    zs.adapter_linear(ctx, z(1), z(128), 0, 8, 16, z(1))
    assert ctx.launches == before


# ---- strides, streams, graphs, threads ------------------------------------------------------------------------
@pytest.mark.parametrize("pad", [4, 3])
def test_append_rows_inside_wider_ones(ctx, pad):
    """k, v and q as slices of a fused projection's rows, q_out with a stride of its own: on 16-byte boundaries and off them."""
    rng = np.random.default_rng(pad)
    h, kv, d, page, new, start = 4, 2, 32, 8, [3, 2], [6, 0]
    t = sum(new) + 1
    paged = Paged(ctx, rng, [9, 2], kv, d, page, False)
    row = (h + 2 * kv) * d + pad
    fused = np.stack([np.concatenate([small(rng, 127, h * d + kv * d), field(rng, kv * d + pad)]) for _ in range(t)])
    q, k, v = (np.ascontiguousarray(fused[:, a:b]) for a, b in ((0, h * d), (h * d, (h + kv) * d), ((h + kv) * d, (h + 2 * kv) * d)))
    buf, out = ctx.upload(fused), ctx.upload(np.full((t, h * d + pad), 9, np.uint32))
    part = lambda at: zk.DeviceBuffer.wrap(ctx, buf_address(buf) + 4 * at, fused.size - at)
    cs = rng.integers(-(1 << 14), 1 << 14, (9, d // 2, 2)).astype(np.int32)
    status = ctx.upload(np.zeros(2, np.uint32))
    rows = np.array([0, 3, 5], np.int32)
    zs.kv_append(paged.cache, part(h * d), part((h + kv) * d), t, paged.table_dev, 2, paged.max_blocks, ctx.upload(words(rows)), ctx.upload(words(np.array(start, np.int32))), status,
                 rotation=zs.Rotation(ctx.upload(words(cs)), 9, d, 14), q=part(0), q_out=out, num_heads=h, k_stride=row, v_stride=row, q_stride=row, q_out_stride=h * d + pad)
    want = np.full((t, h, d), 9, np.int64)
    assert not R.append(paged.k, paged.v, k.reshape(t, kv, d), v.reshape(t, kv, d), paged.table, rows, start, cs, 14, False, q.reshape(t, h, d), want).any()
    got_k, got_v = paged.fetch()
    assert np.array_equal(got_k, paged.k) and np.array_equal(got_v, paged.v)
    got = out.download().reshape(t, -1)
    assert np.array_equal(got[:, :h * d].reshape(t, h, d), want) and (got[:, h * d:] == 9).all() and not status.download().any()


class Decoder:
    """A layer's attention for one new token a sequence: fused projection with adapters, append with rotation, attention, output projection."""

    def __init__(self, ctx, rng, lens, h=4, kv=2, d=32, page=8, model=48, rank=4, adapters=2, room=6):
        self.ctx, self.lens, self.h, self.kv, self.d, self.model, self.b = ctx, list(lens), h, kv, d, model, len(lens)
        self.rank, self.adapters = rank, adapters
        self.paged = Paged(ctx, rng, [n + room for n in lens], kv, d, page, False)
        self.qkv = (h + 2 * kv) * d
        # weights in {-1, 0, 1} with few of them set, so that values stay small and scores inside the table
        sparse = lambda *s: embed(rng.integers(-1, 2, s) * (rng.random(s) < 0.2))
        self.w, self.w_out, self.a, self.bb = sparse(self.qkv, model), sparse(model, h * d), sparse(adapters, rank, model), sparse(adapters, self.qkv, rank)
        self.of = rng.integers(-1, adapters, self.b)
        angle = rng.uniform(0, 6.3, (max(lens) + room, d // 2))
        self.cs = np.round(np.stack([np.cos(angle), np.sin(angle)], -1) * (1 << 14)).astype(np.int32)
        self.table = tables.build_exp_table(1000)
        up, z = ctx.upload, lambda n: ctx.upload(np.zeros(n, np.uint32))
        self.dev = dict(w=up(self.w), w_out=up(self.w_out), a=up(self.a), b=up(self.bb), of=up(words(self.of.astype(np.int32))), cs=up(words(self.cs)), table=up(self.table),
                        rows=up(words(np.arange(self.b + 1, dtype=np.int32))), fused=z(self.b * self.qkv), q=z(self.b * h * d), att=z(self.b * h * d), y=z(self.b * model), status=z(self.b),
                        x=z(self.b * model), start=z(self.b), after=z(self.b))
        self.ws = [z(zs.adapter_linear_workspace(ctx, self.b, self.qkv, model, adapters, rank) // 4 + 64), z(zs.adapter_linear_workspace(ctx, self.b, model, h * d) // 4 + 64),
                   z(zs.paged_attention_workspace(self.paged.cache, self.b, h) // 4 + 64)]

    def set(self, x):
        import ctypes
        from zklm_compile_b200 import _lib
        for name, v in (("x", x), ("start", np.array(self.lens, np.uint32)), ("after", np.array(self.lens, np.uint32) + 1)):
            v = np.ascontiguousarray(v, np.uint32).reshape(-1)
            _lib.check(self.ctx.h, _lib.lib().zkb_buf_upload_u32(self.ctx.h, v.ctypes.data_as(_lib.u32p), ctypes.c_size_t(v.size), self.dev[name].ptr))

    def step(self, workspaces=True):
        ctx, v, h, kv, d, b = self.ctx, self.dev, self.h, self.kv, self.d, self.b
        ws = self.ws if workspaces else [None] * 3
        part = lambda at: zk.DeviceBuffer.wrap(ctx, buf_address(v["fused"]) + 4 * at, b * self.qkv - at)
        zs.adapter_linear(ctx, v["x"], v["w"], b, self.qkv, self.model, v["fused"], adapters=zs.Adapters(v["a"], v["b"], self.adapters, self.rank), adapter_of=v["of"], workspace=ws[0])
        zs.kv_append(self.paged.cache, part(h * d), part((h + kv) * d), b, self.paged.table_dev, b, self.paged.max_blocks, v["rows"], v["start"], v["status"],
                     rotation=zs.Rotation(v["cs"], len(self.cs), d, 14), q=part(0), q_out=v["q"], num_heads=h, k_stride=self.qkv, v_stride=self.qkv, q_stride=self.qkv)
        zs.paged_attention(self.paged.cache, v["q"], self.paged.table_dev, b, self.paged.max_blocks, v["after"], h, v["table"], v["att"], v["status"], score_shift=4, workspace=ws[2])
        zs.adapter_linear(ctx, v["att"], v["w_out"], b, self.model, h * d, v["y"], workspace=ws[1])

    def expect(self, x):
        h, kv, d, b = self.h, self.kv, self.d, self.b
        fused = R.linear(x, self.w, None, self.a, self.bb, self.of).reshape(b, -1, d)
        q = np.zeros((b, h, d), np.int64)
        status = R.append(self.paged.k, self.paged.v, fused[:, h:h + kv], fused[:, h + kv:], self.paged.table, list(range(b + 1)), self.lens, self.cs, 14, False, fused[:, :h], q)
        att, more = R.attend(self.paged.k, self.paged.v, q, self.paged.table, np.array(self.lens) + 1, self.table, 4)
        self.lens = [n + 1 for n in self.lens]
        assert not status.any() and not more.any()
        return R.linear(att.reshape(b, -1), self.w_out)

    def check(self, want):
        zs.check_status(self.ctx, self.dev["status"])
        assert np.array_equal(self.dev["y"].download().reshape(self.b, -1), want)
        got_k, got_v = self.paged.fetch()
        assert np.array_equal(got_k, self.paged.k) and np.array_equal(got_v, self.paged.v)


@pytest.mark.parametrize("workspaces", [False, True])
def test_tokens_one_after_the_other(ctx, workspaces):
    """Projection with adapters, rotation and append, attention, projection, token after token, against the definitions."""
    rng = np.random.default_rng(21)
    dec = Decoder(ctx, rng, [0, 5, 17, 8, 30])
    for _ in range(4):
        x = small(rng, 20, dec.b, dec.model)
        dec.set(x)
        dec.step(workspaces)
        dec.check(dec.expect(x))


def test_captured_steps_replayed(ctx):
    """Two decoders' steps captured once each on the context's stream, with workspaces of their own, and replayed in turn for token after token."""
    import torch
    rng = np.random.default_rng(22)
    stream = torch.cuda.ExternalStream(ctx.stream)
    decs = [Decoder(ctx, rng, [3, 9, 0, 14]), Decoder(ctx, rng, [40, 1], h=6, kv=2, d=64, page=16, model=64)]
    graphs = []
    for dec in decs:
        x = small(rng, 20, dec.b, dec.model)
        dec.set(x)
        dec.step()
        dec.check(dec.expect(x))
        ctx.sync()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="relaxed"):
            dec.step()
        graphs.append(g)
    for _ in range(3):
        xs = [small(rng, 20, dec.b, dec.model) for dec in decs]
        for dec, x in zip(decs, xs):
            dec.set(x)
        with torch.cuda.stream(stream):
            for g in graphs:
                g.replay()
        for dec, x in zip(decs, xs):
            dec.check(dec.expect(x))


def test_captured_call_without_a_workspace_is_refused(ctx):
    import torch
    rng = np.random.default_rng(23)
    dec = Decoder(ctx, rng, [3])
    dec.set(small(rng, 20, 1, dec.model))
    dec.step()
    ctx.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(ctx.stream), capture_error_mode="relaxed"):
        with pytest.raises(zk.ZkbError, match="workspace"):
            dec.step(workspaces=False)


def test_two_contexts_at_once():
    """Two host threads, a context and a decoder each, with nothing between their streams."""
    import threading
    failures = []

    def work(seed, lens):
        try:
            c = zk.Context(0)
            rng = np.random.default_rng(seed)
            dec = Decoder(c, rng, lens, room=9)
            for _ in range(8):
                x = small(rng, 20, dec.b, dec.model)
                dec.set(x)
                dec.step(workspaces=False)
                dec.check(dec.expect(x))
            c.close()
        except BaseException as e:          # noqa: BLE001 - reported by the main thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=(s, lens)) for s, lens in ((31, [0, 70, 3]), (32, [9, 9, 200, 1, 5]))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_tensors_of_another_library(ctx):
    """torch tensors are taken as they are; strided ones, ones of another type and ones on the host are refused."""
    import torch
    x, w, out = (torch.randint(0, P, s, dtype=torch.int32, device="cuda") for s in ((3, 64), (40, 64), (3, 40)))
    torch.cuda.synchronize()
    zs.adapter_linear(ctx, x, w, 3, 40, 64, out)
    ctx.sync()
    assert np.array_equal(out.cpu().numpy(), R.linear(x.cpu().numpy(), w.cpu().numpy()))
    for bad in (x.t(), x.to(torch.int64), x.cpu(), [1, 2]):
        with pytest.raises((ValueError, TypeError)):
            zs.adapter_linear(ctx, bad, w, 3, 40, 64, out)
