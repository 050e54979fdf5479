"""Paged attention on the GPU where a call's blocks are shared between CTAs in every way: rows cut anywhere, many rows a CTA, more sequences than are read
into shared memory, heads of several tiles a CTA.  Results are whole numbers: equal or wrong."""
import numpy as np
import pytest

import zklm_compile_b200 as zk
from tests import serving_ref as R
from tests.test_gpu_serving import P, Paged, field, shift_for, small, words
from zklm_compile_b200 import serving as zs, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = zk.Context(0)
    yield c
    c.close()


class Batch:
    """A cache, queries and what their attention is."""

    def __init__(self, ctx, seed, lens, h, kv, d, page, is_small):
        rng = np.random.default_rng(seed)
        self.ctx, self.lens, self.h, self.d, self.b = ctx, lens, h, d, len(lens)
        self.paged = Paged(ctx, rng, lens, kv, d, page, is_small)
        self.table, self.shift = tables.build_exp_table(1000), shift_for(d)
        q = small(rng, 127, self.b, h, d)
        self.dev = [ctx.upload(q), ctx.upload(words(np.asarray(lens, np.int32))), ctx.upload(self.table), ctx.upload(np.zeros(self.b, np.uint32))]
        self.want, status = R.attend(self.paged.k, self.paged.v, q, self.paged.table, lens, self.table, self.shift)
        assert not status.any()

    def call(self, workspace=None):
        q, lens, table, status = self.dev
        out = self.ctx.upload(np.full(self.b * self.h * self.d, 7, np.uint32))
        zs.paged_attention(self.paged.cache, q, self.paged.table_dev, self.b, self.paged.max_blocks, lens, self.h, table, out, status, score_shift=self.shift, workspace=workspace)
        return out

    def right(self, out):
        return np.array_equal(out.download().reshape(self.want.shape), self.want) and not self.dev[3].download().any()

    def workspace(self):
        return self.ctx.upload(np.zeros(zs.paged_attention_workspace(self.paged.cache, self.b, self.h) // 4, np.uint32))


def attend_exact(k_pages, v_pages, q, table, lens, exp_table, shift):
    """The definition in 64-bit integers, a sequence and key head at a time on the GPU (torch); every score is in the table."""
    import torch
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a).astype(t)).cuda().to(torch.int64)
    k_all, v_all = (dev(a, np.int16 if a.dtype == np.int16 else np.int64) for a in (k_pages, v_pages))
    qs, e_all, n_table = dev(q, np.int64), dev(exp_table, np.int64), len(exp_table)
    (seqs, heads, d), (kv, page) = q.shape, k_pages.shape[1:3]
    out = torch.zeros(seqs, kv, heads // kv, d, dtype=torch.int64, device="cuda")
    for s in range(seqs):
        if not lens[s]:
            continue
        pos = torch.arange(lens[s], device="cuda")
        place = torch.from_numpy(table[s].astype(np.int64)).cuda()[pos // page]
        for h in range(kv):
            k, v = (torch.remainder(a[place, h, pos % page], P) for a in (k_all, v_all))
            for g in range(heads // kv):
                score = (k * qs[s, h * (heads // kv) + g] % P).sum(1) % P
                score = torch.where(score > P // 2, score - P, score)
                score = torch.sign(score) * ((score.abs() + ((1 << shift) >> 1)) >> shift)
                assert bool(((score >= -(n_table // 2)) & (score < n_table // 2)).all())
                e = e_all[torch.remainder(score, n_table)]
                total = int(e.sum()) % P
                assert total
                out[s, h, g] = (e[:, None] * v % P).sum(0) % P * pow(total, P - 2, P) % P
    return out.reshape(seqs, heads, d).cpu().numpy()


class Cut(Batch):
    """The same for more work than numpy does in a moment."""

    def __init__(self, ctx, seed, lens, h, kv, d, page, is_small):
        rng = np.random.default_rng(seed)
        self.ctx, self.lens, self.h, self.d, self.b = ctx, lens, h, d, len(lens)
        self.paged = Paged(ctx, rng, lens, kv, d, page, is_small)
        self.table, self.shift = tables.build_exp_table(1000), shift_for(d)
        q = small(rng, 127, self.b, h, d)
        self.dev = [ctx.upload(q), ctx.upload(words(np.asarray(lens, np.int32))), ctx.upload(self.table), ctx.upload(np.zeros(self.b, np.uint32))]
        self.want = attend_exact(self.paged.k, self.paged.v, q, self.paged.table, lens, self.table, self.shift)


def ragged(rng, seqs, least, most):
    """Lengths spread over the range, about one in seven of them nothing."""
    lens = rng.integers(least, most + 1, seqs)
    lens[rng.random(seqs) < 0.15] = 0
    lens[rng.integers(0, seqs)] = most
    return lens.tolist()


def test_the_two_definitions_agree():
    rng = np.random.default_rng(5)
    k, v = small(rng, 127, 9, 2, 8, 20), field(rng, 9, 2, 8, 20)
    q, table, lens = small(rng, 127, 3, 6, 20), np.array([[4, 0, 8], [1, 2, -1], [3, -1, -1]]), [24, 9, 0]
    want, status = R.attend(k, v, q, table, lens, tables.build_exp_table(1000), shift_for(20))
    assert not status.any() and np.array_equal(attend_exact(k, v, q, table, lens, tables.build_exp_table(1000), shift_for(20)), want)


@pytest.mark.parametrize("is_small", [False, True])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (256, 32), (80, 8)])
@pytest.mark.parametrize("group", [1, 3, 4, 8])
def test_rows_cut_anywhere(ctx, is_small, d, page, group):
    """More rows than CTAs and many blocks a row: CTAs end one row and begin another, most rows have parts in two or more of them and every CTA takes tile after
    tile.  Called again and again without waiting, with the context's counters and with the caller's."""
    rng = np.random.default_rng(d + group)
    b = Cut(ctx, d * 10 + group, ragged(rng, 40, 300, 3000 if group < 8 else 1200), 8 * group, 8, d, page, is_small)
    ws = b.workspace()
    outs = [b.call(w) for w in (None, ws, None, ws, ws)]
    ctx.sync()
    assert all(b.right(o) for o in outs)
    assert not ws.download()[:192].any()


@pytest.mark.parametrize("is_small", [False, True])
@pytest.mark.parametrize("h,kv,d,page,seqs,most", [(2, 2, 64, 16, 300, 1000), (4, 1, 128, 16, 700, 600), (5, 1, 256, 64, 257, 900)])
def test_rows_cut_anywhere_among_many_sequences(ctx, is_small, h, kv, d, page, seqs, most):
    """More sequences than a warp looks at for itself."""
    rng = np.random.default_rng(seqs)
    b = Cut(ctx, seqs, ragged(rng, seqs, 1, most), h, kv, d, page, is_small)
    outs = [b.call() for _ in range(3)]
    ctx.sync()
    assert all(b.right(o) for o in outs)


@pytest.mark.parametrize("is_small,d,group", [(False, 128, 1), (False, 128, 8), (False, 64, 4), (True, 128, 2), (True, 128, 8), (True, 64, 1), (False, 256, 2), (True, 256, 2)])
def test_sums_of_a_stretch_as_long_as_they_may_get(ctx, is_small, d, group):
    """160 key heads over more positions than one CTA adds up before it empties its 32-bit sums (512 blocks), and then some, with the largest digits there are: whole
    rows in one CTA, and rows cut behind that.  All places of the block table name the same page, so the sums are known from it."""
    rng = np.random.default_rng(group)
    kv, page, warps = 160, 64, 12 if is_small and d <= 128 and group <= 4 or d == 64 and group <= 4 else 5 if d == 256 and not is_small else 8
    n = 530 * warps * 16 + 37
    most = 32767 if is_small else P - 1
    k = np.zeros((1, kv, page, d), np.int16 if is_small else np.uint32)
    k[..., 0] = rng.integers(0, 4, (1, kv, page))           # scores of 0 to 3
    v = np.full(k.shape, most, k.dtype)
    v[:, ::3] = rng.integers(-32768 if is_small else 0, most, v[:, ::3].shape)
    q = np.zeros((1, kv * group, d), np.uint32)
    q[..., 0] = 1
    table = np.full(65536, P - 1, np.uint32)
    table[1], table[2] = 0x7fffff7f, 0x7f7fffff
    cache = zs.KvCache(ctx, page, kv, d, 1, is_small, ctx.upload(words(k)), ctx.upload(words(v)))
    blocks = -(-n // page)
    out, status = ctx.upload(np.full(q.size, 7, np.uint32)), ctx.upload(np.zeros(1, np.uint32))
    zs.paged_attention(cache, ctx.upload(q), ctx.upload(np.zeros(blocks, np.uint32)), 1, blocks, ctx.upload(np.array([n], np.uint32)), kv * group, ctx.upload(table), out, status)
    times = np.array([n // page + (r < n % page) for r in range(page)], np.int64)       # how often a row of the page is met
    e = table[k[0, :, :, 0].astype(np.int64)].astype(np.int64) * times % P              # (kv, page)
    total = e.sum(1) % P
    assert total.all()
    want = (e[:, :, None] * (v[0].astype(np.int64) % P) % P).sum(1) % P
    want = want * np.array([pow(int(t), P - 2, P) for t in total], np.int64)[:, None] % P
    got = out.download().reshape(kv, group, d)
    assert not status.download().any()
    assert all(np.array_equal(got[:, g], want) for g in range(group))


@pytest.mark.parametrize("t,m,n", [(2048, 1280, 8192), (2048, 640, 16384), (64, 1280 * 32, 8192), (2048, 700, 20004)])
def test_products_of_a_stretch_as_deep_as_they_may_get(ctx, t, m, n):
    """CTAs that add up all of 8192 columns, and more than one such stretch, before a tile ends, with the largest digits there are.  A row of x and a row of W have one
    value each, so a product is n times the two."""
    rng = np.random.default_rng(m)
    largest = np.array([P - 1, 0x7fffff7f, 0x7f7fffff, 0x7fff7fff, 0x7ffffffe], np.int64)
    xv, wv = (np.where(rng.random(c) < 0.8, rng.choice(largest, c), rng.integers(0, P, c)) for c in (t, m))
    rows = lambda v: ctx.upload(np.broadcast_to(v.astype(np.uint32)[:, None], (len(v), n)))
    out = ctx.upload(np.full(t * m, 7, np.uint32))
    zs.adapter_linear(ctx, rows(xv), rows(wv), t, m, n, out)
    assert np.array_equal(out.download().reshape(t, m), (xv[:, None] * wv % P) * n % P)


def test_counters_are_zero_behind_every_call(ctx):
    """Rows that all CTAs share, rows of their own, none and more than 256 sequences, one behind the other on one workspace without waiting in between."""
    batches = [Batch(ctx, i, lens, 4, 2, 64, 16, i % 2 == 0) for i, lens in enumerate(([20000, 0, 300], [9000] * 6, [0, 0], [1], [50, 0, 200, 130] * 80))]
    ws = max((b.workspace() for b in batches), key=lambda w: w.n)
    outs = [[b.call(ws) for b in batches] for _ in range(3)]
    ctx.sync()
    assert all(b.right(o) for row in outs for b, o in zip(batches, row))
    assert not ws.download()[:192].any()


def test_counters_that_somebody_left_are_reported(ctx):
    """What a call whose lengths changed under it may leave behind: parts of a row that nobody added up.  Every call that finds such counters is reported, whatever
    its own rows are, until the workspace is zeroed again."""
    b, other = Batch(ctx, 1, [20000, 0, 300], 4, 1, 64, 64, True), Batch(ctx, 2, [5], 4, 1, 64, 64, True)
    clean = b.workspace()
    dirty = clean.download()
    dirty[3], dirty[sm_count()] = 2, 2 << 16                # two parts of the row that begins in CTA 3
    ws = ctx.upload(dirty)
    for batch in (other, b, other):
        batch.call(ws)
        with pytest.raises(zk.ZkbError, match="not valid") as e:
            ctx.sync()
        assert e.value.code == 8
    for batch in (b, other, b):
        out = batch.call(clean)
        ctx.sync()
        assert batch.right(out)


def sm_count():
    import torch
    return torch.cuda.get_device_properties(0).multi_processor_count


def test_tokens_one_after_the_other_in_a_16_bit_cache(ctx):
    """Append with rotation and attention for token after token, the values requantised by the caller in between: step by step, then captured once and replayed."""
    import torch
    rng = np.random.default_rng(8)
    h, kv, d, page, room = 8, 2, 64, 16, 7
    lens = [0, 15, 40, 131, 16]
    b = len(lens)
    paged = Paged(ctx, rng, [n + room for n in lens], kv, d, page, True)
    angle = rng.uniform(0, 6.3, (max(lens) + room, d // 2))
    cs = np.round(np.stack([np.cos(angle), np.sin(angle)], -1) * (1 << 14)).astype(np.int32)
    exp, shift = tables.build_exp_table(1000), shift_for(d) + 1         # a turned vector's elements may be the square root of two larger
    stream = torch.cuda.ExternalStream(ctx.stream)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    k, v, q, turned, out, status, start, after = z(b, kv, d), z(b, kv, d), z(b, h, d), z(b, h, d), z(b, h, d), z(b), z(b), z(b)
    rows, cs_dev, exp_dev = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (np.arange(b + 1), cs, exp))
    rotation = zs.Rotation(cs_dev, len(cs), d, 14)
    ws = torch.zeros(zs.paged_attention_workspace(paged.cache, b, h), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def step():
        zs.kv_append(paged.cache, k, v, b, paged.table_dev, b, paged.max_blocks, rows, start, status, rotation=rotation, q=q, q_out=turned, num_heads=h)
        zs.paged_attention(paged.cache, turned, paged.table_dev, b, paged.max_blocks, after, h, exp_dev, out, status, score_shift=shift, workspace=ws)

    graph = None
    for i in range(room):
        new = [small(rng, 127, b, kv, d), small(rng, 32767, b, kv, d), small(rng, 127, b, h, d)]
        with torch.cuda.stream(stream):
            for to, a in zip((k, v, q), new):
                to.copy_(torch.from_numpy(a.view(np.int32)))
            start.copy_(torch.tensor(lens, dtype=torch.int32))
            after.copy_(torch.tensor([n + 1 for n in lens], dtype=torch.int32))
        if i == 3:
            ctx.sync()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
                step()
        if graph:
            with torch.cuda.stream(stream):
                graph.replay()
        else:
            step()
        zs.check_status(ctx, status)
        want_q = np.zeros((b, h, d), np.int64)
        assert not R.append(paged.k, paged.v, new[0], new[1], paged.table, list(range(b + 1)), lens, cs, 14, False, new[2], want_q, True).any()
        lens = [n + 1 for n in lens]
        want, codes = R.attend(paged.k, paged.v, want_q, paged.table, lens, exp, shift)
        assert not codes.any() and np.array_equal(turned.cpu().numpy(), want_q) and np.array_equal(out.cpu().numpy(), want)
        got_k, got_v = paged.fetch()
        assert np.array_equal(got_k, paged.k) and np.array_equal(got_v, paged.v)
