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
