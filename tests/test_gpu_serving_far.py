"""Caches and matrices of more than 2^32 elements: what lies behind the 32-bit offsets is read and written where it is, and what lies at the same offset mod 2^32
is left alone."""
import numpy as np
import pytest

import zklm_compile_b200 as zk
from tests import serving_ref as R
from tests.test_gpu_serving import P, shift_for, small, words
from zklm_compile_b200 import serving as zs, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch
    c = zk.Context(0)
    yield c
    c.close()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("is_small,page,d", [(True, 64, 128), (False, 16, 128), (True, 4, 126)])
def test_cache_of_more_than_32_bits(ctx, is_small, page, d):
    import torch
    rng = np.random.default_rng(d)
    kv, h, lens = 8, 16, [150, 3, 77]
    dense = kv * page * d
    pages = (1 << 32) // dense + 200
    k, v = (torch.zeros(pages, kv, page, d, dtype=torch.int16 if is_small else torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    blocks = [-(-n // page) for n in lens]
    far = (1 << 32) // dense + 1 + rng.permutation(190)         # all behind 2^32 elements
    table, at = np.full((3, max(blocks)), -1, np.int32), 0
    for s, n in enumerate(blocks):
        table[s, :n] = far[at:at + n]
        at += n
    cache = zs.KvCache(ctx, page, kv, d, pages, is_small, k, v)
    t = sum(lens)
    new_k, new_v, q = small(rng, 127, t, kv, d), small(rng, 32767, t, kv, d), small(rng, 127, 3, h, d)
    rows, start = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), np.zeros(3, np.int32)
    status, out, exp = ctx.upload(np.zeros(3, np.uint32)), ctx.upload(np.zeros(3 * h * d, np.uint32)), tables.build_exp_table(1000)
    table_dev = ctx.upload(words(table))
    zs.kv_append(cache, ctx.upload(new_k), ctx.upload(new_v), t, table_dev, 3, table.shape[1], ctx.upload(words(rows)), ctx.upload(words(start)), status)
    zs.paged_attention(cache, ctx.upload(q), table_dev, 3, table.shape[1], ctx.upload(words(np.array(lens, np.int32))), h, ctx.upload(exp), out, status, score_shift=shift_for(d))
    zs.check_status(ctx, status)
    # the same in a cache of the far pages alone, by the definition
    near = np.where(table >= 0, table - (int(far.min())), -1)
    want_k, want_v = (np.zeros((int(far.max() - far.min()) + 1, kv, page, d), np.int16 if is_small else np.uint32) for _ in range(2))
    assert not R.append(want_k, want_v, new_k, new_v, near, rows, start, small=is_small).any()
    want, codes = R.attend(want_k, want_v, q, near, lens, exp, shift_for(d))
    assert not codes.any() and np.array_equal(out.download().reshape(want.shape), want)
    for have, expect in ((k, want_k), (v, want_v)):
        assert np.array_equal(have[int(far.min()):int(far.max()) + 1].cpu().numpy().view(expect.dtype), expect)
        assert not bool(have[:int(far.min())].any())            # nothing came to lie 2^32 elements too early


@pytest.mark.parametrize("m,n", [(300000, 14400), (180001, 24001)])
def test_matrix_of_more_than_32_bits(ctx, m, n):
    import torch
    assert m * n > 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    w = torch.randint(0, P, (m, n), generator=g, dtype=torch.int32, device="cuda")
    x = torch.randint(0, P, (3, n), generator=g, dtype=torch.int32, device="cuda")
    y = torch.zeros(3, m, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    zs.adapter_linear(ctx, x, w, 3, m, n, y)
    ctx.sync()
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        part = w[rows].to(torch.int64)
        for t in range(3):
            assert torch.equal(y[t, rows].to(torch.int64), (part * x[t].to(torch.int64) % P).sum(1) % P)
