"""Tensors of torch that a program drops while a call on the context's stream has yet to read them: the documented way of telling torch's allocator."""
import numpy as np
import pytest

import zklm_compile_b200 as zk
from tests import serving_ref as R
from tests.test_gpu_serving import P
from zklm_compile_b200 import serving as zs

pytestmark = pytest.mark.gpu


def test_dropped_tensors_that_the_allocator_knows_to_be_in_use():
    import torch
    ctx = zk.Context(0)
    stream = torch.cuda.ExternalStream(ctx.stream)
    make = lambda *s: torch.randint(0, P, s, dtype=torch.int32, device="cuda")
    heavy = make(1024, 4096), make(4096, 4096), make(1024, 4096)
    x, w, out = make(5, 2 << 18), make(3, 2 << 18), torch.zeros(5, 3, dtype=torch.int32, device="cuda")
    want = R.linear(x.cpu().numpy(), w.cpu().numpy())
    torch.cuda.synchronize()
    for _ in range(20):                                     # milliseconds in which x waits to be read
        zs.adapter_linear(ctx, heavy[0], heavy[1], 1024, 4096, 4096, heavy[2])
    zs.adapter_linear(ctx, x, w, 5, 3, 2 << 18, out)
    x.record_stream(stream)
    w.record_stream(stream)
    where = {x.data_ptr(), w.data_ptr()}
    del x, w
    others = [torch.full((n, 2 << 18), 7, dtype=torch.int32, device="cuda") for n in (5, 3, 5, 3)]
    assert not where & {o.data_ptr() for o in others}
    ctx.sync()
    assert np.array_equal(out.cpu().numpy(), want)
    ctx.close()
