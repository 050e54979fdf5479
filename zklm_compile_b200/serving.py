"""Token-by-token forward passes in the field: a paged key-value cache, the attention that reads it, projections with adapters.

The reference's forward pass takes a whole sequence (rust/zk_ml_prover/src/pipeline/forward.rs:233-276, 594-640) or one vector
(transformer/mod.rs:140-163); these calls compute the same rows for one new token at a time, in the same exact arithmetic: what
`paged_attention` returns over a cache with score_shift 0 is the row that `attention.row_attention_forward` returns over the whole sequence
(which has neither a shift nor a mask: scores that need a shift to be inputs of the table have no proof there, and a row of a prompt is one
over all of its positions), and what `adapter_linear` returns is the product with the merged matrix W + B A.

Arguments on the GPU are `DeviceBuffer`s, or tensors of another library on the context's GPU (anything with data_ptr, numel,
element_size and is_contiguous, e.g. torch's).  Calls are enqueued on the context's stream (`Context.stream`) and not waited for: a
caller that fills its tensors on another stream orders the two, and changes nothing that a call reads (lengths and block tables included)
before it has run.  Memory is kept until then, too: a DeviceBuffer that is dropped waits for the stream, but torch's allocator hands a dropped
tensor's memory out in the order of its own streams unless it is told, `x.record_stream(torch.cuda.ExternalStream(ctx.stream))`.  What only the
device sees (`STATUS`) is added to the caller's status words, one per sequence, which `check_status` reads.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import check
from .sumcheck import Context, DeviceBuffer

STATUS = {1: "a length or position outside the block table, or a page number outside the pool", 2: "a position that the rotation's table does not have",
          3: "a value that a 16-bit cache cannot hold", 4: "attention: a score is not an input of the exp table", 5: "attention: the weights of a row add up to zero"}


class _Cache(C.Structure):
    _fields_ = [("k_pages", C.c_void_p), ("v_pages", C.c_void_p), ("page_stride", C.c_uint64), ("num_pages", C.c_uint32), ("page_size", C.c_uint32),
                ("num_kv_heads", C.c_uint32), ("d_head", C.c_uint32), ("elem", C.c_int32)]


class _Rotation(C.Structure):
    _fields_ = [("cos_sin", C.c_void_p), ("positions", C.c_uint32), ("rot_dim", C.c_uint32), ("shift", C.c_uint32), ("pairs", C.c_int32)]


_vp, _u32, _sz = C.c_void_p, C.c_uint32, C.c_size_t
_ARGS = {
    "zkb_kv_append": [_vp, _vp, _vp, _sz, _vp, _sz, _u32, _vp, _u32, _u32, _vp, _vp, _vp, _vp, _sz, _u32, _vp, _sz, _vp],
    "zkb_paged_attention": [_vp, _vp, _vp, _sz, _u32, _vp, _u32, _u32, _vp, _vp, _sz, _u32, _vp, _vp, _vp, _sz],
    "zkb_adapter_linear": [_vp, _vp, _sz, _vp, _vp, _u32, _u32, _u32, _vp, _vp, _u32, _u32, _vp, _vp, _sz, _vp, _sz],
    "zkb_paged_attention_workspace": [_vp, _vp, _u32, _u32],
    "zkb_adapter_linear_workspace": [_vp, _u32, _u32, _u32, _u32, _u32],
}
_fns: dict = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(_lib.lib(), name)
        f.argtypes = _ARGS[name]
        f.restype = _sz if name.endswith("_workspace") else C.c_int32
    return f


_MAX = 0xffffffff


def _counts(**sizes) -> None:
    """Every size fits the C interface's unsigned 32 bits (the calls below look at all of them at once first)."""
    for what, v in sizes.items():
        if not 0 <= v <= _MAX:
            raise ValueError(f"{what}: {v} is not in [0, 2^32)")


def _addr(ctx: Context, x, least: int, what: str, size: int = 4) -> int:
    """Address of a device array of at least `least` elements of `size` bytes."""
    if type(x) is not DeviceBuffer:
        try:
            if x.nbytes >= least * size and x.itemsize == size and x.get_device() == ctx.device and x.is_contiguous():
                return x.data_ptr()
        except AttributeError:
            pass
    return _addr_or_why(ctx, x, least, what, size)


def _addr_or_why(ctx: Context, x, least: int, what: str, size: int) -> int:
    """The same for DeviceBuffers and other libraries' tensors, and what is wrong with an array that cannot be taken."""
    if isinstance(x, DeviceBuffer):
        if x.ctx.device != ctx.device:
            raise ValueError(f"{what} lies on another GPU than the context")
        have = 4 * x.n
        at = C.cast(x.ptr, C.c_void_p).value or 0
        if not at:
            raise ValueError(f"{what} has been freed")
    else:
        try:
            at, unit, dense, on = x.data_ptr(), x.element_size(), x.is_contiguous(), x.get_device()
            have = x.numel() * unit
        except AttributeError:
            raise TypeError(f"{what}: a DeviceBuffer or a tensor on the GPU is wanted, not {type(x).__name__}") from None
        if on != ctx.device:
            raise ValueError(f"{what} lies on another device than the context's GPU")
        if not dense or unit != size:
            raise ValueError(f"{what}: a contiguous tensor of {size}-byte elements is wanted")
    if have < least * size:
        raise ValueError(f"{what}: {have // size} elements, {least} are needed")
    return at


def _rows(count: int, row: int, stride: int) -> int:
    """Elements that `count` rows of `row` reach over, `stride` apart (0: dense)."""
    if not stride:
        return count * row
    if stride < row:
        raise ValueError(f"a stride of {stride} is less than a row of {row}")
    return (count - 1) * stride + row if count else 0


class KvCache:
    """Pages of [num_kv_heads][page_size][d_head] elements for K and for V: field elements, or with `small` 16-bit centred integers.
    `k_pages` and `v_pages` are the caller's arrays; without them the cache allocates its own, zeroed.  `page_stride` (elements, 0: dense)
    is the distance between pages, so that one array can hold both in turn.  What a cache is made with is fixed: the library holds its addresses and sizes."""

    def __init__(self, ctx: Context, page_size: int, num_kv_heads: int, d_head: int, num_pages: int, small: bool = False, k_pages=None, v_pages=None,
                 page_stride: int = 0):
        page_size, num_kv_heads, d_head, num_pages, page_stride = int(page_size), int(num_kv_heads), int(d_head), int(num_pages), int(page_stride)
        _counts(page_size=page_size, num_kv_heads=num_kv_heads, d_head=d_head, num_pages=num_pages)
        size, page = (2 if small else 4), num_kv_heads * page_size * d_head
        if (k_pages is None) != (v_pages is None):
            raise ValueError("k_pages and v_pages: both or neither")
        if min(page, num_pages) <= 0:
            raise ValueError("a cache has at least one page, key head and element")
        reach = _rows(num_pages, page, page_stride)
        if k_pages is None:
            import numpy as np
            words = (reach * size + 3) // 4
            k_pages, v_pages = (ctx.upload(np.zeros(words, np.uint32)) for _ in range(2))
        self._pages, self._ctx, self._row, self._d = (k_pages, v_pages), ctx, num_kv_heads * d_head, d_head
        self._c = _Cache(_addr(ctx, k_pages, reach, "k_pages", size), _addr(ctx, v_pages, reach, "v_pages", size), page_stride, num_pages, page_size, num_kv_heads, d_head,
                         int(bool(small)))
        self._at = C.addressof(self._c)

    ctx = property(lambda self: self._ctx)
    k_pages, v_pages = property(lambda self: self._pages[0]), property(lambda self: self._pages[1])
    page_size, num_kv_heads, d_head = property(lambda self: self._c.page_size), property(lambda self: self._c.num_kv_heads), property(lambda self: self._c.d_head)
    num_pages, page_stride, small = property(lambda self: self._c.num_pages), property(lambda self: self._c.page_stride), property(lambda self: bool(self._c.elem))


class Rotation:
    """Rotation by position: `cos_sin` holds (positions, rot_dim / 2, 2) signed integers with `shift` fractional bits; the first rot_dim elements
    of a head turn, element i with i + rot_dim / 2, or 2i with 2i + 1 if `pairs`."""

    def __init__(self, cos_sin, positions: int, rot_dim: int, shift: int = 14, pairs: bool = False):
        self.cos_sin, self.positions, self.rot_dim, self.shift, self.pairs = cos_sin, int(positions), int(rot_dim), int(shift), bool(pairs)
        _counts(positions=self.positions, rot_dim=self.rot_dim, shift=self.shift)
        self._c = _Rotation(None, self.positions, self.rot_dim, self.shift, int(self.pairs))
        self._words = self.positions * self.rot_dim
        self._at = C.addressof(self._c)


class Adapters:
    """Low-rank adapters of one projection: `a` holds (count, rank, n), `b` (count, m, rank) field elements; a scale is part of `b`."""

    def __init__(self, a, b, count: int, rank: int):
        self.a, self.b, self.count, self.rank = a, b, int(count), int(rank)
        _counts(adapters=self.count, rank=self.rank)


def kv_append(cache: KvCache, k, v, num_tokens: int, block_table, num_seqs: int, max_blocks: int, row_start, start, status, rotation: Rotation | None = None,
              q=None, q_out=None, num_heads: int = 0, k_stride: int = 0, v_stride: int = 0, q_stride: int = 0, q_out_stride: int = 0) -> None:
    """Put k, v (num_tokens, num_kv_heads, d_head) into the cache: sequence s brings tokens row_start[s] .. row_start[s + 1] - 1, which get the positions
    from start[s] on; position p is row p % page_size of page block_table[s][p / page_size].  With a rotation K turns by its position, and so does
    q (num_tokens, num_heads, d_head) on its way to q_out (which may be q).  Rows outside every sequence are padding and left alone."""
    ctx, t, s, blocks, heads, row = cache._ctx, num_tokens, num_seqs, max_blocks, num_heads, cache._row
    if not (0 <= t <= _MAX and 0 <= s <= _MAX and 0 <= blocks <= _MAX and 0 <= heads <= _MAX):
        _counts(num_tokens=t, num_seqs=s, max_blocks=blocks, num_heads=heads)
    rot = q_at = q_out_at = None
    if rotation is not None:
        rot = rotation._at
        rotation._c.cos_sin = _addr(ctx, rotation.cos_sin, rotation._words, "the rotation's table") if rotation._c.rot_dim else None
    if q is not None and q_out is not None:
        q_row = heads * cache._d
        q_at = _addr(ctx, q, _rows(t, q_row, q_stride) if q_stride else t * q_row, "q")
        q_out_at = _addr(ctx, q_out, _rows(t, q_row, q_out_stride) if q_out_stride else t * q_row, "q_out")
    elif q is not None or q_out is not None:
        raise ValueError("q and q_out: both or neither")
    st = _fn("zkb_kv_append")(
        ctx.h, cache._at, _addr(ctx, k, _rows(t, row, k_stride) if k_stride else t * row, "k"), k_stride,
        _addr(ctx, v, _rows(t, row, v_stride) if v_stride else t * row, "v"), v_stride, t, _addr(ctx, block_table, s * blocks, "block_table"), s, blocks,
        _addr(ctx, row_start, s + 1, "row_start"), _addr(ctx, start, s, "start"), rot, q_at, q_stride, heads, q_out_at, q_out_stride, _addr(ctx, status, s, "status"))
    if st:
        check(ctx.h, st)


def paged_attention_workspace(cache: KvCache, num_seqs: int, num_heads: int) -> int:
    """Bytes of workspace for calls of this size: a captured call needs one of its own, 256-byte aligned, zeroed once before its first call and used by this
    operator alone from then on (and zeroed again if a call on it gave up, ZkbError of code 8)."""
    _counts(num_seqs=num_seqs, num_heads=num_heads)
    return int(_fn("zkb_paged_attention_workspace")(cache.ctx.h, cache._at, num_seqs, num_heads))


def paged_attention(cache: KvCache, q, block_table, num_seqs: int, max_blocks: int, lens, num_heads: int, exp_table, out, status, score_shift: int = 0,
                    q_stride: int = 0, workspace=None, n_table: int = 65536) -> None:
    """One new token per sequence: q (num_seqs, num_heads, d_head) over the first lens[s] positions of the cache, into out (num_seqs, num_heads, d_head).
    The score q . k_j, divided by 2^score_shift and rounded half away from zero, must be an input of the exp table; a sequence of length 0 and a
    row that is refused (status) give zeros.  `out` overlaps no input."""
    ctx, s, blocks, heads, row = cache._ctx, num_seqs, max_blocks, num_heads, num_heads * cache._d
    if not (0 <= s <= _MAX and 0 <= blocks <= _MAX and 0 <= heads <= _MAX and 0 <= score_shift <= _MAX):
        _counts(num_seqs=s, max_blocks=blocks, num_heads=heads, score_shift=score_shift)
    at, size = _workspace(ctx, workspace) if workspace is not None else (None, 0)
    st = _fn("zkb_paged_attention")(
        ctx.h, cache._at, _addr(ctx, q, _rows(s, row, q_stride) if q_stride else s * row, "q"), q_stride, heads, _addr(ctx, block_table, s * blocks, "block_table"), s, blocks,
        _addr(ctx, lens, s, "lens"), _addr(ctx, exp_table, n_table, "exp_table"), n_table, score_shift, _addr(ctx, out, s * row, "out"),
        _addr(ctx, status, s, "status"), at, size)
    if st:
        check(ctx.h, st)


def adapter_linear_workspace(ctx: Context, tokens: int, m: int, n: int, num_adapters: int = 0, rank: int = 0) -> int:
    """Bytes of workspace for calls of this size; more tokens may need less than fewer, so ask for the size that is called."""
    _counts(tokens=tokens, m=m, n=n, num_adapters=num_adapters, rank=rank)
    return int(_fn("zkb_adapter_linear_workspace")(ctx.h, tokens, m, n, num_adapters, rank))


def adapter_linear(ctx: Context, x, w, tokens: int, m: int, n: int, out, bias=None, adapters: Adapters | None = None, adapter_of=None, x_stride: int = 0,
                   out_stride: int = 0, workspace=None) -> None:
    """out[t] = W x[t] + bias + B[a] (A[a] x[t]), a = adapter_of[t] (outside the adapters: none), for `tokens` rows x of n words; W is m x n, row-major.
    `out` overlaps no input; rows of x and of out may alternate in one array."""
    if not (0 <= tokens <= _MAX and 0 <= m <= _MAX and 0 <= n <= _MAX):
        _counts(tokens=tokens, m=m, n=n)
    if (adapters is None) != (adapter_of is None):
        raise ValueError("adapters and adapter_of: both or neither")
    at, size = _workspace(ctx, workspace) if workspace is not None else (None, 0)
    a = b = of = None
    count = rank = 0
    if adapters is not None:
        count, rank = adapters.count, adapters.rank
        a, b, of = _addr(ctx, adapters.a, count * rank * n, "A"), _addr(ctx, adapters.b, count * m * rank, "B"), _addr(ctx, adapter_of, tokens, "adapter_of")
    st = _fn("zkb_adapter_linear")(
        ctx.h, _addr(ctx, x, _rows(tokens, n, x_stride) if x_stride else tokens * n, "x"), x_stride, _addr(ctx, w, m * n, "w"),
        _addr(ctx, bias, m, "bias") if bias is not None else None, tokens, m, n, a, b, count, rank, of,
        _addr(ctx, out, _rows(tokens, m, out_stride) if out_stride else tokens * m, "out"), out_stride, at, size)
    if st:
        check(ctx.h, st)


def _workspace(ctx, w):
    """A workspace may have elements of any size."""
    size = 4 if isinstance(w, DeviceBuffer) else getattr(w, "itemsize", 1)
    at = _addr(ctx, w, 0, "workspace", size)
    return at, (4 * w.n if isinstance(w, DeviceBuffer) else w.numel() * size)


def check_status(ctx: Context, status) -> None:
    """Wait for the context's stream and raise ZkbError for the first sequence whose status word is set."""
    ctx.sync()
    words = status.download().reshape(-1) if isinstance(status, DeviceBuffer) else status.reshape(-1).tolist()
    for s, code in enumerate(words):
        if code:
            raise _lib.ZkbError(2, f"sequence {s}: {STATUS.get(int(code), f'status {int(code)}')}")
