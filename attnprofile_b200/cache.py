"""A paged cache of keys and values held in 8 bits, and attention over it.

Python face of the cache entry points of the C ABI (include/attnprof.h):

  block_tables   block tables and slot maps of a step from request lengths
  block_trim     blocks of ended or shortened requests back to the pool
  cache_append   keys and values of new tokens quantised into the cache
  attn_cached    attention of each request's newest tokens over its cache

and CacheBatch, which runs them together for the requests of a server.  All
work is asynchronous on `stream` (default: the current stream of the tensors'
device), never synchronises, and can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _check, lib

__all__ = ["PagedCache", "BlockPool", "BlockPlan", "CacheBatch", "block_tables", "block_trim",
           "cache_append", "attn_cached", "cached_workspace", "BLOCK_SIZES", "BLOCKS", "MAX_BATCH"]

BLOCK_SIZES = (16, 32, 64, 128)
#: Values of the status word that block_tables and block_trim write.
BLOCKS = {"OK": 0, "POOL": 1, "ROW": 2, "SLOTS": 3, "NEGATIVE": 4}
MAX_BATCH = 16384
_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_INT32 = torch.int32
_workspace_bytes: dict = {}
_functions: dict = {}


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The same without building a Stream object (2 us less per call), where this
# torch offers it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
# And the current device (CUDA is initialised: there are tensors).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream(index, stream) -> int:
    """The handle of a stream that a call was given."""
    if stream.device.index != index:
        raise ValueError(f"the stream is on {stream.device}, the tensors on cuda:{index}")
    return stream.cuda_stream


# The argument structs of include/attnprof.h, field by field in their order ("0q":
# and the padding behind the last one).
_TABLES = struct.Struct("@10Qq5i0q").pack
_TRIM = struct.Struct("@8Qq4i0q").pack
_APPEND = struct.Struct("@7Q4q7i0q").pack
_CACHED = struct.Struct("@11Q5q12if0q").pack


def _call(name, index, *args):
    """A C entry point with the tensors' device current."""
    if _current_device() != index:
        with torch.cuda.device(index):
            return _call(name, index, *args)
    function = _functions.get(name)
    if function is None:
        function = _functions[name] = getattr(lib(), name)
    rc = function(*args)
    if rc:
        _check(rc, name)


def _empty(shape, dtype, device, stream):
    """A new tensor for work on `stream` that the current stream may use too."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        x = torch.empty(shape, dtype=dtype, device=device)
    x.record_stream(torch.cuda.current_stream(device))
    return x


def _ints(name, t, index, n):
    """Checks an int32 vector of n; its address."""
    if t.dtype is not _INT32:
        raise TypeError(f"{name} must be int32")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of shape ({n},)")
    return t.data_ptr()


def _table(tables, index, batch):
    if tables.dtype is not _INT32:
        raise TypeError("tables must be int32")
    if tables.get_device() != index:
        raise ValueError(f"tables must be on cuda:{index}")
    shape = tables.shape
    if len(shape) != 2 or shape[0] != batch:
        raise ValueError(f"tables must be [{batch}, width]")
    width = shape[1]
    row, one = tables.stride()
    if (width > 1 and one != 1) or (batch > 1 and row < width):
        raise ValueError("rows of tables must be contiguous and may not overlap")
    return tables.data_ptr(), width, row if batch > 1 else width


class _Checked:
    """Tensors that are checked when they are first used, and again once one was
    replaced or has other memory."""

    __slots__ = ("_seen", "_at", "_held")

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        for kept in _Checked.__slots__:  # (the memory of the tensor before too)
            object.__setattr__(self, kept, None)

    def _keep(self, tensors, *seen):
        """Remembers what a check gave, the tensors' addresses last.  It holds as
        long as _at, which reads them, gives the same: their memory is held until
        then, so that no other tensor can get the same address."""
        seen += (tuple(t.data_ptr() for t in tensors),)
        object.__setattr__(self, "_seen", seen)
        object.__setattr__(self, "_at", tuple(t.data_ptr for t in tensors))
        object.__setattr__(self, "_held", tuple(t.untyped_storage() for t in tensors))
        return seen


class PagedCache(_Checked):
    """Keys and values of one layer in a pool of blocks.

    k, v: codes [num_blocks, kv_heads, block_size, D], float8_e4m3fn or int8;
    k_scale, v_scale: float32 [num_blocks, kv_heads], all contiguous CUDA
    tensors of one device.  A code c of block b, head h stands for
    c * scale[b, h].  The object holds the tensors and nothing else; they may
    be replaced by others (all that belong together, before the next call)."""

    __slots__ = ("k", "v", "k_scale", "v_scale")

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._now()

    def _now(self):
        """(device index, num_blocks, kv_heads, block_size, D, code, addresses)."""
        seen = self._seen
        if seen is not None:
            k, v, k_scale, v_scale = self._at
            if seen[6] == (k(), v(), k_scale(), v_scale()):
                return seen
        k, v, k_scale, v_scale = tensors = self.k, self.v, self.k_scale, self.v_scale
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must share one [num_blocks, kv_heads, block_size, D] shape "
                             "and dtype")
        if k.dtype not in _CODES:
            raise TypeError(f"unsupported codes {k.dtype} (float8_e4m3fn or int8)")
        num_blocks, kv_heads, block_size, dim = k.shape
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size {block_size} is not one of {BLOCK_SIZES}")
        if dim not in (64, 128):
            raise ValueError(f"D = {dim} is not 64 or 128")
        if not k.is_cuda:
            raise ValueError("k must be a CUDA tensor")
        for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t.device != k.device:
                raise ValueError(f"{name} must be on {k.device}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32")
            if t.shape != k.shape[:2]:
                raise ValueError(f"{name} must be [num_blocks, kv_heads]")
        return self._keep(tensors, k.get_device(), num_blocks, kv_heads, block_size, dim,
                          _CODES[k.dtype])

    device = property(lambda self: self.k.device)
    num_blocks = property(lambda self: self._now()[1])
    kv_heads = property(lambda self: self._now()[2])
    block_size = property(lambda self: self._now()[3])
    dim = property(lambda self: self._now()[4])
    code = property(lambda self: self._now()[5])
    ptrs = property(lambda self: self._now()[6])

    @classmethod
    def empty(cls, num_blocks: int, kv_heads: int, dim: int, *, block_size: int = 32,
              dtype=torch.float8_e4m3fn, device="cuda"):
        """A cache that holds nothing yet."""
        shape = (num_blocks, kv_heads, block_size, dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        ks, vs = (torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


class BlockPool(_Checked):
    """The free blocks of a pool: the stack free[0 : free_count[0]] of block
    ids (int32, capacity = the number of blocks)."""

    __slots__ = ("free", "free_count", "block_size")

    def __init__(self, free, free_count, block_size: int):
        self.free, self.free_count, self.block_size = free, free_count, block_size
        self._now()

    def _now(self):
        """(device index, num_blocks, block_size, addresses of free and free_count)."""
        seen = self._seen
        if seen is not None:
            free, free_count = self._at
            if seen[3] == (free(), free_count()):
                return seen
        free, free_count, block_size = self.free, self.free_count, self.block_size
        if not free.is_cuda or free.dim() != 1 or free.numel() == 0:
            raise ValueError("free must be a CUDA tensor [num_blocks]")
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"block_size {block_size} is not one of {BLOCK_SIZES}")
        index, num_blocks = free.get_device(), free.numel()
        _ints("free", free, index, num_blocks)
        _ints("free_count", free_count, index, 1)
        return self._keep((free, free_count), index, num_blocks, block_size)

    device = property(lambda self: self.free.device)
    num_blocks = property(lambda self: self._now()[1])

    @classmethod
    def full(cls, num_blocks: int, block_size: int, device="cuda"):
        """All blocks free, block 0 on top."""
        free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(free, torch.full((1,), num_blocks, dtype=torch.int32, device=device),
                   block_size)


class BlockPlan(_Checked):
    """What block_tables writes: kv_lens [batch], starts [batch + 1], slots
    [tokens] and the status word [1] (BLOCKS), all int32."""

    __slots__ = ("kv_lens", "starts", "slots", "status")

    def __init__(self, kv_lens, starts, slots, status):
        self.kv_lens, self.starts, self.slots, self.status = kv_lens, starts, slots, status

    def _ptrs(self, index, batch, tokens):
        """Addresses of the four for `batch` requests on device `index`."""
        seen, want = self._seen, (index, batch, tokens)
        if seen is not None and seen[0] == want:
            kv_lens, starts, slots, status = self._at
            if seen[1] == (kv_lens(), starts(), slots(), status()):
                return seen[1]
        _ints("plan.kv_lens", self.kv_lens, index, batch)
        _ints("plan.starts", self.starts, index, batch + 1)
        _ints("plan.slots", self.slots, index, tokens)
        _ints("plan.status", self.status, index, 1)
        return self._keep((self.kv_lens, self.starts, self.slots, self.status), want)[1]

    @classmethod
    def empty(cls, batch: int, tokens: int, device="cuda"):
        new = lambda n: torch.empty(n, dtype=torch.int32, device=device)  # noqa: E731
        return cls(new(batch), new(batch + 1), new(tokens), new(1))


def block_tables(pool: BlockPool, lens, new_lens, tables, tokens: int, *, plan=None,
                 free_left=None, stream=None) -> BlockPlan:
    """Blocks, slots and lengths of one step: request r holds lens[r] tokens
    and gets new_lens[r] more.  New blocks come from the pool and are written
    into `tables` [batch, width]; the rest goes into `plan` (a new one by
    default; its kv_lens may be `lens`).  `tokens` is the length of the slot
    map, at least the number of new tokens; behind them slots are -1.
    pool.free_count becomes what is left, or keeps its value if free_left
    takes it.  All or nothing: plan.status tells (on the device) whether the
    pool, the table rows and the slot map were large enough."""
    index, num_blocks, block_size, stack = pool._now()
    batch = lens.shape[0]
    s = _raw_stream(index) if stream is None else _stream(index, stream)
    if plan is None:
        plan = BlockPlan(*(_empty(n, torch.int32, pool.device, stream)
                           for n in (batch, batch + 1, tokens, 1)))
    left = stack[1] if free_left is None else _ints("free_left", free_left, index, 1)
    t, width, stride = _table(tables, index, batch)
    kv_lens, starts, slots, status = plan._ptrs(index, batch, tokens)
    _call("attn_block_tables", index, _TABLES(
        _ints("lens", lens, index, batch), _ints("new_lens", new_lens, index, batch), t,
        *stack, kv_lens, starts, slots, left, status, stride, batch, width, num_blocks,
        block_size, tokens), s)
    return plan


def block_trim(pool: BlockPool, lens, keep, tables, *, lens_left=None, free_left=None,
               status=None, stream=None):
    """Request r keeps its first min(lens[r], keep[r]) tokens; the blocks
    behind them go back to the pool.  Writes lens_left (default: `lens`
    itself) and free_left (default: pool.free_count); returns the status word
    [1] (BLOCKS; anything but OK: nothing was changed).  A block that is kept in
    part keeps its scale, which the tokens given up may have made larger, or
    NaN (where they were not finite), until it is begun anew."""
    index, num_blocks, block_size, stack = pool._now()
    batch = lens.shape[0]
    s = _raw_stream(index) if stream is None else _stream(index, stream)
    if lens_left is None:
        lens_left = lens
    left = stack[1] if free_left is None else _ints("free_left", free_left, index, 1)
    if status is None:
        status = _empty(1, torch.int32, pool.device, stream)
    t, width, stride = _table(tables, index, batch)
    _call("attn_block_trim", index, _TRIM(
        _ints("lens", lens, index, batch), _ints("keep", keep, index, batch), t,
        *stack, _ints("lens_left", lens_left, index, batch), left,
        _ints("status", status, index, 1), stride, batch, width, num_blocks, block_size), s)
    return status


def _rows(name, x, index, heads, dim):
    """Checks a [tokens, heads, D] tensor; its dtype code, shape, strides, and the
    strides of tokens and heads (0 where there is one only, whose stride means
    nothing)."""
    kind = _DTYPES.get(x.dtype)
    if kind is None:
        raise TypeError(f"unsupported dtype {x.dtype} of {name} (float16 or bfloat16)")
    if x.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}")
    shape = x.shape
    tokens, many, last = shape if len(shape) == 3 else (0, 0, 0)
    if last != dim or (heads and many != heads):
        raise ValueError(f"{name} must be [tokens, {heads or 'heads'}, {dim}]")
    token, head, one = strides = x.stride()
    if one != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return kind, shape, strides, token if tokens > 1 else 0, head if many > 1 else 0


def cache_append(cache: PagedCache, k, v, slots, *, stream=None) -> None:
    """Writes k and v [tokens, kv_heads, D] (float16 or bfloat16; slices of a
    larger projection are fine) into the cache at `slots` [tokens] int32.

    A block's scale per head is the least power of two that holds its largest
    number; it grows when new tokens need that, and the block's older codes are
    rounded again.  Negative slots (padding) are skipped.  A number that is not
    finite makes that block's k_scale NaN for its head.  The tokens of
    one block follow each other with consecutive slots, as block_tables gives
    them: no gap, no skipped token between them, and no block twice (pieces of a
    block go into calls of their own)."""
    index, num_blocks, heads, block_size, dim, code, ptrs = cache._now()
    kind, shape, strides, k_token, k_head = _rows("k", k, index, heads, dim)
    if (v.dtype is k.dtype and v.shape == shape and v.get_device() == index
            and v.stride() == strides):  # the usual: slices of one projection
        v_token, v_head = k_token, k_head
    else:
        v_kind, v_shape, _, v_token, v_head = _rows("v", v, index, heads, dim)
        if v_kind != kind or v_shape != shape:
            raise ValueError("k and v must share one shape and dtype")
    tokens = shape[0]
    _call("attn_cache_append", index, _APPEND(
        k.data_ptr(), v.data_ptr(), _ints("slots", slots, index, tokens), *ptrs, k_token, k_head,
        v_token, v_head, tokens, heads, dim, kind, code, num_blocks, block_size),
        _raw_stream(index) if stream is None else _stream(index, stream))


def _workspace(index, heads, kv_heads, dim, max_new, block_size, width) -> int:
    key = (index, heads, kv_heads, dim, max_new, block_size, width)
    n = _workspace_bytes.get(key)
    if n is None:
        if len(_workspace_bytes) > 4096:
            _workspace_bytes.clear()
        out = ctypes.c_ulonglong()
        _call("attn_cached_workspace", index, heads, kv_heads, dim, max_new, block_size, width,
              ctypes.byref(out))
        n = _workspace_bytes[key] = out.value
    return n


def cached_workspace(cache: PagedCache, heads: int, max_new: int, width: int) -> int:
    """Bytes of workspace that attn_cached needs with `heads` query heads and
    tables of `width` entries, whatever the lengths (0: none)."""
    index, _, kv_heads, block_size, dim, _, _ = cache._now()
    return _workspace(index, heads, kv_heads, dim, max_new, block_size, width)


def attn_cached(q, cache: PagedCache, tables, kv_lens, starts, *, max_new: int,
                causal: bool = True, scale: float | None = None, out=None, workspace=None,
                stream=None):
    """Attention of each request's newest tokens over its cache; returns out.

    q, out: [tokens, heads, D], heads a multiple of the cache's; rows
    starts[r] .. starts[r + 1) (starts may not decrease) are the last tokens of
    request r, whose kv_lens[r] tokens lie in the blocks tables[r] (they are in
    the cache already).  Row i of n sees the first kv_lens[r] - n + i + 1 tokens
    (causal) or all of them; a row that sees none becomes 0.  max_new: the most
    rows of any request; n counts those beyond it too.  scale: of the scores,
    1 / sqrt(D) by default.  Rows of `out` beyond max_new and behind starts[-1]
    are left as they were (with out=None: undefined); out must not overlap q.
    Weights are rounded to f16, by up to 2^-11 of themselves or 2^-32 of the
    row's largest.  With many rows values are rounded once more, by up to 2^-11 of themselves,
    where the V scales are no powers of two, and those of a block whose V scale is
    below 2^-22 of the request's largest (of that head) keep an absolute accuracy
    only, 2^-32 of that scale.
    workspace: a uint8 tensor to use instead of a new one per call, of
    cached_workspace(...) bytes; calls that may overlap on the GPU need one
    each."""
    index, num_blocks, kv_heads, block_size, dim, code, ptrs = cache._now()
    kind, shape, _, q_token, q_head = _rows("q", q, index, 0, dim)
    tokens, heads, _ = shape
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of the cache's {kv_heads}")
    if scale is None:
        scale = 0.0
    elif not scale > 2.0 ** -150:  # (in 32 bits that is 0, which stands for the default)
        raise ValueError("scale must be positive in 32 bits")
    if max_new < 0:
        raise ValueError("max_new must not be negative")
    batch = kv_lens.shape[0]
    t, width, stride = _table(tables, index, batch)
    lens_ptr = _ints("kv_lens", kv_lens, index, batch)
    starts_ptr = _ints("starts", starts, index, batch + 1)
    s = _raw_stream(index) if stream is None else _stream(index, stream)
    if out is None:
        out = _empty(shape, q.dtype, q.device, stream)
        o_token, o_head = heads * dim, dim
    else:
        o_kind, o_shape, _, o_token, o_head = _rows("out", out, index, heads, dim)
        if o_kind != kind or o_shape != shape:
            raise ValueError("out must have the shape and dtype of q")
    if workspace is None:
        need = _workspace(index, heads, kv_heads, dim, max_new, block_size, width)
        if need:
            workspace = _empty(need, torch.uint8, q.device, stream)
    else:
        if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
            raise TypeError("workspace must be a contiguous uint8 tensor")
        if workspace.get_device() != index:
            raise ValueError(f"workspace must be on {q.device}")
        need = workspace.numel()
    _call("attn_cached", index, _CACHED(
        q.data_ptr(), out.data_ptr(), *ptrs, t, lens_ptr, starts_ptr,
        workspace.data_ptr() if need else 0, need, q_token, q_head, o_token, o_head, stride, tokens, heads, kv_heads, dim, kind,
        code, num_blocks, block_size, width, batch, max_new, 1 if causal else 0, scale), s)
    return out


class CacheBatch:
    """The requests of a server: `rows` of them, each with a table row of up to
    max_len tokens, over one pool of blocks shared by any number of layers.

    A step is advance() once, then attend() for each layer:

        batch = CacheBatch(BlockPool.full(num_blocks, 32), rows=64, max_len=8192,
                           max_tokens=4096)
        cache = [PagedCache.empty(num_blocks, 8, 128) for _ in layers]
        batch.advance(new_lens, tokens=q.shape[0])
        for each layer: o = batch.attend(cache[i], q, k, v, max_new=1)
        batch.trim(keep)        # ended requests: 0, refused drafts: fewer

    q, k, v hold the new tokens of all requests, request after request;
    padding may follow the last one.  max_tokens: the most rows of any step.
    Nothing waits for the GPU: `status` holds the last advance()'s word (BLOCKS)
    there.  Where it is not OK the step has no tokens: nothing is appended, and
    attend() leaves its output alone.  All arrays are made here and stay where
    they are, so steps can be captured into CUDA graphs (after one step outside);
    the steps of one batch follow each other on the GPU."""

    def __init__(self, pool: BlockPool, rows: int, max_len: int, max_tokens: int):
        device, bs = pool.device, pool.block_size
        if rows <= 0 or max_len <= 0 or max_tokens <= 0:
            raise ValueError("rows, max_len and max_tokens must be positive")
        if rows > MAX_BATCH:
            raise ValueError(f"at most {MAX_BATCH} rows")
        self.pool = pool
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.tables = torch.full((rows, -(-max_len // bs)), -1, dtype=torch.int32, device=device)
        self.starts = torch.zeros(rows + 1, dtype=torch.int32, device=device)
        self.slots = torch.full((max_tokens,), -1, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.trim_status = torch.zeros(1, dtype=torch.int32, device=device)
        self.plan = None

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        if name in ("lens", "starts", "slots", "status"):  # a plan holds these
            self.plan = None

    def advance(self, new_lens, tokens: int, *, stream=None) -> BlockPlan:
        """new_lens[r] tokens more for request r, in a slot map of `tokens`."""
        if not 0 <= tokens <= self.slots.shape[0]:
            raise ValueError(f"tokens must be at most max_tokens = {self.slots.shape[0]}")
        if self.plan is None or self.plan.slots.shape[0] != tokens:
            self.plan = BlockPlan(self.lens, self.starts, self.slots[:tokens], self.status)
        return block_tables(self.pool, self.lens, new_lens, self.tables, tokens, plan=self.plan,
                            stream=stream)

    def attend(self, cache: PagedCache, q, k, v, *, max_new: int, causal: bool = True,
               scale: float | None = None, out=None, stream=None):
        """Appends k and v of the step's tokens, then attends with q.  With
        out=None the rows of padding, of a refused step and beyond max_new are
        undefined."""
        if self.plan is None:
            raise RuntimeError("advance() first")
        if cache.block_size != self.pool.block_size or cache.num_blocks != self.pool.num_blocks:
            raise ValueError("the cache's blocks are not the pool's")
        cache_append(cache, k, v, self.plan.slots, stream=stream)
        return attn_cached(q, cache, self.tables, self.lens, self.starts, max_new=max_new,
                           causal=causal, scale=scale, out=out, stream=stream)

    def trim(self, keep, *, stream=None):
        """Requests keep their first keep[r] tokens; returns the status word.
        (See block_trim for the scales of blocks that are kept in part.)"""
        return block_trim(self.pool, self.lens, keep, self.tables, status=self.trim_status,
                          stream=stream)
