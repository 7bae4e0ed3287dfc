"""The paged 8-bit cache at the limits of what its calls allow: fewer rows than
requests have, scales far from one and from each other, batches next to the
shared memory's limits, arrays that are replaced, every call on a stream given
by name.  Against plain implementations in 64 bits (tests/cache_ref.py)."""
import math
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from tests import cache_ref as ref  # noqa: E402
from tests.test_gpu_cache import CODES, E4M3, TYPES, check_append, ints, make_cache  # noqa: E402

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def ap(engine):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return engine


def rows_of(kv_lens, bs):
    """Table rows for requests of these lengths, one after the other."""
    counts = [ref.blocks_of(n, bs) for n in kv_lens]
    tables, at = [], 0
    for n in counts:
        tables.append(list(range(at, at + n)) + [-1] * (max(counts) - n))
        at += n
    return tables, at


# --------------------------------------------------------------------------- rows beyond max_new
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads,max_new,kv_lens,given", [
    (64, 2, 1, 3, [640], [203]), (128, 4, 1, 2, [300, 77, 5], [9, 2, 5]),   # the split kernel
    (64, 2, 2, 5, [3000, 64], [12, 1]),                                     # its joining kernels
    (64, 2, 1, 50, [640], [250]), (128, 2, 1, 50, [400, 90], [120, 3]),     # the tiled kernel
    (128, 3, 1, 40, [4100], [300]), (64, 2, 2, 150, [700, 400], [400, 150]),
])
def test_rows_beyond_max_new_leave_the_others_as_they_are(ap, kind, dim, heads, kv_heads, max_new,
                                                          kv_lens, given):
    """Causal rows see the tokens up to their own, however many rows follow them."""
    bs = 16
    tables, blocks = rows_of(kv_lens, bs)
    cache, host = make_cache(ap, blocks, kv_heads, bs, dim, E4M3, dim + max_new)
    starts = [sum(given[:i]) for i in range(len(given) + 1)]
    gen = torch.Generator().manual_seed(max_new)
    q = torch.randn(starts[-1], heads, dim, generator=gen).to(kind)
    want, tol = ref.attend_ref(q, *host, tables, kv_lens, starts, True)
    out = torch.full(q.shape, 3.0, dtype=kind, device="cuda")
    ap.attn_cached(q.cuda(), cache, ints(tables), ints(kv_lens), ints(starts), max_new=max_new,
                   out=out)
    got = out.double().cpu()
    for a, b in zip(starts, starts[1:]):
        m = min(b, a + max_new)
        off = (got[a:m] - want[a:m]).abs() / tol[a:m]
        assert torch.all(off <= 1), f"off by {off.max():.3g} times"
        assert torch.all(got[m:b] == 3)


# --------------------------------------------------------------------------- batches and shared memory
TABLES_OF = """
import sys, torch
sys.path.insert(0, {root!r})
import attnprofile_b200 as ap
new = lambda n, x: torch.full((n,), x, dtype=torch.int32, device="cuda")
for batch in {batches}:
    pool, tables = ap.BlockPool.full(2 * batch, 16), new(2 * batch, -1).view(batch, 2)
    lens = new(batch, 0)
    if {trim}:
        lens.fill_(32)
        tables.copy_(torch.arange(2 * batch, device="cuda").view(batch, 2))
        pool.free_count.fill_(0)
        status = ap.block_trim(pool, lens, new(batch, 16), tables)
        ok = bool((lens == 16).all()) and pool.free_count.item() == batch
        ok &= bool((pool.free[:batch] == tables[:, 1]).all())
    else:
        plan = ap.block_tables(pool, lens, new(batch, 1), tables, batch)
        status = plan.status
        ok = bool((plan.kv_lens == 1).all()) and pool.free_count.item() == batch
        ok &= bool((plan.slots == 16 * torch.arange(batch, device="cuda")).all())
    assert ok and status.item() == 0, batch
print("fine")
"""


@pytest.mark.parametrize("trim,batches", [
    (False, [4053, 4054]), (False, [4096]), (False, [4097, 4096, 16384, 4060]),
    (True, [6080, 6081]), (True, [6144]), (True, [6145, 6144, 16384, 6100]),
])
def test_tables_and_trim_of_batches_that_fill_48_kb(ap, trim, batches):
    """In a process of its own: no larger batch has been there before."""
    code = TABLES_OF.format(root=str(ROOT), batches=batches, trim=trim)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-800:]


# --------------------------------------------------------------------------- scales of V
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim,heads,kv_lens,new", [
    (64, 2, [700, 90], [1, 1]), (64, 2, [700, 90], [70, 1]), (128, 2, [300], [200]),
    (128, 1, [5000], [40]),
])
@pytest.mark.parametrize("factor", [2.0 ** -118, 0.37 * 2.0 ** -113, 2.0 ** -130])
def test_values_of_the_smallest_scales(ap, code, dim, heads, kv_lens, new, factor):
    """V scales down to the least numbers of 32 bits: results follow them as far
    as bf16 reaches.  Checked after both sides are multiplied by 2^118, so that
    the allowance keeps its meaning; it grows by half the least step of bf16
    (2^-134) and, for scales below 2^-126, by what a product of theirs may be
    rounded in 32 bits: n tokens' steps of 2^-150 and codes up to 448."""
    bs = 16
    tables, blocks = rows_of(kv_lens, bs)
    cache, host = make_cache(ap, blocks, 1, bs, dim, code, 3)
    host = list(host)
    host[3] = host[3] * factor
    cache.v_scale.copy_(host[3])
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn(starts[-1], heads, dim, generator=torch.Generator().manual_seed(5)).bfloat16()
    lift = 2.0 ** 118
    host[3] = host[3].double() * lift
    want, tol = ref.attend_ref(q, *host, tables, kv_lens, starts, True)
    out = ap.attn_cached(q.cuda(), cache, ints(tables), ints(kv_lens), ints(starts),
                         max_new=max(new))
    # A sum in 32 bits of p v, each term a multiple of 2^-149 at worst: half a
    # step for every partial sum of 16 keys and for each later factor.
    steps = (max(kv_lens) / 16 + 64) * 2.0 ** -150 * lift
    off = (out.double().cpu() * lift - want).abs() / (tol + 2.0 ** -134 * lift + steps)
    assert torch.all(off <= 1), f"off by {off.max():.3g} times"


# --------------------------------------------------------------------------- scales of V far apart
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("power", [20, 22, 24, 25, 27, 30, 33])
def test_values_far_below_the_largest_scale(ap, code, dim, new, power):
    """All weight lies on blocks whose V scale is 2^-power of the largest one's:
    values keep the stated absolute accuracy, 2^-32 of the largest scale."""
    bs, n_kv, r = 16, 64, 2.0 ** 6
    cache, host = make_cache(ap, 4, 1, bs, dim, code, power)
    k, v, ks, vs = host
    k.zero_()
    k[0, :, :, 0] = -100  # block 0: scores of -100 * 8 * D^-1/2, no weight is left
    ks.fill_(1.0)
    v.copy_(v.float().abs().clamp(min=64).to(v.dtype))
    vs.fill_(r * 2.0 ** -power)
    vs[0] = r
    for mine, x in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), host):
        mine.copy_(x)
    q = torch.zeros(new, 1, dim).bfloat16()
    q[:, 0, 0] = 8.0
    want, tol = ref.attend_ref(q, *host, [[0, 1, 2, 3]], [n_kv], [0, new], False)
    out = ap.attn_cached(q.cuda(), cache, ints([[0, 1, 2, 3]]), ints([n_kv]), ints([0, new]),
                         max_new=new, causal=False)
    # (the allowance of the reference has an absolute part of 2^-25, which values
    # of 2^-27 and more may not hide behind)
    tol = tol - 2.0 ** -25 + 2.0 ** -32 * r
    assert torch.all(want[:, 0] > 64 * r * 2.0 ** -power * 0.99)
    off = (out.double().cpu() - want).abs() / tol
    assert torch.all(off <= 1), f"off by {off.max():.3g} times"


# --------------------------------------------------------------------------- scale of the scores
@pytest.mark.parametrize("new", [1, 50])
def test_a_scale_of_the_scores_is_never_taken_for_none(ap, new):
    """A scale that is 0 in 32 bits would mean 1 / sqrt(D): it is refused; the
    least one that is not makes all weights alike."""
    cache, host = make_cache(ap, 3, 1, 16, 64, E4M3, 4)
    q = torch.randn(new, 1, 64, device="cuda").half()
    args = (q, cache, ints([[0, 1, 2]]), ints([48]), ints([0, new]))
    for scale in (1e-46, 2.0 ** -150, 0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="scale"):
            ap.attn_cached(*args, max_new=new, scale=scale)
    want, tol = ref.attend_ref(q.cpu(), *host, [[0, 1, 2]], [48], [0, new], False, 2.0 ** -149)
    out = ap.attn_cached(*args, max_new=new, causal=False, scale=2.0 ** -149)
    assert torch.all((out.double().cpu() - want).abs() <= tol)


# --------------------------------------------------------------------------- arrays that are replaced
def other_cache(ap, blocks, seed):
    return make_cache(ap, blocks, 2, 16, 64, E4M3, seed)[0]


@pytest.mark.parametrize("how", ["attribute", "set_"])
@pytest.mark.parametrize("new", [1, 40])
def test_a_cache_follows_tensors_that_are_replaced(ap, how, new):
    """Every call reads and writes the tensors that the cache has now."""
    cache, want_from = other_cache(ap, 6, 1), other_cache(ap, 20, 2)
    kept = [x.detach() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    before = [x.clone() for x in kept]
    for name in cache.__slots__:
        mine = getattr(want_from, name).clone()
        if how == "attribute":
            setattr(cache, name, mine)
        else:
            getattr(cache, name).set_(mine)
    assert cache.num_blocks == 20
    q = torch.randn(new, 4, 64, device="cuda").half()
    args = ints([list(range(19, 3, -1))]), ints([250]), ints([0, new])
    got = ap.attn_cached(q, cache, *args, max_new=new)
    assert torch.equal(got, ap.attn_cached(q, want_from, *args, max_new=new))
    k, v = (torch.randn(3, 2, 64, device="cuda").half() for _ in range(2))
    for c in (cache, want_from):
        ap.cache_append(c, k, v, ints([16 * 18, 16 * 18 + 1, 0]))
    for name in cache.__slots__:
        assert torch.equal(getattr(cache, name).float(), getattr(want_from, name).float())
    for x, y in zip(kept, before):
        assert torch.equal(x.float(), y.float())


def test_a_cache_of_tensors_that_do_not_belong_together_is_refused(ap):
    cache = other_cache(ap, 6, 1)
    q = torch.randn(1, 4, 64, device="cuda").half()
    args = ints([[0, 1]]), ints([20]), ints([0, 1])
    first = cache.k
    cache.k = other_cache(ap, 7, 2).k
    with pytest.raises(ValueError, match="share one"):
        ap.attn_cached(q, cache, *args, max_new=1)
    with pytest.raises(ValueError, match="share one"):
        ap.cache_append(cache, q[:, :2], q[:, :2], ints([0]))
    cache.k = first
    cache.v_scale = cache.v_scale[:5]
    with pytest.raises(ValueError, match="v_scale"):
        ap.attn_cached(q, cache, *args, max_new=1)
    cache.v_scale = torch.ones(6, 2, device="cuda", dtype=torch.float64)
    with pytest.raises(TypeError, match="v_scale"):
        ap.attn_cached(q, cache, *args, max_new=1)
    cache.v_scale = torch.ones(6, 2, device="cuda")
    ap.attn_cached(q, cache, *args, max_new=1)
    with pytest.raises(AttributeError):
        cache.num_blocks = 9


@pytest.mark.parametrize("how", ["attribute", "set_"])
def test_a_pool_follows_a_list_that_is_replaced(ap, how):
    """A shorter free list takes no more blocks than it has room for."""
    pool = ap.BlockPool.full(32, 16)
    kept = pool.free.detach()
    buffer = torch.full((32,), -5, dtype=torch.int32, device="cuda")
    if how == "attribute":
        pool.free = buffer[:4]
    else:
        pool.free.set_(buffer[:4])
    assert pool.num_blocks == 4
    pool.free_count = ints([0])
    lens, tables = ints([90]), ints([[9, 8, 7, 6, 5, 4]])
    assert ap.block_trim(pool, lens, ints([0]), tables).item() == 1
    assert (buffer == -5).all() and kept[0].item() == 31 and lens.item() == 90
    lens.fill_(60)
    assert ap.block_trim(pool, lens, ints([0]), tables).item() == 0
    assert buffer[:4].tolist() == [9, 8, 7, 6] and (buffer[4:] == -5).all()
    pool.block_size = 32
    pool.free, pool.free_count = ints([3, 2, 1, 0]), ints([4])
    plan = ap.block_tables(pool, ints([0]), ints([33]), ints([[-1, -1]]), 33)
    assert plan.slots[32].item() == 32 and pool.free_count.item() == 2
    pool.free = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="free"):
        ap.block_tables(pool, ints([0]), ints([0]), ints([[-1]]), 0)


def test_a_plan_follows_memory_that_is_replaced(ap):
    pool, lens, new = ap.BlockPool.full(8, 16), ints([0, 3]), ints([5, 1])
    tables, plan = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), ap.BlockPlan.empty(2, 6)
    ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    kept = plan.slots.detach()
    buffer = torch.full((12,), -5, dtype=torch.int32, device="cuda")
    plan.slots.set_(buffer[:4])
    with pytest.raises(ValueError, match="plan.slots"):
        ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    kept.fill_(-9)
    plan.slots.set_(buffer[4:10])
    ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    assert (kept == -9).all() and (buffer[4:10] >= 0).all()
    assert (buffer[:4] == -5).all() and (buffer[10:] == -5).all()


def test_a_tensor_that_was_replaced_is_not_held(ap):
    pool = ap.BlockPool.full(1 << 20, 16)
    cache = ap.PagedCache.empty(64, 8, 128, block_size=128)
    size = cache.k.numel()
    ap.cache_append(cache, *torch.zeros(2, 1, 8, 128, device="cuda").half(), ints([0]))
    before = torch.cuda.memory_allocated()
    cache.v = cache.k
    assert torch.cuda.memory_allocated() <= before - size
    ap.block_trim(pool, ints([0]), ints([0]), ints([[0]]))
    before = torch.cuda.memory_allocated()
    pool.free = pool.free[:4].clone()
    assert torch.cuda.memory_allocated() <= before - (4 << 20) + 512


@pytest.mark.parametrize("name", ["lens", "starts", "slots", "status"])
def test_a_batch_follows_arrays_that_are_replaced(ap, name):
    """The next step writes into the array that the batch has now."""
    batch = ap.CacheBatch(ap.BlockPool.full(20, 16), rows=2, max_len=64, max_tokens=8)
    cache = ap.PagedCache.empty(20, 1, 64, block_size=16)
    x = torch.randn(8, 1, 64, device="cuda").half()
    batch.advance(ints([5, 3]), 8)
    batch.attend(cache, x, x, x, max_new=5)
    old = getattr(batch, name)
    was = old.clone()
    setattr(batch, name, old.clone() if name == "lens" else torch.full_like(old, -5))
    with pytest.raises(RuntimeError, match="advance"):
        batch.attend(cache, x, x, x, max_new=5)
    batch.advance(ints([2, 6]), 8)
    assert batch.lens.tolist() == [7, 9] and batch.starts.tolist() == [0, 2, 8]
    assert batch.slots.tolist() == [5, 6] + [16 + i for i in range(3, 9)]
    assert batch.status.item() == 0 and torch.equal(old, was)


# --------------------------------------------------------------------------- the longest requests
def test_tables_and_trim_of_the_longest_requests(ap):
    """Lengths up to the last that 31 bits hold, in a table of 2^24 entries."""
    bs, width = 128, 2 ** 24
    tables = torch.full((1, width), 7, dtype=torch.int32, device="cuda")
    tables[0, -1] = 250
    pool = ap.BlockPool(torch.arange(300, dtype=torch.int32, device="cuda"), ints([5]), bs)
    lens, new = ints([2 ** 31 - 10]), ints([9])
    plan = ap.block_tables(pool, lens, new, tables, 10)  # all in the last block, which is held
    assert plan.status.item() == 0 and pool.free_count.item() == 5
    assert plan.kv_lens.item() == 2 ** 31 - 1
    assert plan.slots.tolist() == [250 * bs + 118 + i for i in range(9)] + [-1]
    new.fill_(10)
    plan = ap.block_tables(pool, lens, new, tables, 10)  # one token too many
    assert plan.status.item() == 2 and plan.slots.tolist() == [-1] * 10
    lens.fill_(2 ** 31 - 131)
    new.fill_(7)
    plan = ap.block_tables(pool, lens, new, tables, 7)  # over the border into a new block
    assert plan.status.item() == 0 and pool.free_count.item() == 4
    assert plan.slots.tolist() == [7 * bs + 125 + i for i in range(3)] + [4 * bs + i for i in range(4)]
    assert tables[0, -2:].tolist() == [7, 4]
    lens.fill_(2 ** 31 - 1)
    assert ap.block_trim(pool, lens, ints([2 ** 31 - 128]), tables).item() == 0
    assert pool.free[:5].tolist() == [0, 1, 2, 3, 4] and pool.free_count.item() == 5
    assert lens.item() == 2 ** 31 - 128
    lens.fill_(2 ** 31 - 1)
    assert ap.block_trim(pool, lens, ints([2 ** 31 - 2]), tables).item() == 0
    assert pool.free_count.item() == 5 and lens.item() == 2 ** 31 - 2
    assert ap.block_trim(pool, lens, ints([0]), tables).item() == 1  # more than the pool has


# --------------------------------------------------------------------------- pieces of a block
@pytest.mark.parametrize("code", CODES)
def test_pieces_of_a_block_in_calls_of_their_own(ap, code):
    """Slots with a gap, or with padding between them, are appended piece by
    piece; each piece finds the scale that the one before it left."""
    bs, dim = 16, 64
    cache, host = make_cache(ap, 3, 2, bs, dim, code, 5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i, slots in enumerate(([16, 17, -1, 32], [-1, 18, 35], [21, 22, -1], [23, 37, 38, 39])):
        k, v = ((torch.randn(len(slots), 2, dim, generator=gen, device="cuda") * 4 ** i).half()
                for _ in range(2))
        check_append(cache, host, k, v, slots, bs, code)
        host = tuple(x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale))


# --------------------------------------------------------------------------- streams given by name
def test_every_call_on_a_stream_given_by_name(ap):
    """A step of single calls, and of CacheBatch, on a stream that waits behind
    a long kernel of its own while the current stream is idle: the results are
    those of the current stream, and are there once the named one has ended."""
    bs, heads, kv_heads, dim, rows = 16, 4, 2, 64, 3
    gen = torch.Generator(device="cuda").manual_seed(9)
    new = [70, 1, 40]
    tokens = sum(new) + 2
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=gen, device="cuda").half()
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    new_t, keep = ints(new), ints([66, 0, 40])
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")

    def single(stream):
        pool, lens = ap.BlockPool.full(30, bs), ints([0] * rows)
        tables = torch.full((rows, 9), -1, dtype=torch.int32, device="cuda")
        cache = ap.PagedCache.empty(30, kv_heads, dim, block_size=bs)
        out = torch.zeros(tokens, heads, dim, device="cuda").half()
        torch.cuda.synchronize()
        if stream is not None:
            with torch.cuda.stream(stream):
                for _ in range(8):
                    torch.mm(busy, busy)
        plan = ap.block_tables(pool, lens, new_t, tables, tokens, stream=stream)
        ap.cache_append(cache, k, v, plan.slots, stream=stream)
        ap.attn_cached(q, cache, tables, plan.kv_lens, plan.starts, max_new=70, out=out,
                       stream=stream)
        status = ap.block_trim(pool, plan.kv_lens, keep, tables, stream=stream)
        (stream or torch.cuda.current_stream()).synchronize()
        n = int(pool.free_count)
        return [plan.kv_lens, plan.starts, plan.slots, plan.status, status, tables, pool.free[:n],
                cache.k_scale[tables[2, :3].long()], cache.v_scale[tables[2, :3].long()], out]

    def batch(stream):
        b = ap.CacheBatch(ap.BlockPool.full(30, bs), rows, 9 * bs, tokens)
        cache = ap.PagedCache.empty(30, kv_heads, dim, block_size=bs)
        out = torch.zeros(tokens, heads, dim, device="cuda").half()
        torch.cuda.synchronize()
        if stream is not None:
            with torch.cuda.stream(stream):
                for _ in range(8):
                    torch.mm(busy, busy)
        b.advance(new_t, tokens, stream=stream)
        b.attend(cache, q, k, v, max_new=70, out=out, stream=stream)
        got = b.attend(cache, q, k, v, max_new=70, stream=stream)  # (a second layer, with a new output)
        status = b.trim(keep, stream=stream)
        (stream or torch.cuda.current_stream()).synchronize()
        return [b.lens, b.starts, b.slots, b.status, status, b.tables,
                b.pool.free[:int(b.pool.free_count)], out, got[:sum(new)]]

    for step in (single, batch):
        want = step(None)
        for a, b in zip(step(side), want):
            assert torch.equal(a, b)
        assert want[4].item() == 0 and want[3].item() == 0
        assert want[-1][:sum(new)].abs().sum() > 0


def test_a_stream_of_the_tensors_device_is_asked_for(ap):
    """(with one device: a stream that says it is another's)"""
    class Other:
        device = torch.device("cuda", 7)
        cuda_stream = 0
    batch = ap.CacheBatch(ap.BlockPool.full(4, 16), 1, 64, 4)
    cache = ap.PagedCache.empty(4, 1, 64, block_size=16)
    x = torch.zeros(4, 1, 64, device="cuda").half()
    batch.advance(ints([4]), 4)
    for call in (lambda: batch.advance(ints([0]), 4, stream=Other),
                 lambda: batch.trim(ints([0]), stream=Other),
                 lambda: ap.cache_append(cache, x, x, batch.slots, stream=Other),
                 lambda: ap.attn_cached(x, cache, batch.tables, batch.lens, batch.starts, max_new=4,
                                        stream=Other)):
        with pytest.raises(ValueError, match="stream"):
            call()
    assert batch.lens.tolist() == [4]


# --------------------------------------------------------------------------- weights far below the largest
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 70])
def test_weights_far_below_the_largest(ap, code, dim, new):
    """The largest weight lies on values of 2^-20 of the others': what the small
    weights add keeps the stated accuracy, 2^-32 of the largest weight each."""
    bs, n_kv = 16, 160
    cache, host = make_cache(ap, 10, 1, bs, dim, code, dim)
    k, v, ks, vs = host
    k.zero_()
    k[:, 0, :, 0] = (-torch.arange(1.0, n_kv + 1).view(10, bs)).clamp(min=-120).to(k.dtype)
    k[0, 0, 0, 0] = 0
    ks.fill_(2.0 ** -2)   # scores of 0 and about -0.25, -0.5, ... -30 (weights down to 2^-43)
    vs.fill_(1.0)
    vs[0] = 2.0 ** -20
    for mine, x in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), host):
        mine.copy_(x)
    q = torch.zeros(new, 1, dim).bfloat16()
    q[:, 0, 0] = 1.0
    table = [list(range(10))]
    want, tol = ref.attend_ref(q, *host, table, [n_kv], [0, new], False, 1.0)
    tol = tol - 2.0 ** -25 + 2.0 ** -32 * (v.double() * vs.double()[:, :, None, None]).abs().sum((0, 2))
    out = ap.attn_cached(q.cuda(), cache, ints(table), ints([n_kv]), ints([0, new]), max_new=new,
                         causal=False, scale=1.0)
    off = (out.double().cpu() - want).abs() / tol
    assert torch.all(off <= 1), f"off by {off.max():.3g} times"
