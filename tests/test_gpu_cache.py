"""The paged 8-bit cache on a GPU: block tables, trim, append and attention
against plain implementations in 64 bits (tests/cache_ref.py)."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from tests import cache_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
CODES = [E4M3, INT8]
TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ap(engine):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return engine


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------- tables and trim
def batch_state(rng, batch, longest, most_new, bs, spare=5):
    """Lengths, new lengths, table rows with the blocks held, the free list."""
    lens = [rng.choice([0, rng.randint(0, longest)]) for _ in range(batch)]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(batch)]
    held = [ref.blocks_of(a, bs) for a in lens]
    width = max([ref.blocks_of(a + b, bs) for a, b in zip(lens, new)] + [1]) + rng.randint(0, 2)
    need = sum(ref.blocks_of(a + b, bs) for a, b in zip(lens, new)) - sum(held)
    blocks = sum(held) + need + spare
    ids = list(range(blocks))
    rng.shuffle(ids)
    tables, at = [], 0
    for n in held:
        tables.append(ids[at:at + n] + [-7] * (width - n))
        at += n
    free = ids[at:]
    return lens, new, tables, free + [-3] * (blocks - len(free)), len(free)


def run_tables(ap, lens, new, tables, free, count, bs, tokens, in_place):
    pool = ap.BlockPool(ints(free), ints([count]), bs)
    t = ints(tables) if tables else torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    lens_t = ints(lens)
    plan = ap.BlockPlan.empty(len(lens), tokens)
    left = None
    if in_place:
        plan.kv_lens = lens_t
    else:
        left = torch.empty(1, dtype=torch.int32, device="cuda")
    ap.block_tables(pool, lens_t, ints(new), t, tokens, plan=plan, free_left=left)
    left = pool.free_count if in_place else left
    if not in_place:
        assert lens_t.tolist() == lens and pool.free_count.item() == count
    assert pool.free.tolist() == free
    return (t.tolist(), plan.kv_lens.tolist(), plan.starts.tolist(), plan.slots.tolist(),
            left.item(), plan.status.item())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,longest,most_new,bs,pad", [
    (1, 0, 1, 16, 0), (1, 100, 300, 64, 3), (3, 40, 17, 16, 0), (64, 500, 1, 32, 5),
    (37, 90, 700, 128, 11), (1024, 70, 2, 16, 0), (1025, 70, 9, 32, 1), (3001, 40, 3, 16, 4),
])
def test_block_tables(ap, batch, longest, most_new, bs, pad, in_place):
    rng = random.Random(batch * 7 + bs)
    state = batch_state(rng, batch, longest, most_new, bs)
    tokens = sum(state[1]) + pad
    assert run_tables(ap, *state, bs, tokens, in_place) == ref.tables_ref(*state, bs, tokens)


def test_block_tables_and_trim_of_the_largest_batch(ap):
    rng = random.Random(2)
    state = batch_state(rng, 16384, 30, 3, 16)
    tokens = sum(state[1])
    got = run_tables(ap, *state, 16, tokens, True)
    assert got == ref.tables_ref(*state, 16, tokens)
    lens, tables, free, count = got[1], got[0], state[3], got[4]
    keep = [rng.choice([0, n, n - 1 if n else 0]) for n in lens]
    pool = ap.BlockPool(ints(free), ints([count]), 16)
    lens_t = ints(lens)
    status = ap.block_trim(pool, lens_t, ints(keep), ints(tables))
    assert (pool.free.tolist(), lens_t.tolist(), pool.free_count.item(), status.item()) \
        == ref.trim_ref(lens, keep, tables, free, count, 16)
    with pytest.raises(ap.AttnError):
        ap.block_tables(pool, torch.zeros(16385, dtype=torch.int32, device="cuda"),
                        torch.zeros(16385, dtype=torch.int32, device="cuda"),
                        torch.zeros(16385, 1, dtype=torch.int32, device="cuda"), 4)


def test_block_tables_of_no_requests_and_of_no_tokens(ap):
    for batch in (0, 4):
        lens, new = [16 * i for i in range(batch)], [0] * batch
        tables = [[9, 8, 7] for _ in range(batch)]
        state = (lens, new, tables, [0, 1, 2, 3], 2)
        assert run_tables(ap, *state, 16, 6, False) == ref.tables_ref(*state, 16, 6)
        assert run_tables(ap, *state, 16, 0, False) == ref.tables_ref(*state, 16, 0)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case,status", [("pool", 1), ("row", 2), ("slots", 3), ("negative", 4),
                                         ("count", 1), ("huge", 3)])
def test_block_tables_refuses_as_a_whole(ap, case, status, in_place):
    rng = random.Random(5)
    lens, new, tables, free, count = batch_state(rng, 40, 200, 50, 16, spare=0)
    tokens = sum(new)
    if case == "pool":
        new[3] += 16
        tokens += 16
        tables = [t + [-7, -7] for t in tables]
    elif case == "row":
        new[lens.index(max(lens))] += 16 * len(tables[0])
        tokens = sum(new)
    elif case == "slots":
        tokens -= 1
    elif case == "negative":
        new[7] = -1
    elif case == "count":
        count = len(free) + 1
    elif case == "huge":
        new[3] = new[9] = 2 ** 31 - 1
    got = run_tables(ap, lens, new, tables, free, count, 16, tokens, in_place)
    if case == "count":  # the reference takes the count as it is
        assert got == (tables, lens, [0] * 41, [-1] * tokens, count, 1)
        return
    want = ref.tables_ref(lens, new, tables, free, count, 16, tokens)
    assert got == want and want[-1] == status


def test_block_tables_gives_no_slot_for_a_bad_id(ap):
    got = run_tables(ap, [16, 3], [2, 2], [[0, -7], [99, -7]], [5, -1, 7, 8], 2, 16, 4, False)
    assert got[3] == [-1, -1, -1, -1] and got[5] == 0  # free id -1, table id 99 of 4 blocks


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,longest,bs", [(1, 0, 16), (1, 90, 16), (5, 100, 32), (64, 700, 64),
                                              (1024, 40, 16), (2500, 300, 16)])
def test_block_trim(ap, batch, longest, bs, in_place):
    rng = random.Random(batch + bs)
    lens, _, tables, free, count = batch_state(rng, batch, longest, 0, bs)
    keep = [rng.choice([0, a, max(0, a - rng.randint(1, 9)), a + 3]) for a in lens]
    pool = ap.BlockPool(ints(free), ints([count]), bs)
    lens_t, table_t = ints(lens), ints(tables)
    out = {} if in_place else {"lens_left": ints([9] * batch), "free_left": ints([9])}
    status = ap.block_trim(pool, lens_t, ints(keep), table_t, **out)
    got = (pool.free.tolist(), out.get("lens_left", lens_t).tolist(),
           out.get("free_left", pool.free_count).item(), status.item())
    assert got == ref.trim_ref(lens, keep, tables, free, count, bs)
    assert table_t.tolist() == tables


@pytest.mark.parametrize("case,status", [("twice", 1), ("row", 2), ("negative", 4)])
def test_block_trim_refuses_as_a_whole(ap, case, status):
    lens, keep, tables = [40, 33, 5], [0, 20, 5], [[4, 5, 6], [7, 8, 9], [3, -7, -7]]
    free, count = [0, 1, 2] + [-3] * 7, 3
    if case == "twice":
        count = 8
    elif case == "row":
        lens[0] = 49
    else:
        keep[2] = -1
    pool = ap.BlockPool(ints(free), ints([count]), 16)
    lens_t = ints(lens)
    got = ap.block_trim(pool, lens_t, ints(keep), ints(tables))
    assert (pool.free.tolist(), lens_t.tolist(), pool.free_count.item(), got.item()) \
        == (free, lens, count, status)


# --------------------------------------------------------------------------- append
def make_cache(ap, blocks, heads, bs, dim, code, seed):
    """A cache of random codes and power-of-two scales, and its 64-bit copy."""
    gen = torch.Generator().manual_seed(seed)
    parts = []
    for _ in range(2):
        if code is INT8:
            c = torch.randint(-127, 128, (blocks, heads, bs, dim), generator=gen).to(INT8)
        else:
            c = (torch.randn(blocks, heads, bs, dim, generator=gen) * 60).clamp(-448, 448).to(E4M3)
        s = 2.0 ** torch.randint(-9, -4, (blocks, heads), generator=gen).float()
        parts.append((c, s))
    (k, ks), (v, vs) = parts
    return ap.PagedCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda()), (k, v, ks, vs)


def check_append(cache, host, k, v, slots, bs, code, **kw):
    import attnprofile_b200 as ap
    ap.cache_append(cache, k, v, ints(slots), **kw)
    torch.cuda.synchronize()
    kc, vc, ks, vs = host
    want = [c.double() for c in (kc, vc, ks, vs)]
    kd, vd = k.double().cpu(), v.double().cpu()
    ref.append_ref(want[0], want[2], kd, slots, bs, code, vd)
    ref.append_ref(want[1], want[3], vd, slots, bs, code, None)
    assert torch.equal(torch.nan_to_num(cache.k_scale.double().cpu(), -1.0),
                       torch.nan_to_num(want[2], -1.0))
    assert torch.equal(cache.v_scale.double().cpu(), want[3])
    dead = torch.isnan(want[2])[:, :, None, None]  # K codes under a NaN scale mean nothing
    assert torch.equal(torch.where(dead, 0.0, cache.k.double().cpu()),
                       torch.where(dead, 0.0, want[0]))
    assert torch.equal(cache.v.double().cpu(), want[1])


def slots_of(spec, bs):
    """[(block, first offset, tokens)] -> slots; (None, 0, n): n padding tokens."""
    return [s for b, off, n in spec
            for s in ([-1] * n if b is None else range(b * bs + off, b * bs + off + n))]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,bs,heads", [(128, 16, 3), (64, 32, 2), (128, 64, 1), (64, 128, 5),
                                          (128, 32, 8)])
def test_cache_append(ap, kind, code, dim, bs, heads):
    cache, host = make_cache(ap, 12, heads, bs, dim, code, dim + bs)
    spec = [(3, 0, bs), (7, 0, 1), (2, bs - 1, 1), (None, 0, 2), (5, 3, bs - 3), (9, 0, 5),
            (11, 1, 2), (0, 7, 1)]
    slots = slots_of(spec, bs)
    gen = torch.Generator(device="cuda").manual_seed(bs)
    qkv = torch.randn(len(slots), 3, heads, dim, generator=gen, device="cuda")
    qkv *= torch.exp(1.5 * torch.randn(len(slots), 3, heads, 1, generator=gen, device="cuda"))
    qkv = qkv.to(kind)
    check_append(cache, host, qkv[:, 1], qkv[:, 2], slots, bs, code)


@pytest.mark.parametrize("code", CODES)
def test_cache_append_many_tokens(ap, code):
    """Enough tokens that a warp looks at a block's worth of them."""
    bs, heads, dim = 16, 4, 64
    cache, host = make_cache(ap, 150, heads, bs, dim, code, 3)
    spec = [(i, 0, bs) for i in range(60)] + [(60, 5, 11), (61, 0, 16), (62, 0, 3), (None, 0, 40),
            (70, 2, 1), (71, 15, 1)] + [(80 + i, i % bs, 1) for i in range(50)] + [(140, 0, 16)]
    slots = slots_of(spec, bs)
    assert len(slots) * heads > 148 * 16
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(len(slots), heads, dim, generator=gen, device="cuda").half()
            for _ in range(2))
    check_append(cache, host, k, v, slots, bs, code)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
def test_cache_append_extremes(ap, kind, code):
    """Zeros, the largest and smallest numbers of the type, numbers at the
    border between two scales, rounding ties; slots outside the pool."""
    bs, dim = 16, 64
    cache, host = make_cache(ap, 9, 1, bs, dim, code, 1)
    top = torch.finfo(kind).max
    c = ref.LARGEST[code]
    rows = [0.0, top, 2.0 ** -24, c, c * (1 + 2.0 ** -7), c / 8, 1.0, torch.finfo(kind).tiny]
    k = torch.zeros(len(rows) + 3, 1, dim, device="cuda")
    for i, x in enumerate(rows):
        k[i] = torch.linspace(-1, 1, dim, device="cuda") * x
        k[i, 0, 5] = x
    k[-3:] = torch.arange(dim, device="cuda") + 0.5  # ties of int8, and of e4m3 above 16
    slots = [i * bs for i in range(len(rows))] + [-1, 9 * bs, 8 * bs + 4]
    check_append(cache, host, k.to(kind), (-k).to(kind), slots, bs, code)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
def test_cache_append_numbers_that_are_not_finite(ap, kind, code):
    bs, dim, heads = 16, 128, 2
    cache, host = make_cache(ap, 5, heads, bs, dim, code, 2)
    slots = slots_of([(0, 0, 4), (1, 3, 2), (2, 0, 1), (3, 5, 1), (4, 0, 16)], bs)
    k, v = (torch.randn(len(slots), heads, dim, device="cuda").to(kind) for _ in range(2))
    k[1, 0, 7], k[4, 1, 0], v[6, 0, 3], v[7, 1, 127] = math.nan, math.inf, -math.inf, math.nan
    check_append(cache, host, k, v, slots, bs, code)
    assert torch.isnan(cache.k_scale).sum() == 4
    # a NaN scale stays while the block goes on, and ends when it is begun anew
    host = tuple(x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale))
    slots = slots_of([(0, 4, 3), (1, 0, 2)], bs)
    k, v = (torch.randn(len(slots), heads, dim, device="cuda").to(kind) for _ in range(2))
    check_append(cache, host, k, v, slots, bs, code)
    assert torch.isnan(cache.k_scale[0, 0]) and not torch.isnan(cache.k_scale[1]).any()


@pytest.mark.parametrize("code", CODES)
def test_cache_append_token_by_token(ap, code):
    """One call a token: the scale grows as larger ones come."""
    bs, dim, heads = 32, 64, 2
    cache, host = make_cache(ap, 2, heads, bs, dim, code, 6)
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(bs, 2, heads, dim, generator=gen, device="cuda")
    x = (x * torch.logspace(-3, 2, bs, device="cuda")[:, None, None, None]).half()
    for t in range(bs):
        check_append(cache, host, x[t:t + 1, 0], x[t:t + 1, 1], [bs + t], bs, code)
        host = tuple(y.cpu() for y in (cache.k, cache.v, cache.k_scale, cache.v_scale))


def test_cache_append_keeps_a_scale_that_is_no_power_of_two(ap):
    bs, dim = 16, 64
    cache, host = make_cache(ap, 2, 1, bs, dim, INT8, 9)
    host[2].fill_(0.37)
    cache.k_scale.fill_(0.37)
    k, v = (torch.randn(3, 1, dim, device="cuda").half() for _ in range(2))
    import attnprofile_b200 as m
    m.cache_append(cache, k, v, ints([4, 5, 6]))
    assert cache.k_scale[0, 0].item() == pytest.approx(0.37, abs=1e-7)
    want = (k.cpu().float()[:, 0] / torch.tensor(0.37)).round()
    assert torch.equal(cache.k[0, 0, 4:7].float().cpu(), want)


# --------------------------------------------------------------------------- attention
def attend_case(ap, kind, code, dim, bs, heads, kv_heads, kv_lens, new, causal=True, seed=0,
                scale=None, pad=0, spread=1.0, prepare=None, **kw):
    """Runs attn_cached on random data and checks it; returns the output."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    counts = [ref.blocks_of(n, bs) for n in kv_lens]
    blocks = sum(counts) + 3
    cache, host = make_cache(ap, blocks, kv_heads, bs, dim, code, seed)
    ids = list(range(blocks))
    rng.shuffle(ids)
    width = max(counts + [1]) + rng.randint(0, 1)
    tables, at = [], 0
    for n in counts:
        tables.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1] + pad, heads, dim, generator=gen) * spread).to(kind)
    # codes of about one: as e4m3 60 * 2^-6, as int8 127 * 2^-6
    if prepare is not None:
        q = prepare(q, cache, host, tables) or q
    want, tol = ref.attend_ref(q, *host, tables, kv_lens, starts, causal, scale)
    out = torch.full(q.shape, 7.0, dtype=kind, device="cuda")
    got = ap.attn_cached(q.cuda(), cache, ints(tables), ints(kv_lens), ints(starts),
                         max_new=max(new + [0]), causal=causal, scale=scale, out=out, **kw)
    torch.cuda.synchronize()
    assert got is out
    got = got.double().cpu()
    assert torch.all(got[starts[-1]:] == 7.0)
    live, nan = slice(0, starts[-1]), torch.isnan(want[:starts[-1]])
    assert torch.equal(torch.isnan(got[live]), nan)
    off = (got[live] - want[live]).abs()[~nan]
    assert torch.all(off <= tol[live][~nan]), f"off by {(off / tol[live][~nan]).max():.3g} times"
    return out


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1), (15, 3)])
def test_attn_cached_single_tokens(ap, kind, code, dim, bs, heads, kv_heads):
    attend_case(ap, kind, code, dim, bs, heads, kv_heads, [1, 15, 16, 17, 333, 0, 1000, 257],
                [1] * 8, seed=bs + dim + heads)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,new", [
    (2, 2, 7), (6, 2, 5), (16, 1, 1), (16, 1, 2), (32, 1, 1), (10, 2, 6), (40, 1, 1), (71, 1, 1),
    (48, 1, 3),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_cached_some_tokens(ap, code, dim, heads, kv_heads, new, causal):
    kv = [new, 300, new + 1, 64, 513]
    attend_case(ap, torch.float16, code, dim, 32, heads, kv_heads, kv,
                [new, max(1, new - 1), new, 1, new], causal, seed=heads + new)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,bs,heads,kv_heads,kv_lens,new", [
    (128, 16, 4, 2, [130], [130]), (64, 32, 2, 2, [400], [257]), (128, 64, 3, 1, [700, 129], [64, 129]),
    (64, 128, 5, 5, [300, 1, 90], [200, 1, 33]), (128, 32, 8, 2, [1100, 40], [300, 1]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_cached_prompts(ap, kind, code, dim, bs, heads, kv_heads, kv_lens, new, causal):
    attend_case(ap, kind, code, dim, bs, heads, kv_heads, kv_lens, new, causal, seed=dim + bs)


def test_attn_cached_long_keys(ap):
    """One long request among short ones: cut into many parts."""
    attend_case(ap, torch.float16, E4M3, 128, 64, 4, 1, [20000, 3, 5000], [1, 1, 1], seed=3)
    attend_case(ap, torch.bfloat16, INT8, 64, 16, 8, 2, [9000], [2], seed=4)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,heads,kv_heads,kv_lens,new", [
    (128, 4, 2, [5000], [40]), (64, 4, 2, [5000, 700], [40, 33]), (128, 1, 1, [4100], [257]),
    (64, 3, 1, [3000, 2900], [170, 1]), (128, 8, 1, [2500], [16]), (64, 2, 2, [1030], [129]),
    (128, 32, 1, [3000, 20], [1, 1]), (64, 71, 1, [2100], [1]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_cached_few_rows_and_many_keys(ap, kind, code, dim, heads, kv_heads, kv_lens, new,
                                            causal):
    """More rows than the split kernel takes and fewer units than SMs: the
    keys of a unit are cut, and units of up to 128 rows use both tiles."""
    attend_case(ap, kind, code, dim, 16, heads, kv_heads, kv_lens, new, causal, seed=heads)


@pytest.mark.parametrize("batch,longest", [(33, 1500), (129, 900), (200, 1500), (700, 300)])
def test_attn_cached_many_requests(ap, batch, longest):
    """One token each: more requests than the lanes of a warp hold, than the
    threads of a CTA, units cut between ranges and short ones whole."""
    rng = random.Random(batch)
    kv = [rng.choice([1, rng.randint(1, longest)]) for _ in range(batch)]
    attend_case(ap, torch.float16, E4M3, 64, 32, 4, 2, kv, [1] * batch, seed=batch)


def test_attn_cached_more_prompts_than_threads(ap):
    rng = random.Random(3)
    new = [rng.choice([1, 33, 40]) for _ in range(600)]
    attend_case(ap, torch.bfloat16, INT8, 64, 16, 1, 1, [n + rng.randint(0, 60) for n in new], new,
                seed=4)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128])
def test_attn_cached_single_tokens_beside_prompts(ap, dim, code):
    """Both kernels in one call, each on its own requests."""
    attend_case(ap, torch.float16, code, dim, 32, 6, 2, [1500, 130, 1, 0, 600, 77, 300],
                [1, 130, 1, 2, 4, 40, 300], seed=12)


@pytest.mark.parametrize("new", [[3, 0, 0, 1], [40, 0, 90, 1]])
def test_attn_cached_rows_without_keys(ap, new):
    """No cache, fewer tokens than rows, requests without rows, padding."""
    for causal in (True, False):
        out = attend_case(ap, torch.float16, E4M3, 128, 16, 4, 2, [0, 50, 20, 0], new, causal,
                          pad=9, seed=1)
        assert torch.all(out[:new[0]] == 0) and torch.all(out[-10] == 0)
    # causal rows in front of the first token
    out = attend_case(ap, torch.float16, E4M3, 128, 16, 4, 2, [2, 50, 20, 0], new, True, seed=2)
    assert torch.all(out[0] == 0)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("new", [1, 70])
def test_attn_cached_never_uses_slots_without_tokens(ap, code, new):
    """Codes behind the last token, blocks of nobody and table entries behind
    the end hold NaN or the largest numbers; scales of free blocks are NaN."""
    def poison(q, cache, host, tables):
        kv = [333, 77]
        used = {tables[r][i // 16]: 0 for r in (0, 1) for i in range(kv[r])}
        for b in range(cache.num_blocks):
            if b not in used:
                cache.k_scale[b] = cache.v_scale[b] = math.nan
        for r in (0, 1):
            last, held = tables[r][(kv[r] - 1) // 16], (kv[r] - 1) % 16 + 1
            for c in (cache.k, cache.v):
                c.view(torch.uint8)[last, :, held:] = 0x7f  # NaN of e4m3, 127 of int8
            tables[r][len(tables[r]) - 1] = 2 ** 30 if len(tables[r]) * 16 > kv[r] + 16 \
                else tables[r][-1]
    attend_case(ap, torch.float16, code, 128, 16, 4, 2, [333, 77], [new, 1], seed=11,
                prepare=poison)


@pytest.mark.parametrize("new", [1, 70])
def test_attn_cached_leaves_out_blocks_that_are_none(ap, new):
    """A table entry outside the pool: its tokens are left out, the rest
    attended (checked on one request against a cache without those tokens)."""
    cache, host = make_cache(ap, 9, 1, 16, 64, E4M3, 4)
    q = torch.randn(new, 2, 64, device="cuda").half()
    lens, starts = ints([128]), ints([0, new])
    for bad in (-1, 9, 2 ** 31 - 1, -2 ** 31):
        a = ap.attn_cached(q, cache, ints([[0, 1, bad, 3, bad, 5, 6, 7]]), lens, starts,
                           max_new=new, causal=False)
        b = ap.attn_cached(q, cache, ints([[0, 1, 3, 5, 6, 7]]), ints([96]), starts, max_new=new,
                           causal=False)
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -9, atol=2 ** -9)


@pytest.mark.parametrize("new", [1, 80])
def test_attn_cached_lengths_out_of_range(ap, new):
    """Lengths above the table's width, starts outside the rows: taken as the
    nearest that is there, never read or written outside."""
    cache, host = make_cache(ap, 6, 1, 16, 64, E4M3, 4)
    q = torch.randn(new, 2, 64, device="cuda").half()
    table = ints([[0, 1, 2, 3, 4, 5]])
    want = ap.attn_cached(q, cache, table, ints([96]), ints([0, new]), max_new=new, causal=False)
    for kv, starts in ((1000, [0, new]), (2 ** 31 - 1, [-5, new + 100]), (97, [0, 2 ** 31 - 1])):
        got = ap.attn_cached(q, cache, table, ints([kv]), ints(starts), max_new=new, causal=False)
        assert torch.equal(got, want)
    out = torch.full_like(q, 3.0)
    ap.attn_cached(q, cache, table, ints([-4]), ints([0, new]), max_new=new, out=out)
    assert torch.all(out == 0)
    out.fill_(3.0)
    ap.attn_cached(q, cache, table, ints([96]), ints([new, 0]), max_new=new, out=out)
    assert torch.all(out == 3)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new", [1, 70])
def test_attn_cached_scales_far_apart(ap, kind, new):
    """Block scales over 2^-20 .. 2^6 and one that is no power of two."""
    def spread(q, cache, host, tables):
        gen = torch.Generator().manual_seed(1)
        for i in (2, 3):
            s = 2.0 ** torch.randint(-20, -5, host[i].shape, generator=gen).float()
            if i == 2:
                s = s.clamp(max=2.0 ** -6)
            else:
                s[::5] = 2.0 ** 6
                s[1::5] = 0.37
            host[i].copy_(s)
            (cache.k_scale, cache.v_scale)[i - 2].copy_(s)
    attend_case(ap, kind, E4M3, 128, 16, 4, 2, [700, 90], [new, 1], seed=5, prepare=spread)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new", [2, 70])
def test_attn_cached_large_and_small_queries(ap, kind, new):
    """One-hot weights from large scores, rows of zeros, rows of tiny numbers."""
    def rows(q, cache, host, tables):
        q[0] *= 30
        q[1] = 0
        q[-1] *= 2.0 ** -12
        q[-2, 0, 1:] *= 2.0 ** -10
    attend_case(ap, kind, INT8, 64, 32, 4, 2, [400], [new], seed=6, prepare=rows)


@pytest.mark.parametrize("new", [1, 70])
def test_attn_cached_marks_only_rows_that_see_a_bad_block(ap, new):
    """A NaN K scale reaches the rows that see the block, and no others."""
    def bad(q, cache, host, tables):
        cache.k_scale[tables[0][(300 - 1) // 16], 0] = math.nan
        host[2][tables[0][(300 - 1) // 16], 0] = math.nan
    if new == 1:
        out = attend_case(ap, torch.float16, E4M3, 128, 16, 4, 2, [300, 40], [new, 1], seed=7,
                          prepare=bad)
        assert torch.isnan(out[0, :2]).all() and not torch.isnan(out[0, 2:]).any()
        return
    # a block that the first rows do not see
    cache, host = make_cache(ap, 20, 1, 16, 128, E4M3, 4)
    cache.k_scale[19] = math.nan  # tokens 288 .. 299
    table = ints([[(i + 1) % 20 for i in range(19)]])
    q = torch.randn(new, 2, 128, device="cuda").half()
    out = ap.attn_cached(q, cache, table, ints([300]), ints([0, new]), max_new=new)
    bad_rows = torch.isnan(out).all(-1).all(-1)
    assert bad_rows.tolist() == [300 - new + i >= 288 for i in range(new)]
    assert not torch.isnan(out[~bad_rows]).any()


@pytest.mark.parametrize("new", [3, 90])
def test_attn_cached_strides_and_scale(ap, new):
    """q inside a fused projection, out inside a wider buffer, another scale."""
    cache, host = make_cache(ap, 30, 2, 16, 64, E4M3, 4)
    qkv = torch.randn(new, 4 + 2 + 2, 64, device="cuda").half()
    wide = torch.full((4, new, 80), 5.0, device="cuda").half()  # heads first
    q, out = qkv[:, :4], wide[:, :, 8:72].transpose(0, 1)
    table, lens, starts = ints([list(range(29, -1, -1))]), ints([411]), ints([0, new])
    ap.attn_cached(q, cache, table, lens, starts, max_new=new, scale=0.3, out=out)
    want, tol = ref.attend_ref(q.cpu(), *host, table.tolist(), [411], [0, new], True, 0.3)
    assert torch.all((out.double().cpu() - want).abs() <= tol)
    assert torch.all(wide[:, :, :8] == 5) and torch.all(wide[:, :, 72:] == 5)
    # a table that is a slice of a wider one
    both = ints([list(range(29, -1, -1)) + [0] * 7] * 2)
    again = ap.attn_cached(q, cache, both[:1, :30], lens, starts, max_new=new, scale=0.3)
    assert torch.equal(again, out)


@pytest.mark.parametrize("new", [1, 70])
def test_attn_cached_one_token_or_head_of_any_stride(ap, new):
    """The stride of a dimension of size one means nothing."""
    cache, host = make_cache(ap, 6, 1, 16, 64, E4M3, 4)
    table, lens, starts = ints([[0, 1, 2, 3, 4, 5]]), ints([90]), ints([0, new])
    base = torch.randn(new * 64 + 70, device="cuda").half()
    q = base.as_strided((new, 1, 64), (64, 7, 1))
    out = torch.empty(new * 64, device="cuda").half().as_strided((new, 1, 64), (64, 13, 1))
    ap.attn_cached(q, cache, table, lens, starts, max_new=new, out=out)
    want = ap.attn_cached(q.contiguous(), cache, table, lens, starts, max_new=new)
    assert torch.equal(out, want)
    with pytest.raises(ap.AttnError):  # rows written over each other
        ap.attn_cached(q, cache, table, lens, starts, max_new=new, out=q)


@pytest.mark.parametrize("new", [3, 50])
def test_attn_cached_takes_no_more_rows_than_max_new(ap, new):
    cache, host = make_cache(ap, 40, 1, 16, 64, E4M3, 4)
    q = torch.randn(new + 200, 2, 64, device="cuda").half()
    out = torch.full_like(q, 3.0)
    ap.attn_cached(q, cache, ints([list(range(40))]), ints([640]), ints([0, new + 200]),
                   max_new=new, causal=False, out=out)
    want = ap.attn_cached(q[:new], cache, ints([list(range(40))]), ints([640]), ints([0, new]),
                          max_new=new, causal=False)
    assert torch.equal(out[:new], want) and torch.all(out[new:] == 3)


@pytest.mark.parametrize("new", [1, 4, 100])
def test_attn_cached_gives_the_same_bits_again(ap, new):
    outs = [attend_case(ap, torch.float16, E4M3, 128, 32, 8, 2, [3000, 100, 777], [new, 1, new],
                        seed=8) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_offsets_beyond_32_bits(ap):
    """A pool of more than 2^32 bytes of keys: its last blocks are used."""
    bs, heads, dim = 128, 8, 128
    blocks = (2 ** 32) // (bs * heads * dim) + 40
    cache = ap.PagedCache.empty(blocks, heads, dim, block_size=bs)
    slots = [(blocks - 2) * bs + i for i in range(bs)] + [(blocks - 1) * bs + i for i in range(9)]
    gen = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(len(slots), heads, dim, generator=gen, device="cuda").half()
            for _ in range(2))
    ap.cache_append(cache, k, v, ints(slots))
    for new in (1, 100):
        q = torch.randn(new, heads, dim, generator=gen, device="cuda").half()
        out = ap.attn_cached(q, cache, ints([[blocks - 2, blocks - 1]]), ints([len(slots)]),
                             ints([0, new]), max_new=new)
        host = [x[blocks - 2:].cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        want, tol = ref.attend_ref(q.cpu(), *host, [[0, 1]], [len(slots)], [0, new], True)
        assert torch.all((out.double().cpu() - want).abs() <= tol)


# --------------------------------------------------------------------------- streams, graphs, steps
def test_another_stream(ap):
    """Everything on a stream given by name, while the current one is busy."""
    cache, host = make_cache(ap, 30, 2, 16, 64, E4M3, 4)
    s = torch.cuda.Stream()
    table, lens = ints([list(range(30))]), ints([400])
    for new in (1, 90):
        q = torch.randn(new, 4, 64, device="cuda").half()
        starts = ints([0, new])
        want = ap.attn_cached(q, cache, table, lens, starts, max_new=new)
        torch.cuda.synchronize()
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(5):
            busy = busy @ busy
        got = ap.attn_cached(q, cache, table, lens, starts, max_new=new, stream=s)
        s.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 70])
def test_captured_and_replayed_with_other_lengths(ap, new):
    """A graph of a whole step follows the lengths that it finds."""
    bs, heads, dim = 16, 2, 64
    cache = ap.PagedCache.empty(80, heads, dim, block_size=bs)
    batch = ap.CacheBatch(ap.BlockPool.full(80, bs), rows=3, max_len=600,
                          max_tokens=2 * new + 1)
    new_lens = ints([new, 0, 1])
    tokens = 2 * new + 1
    qkv = torch.zeros(tokens, 8, dim, device="cuda").half()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    out = torch.zeros(tokens, 4, dim, device="cuda").half()

    def step():
        batch.advance(new_lens, tokens)
        batch.attend(cache, q, k, v, max_new=new, out=out)

    saved = [x.clone() for x in (batch.lens, batch.pool.free_count)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    batch.lens.copy_(saved[0])
    batch.pool.free_count.copy_(saved[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens = [0, 0, 0]
    kept = [[[], []] for _ in range(3)]
    rng = random.Random(1)
    for _ in range(4):
        add = [rng.randint(0, new), rng.randint(0, new), 1]
        new_lens.copy_(ints(add))
        qkv.copy_(torch.randn(qkv.shape, device="cuda"))
        graph.replay()
        lens = [a + b for a, b in zip(lens, add)]
        assert batch.status.item() == 0 and batch.lens.tolist() == lens
        starts = [0, add[0], add[0] + add[1], sum(add)]
        host = [x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        want, tol = ref.attend_ref(q.cpu(), *host, batch.tables.tolist(), lens, starts, True)
        n = sum(add)
        assert torch.all((out[:n].double().cpu() - want[:n]).abs() <= tol[:n])


def test_waits_that_run_out_are_reported(ap):
    """Nothing is fetched: the bounded waits expire, the status word says so,
    and the next call is right again."""
    cache, host = make_cache(ap, 30, 1, 16, 64, E4M3, 4)
    table, lens = ints([list(range(30))]), ints([470])
    assert ap.get_status(0)[0] == 0
    for new in (1, 40, 200):  # the split kernel; the tiled one with one and two tiles of rows
        q = torch.randn(new, 1, 64, device="cuda").half()
        want = ap.attn_cached(q, cache, table, lens, ints([0, new]), max_new=new)
        ap.set_timeout_ns(50_000_000)
        ap.debug_fault(1)
        try:
            ap.attn_cached(q, cache, table, lens, ints([0, new]), max_new=new)
            rc, site = ap.get_status(0, reset=True)
        finally:
            ap.debug_fault(0)
            ap.set_timeout_ns(2_000_000_000)
        assert rc == ap.ERR["DEVICE_TIMEOUT"] and site != 0
        got = ap.attn_cached(q, cache, table, lens, ints([0, new]), max_new=new)
        assert ap.get_status(0)[0] == 0
        assert torch.equal(got, want)


def test_a_workspace_given_and_one_too_small(ap):
    cache, _ = make_cache(ap, 100, 1, 16, 64, E4M3, 4)
    table, lens = ints([list(range(100))]), ints([1600])
    for new in (1, 40):
        q = torch.randn(new, 1, 64, device="cuda").half()
        starts = ints([0, new])
        want = ap.attn_cached(q, cache, table, lens, starts, max_new=new)
        need = ap.cached_workspace(cache, 1, new, 100)
        ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")  # any contents
        got = ap.attn_cached(q, cache, table, lens, starts, max_new=new, workspace=ws)
        assert torch.equal(got, want)
        with pytest.raises(ap.AttnError) as e:
            ap.attn_cached(q, cache, table, lens, starts, max_new=new, workspace=ws[:16])
        assert e.value.code == ap.ERR["WORKSPACE"]
    assert ap.cached_workspace(cache, 1, 1, 4) == 0


def test_two_graphs_at_once(ap):
    """Two captured calls replayed side by side do not share scratch memory."""
    cache, _ = make_cache(ap, 700, 1, 16, 128, E4M3, 4)
    jobs = []
    for i in range(2):
        q = torch.randn(1, 4, 128, device="cuda").half()
        table = ints([list(range(i, 700, 2))[:300]])
        lens, starts = ints([4700 - i]), ints([0, 1])
        want = ap.attn_cached(q, cache, table, lens, starts, max_new=1)
        torch.cuda.synchronize()
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
        with torch.cuda.graph(graph):
            for _ in range(20):
                ap.attn_cached(q, cache, table, lens, starts, max_new=1, out=out)
        jobs.append((graph, out, want, torch.cuda.Stream(), (q, table, lens, starts)))
    for _ in range(5):
        for graph, out, _, s, _ in jobs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, _, _, s, _ in jobs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _, _ in jobs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("code", CODES)
def test_steps_of_a_server(ap, code):
    """Prompts, single tokens, drafts refused, requests that end and begin
    again, a pool that runs dry: the cache's contents and every output against
    plain 64-bit ones."""
    bs, heads, kv_heads, dim, rows, blocks = 16, 4, 2, 64, 4, 30
    cache = ap.PagedCache.empty(blocks, kv_heads, dim, block_size=bs, dtype=code)
    batch = ap.CacheBatch(ap.BlockPool.full(blocks, bs), rows=rows, max_len=300,
                          max_tokens=400)
    state = [x.cpu() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    want_kv = [x.double() for x in state]
    lens, tables = [0] * rows, [[-1] * 19 for _ in range(rows)]
    free, count = list(range(blocks - 1, -1, -1)), blocks
    gen = torch.Generator(device="cuda").manual_seed(3)
    steps = [([70, 1, 0, 33], None), ([1, 1, 1, 1], [68, 2, 1, 0]), ([5, 4, 90, 40], [71, 3, 91, 40]),
             ([1, 0, 1, 1], None), ([300, 0, 0, 0], None), ([1, 16, 1, 1], [0, 19, 92, 42]),
             ([120, 1, 1, 1], None)]
    for new, keep in steps:
        tokens = sum(new) + 3
        qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=gen, device="cuda")
        qkv *= torch.exp(torch.randn(tokens, 1, 1, generator=gen, device="cuda"))
        qkv = qkv.half()
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        plan = batch.advance(ints(new), tokens)
        out = batch.attend(cache, q, k, v, max_new=max(new))
        tables, lens, starts, slots, count, status = ref.tables_ref(lens, new, tables, free, count,
                                                                    bs, tokens)
        assert (plan.status.item(), plan.slots.tolist(), batch.lens.tolist()) == (status, slots, lens)
        assert batch.tables.tolist() == tables and batch.pool.free_count.item() == count
        assert (status != 0) == (new[0] == 300)
        kd, vd = k.double().cpu(), v.double().cpu()
        ref.append_ref(want_kv[0], want_kv[2], kd, slots, bs, code, vd)
        ref.append_ref(want_kv[1], want_kv[3], vd, slots, bs, code, None)
        for r in range(rows):  # the tokens held
            for h in range(kv_heads):
                for i, (c, s) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
                    got = ref.gather_ref(c.cpu(), s.cpu(), tables[r], lens[r], bs, h)
                    assert torch.equal(got, ref.gather_ref(want_kv[i], want_kv[i + 2], tables[r],
                                                           lens[r], bs, h))
        want, tol = ref.attend_ref(q.cpu(), *want_kv, tables, lens, starts, True)
        n = starts[-1]
        assert torch.all((out[:n].double().cpu() - want[:n]).abs() <= tol[:n])
        if keep is not None:
            assert batch.trim(ints(keep)).item() == 0
            free, lens, count, _ = ref.trim_ref(lens, keep, tables, free, count, bs)
            assert batch.lens.tolist() == lens and batch.pool.free.tolist()[:count] == free[:count]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("max_len", [400, 4000])
def test_calls_that_follow_each_other_at_once(ap, dim, code, max_len):
    """Steps whose calls are issued without any wait, on one buffer that is
    overwritten between them, give the bits of steps that wait after every call
    (up to 512 tokens nothing is joined, beyond that parts are)."""
    bs, heads, kv_heads, rows = 32, 8, 2, 3
    most = max_len // 4
    gen = torch.Generator(device="cuda").manual_seed(max_len)
    prompts = [[most, most // 2, 1], [1, 1, 1], [2, 1, 3], [most, 7, most // 3]] + [[1, 1, 1]] * 6
    keeps = {3: [most + 2, 5, most], 7: [0, 9, most + 1]}
    inputs = [torch.randn(sum(n) + 2, heads + 2 * kv_heads, dim, generator=gen,
                          device="cuda").half() for n in prompts]
    new = [ints(n) for n in prompts]
    keeps = {i: ints(n) for i, n in keeps.items()}

    def run(wait):
        blocks = rows * (max_len // bs + 1)
        batch = ap.CacheBatch(ap.BlockPool.full(blocks, bs), rows, max_len, len(inputs[0]))
        cache = ap.PagedCache.empty(blocks, kv_heads, dim, block_size=bs, dtype=code)
        buffer, outs = torch.zeros_like(inputs[0]), []
        torch.cuda.synchronize()
        for i, x in enumerate(inputs):
            qkv = buffer[:len(x)]
            qkv.copy_(x)
            out = torch.zeros_like(x[:, :heads])
            wait()
            batch.advance(new[i], len(x))
            wait()
            batch.attend(cache, qkv[:, :heads], qkv[:, heads:heads + kv_heads],
                         qkv[:, heads + kv_heads:], max_new=max(prompts[i]), out=out)
            wait()
            if i in keeps:
                batch.trim(keeps[i])
                wait()
            buffer.fill_(float("nan"))
            outs.append(out)
        torch.cuda.synchronize()
        assert batch.status.item() == 0
        return outs + [batch.lens, batch.pool.free_count]

    want = run(torch.cuda.synchronize)
    assert all(torch.isfinite(x).all() for x in want) and any(x.any() for x in want)
    for _ in range(3):
        for a, b in zip(run(lambda: None), want):
            assert torch.equal(a, b)


def test_a_plan_is_checked_again_where_it_changed(ap):
    pool, lens, new = ap.BlockPool.full(8, 16), ints([0, 3]), ints([5, 1])
    tables, plan = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), ap.BlockPlan.empty(2, 6)
    for _ in range(2):
        ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    with pytest.raises(ValueError, match="plan.slots"):
        ap.block_tables(pool, lens, new, tables, 7, plan=plan)
    with pytest.raises(ValueError, match="plan.kv_lens"):
        ap.block_tables(pool, lens[:1], new[:1], tables[:1], 6, plan=plan)
    plan.slots = torch.empty(12, dtype=torch.int32, device="cuda")[::2]
    with pytest.raises(ValueError, match="plan.slots"):
        ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    plan.slots = torch.empty(6, dtype=torch.int32, device="cuda")
    plan.status = torch.empty(1, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="plan.status"):
        ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    plan.status = torch.full((1,), 9, dtype=torch.int32, device="cuda")
    plan.slots = slots = torch.full((6,), 77, dtype=torch.int32, device="cuda")
    ap.block_tables(pool, lens, new, tables, 6, plan=plan)
    assert plan.status.item() == 0 and (slots >= 0).all() and (slots < 128).all()


@pytest.mark.parametrize("max_len", [400, 4000])
def test_captured_behind_copies_and_another_stream(ap, max_len):
    """A graph in which copies, a cleared buffer and a kernel of another stream
    come right before the calls gives the bits of calls outside a graph."""
    bs, heads, kv_heads, dim, rows, most = 16, 4, 2, 64, 2, max_len // 8
    tokens = 2 * most
    gen = torch.Generator(device="cuda").manual_seed(2)
    staged = torch.zeros(tokens, heads + 2 * kv_heads, dim, device="cuda").half()
    staged_lens, factor = ints([0, 0]), torch.ones(1, device="cuda").half()

    def fresh():
        blocks = rows * (max_len // bs + 1)
        batch = ap.CacheBatch(ap.BlockPool.full(blocks, bs), rows, max_len, tokens)
        cache = ap.PagedCache.empty(blocks, kv_heads, dim, block_size=bs)
        return batch, cache, torch.zeros_like(staged), torch.zeros_like(staged[:, :heads]), ints([0, 0])

    side = torch.cuda.Stream()

    def step(batch, cache, qkv, out, new):
        here = torch.cuda.current_stream()
        qkv.copy_(staged)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            qkv.mul_(factor)
        new.copy_(staged_lens)
        out.zero_()
        batch.advance(new, tokens)
        here.wait_stream(side)
        batch.attend(cache, qkv[:, :heads], qkv[:, heads:heads + kv_heads],
                     qkv[:, heads + kv_heads:], max_new=most, out=out)

    plain, caught = fresh(), fresh()
    step(*caught)  # (no tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*caught)
    for new in ([most, 3], [1, most], [1, 1], [2, 1], [most, most], [1, 1]):
        staged.copy_(torch.randn(staged.shape, generator=gen, device="cuda"))
        factor.fill_(0.5 + new[0] % 3)
        staged_lens.copy_(ints(new))
        step(*plain)
        graph.replay()
        torch.cuda.synchronize()
        assert plain[0].status.item() == 0 and torch.equal(plain[0].lens, caught[0].lens)
        assert torch.equal(plain[3], caught[3]) and caught[3][:sum(new)].isfinite().all()
        assert caught[3][:sum(new)].abs().sum() > 0
