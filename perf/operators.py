"""Workloads of the operators that serve requests from a paged cache held in 8 bits.

Four operators: `attend` (attention over the cache), `append` (new keys and
values quantised into it), `tables` (block tables and slot maps from request
lengths) and `trim` (blocks given back to the pool).  With `own` false, run()
computes them with elementary torch operations; with `own` true it calls
attnprofile_b200.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}  # largest finite value of a code
LEAST_EXPONENT = -100  # of a block's scale


def listed():
    return [
        # One user's chat, one token: the launch and the chain of one short read are all there is.
        {"name": "attend one request", "op": "attend", "batch": 1, "longest": 333, "shortest": 333, "new": 1,
         "heads": 16, "kv_heads": 4, "dim": 128, "block": 16, "type": "f16", "code": "e4m3", "causal": True},
        # A full decode batch of a server, lengths from a few tokens to eight thousand.
        {"name": "attend batch", "op": "attend", "batch": 64, "longest": 8191, "shortest": 5, "new": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "type": "bf16", "code": "e4m3", "causal": True},
        # Three long documents, one token each: few rows, so the keys have to be split.
        {"name": "attend long", "op": "attend", "batch": 3, "longest": 131072, "shortest": 40001, "new": 1,
         "heads": 32, "kv_heads": 4, "dim": 128, "block": 64, "type": "f16", "code": "int8", "causal": True},
        # Up to five drafted tokens a request are checked at once; ungrouped heads of 64.
        {"name": "attend drafts", "op": "attend", "batch": 24, "longest": 2047, "shortest": 64, "new": 5,
         "heads": 16, "kv_heads": 16, "dim": 64, "block": 16, "type": "bf16", "code": "int8", "causal": True},
        # A whole prompt of 4096 tokens on the engine's 16 heads of 64.
        {"name": "attend prompt", "op": "attend", "batch": 1, "longest": 4096, "shortest": 4096, "new": 4096,
         "heads": 16, "kv_heads": 16, "dim": 64, "block": 32, "type": "f16", "code": "e4m3", "causal": True},
        # Chunks of long prompts of several requests, grouped heads: the largest.
        {"name": "attend chunks", "op": "attend", "batch": 3, "longest": 16000, "shortest": 3000, "new": 2048,
         "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "type": "bf16", "code": "e4m3", "causal": True},
        # One decode step's keys and values, one token a request.
        {"name": "append tokens", "op": "append", "batch": 64, "longest": 1900, "shortest": 0, "new": 1,
         "kv_heads": 8, "dim": 128, "block": 32, "type": "bf16", "code": "e4m3"},
        # The keys and values of prompts, 16 thousand tokens in all.
        {"name": "append prompts", "op": "append", "batch": 5, "longest": 700, "shortest": 0, "new": 6000,
         "kv_heads": 8, "dim": 128, "block": 64, "type": "f16", "code": "int8"},
        # A decode step of 256 requests: one in sixteen needs a block.
        {"name": "tables for tokens", "op": "tables", "batch": 256, "longest": 8000, "shortest": 1, "new": 1,
         "block": 16},
        # Prompts come in: about 60 thousand slots.
        {"name": "tables for prompts", "op": "tables", "batch": 40, "longest": 500, "shortest": 0, "new": 3001,
         "block": 64},
        # After a step: some requests have ended, some drafts were refused.
        {"name": "trim batch", "op": "trim", "batch": 256, "longest": 4000, "shortest": 1, "block": 16},
        # A server is drained of two thousand requests.
        {"name": "trim many", "op": "trim", "batch": 2000, "longest": 900, "shortest": 1, "block": 32},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    op = rng.choice(["attend"] * 5 + ["append"] * 2 + ["tables", "trim"])
    block = rng.choice([16, 32, 64, 128])
    if op in ("tables", "trim"):
        case = {"op": op, "batch": _log(rng, 1, 2000), "longest": _log(rng, 1, 4000), "shortest": 0, "block": block}
        if op == "tables":
            case["new"] = rng.choice([1, _log(rng, 1, max(1, 60000 // case["batch"]))])
        return case
    case = {"op": op, "kv_heads": rng.choice([1, 2, 4, 5, 8, 16]), "dim": rng.choice([64, 128]), "block": block,
            "type": rng.choice(["f16", "bf16"]), "code": rng.choice(["e4m3", "int8"])}
    width = case["kv_heads"] * case["dim"]
    if op == "append":
        case["batch"] = _log(rng, 1, 128)
        case["new"] = rng.choice([1, 4, _log(rng, 1, max(1, 16000 * 1024 // width // case["batch"]))])
        case["longest"] = _log(rng, 1, 2000)
        case["shortest"] = 0
        return case
    kind = rng.choice(["token", "drafts", "prompt"])
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 7, 8, 16] if width < 1024 else [1, 2, 3, 4, 7])
    case["causal"] = rng.random() < 0.8
    if kind == "prompt":
        case["batch"] = rng.choice([1, 2, 3, 4])
        case["new"] = _log(rng, 33, 2048)
        case["longest"] = case["new"] + rng.choice([0, _log(rng, 1, 8000)])
    else:
        case["batch"] = _log(rng, 1, 96)
        case["new"] = 1 if kind == "token" else rng.randint(2, 8)
        case["longest"] = case["new"] + _log(rng, 1, min(100000, 250000 * 1024 // width // case["batch"]))
    # no more than the largest listed case, in the maps that a plain form holds too
    while case["batch"] * case["heads"] * case["new"] * case["longest"] > 3_000_000_000:
        case["new"] = max(1, case["new"] // 2 + 1)
        case["longest"] = max(case["new"], case["longest"] // 2 + 1)
    case["shortest"] = rng.choice([case["new"], max(case["new"], case["longest"] // 3)])
    return case


def _lengths(case):
    """(tokens of each request after the step, new ones among them): by the case alone, spread over its range."""
    n = case["batch"]
    part = [(i * 0.6180339887) % 1.0 for i in range(n)]
    after = [int(round(case["longest"] - (case["longest"] - case["shortest"]) * p)) for p in part]
    most = case.get("new", 0)
    new = [most if i == 0 else 1 + int((most - 1) * ((i * 0.7548776662) % 1.0)) for i in range(n)] if most else [0] * n
    if case["op"] != "attend":  # there the lengths are those before the step
        after = [a + b for a, b in zip(after, new)]
    return [max(a, b) for a, b in zip(after, new)], new


def _blocks(tokens, block):
    return -(-tokens // block)


def _ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _two_to(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale_of(largest, code):
    """The least power of two, no less than 2^LEAST_EXPONENT, that brings `largest` into the code's range."""
    mantissa, exponent = torch.frexp(largest / LARGEST[code])
    e = torch.where(mantissa > 0.5, exponent, exponent - 1)
    return _two_to(torch.where(largest > 0, e, LEAST_EXPONENT).clamp(min=LEAST_EXPONENT))


def _codes(x, code):
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _pool(case, blocks, gen):
    """Codes and scales of `blocks` blocks of keys or values: each block and head has its own level."""
    shape = (blocks, case["kv_heads"], case["block"], case["dim"])
    codes = torch.empty(shape, dtype=CODES[case["code"]], device="cuda")
    scales = torch.empty(shape[:2], dtype=torch.float32, device="cuda")
    some = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, blocks, some):
        part = scales[at:at + some]
        x = torch.randn((part.shape[0],) + shape[1:], generator=gen, device="cuda")
        x *= torch.exp(0.4 * torch.randn(x.shape[:2] + (1, 1), generator=gen, device="cuda"))
        s = _scale_of(x.abs().amax((2, 3)), case["code"])
        part.copy_(s)
        codes[at:at + some] = _codes(x / s[..., None, None], case["code"])
    return codes, scales


def _tables(case, counts, blocks, gen):
    """A table row of each request: its blocks lie anywhere in the pool."""
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    width = max(1, max(counts))
    index, at = torch.zeros(len(counts), width, dtype=torch.int64), 0
    for i, n in enumerate(counts):
        index[i, :n] = torch.arange(at, at + n)
        at += n
    return order[index.cuda()].contiguous(), order[at:].flip(0).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    after, new = _lengths(case)
    before = [a - b for a, b in zip(after, new)]
    bs = case["block"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["tokens"] = starts[-1]
    if case["op"] in ("tables", "trim"):
        held = [_blocks(n, bs) for n in before]
        want = sum(_blocks(n, bs) for n in after) - sum(held)
        s["blocks"] = sum(held) + want + 37
        tables, free = _tables(case, held, s["blocks"], gen)
        width = max(1, max(_blocks(n, bs) for n in after)) + 3
        s["tables"] = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
        s["tables"][:, :tables.shape[1]] = tables
        s["free"] = torch.zeros(s["blocks"], dtype=torch.int32, device="cuda")
        s["free"][:free.numel()] = free
        s["free_count"] = _ints([free.numel()])
        s["lens"], s["new_lens"] = _ints(before), _ints(new)
        if case["op"] == "trim":  # a quarter has ended, a quarter loses drafts
            kind = torch.randint(0, 4, (len(held),), generator=gen, device="cuda")
            back = torch.randint(1, 6, (len(held),), generator=gen, device="cuda")
            lens = s["lens"]
            s["keep"] = torch.where(kind == 0, 0, torch.where(kind == 1, (lens - back).clamp(min=0), lens)).to(torch.int32)
        if own:  # the pool that a server keeps, and the arrays that it hands over each step
            import attnprofile_b200 as ap
            s["pool"] = ap.BlockPool(s["free"], s["free_count"], bs)
            s["free_left"], s["lens_left"] = torch.empty_like(s["free_count"]), torch.empty_like(s["lens"])
            if case["op"] == "tables":
                s["plan"] = ap.BlockPlan.empty(len(held), s["tokens"], device="cuda")
            s["status"] = torch.empty(1, dtype=torch.int32, device="cuda")
        return s
    counts = [_blocks(n, bs) for n in after]
    s["blocks"] = sum(counts) + 3
    s["k_codes"], s["k_scale"] = _pool(case, s["blocks"], gen)
    s["v_codes"], s["v_scale"] = _pool(case, s["blocks"], gen)
    s["tables"], _ = _tables(case, counts, s["blocks"], gen)
    s["kv_lens"], s["starts"] = _ints(after), _ints(starts)
    kind = TYPES[case["type"]]
    if case["op"] == "attend":
        s["q"] = torch.randn(s["tokens"], case["heads"], case["dim"], generator=gen, device="cuda").to(kind)
        s["out"] = torch.zeros_like(s["q"])
    else:
        # k and v are slices of one projection's output, as a model has them
        both = torch.randn(s["tokens"], 2, case["kv_heads"], case["dim"], generator=gen, device="cuda")
        both *= torch.exp(0.7 * torch.randn(s["tokens"], 2, case["kv_heads"], 1, generator=gen, device="cuda"))
        both = both.to(kind)
        s["k"], s["v"] = both[:, 0], both[:, 1]
        rows = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], device="cuda")
        pos = torch.tensor([a + j for a, n in zip(before, new) for j in range(n)], device="cuda")
        s["slots"] = (s["tables"][rows, pos // bs] * bs + pos % bs).to(torch.int32)
    if own:  # the handle of the cache, kept from step to step
        import attnprofile_b200 as ap
        s["cache"] = ap.PagedCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    return s


def run(s):
    return {"attend": _attend, "append": _append, "tables": _block_tables, "trim": _block_trim}[s["op"]](s)


def _attend(s):
    if own:
        import attnprofile_b200 as ap
        return ap.attn_cached(s["q"], s["cache"], s["tables"], s["kv_lens"], s["starts"], max_new=s["new"],
                              causal=s["causal"], out=s["out"])
    heads, kv, dim, new = s["heads"], s["kv_heads"], s["dim"], s["new"]
    kv_lens, starts, tables = s["kv_lens"].long(), s["starts"].long(), s["tables"].long()
    batch, keys = tables.shape[0], tables.shape[1] * s["block"]
    place = torch.arange(keys, device="cuda")
    held = (place < kv_lens[:, None])[:, None, :, None]

    def read(codes, scale):  # [batch, kv, keys, dim], zeros where no token is held
        x = codes[tables].float() * scale[tables][..., None, None]
        return torch.where(held, x.transpose(1, 2).reshape(batch, kv, keys, dim), 0.0)

    count = starts[1:] - starts[:-1]
    row = torch.arange(new, device="cuda")
    at = (starts[:-1, None] + row).clamp(max=s["tokens"] - 1)
    q = s["q"][at].float().reshape(batch, new, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, kv, -1, dim)
    score = (q @ read(s["k_codes"], s["k_scale"]).transpose(-1, -2)) / math.sqrt(dim)
    score = score.view(batch, kv, heads // kv, new, keys)
    last = kv_lens[:, None] - 1
    if s["causal"]:
        last = last - count[:, None] + 1 + row
    seen = (place <= last[..., None])[:, None, None]
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = p.view(batch, kv, -1, keys) @ read(s["v_codes"], s["v_scale"])
    o = o.view(batch, kv, heads // kv, new, dim).permute(0, 3, 1, 2, 4).reshape(batch, new, heads, dim)
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(starts[1:], token, right=True)
    s["out"].copy_(o[request, token - starts[request]])
    return s["out"]


def _append(s):
    if own:
        import attnprofile_b200 as ap
        ap.cache_append(s["cache"], s["k"], s["v"], s["slots"])
    else:
        _append_plain(s, s["k"], s["k_codes"], s["k_scale"])
        _append_plain(s, s["v"], s["v_codes"], s["v_scale"])
    # Codes are returned as what they are (e4m3 numbers, whole numbers), each scale beside them.
    return {"k": s["k_codes"], "v": s["v_codes"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _append_plain(s, x, codes, scale):
    bs, blocks, heads, dim = s["block"], s["blocks"], s["kv_heads"], s["dim"]
    slots = s["slots"].long()
    block = slots // bs
    x = x.float()
    largest = torch.zeros(blocks, heads, device="cuda").index_reduce_(0, block, x.abs().amax(-1), "amax")
    first = torch.full((blocks,), bs, device="cuda").index_reduce_(0, block, slots % bs, "amin")
    wanted = _scale_of(largest, s["code"])
    grown = torch.where((first == 0)[:, None], wanted, torch.maximum(scale, wanted))
    grown = torch.where((first < bs)[:, None], grown, scale)
    kept = codes.float()
    before = torch.arange(bs, device="cuda") < first[:, None]
    moved = kept * (scale / grown)[..., None, None]
    kept = torch.where(before[:, None, :, None], moved, kept)
    source = torch.full((blocks * bs,), -1, dtype=torch.int64, device="cuda")
    source[slots] = torch.arange(slots.numel(), device="cuda")
    fresh = x[source.clamp(min=0)].view(blocks, bs, heads, dim).transpose(1, 2) / grown[..., None, None]
    fresh = torch.where((source >= 0).view(blocks, 1, bs, 1), fresh, kept)
    codes.copy_(_codes(fresh, s["code"]))
    scale.copy_(grown)


def _block_tables(s):
    if own:
        import attnprofile_b200 as ap
        plan = ap.block_tables(s["pool"], s["lens"], s["new_lens"], s["tables"], s["tokens"], plan=s["plan"],
                               free_left=s["free_left"])
        return {"tables": s["tables"], "kv_lens": plan.kv_lens, "starts": plan.starts, "slots": plan.slots,
                "free_left": s["free_left"], "status": plan.status}
    bs, tokens = s["block"], s["tokens"]
    lens, new, tables = s["lens"].long(), s["new_lens"].long(), s["tables"]
    held, after = (lens + bs - 1) // bs, (lens + new + bs - 1) // bs
    need = after - held
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    total = need.sum()
    status = torch.where(total > s["free_count"][0], 1, 0)
    status = torch.where((after > tables.shape[1]).any(), 2, status)
    status = torch.where(ends[-1] > tokens, 3, status)
    status = torch.where(((lens < 0) | (new < 0)).any(), 4, status)
    ok = status == 0
    first = torch.cumsum(need, 0) - need
    column = torch.arange(tables.shape[1], device="cuda") - held[:, None]
    taken = s["free_count"].long() - 1 - first[:, None] - column
    mine = (column >= 0) & (column < need[:, None]) & ok
    tables.copy_(torch.where(mine, s["free"][taken.clamp(0, s["blocks"] - 1)], tables))
    token = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(ends, token, right=True).clamp(max=lens.numel() - 1)
    pos = lens[row] + token - starts[row]
    slot = tables[row, (pos // bs).clamp(0, tables.shape[1] - 1)] * bs + pos % bs
    slots = torch.where((token < ends[-1]) & ok, slot, -1).int()
    return {"tables": tables, "kv_lens": torch.where(ok, lens + new, lens).int(),
            "starts": torch.where(ok, starts, 0).int(), "slots": slots,
            "free_left": (s["free_count"] - torch.where(ok, total, 0)).int(), "status": status.int().view(1)}


def _block_trim(s):
    if own:
        import attnprofile_b200 as ap
        ap.block_trim(s["pool"], s["lens"], s["keep"], s["tables"], lens_left=s["lens_left"],
                      free_left=s["free_left"], status=s["status"])
        return {"free": s["free"], "lens": s["lens_left"], "free_left": s["free_left"], "status": s["status"]}
    bs = s["block"]
    lens, keep, tables = s["lens"].long(), s["keep"].long(), s["tables"]
    left = torch.minimum(lens, keep)
    held, kept = (lens + bs - 1) // bs, (left + bs - 1) // bs
    ends = torch.cumsum(held - kept, 0)
    count = s["free_count"].long()
    status = torch.where(count[0] + ends[-1] > s["blocks"], 1, 0)
    status = torch.where((held > tables.shape[1]).any(), 2, status)
    status = torch.where(((lens < 0) | (keep < 0)).any(), 4, status)
    ok = status == 0
    rank = torch.arange(s["blocks"], device="cuda") - count
    row = torch.searchsorted(ends, rank, right=True).clamp(max=lens.numel() - 1)
    column = kept[row] + rank - (ends - (held - kept))[row]
    back = tables[row, column.clamp(0, tables.shape[1] - 1)]
    s["free"].copy_(torch.where((rank >= 0) & (rank < ends[-1]) & ok, back, s["free"]))
    return {"free": s["free"], "lens": torch.where(ok, left, lens).int(),
            "free_left": (s["free_count"] + torch.where(ok, ends[-1], 0)).int(), "status": status.int().view(1)}


def work(case):
    after, new = _lengths(case)
    bs = case["block"]
    tokens = sum(new)
    if case["op"] == "tables":
        taken = sum(_blocks(a, bs) for a in after) - sum(_blocks(a - n, bs) for a, n in zip(after, new))
        return {"bytes": 4 * (4 * case["batch"] + tokens + 2 * taken + 3), "flops": 0}
    if case["op"] == "trim":  # a quarter of the blocks go back: read in the table, written to the list
        return {"bytes": 4 * (3 * case["batch"] + 2 * sum(_blocks(a, bs) for a in after) // 4 + 3), "flops": 0}
    width = case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        touched = sum(_blocks(a, bs) - (a - n) // bs for a, n in zip(after, new))
        return {"bytes": 2 * (3 * tokens * width + 8 * touched * case["kv_heads"]) + 4 * tokens, "flops": 4 * tokens * width}
    pairs = sum(n * a - (n * (n - 1) // 2 if case["causal"] else 0) for a, n in zip(after, new))
    held = sum(2 * width * a + 8 * case["kv_heads"] * _blocks(a, bs) + 4 * _blocks(a, bs) for a in after)
    return {"bytes": held + 4 * tokens * case["heads"] * case["dim"], "flops": 4 * pairs * case["heads"] * case["dim"]}


def exact(case, seed):
    if case["op"] in ("tables", "trim"):
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_attend(s) if case["op"] == "attend" else _exact_append(s)


def _exact_attend(s):
    """Request by request and head by head, in 64 bits."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = s["heads"] // s["kv_heads"]
    for r, length in enumerate(s["kv_lens"].tolist()):
        a, b = s["starts"][r:r + 2].tolist()
        ids = s["tables"][r, :_blocks(length, s["block"])].long()
        limit = torch.full((b - a,), length, device="cuda")
        if s["causal"]:
            limit = length - (b - a) + 1 + torch.arange(b - a, device="cuda")
        hidden = (torch.arange(length, device="cuda") >= limit[:, None]).repeat_interleave(group, 0)
        for h in range(s["kv_heads"]):
            k, v = ((c[ids, h].double() * f[ids, h].double()[:, None, None]).flatten(0, 1)[:length]
                    for c, f in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])))
            q = s["q"][a:b, h * group:(h + 1) * group].double().flatten(0, 1)
            weight = torch.softmax(((q @ k.T) * s["dim"] ** -0.5).masked_fill_(hidden, -math.inf), -1)
            out[a:b, h * group:(h + 1) * group] = (weight @ v).view(b - a, group, -1)
    return out


def _exact_append(s):
    """Block by block: the tokens that fall into it are looked up, and the whole block is written anew."""
    done = {}
    bs, top = s["block"], LARGEST[s["code"]]
    slots = s["slots"].tolist()
    tokens_of = {}
    for t, slot in enumerate(slots):
        tokens_of.setdefault(slot // bs, []).append(t)
    for name in ("k", "v"):
        values, scales = s[name + "_codes"].double(), s[name + "_scale"].double()
        for block, tokens in tokens_of.items():
            x = s[name][tokens].double()  # [tokens, heads, dim]
            at = [slots[t] % bs for t in tokens]
            largest = x.abs().amax((0, 2))
            e = torch.round(torch.log2(largest.clamp(min=1e-300) / top))  # within one of the least exponent
            e = torch.where(largest > top * _power(e), e + 1, torch.where(largest <= top * _power(e - 1), e - 1, e))
            scale = _power(e.clamp(min=LEAST_EXPONENT))
            if min(at) > 0:
                scale = torch.maximum(scale, scales[block])
                values[block, :, :min(at)] = _rounded(values[block, :, :min(at)] * (scales[block] / scale)[:, None, None], s["code"])
            scales[block] = scale
            values[block][:, at] = _rounded(x.transpose(0, 1) / scale[:, None, None], s["code"])
        done[name], done[name + "_scale"] = (values if s["code"] == "e4m3" else values.to(torch.int8)), scales
    return done


def _power(e):
    """2^e in 64 bits, from the number's bits: exp2() and pow() of whole numbers may be a step off there."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rounded(x, code):
    if code == "int8":
        return x.round()
    step = _power(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)  # three bits behind the first
    return (x / step).round() * step
