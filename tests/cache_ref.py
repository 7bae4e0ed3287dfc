"""Plain implementations of the cache operators, request by request: whole
numbers in Python, numbers in 64 bits.  Used by the tests only."""
import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def blocks_of(tokens, bs):
    return -(-tokens // bs)


def tables_ref(lens, new, tables, free, count, bs, tokens):
    """(tables, kv_lens, starts, slots, free_left, status) as lists."""
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    need = [blocks_of(a + b, bs) - blocks_of(a, bs) if a >= 0 and b >= 0 else 0
            for a, b in zip(lens, new)]
    good = [(a, b) for a, b in zip(lens, new) if a >= 0 and b >= 0]
    status = 0
    if sum(need) > count:
        status = 1
    if any(blocks_of(a + b, bs) > width for a, b in good):
        status = 2
    if sum(b for _, b in good) > tokens:
        status = 3
    if len(good) < len(lens):
        status = 4
    if status:
        return tables, list(lens), [0] * (len(lens) + 1), [-1] * tokens, count, status
    slots, starts = [], [0]
    for r, (a, b) in enumerate(zip(lens, new)):
        for column in range(blocks_of(a, bs), blocks_of(a + b, bs)):
            count -= 1
            tables[r][column] = free[count]
        slots += [tables[r][p // bs] * bs + p % bs for p in range(a, a + b)]
        starts.append(len(slots))
    return (tables, [a + b for a, b in zip(lens, new)], starts,
            slots + [-1] * (tokens - len(slots)), count, 0)


def trim_ref(lens, keep, tables, free, count, bs):
    """(free list, lens, free_left, status) as lists."""
    free, capacity = list(free), len(free)
    width = len(tables[0]) if tables else 0
    status = 0
    back = [c for r, (a, k) in enumerate(zip(lens, keep)) if a >= 0 and k >= 0
            and blocks_of(a, bs) <= width
            for c in tables[r][blocks_of(min(a, k), bs):blocks_of(a, bs)]]
    if count + len(back) > capacity:
        status = 1
    if any(blocks_of(a, bs) > width for a in lens if a >= 0):
        status = 2
    if any(a < 0 or k < 0 for a, k in zip(lens, keep)):
        status = 4
    if status:
        return free, list(lens), count, status
    free[count:count + len(back)] = back
    return free, [min(a, k) for a, k in zip(lens, keep)], count + len(back), 0


def scale_for(largest, code):
    """The least power of two >= 2^-100 with largest <= LARGEST * it."""
    if largest == 0:
        return 2.0 ** -100
    m, e = math.frexp(largest / LARGEST[code])  # in 64 bits: exact enough for 16-bit inputs
    return 2.0 ** max(-100, e - 1 if m == 0.5 else e)


def encode(x, code):
    """float64 -> code values (float64), to nearest even."""
    if code is torch.int8:
        return x.round().clamp(-127, 127)
    e = torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4
    step = torch.ldexp(torch.ones_like(x), e)
    return ((x / step).round() * step).clamp(-448, 448)


def append_ref(values, scales, x, slots, bs, code, other):
    """One of K and V, on the CPU in float64, in place: values [N, H, bs, D]
    code values, scales [N, H], x [T, H, D].  `other` (for K only) is V's x: a
    number that is not finite in either makes K's scale NaN."""
    runs = []
    for t, s in enumerate(slots):
        if not 0 <= s < values.shape[0] * bs:
            continue
        if t and runs and runs[-1][-1] == t - 1 and slots[t - 1] == s - 1 and s % bs:
            runs[-1].append(t)
        else:
            runs.append([t])
    for run in runs:
        b, off = slots[run[0]] // bs, slots[run[0]] % bs
        for h in range(x.shape[1]):
            y = x[run, h].clone()
            bad = not bool(torch.isfinite(y).all())
            if other is not None:
                bad |= not bool(torch.isfinite(other[run, h]).all())
            y[~torch.isfinite(y)] = 0
            old = float(scales[b, h]) if off else 0.0
            dead = off > 0 and math.isnan(old)
            want = scale_for(float(y.abs().max()), code)
            now = old if off and old > want else want
            if off and not dead and now > old:
                values[b, h, :off] = encode(values[b, h, :off] * (old / now), code)
            values[b, h, off:off + len(run)] = encode(y / now, code)
            scales[b, h] = math.nan if dead or (bad and other is not None) else now


def gather_ref(codes, scales, table, length, bs, head):
    """Tokens [length, D] of one request and head in float64."""
    ids = torch.tensor(table[:blocks_of(length, bs)], dtype=torch.int64)
    x = codes[ids, head].double() * scales[ids, head].double()[:, None, None]
    return x.reshape(-1, codes.shape[3])[:length]


def attend_ref(q, k_codes, v_codes, k_scale, v_scale, tables, kv_lens, starts, causal,
               scale=None):
    """(exact output, allowance per element) [T, H, D] in float64 on the CPU;
    rows behind the last request are NaN in both.

    The allowance counts, relative to A = sum_j p_j |v_j|: the rounding of each
    weight to f16 (eps / 2 = 2^-11); the same again for values that are scaled
    and rounded to f16 (a kernel may hold v * scale / power of two in f16, exact
    for power-of-two scales); errors of the scores, whose f32 sums of D products
    are off by at most 2 D 2^-24 of the sum of magnitudes, as an error of p, with
    the division by the sum of all p: twice; the f32 sums over n keys, n 2^-24
    where every addition is rounded one after the other, 32 keys at a time and a
    few joins: (n / 32 + 64) 2^-24, twice for sum and division; exp2 to 2^-20.
    The result's own rounding is eps / 2 of its type."""
    T, H, D = q.shape
    group = H // k_codes.shape[1]
    bs = k_codes.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, D), math.nan, dtype=torch.float64)
    tol = out.clone()
    half = torch.finfo(q.dtype).eps / 2
    for r, n_kv in enumerate(kv_lens):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        for h in range(H):
            k = gather_ref(k_codes, k_scale, tables[r], n_kv, bs, h // group)
            v = gather_ref(v_codes, v_scale, tables[r], n_kv, bs, h // group)
            y = q[a:b, h].double()
            s = (y @ k.T) * scale
            size = ((y.abs() @ k.abs().T) * scale).amax(1, keepdim=True) if n_kv else 0.0
            last = n_kv - (b - a) + 1 + torch.arange(b - a) if causal \
                else torch.full((b - a,), n_kv)
            seen = torch.arange(n_kv) < last[:, None]
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True) if n_kv else torch.zeros(b - a, 1, dtype=s.dtype)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            o, A = p @ v, p @ v.abs()
            delta = 2 * D * 2.0 ** -24 * size
            part = 2 * 2.0 ** -11 + 2 * delta + 2 * (n_kv / 32 + 64) * 2.0 ** -24 + 2.0 ** -20
            out[a:b, h], tol[a:b, h] = o, A * part * (1 + half) + half * o.abs() + 2.0 ** -25
    return out, tol
