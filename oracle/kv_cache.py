"""Plain restatement, in numpy, of the calls over an 8-bit paged key/value cache: one sequence, block, head and
page after the other, integers in Python, sums in 64 bits.  Codes travel as uint8 (f8e4m3fn) or int8 (s8)."""
import math

import numpy as np

from xla_amd import dtypes

QMAX = {"s8": np.float32(127.0), "f8": np.float32(448.0)}


def values(codes, kind):
    return codes.astype(np.float32) if kind == "s8" else dtypes.f8e4m3fn_to_f32(codes)


def to_codes(x, kind):
    """f32 -> codes: clamped, rounded to nearest even; a NaN gives code 0."""
    x = np.where(np.isnan(x), np.float32(0), x).astype(np.float32)
    x = np.clip(x, -QMAX[kind], QMAX[kind])
    return np.rint(x).astype(np.int8) if kind == "s8" else dtypes.f32_to_f8e4m3fn(x)


def sequences(rows, q_offsets, kv_lens, width, page):
    """(first row, rows, length) of each sequence, clamped as the kernels clamp them."""
    for b in range(len(kv_lens)):
        row0 = min(max(int(q_offsets[b]), 0), rows)
        n = min(max(int(q_offsets[b + 1]), row0), rows) - row0
        yield row0, n, min(max(int(kv_lens[b]), 0), width * page)


def write(x, codes, scales, kind, page_table, kv_lens, q_offsets):
    """x f32 [rows, heads, head] into copies of codes [pages, heads, page, head], scales; returns both."""
    codes, scales = codes.copy(), scales.copy()
    pages, heads, page, _ = codes.shape
    block = page // scales.shape[2]
    with np.errstate(all="ignore"):
        for b, (row0, n, length) in enumerate(sequences(x.shape[0], q_offsets, kv_lens, page_table.shape[1], page)):
            pos = max(length - n, 0)
            while pos < length and n > 0:
                first = pos // block * block
                end = min(length, first + block)
                pg, o = int(page_table[b, pos // page]), first % page
                if 0 <= pg < pages:
                    for h in range(heads):
                        new = x[row0 + n - (length - pos):row0 + n - (length - end), h]
                        s = np.float32(np.max(np.abs(new))) / QMAX[kind]
                        if pos > first:
                            old = scales[pg, h, o // block]
                            s = np.float32(np.nan) if np.isnan(s) or np.isnan(old) else max(s, old)
                            if not s == old:
                                held = values(codes[pg, h, o:o + pos - first], kind)
                                codes[pg, h, o:o + pos - first] = to_codes(held * np.float32(old / s), kind)
                        q = new / s if s > 0 else np.zeros_like(new)
                        codes[pg, h, o + pos - first:o + end - first] = to_codes(q, kind)
                        scales[pg, h, o // block] = s
                pos = end
    return codes, scales


def attention(q, k_codes, v_codes, k_scales, v_scales, kind, page_table, kv_lens, q_offsets, scale, causal=True, window=0,
              softcap=0.0):
    """(out, lse, spread, slack, largest) in 64 bits for q [rows, q_heads, head].  spread [rows, q_heads, head] is
    sum_j w_j |v_j|, the size that errors of the weights act on; slack [rows, q_heads] bounds how far f32 sums
    of head products, in any order, leave a score: (head + 8) 2^-24 max_j sum_d |q_d k_jd| scale, and three
    roundings of the score itself; largest [rows, q_heads] is max_j w_j |scale of v_j|."""
    rows, q_heads, head = q.shape
    pages, heads, page, _ = k_codes.shape
    block = page // k_scales.shape[2]
    group = q_heads // heads
    out = np.zeros((rows, q_heads, head))
    spread, slack = np.zeros_like(out), np.zeros((rows, q_heads))
    lse, largest = np.full((rows, q_heads), -np.inf), np.zeros((rows, q_heads))
    for b, (row0, n, length) in enumerate(sequences(rows, q_offsets, kv_lens, page_table.shape[1], page)):
        if n == 0 or length == 0:
            continue
        j = np.arange(length)
        pg = page_table[b, j // page].astype(np.int64)
        there = (pg >= 0) & (pg < pages)
        pg = np.where(there, pg, 0)
        p = length - n + np.arange(n)
        seen = np.broadcast_to(there[None, :], (n, length)).copy()
        if causal:
            seen &= j[None, :] <= p[:, None]
        if window > 0:
            seen &= j[None, :] > p[:, None] - window
        any_row = seen.any(0)  # what no row sees may hold anything
        for h in range(heads):
            def read(codes, scales):
                x = values(codes[pg, h, j % page], kind).astype(np.float64)
                x = x * scales[pg, h, j % page // block].astype(np.float64)[:, None]
                return np.where(any_row[:, None], x, 0.0)
            k, v = read(k_codes, k_scales), read(v_codes, v_scales)
            vs = np.where(any_row, np.abs(v_scales[pg, h, j % page // block].astype(np.float64)), 0.0)
            for g in range(group):
                qq = q[row0:row0 + n, h * group + g].astype(np.float64)
                x = qq @ k.T * scale
                size = (np.abs(qq) @ np.abs(k).T) * abs(scale)
                room = (head + 8) * 2.0 ** -24 * size + 3 * 2.0 ** -23 * np.abs(x)
                if softcap > 0:
                    x = softcap * np.tanh(x / softcap)
                    room = room + 2.0 ** -20 * softcap
                x = np.where(seen, x, -np.inf)
                some = seen.any(1)
                top = np.where(some, x.max(1, initial=-np.inf), 0.0)
                w = np.exp(x - top[:, None])
                total = w.sum(1)
                at = (slice(row0, row0 + n), h * group + g)
                safe = np.where(some, total, 1.0)[:, None]
                out[at] = np.where(some[:, None], w @ v / safe, 0.0)
                spread[at] = np.where(some[:, None], w @ np.abs(v) / safe, 0.0)
                lse[at] = np.where(some, top + np.log(np.where(some, total, 1.0)), -np.inf)
                slack[at] = np.where(seen, room, 0.0).max(1, initial=0.0)
                largest[at] = np.where(some, (w * vs[None, :]).max(1, initial=0.0) / safe[:, 0], 0.0)
    return out, lse, spread, slack, largest


def attention_tolerance(out, lse, spread, slack, largest, positions):
    """Bounds on |out - exact| and |lse - exact| for a bf16 result of f32 sums whose weights times scales are rounded to
    f16: half a bf16 step (2^-8) of the result, half an f16 step (2^-11) of every weight, or 2^-24 of the row's largest
    where that is more (f16's smallest step is 2^-24, the largest is kept at 1/2 or above), times a code (up to 448) for
    each of `positions`; a weight is off by its score's slack
    against the maximum's (2 slack) and by the exponential (2^-21); sums of `positions` weights by their
    number of 2^-24 roundings, in the numerator and in the denominator."""
    sums = (positions + 16) * 2.0 ** -24
    # above the formula's terms stands only their product, below 2^-8 of each: the factor 1.01
    tol = 1.01 * (2.0 ** -8 * np.abs(out) + (2.0 ** -11 + 2.0 ** -20 + 2 * sums) * spread
                  + 4 * slack[..., None] * spread + positions * 448 * 2.0 ** -24 * largest[..., None]) + 1e-37
    fine = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    return tol, 1.01 * (2 * slack + sums + 2.0 ** -20 + 2.0 ** -23 * fine)


def pages(op, page_table, kv_lens, ref_counts, request, page):
    """(page_table, kv_lens, ref_counts, moves, status), one request after the other."""
    batch, width = page_table.shape
    table, lens, refs = page_table.copy(), kv_lens.copy(), ref_counts.copy()
    count = refs.shape[0]
    held = [min(max(0, math.ceil(int(n) / page)), width) for n in kv_lens]
    for b in range(batch):
        table[b, held[b]:] = -1
    free = [p for p in range(count) if ref_counts[p] == 0]
    moves, status = [], []
    full = False  # a request that did not fit closes the pool for those behind it
    if op == "RESERVE":
        for b in range(batch):
            want = int(request[b])
            ok = int(kv_lens[b]) <= want <= width * page
            need = math.ceil(want / page) - held[b] if ok else 0
            if ok and need > 0:
                full = full or need > len(free)
                ok = not full
            if ok:
                for j in range(need):
                    table[b, held[b] + j] = free.pop(0)
                    refs[table[b, held[b] + j]] = 1
                lens[b] = want
            status.append(int(ok))
    elif op == "FORK":
        named = set()
        for src, dst in request.tolist():
            inside = 0 <= dst < batch
            ok = inside and 0 <= src < batch and src != dst and kv_lens[dst] <= 0 and dst not in named
            if inside:
                named.add(dst)
            n = held[src] if ok else 0
            own = ok and 0 < kv_lens[src] <= width * page and kv_lens[src] % page != 0
            if own:
                full = full or not free
                ok = not full
            if ok:
                row = page_table[src].copy()
                row[n:] = -1
                for j in range(n):
                    if own and j == n - 1:
                        new = free.pop(0)
                        moves.append((row[j], new))
                        row[j], refs[new] = new, 1
                    elif 0 <= row[j] < count:
                        refs[row[j]] += 1
                table[dst], lens[dst] = row, kv_lens[src]
            status.append(int(ok))
        moves += [(-1, -1)] * (len(request) - len(moves))
    elif op == "FREE":
        named = set()
        for b in request.tolist():
            ok = 0 <= b < batch and b not in named
            if ok:
                named.add(b)
                for j in range(held[b]):
                    if 0 <= page_table[b, j] < count:
                        refs[page_table[b, j]] -= 1
                table[b], lens[b] = -1, 0
            status.append(int(ok))
    else:
        used = int((ref_counts != 0).sum())
        to = {}
        for p in range(used, count):
            if ref_counts[p] != 0:
                to[p] = free.pop(0)
                moves.append((p, to[p]))
                refs[to[p]], refs[p] = refs[p], 0
        for b in range(batch):
            for j in range(held[b]):
                table[b, j] = to.get(int(page_table[b, j]), page_table[b, j])
        moves += [(-1, -1)] * (count // 2 - len(moves))
    return table, lens, refs, np.array(moves, np.int32).reshape(-1, 2), np.array(status, np.int32)
