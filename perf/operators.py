"""The 8-bit paged key/value cache of a decoder: what its four operators are measured on.

A cache layer is a pool of pages.  `k_cache` and `v_cache` hold 8-bit codes [pages, kv_heads, page, head],
`k_scales` and `v_scales` one f32 for each block of tokens and head [pages, kv_heads, page / block]; a value
is code * scale.  `page_table` [batch, table] lists each sequence's pages in order, `kv_lens` [batch] how many
tokens it holds, and the tokens of a call lie ragged behind each other, sequence b owning the rows
[q_offsets[b], q_offsets[b + 1]), which are its last ones.

write    quantises new keys and values into the pages; a block that already holds tokens keeps its scale
         unless the new ones are larger, and is then re-scaled
attend   softmax attention of query rows over the pages, grouped heads, causal, sliding window, soft cap
pages    the pool's book-keeping (RESERVE, FORK, FREE, COMPACT) with no step on the host
copy     moves whole pages inside every buffer of the pool, as FORK and COMPACT ask for
"""
import math

import torch

own = False

DEV = "cuda"
QMAX = {"s8": 127.0, "f8": 448.0}


# ---- cases -----------------------------------------------------------------------------------------

def listed():
    return [
        # a server's decode step: one new token for each of 128 sequences in mid-generation
        dict(name="write_decode", op="write", dtype="s8", batch=128, new_lo=1, new_hi=1, ctx_lo=40, ctx_hi=4000,
             kv_heads=8, head=128, page=64, block=64, pad=0),
        # prompts of very different lengths, written whole in one call
        dict(name="write_prompts", op="write", dtype="f8", batch=16, new_lo=33, new_hi=2011, ctx_lo=33, ctx_hi=2011,
             kv_heads=8, head=128, page=64, block=16, pad=7),
        # one user, a short conversation: latency is all that counts
        dict(name="attend_one", op="attend", dtype="f8", batch=1, new_lo=1, new_hi=1, ctx_lo=777, ctx_hi=777,
             q_heads=32, kv_heads=8, head=128, page=64, block=16, causal=True, window=0, softcap=0.0, lse=False, pad=0),
        # a server's decode step over contexts of mixed length
        dict(name="attend_decode", op="attend", dtype="s8", batch=64, new_lo=1, new_hi=1, ctx_lo=300, ctx_hi=8192,
             q_heads=32, kv_heads=8, head=128, page=64, block=64, causal=True, window=0, softcap=0.0, lse=False, pad=0),
        # few sequences with very long contexts: the work is split over the keys
        dict(name="attend_long", op="attend", dtype="f8", batch=4, new_lo=1, new_hi=1, ctx_lo=100001, ctx_hi=131072,
             q_heads=64, kv_heads=8, head=128, page=128, block=32, causal=True, window=0, softcap=0.0, lse=True, pad=0),
        # speculative decoding: a handful of drafted tokens each, a head size between the usual ones
        dict(name="attend_drafts", op="attend", dtype="s8", batch=24, new_lo=3, new_hi=5, ctx_lo=900, ctx_hi=6000,
             q_heads=40, kv_heads=8, head=96, page=16, block=8, causal=True, window=2048, softcap=50.0, lse=False, pad=5),
        # one long prompt
        dict(name="attend_prompt", op="attend", dtype="f8", batch=1, new_lo=8192, new_hi=8192, ctx_lo=8192, ctx_hi=8192,
             q_heads=32, kv_heads=8, head=128, page=64, block=16, causal=True, window=0, softcap=0.0, lse=False, pad=0),
        # chunks of prompts on top of earlier chunks, ragged
        dict(name="attend_chunks", op="attend", dtype="s8", batch=6, new_lo=100, new_hi=700, ctx_lo=1500, ctx_hi=5003,
             q_heads=16, kv_heads=4, head=64, page=32, block=32, causal=True, window=0, softcap=0.0, lse=True, pad=0),
        # a batch whose sequences each grow past a page's end now and then
        dict(name="pages_reserve", op="pages", kind="RESERVE", batch=256, pages=16384, page=64, table=128, share=0.0),
        # the pool of a long-running server: holes everywhere, pages shared between forks
        dict(name="pages_compact", op="pages", kind="COMPACT", batch=512, pages=131072, page=16, table=512, share=0.3),
        # best-of-n sampling: the last page of each forked sequence is copied
        dict(name="copy_forks", op="copy", dtype="f8", pages=512, moves=24, slots=32, kv_heads=8, head=128, page=64, block=16),
        # compaction of a half empty pool
        dict(name="copy_compact", op="copy", dtype="s8", pages=16384, moves=4096, slots=8192, kv_heads=8, head=128,
             page=64, block=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["write", "write", "attend", "attend", "attend", "attend", "pages", "copy"])
    page = rng.choice([16, 32, 64, 128])
    head = rng.choice([64, 80, 96, 112, 128, 128, 128, 192, 256])
    c = dict(op=op, dtype=rng.choice(["s8", "f8"]), page=page, block=rng.choice([b for b in (1, 4, 8, 16, 32, 64, 128) if b <= page]))
    if op == "pages":
        kind = rng.choice(["RESERVE", "FORK", "FREE", "COMPACT"])
        batch, table = _log(rng, 1, 512), _log(rng, 4, 512)
        pages = max(64, min(131072, int(batch * table * rng.uniform(0.4, 0.9))))
        return dict(op=op, kind=kind, batch=batch, pages=pages, page=page, table=table, share=round(rng.uniform(0, 0.5), 2))
    kv = rng.choice([1, 2, 4, 5, 8])
    c.update(kv_heads=kv, head=head)
    if op == "copy":
        moves = _log(rng, 1, 4096)
        room = max(1, (2 << 30) // (kv * page * head * 2))
        moves = min(moves, max(1, room // 4))
        c.update(moves=moves, slots=int(moves * rng.uniform(1, 2)), pages=2 * moves + rng.randrange(1, 64))
        return c
    if op == "write":
        new_hi = rng.choice([1, 1, _log(rng, 2, 4096)])
        batch = _log(rng, 1, 256 if new_hi == 1 else max(1, min(32, 16384 // new_hi)))
        ctx_hi = new_hi + _log(rng, 1, 4000)
        new_lo = max(1, int(new_hi * rng.uniform(0.2, 1)))
        c.update(batch=batch, new_lo=new_lo, new_hi=new_hi, ctx_lo=max(new_hi, int(ctx_hi * rng.uniform(0.1, 1))),
                 ctx_hi=ctx_hi, pad=rng.choice([0, 0, 3]))
        return c
    group = rng.choice([1, 2, 4, 5, 8, 16])
    c.update(q_heads=group * kv, causal=rng.random() < 0.85, window=0, softcap=rng.choice([0.0, 0.0, 30.0]),
             lse=rng.random() < 0.5, pad=rng.choice([0, 0, 4]))
    kind = rng.choice(["decode", "decode", "drafts", "prompt"])
    if kind == "prompt":
        new_hi = _log(rng, 33, 4096)
        batch = max(1, min(6, 4096 // new_hi))
        ctx_hi = new_hi + rng.choice([0, _log(rng, 1, 3000)])
    else:
        new_hi = 1 if kind == "decode" else rng.randrange(2, 9)
        batch = _log(rng, 1, 64)
        ctx_hi = max(new_hi, _log(rng, 20, max(256, min(65536, 320000 // batch))))
    new_lo = max(1, int(new_hi * rng.uniform(0.3, 1)))
    if c["causal"] and rng.random() < 0.3:
        c["window"] = _log(rng, 16, ctx_hi + 16)
    c.update(batch=batch, new_lo=new_lo, new_hi=new_hi, ctx_lo=max(new_hi, int(ctx_hi * rng.uniform(0.1, 1))), ctx_hi=ctx_hi)
    return c


def _spread(lo, hi, n, step):
    """n whole numbers from lo to hi, the last one hi, in an order that is not sorted; the same for every seed."""
    return [hi if i == n - 1 else lo + (i * step * 7919 + 13 * i) % (hi - lo + 1) for i in range(n)]


def _lens(c):
    return _spread(c["ctx_lo"], c["ctx_hi"], c["batch"], 31), _spread(c["new_lo"], c["new_hi"], c["batch"], 17)


# ---- inputs ----------------------------------------------------------------------------------------

def _codes(c, pages, g):
    """8-bit codes of normally distributed values, whose largest of a block is about 4 standard deviations."""
    x = torch.empty((pages, c["kv_heads"], c["page"], c["head"]), dtype=torch.float16, device=DEV)
    x.normal_(0.0, QMAX[c["dtype"]] / 4.0, generator=g).clamp_(-QMAX[c["dtype"]], QMAX[c["dtype"]])
    return x.round_().to(torch.int8) if c["dtype"] == "s8" else x.to(torch.float8_e4m3fn)


def _scales(c, pages, g):
    x = torch.rand((pages, c["kv_heads"], c["page"] // c["block"]), generator=g, device=DEV)
    return (x * 0.6 + 0.7) * (4.0 / QMAX[c["dtype"]])


def _pool(c, g):
    ctx, new = _lens(c)
    per = [-(-n // c["page"]) for n in ctx]
    table = max(per) + 1
    pages = sum(per) + max(2, sum(per) // 10)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    j = torch.arange(table, device=DEV)
    first = torch.tensor([sum(per[:b]) for b in range(len(per))], device=DEV)
    have = torch.tensor(per, device=DEV)
    at = (first[:, None] + j).clamp(max=pages - 1)
    page_table = torch.where(j < have[:, None], order[at], torch.full_like(order[at], -1))
    offsets = [sum(new[:b]) for b in range(len(new) + 1)]
    return dict(case=c, k_cache=_codes(c, pages, g), v_cache=_codes(c, pages, g), k_scales=_scales(c, pages, g),
                v_scales=_scales(c, pages, g), page_table=page_table.contiguous(), tokens=offsets[-1] + c["pad"],
                kv_lens=torch.tensor(ctx, dtype=torch.int32, device=DEV),
                q_offsets=torch.tensor(offsets, dtype=torch.int32, device=DEV), max_new=max(new), max_ctx=max(ctx))


def _book(c, g):
    """Tables, lengths and reference counts that fit together: shared full pages, holes, empty sequences."""
    batch, pages, page, table = c["batch"], c["pages"], c["page"], c["table"]
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    per = max(1, min(table - 1, int(pages * 0.55) // batch))
    full = torch.randint(0, per + 1, (batch,), generator=g, device=DEV)
    part = torch.randint(0, page, (batch,), generator=g, device=DEV)
    lens = full * page + part
    if c["kind"] == "FORK":
        lens[batch // 2:] = 0  # slots for the children
    have = (lens + page - 1) // page
    first = have.cumsum(0) - have
    j = torch.arange(table, device=DEV)
    tab = torch.where(j < have[:, None], order[(first[:, None] + j).clamp(max=pages - 1)], torch.full_like(order[:1], -1))
    # some sequences start with the full pages of their neighbour: a shared prompt
    share = torch.rand((batch,), generator=g, device=DEV) < c["share"]
    share[0] = False
    common = torch.minimum(lens // page, (lens // page).roll(1))
    take = share[:, None] & (j < common[:, None]) & ~share.roll(1)[:, None]
    tab = torch.where(take, tab.roll(1, 0), tab)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    used = tab[j < have[:, None]].long()
    refs.index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
    s = dict(case=c, page_table=tab.contiguous(), kv_lens=lens.to(torch.int32), ref_counts=refs, request=None)
    if c["kind"] == "RESERVE":
        s["request"] = (s["kv_lens"] + torch.randint(0, page + 1, (batch,), generator=g, device=DEV)).to(torch.int32)
    elif c["kind"] == "FORK":
        n = max(1, batch // 2)
        src = torch.randint(0, max(1, batch // 2), (n,), generator=g, device=DEV)
        dst = batch // 2 + torch.randperm(batch - batch // 2, generator=g, device=DEV)[:n]
        s["request"] = torch.stack([src, dst], 1).to(torch.int32).contiguous()
    elif c["kind"] == "FREE":
        s["request"] = torch.randperm(batch, generator=g, device=DEV)[:max(1, batch // 3)].to(torch.int32).contiguous()
    return s


def _inputs(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if c["op"] == "pages":
        return _book(c, g)
    if c["op"] == "copy":
        pages = c["pages"]
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        moves = torch.full((c["slots"], 2), -1, dtype=torch.int32, device=DEV)
        moves[:c["moves"]] = order[:2 * c["moves"]].reshape(-1, 2)
        return dict(case=c, moves=moves, buffers=[_codes(c, pages, g), _codes(c, pages, g), _scales(c, pages, g), _scales(c, pages, g)])
    s = _pool(c, g)
    rows = (s["tokens"], c["kv_heads"], c["head"])
    if c["op"] == "write":
        s["k"] = torch.randn(rows, generator=g, device=DEV).to(torch.bfloat16)
        s["v"] = torch.randn(rows, generator=g, device=DEV).to(torch.bfloat16)
    else:
        s["q"] = torch.randn((s["tokens"], c["q_heads"], c["head"]), generator=g, device=DEV).to(torch.bfloat16)
        s["scale"] = c["head"] ** -0.5
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        # the prepared custom call, which a program keeps like an executable: it names the buffers, and every
        # run() works on what they hold then
        from xla_amd import ops
        c = case
        cache = [s.get(k) for k in ("k_cache", "v_cache", "k_scales", "v_scales", "page_table", "kv_lens", "q_offsets")]
        if c["op"] == "write":
            s["call"] = ops.kv_cache_write(s["k"], s["v"], *cache, build_only=True)
        elif c["op"] == "attend":
            s["call"] = ops.kv_cache_attention(s["q"], *cache, scale=s["scale"], causal=c["causal"], window=c["window"],
                                               softcap=c["softcap"], lse=c["lse"], build_only=True)
        elif c["op"] == "pages":
            s["call"] = ops.kv_cache_pages(c["kind"], s["page_table"], s["kv_lens"], s["ref_counts"], s["request"],
                                           page_size=c["page"], build_only=True)
        else:
            s["call"] = ops.kv_cache_copy_pages(s["moves"], s["buffers"], build_only=True)
    return s


def run(state):
    if own:
        return state["call"].run()
    return {"write": _write, "attend": _attend, "pages": _pages, "copy": _copy}[state["case"]["op"]](state)


# ---- the plain forms -------------------------------------------------------------------------------

def _owner(s):
    """For every row of the call: its sequence, its place among that sequence's rows, and whether it has one."""
    t = torch.arange(s["tokens"], device=DEV)
    seq = (t[:, None] >= s["q_offsets"][None, 1:]).sum(1)
    valid = seq < s["case"]["batch"]
    seq = seq.clamp(max=s["case"]["batch"] - 1)
    return seq, t - s["q_offsets"].long()[seq], valid


def _quantise(x, scale, c):
    """Codes of x at `scale`: the f32 quotient, rounded to the nearest even code; zero where the scale is zero."""
    q = (x.double() / scale.double()).float()  # the f32 quotient, rounded once
    q = torch.where(scale > 0, q, torch.zeros_like(q)).clamp(-QMAX[c["dtype"]], QMAX[c["dtype"]])
    return q.round().to(torch.int8) if c["dtype"] == "s8" else q.to(torch.float8_e4m3fn).view(torch.int8)


def _write(s):
    c = s["case"]
    page, block = c["page"], c["block"]
    seq, i, valid = _owner(s)
    seq, i = seq[valid], i[valid]
    lens, off = s["kv_lens"].long(), s["q_offsets"].long()
    start = lens - (off[1:] - off[:-1])  # tokens that the sequence held before
    pos = start[seq] + i
    where = s["page_table"][seq, pos // page].long() * (page // block) + pos % page // block
    # a sequence's first block may hold tokens already
    b0 = start // block * block
    held = start - b0
    old_page = s["page_table"].gather(1, (b0 // page)[:, None])[:, 0].long().clamp(min=0)
    old_at = old_page * (page // block) + b0 % page // block
    at = (b0 % page)[:, None] + torch.arange(block, device=DEV)
    for x, codes, scales in ((s["k"], s["k_cache"], s["k_scales"]), (s["v"], s["v_cache"], s["v_scales"])):
        x = x[valid].float()
        flat = scales.permute(0, 2, 1).reshape(-1, c["kv_heads"])  # a copy: one row of heads for each block
        was = flat[old_at]
        new = torch.zeros_like(flat)
        amax = (x.abs().amax(-1).double() / QMAX[c["dtype"]]).float()
        new.scatter_reduce_(0, where[:, None].expand(-1, c["kv_heads"]), amax, "amax")
        grown = torch.where(held[:, None] > 0, torch.maximum(was, new[old_at]), new[old_at])
        new[old_at] = torch.where((start < lens)[:, None], grown, was)
        # what the first block holds, at its new scale
        ratio = torch.where(grown > 0, (was.double() / grown.double()).float(), torch.zeros_like(was))
        bytes_ = codes.view(torch.int8)
        old = codes.view(torch.int8)[old_page[:, None], :, at]  # [batch, block, heads, head]
        val = old.float() if c["dtype"] == "s8" else old.view(torch.float8_e4m3fn).float()
        val = (val * ratio[:, None, :, None]).clamp(-QMAX[c["dtype"]], QMAX[c["dtype"]])
        val = val.round().to(torch.int8) if c["dtype"] == "s8" else val.to(torch.float8_e4m3fn).view(torch.int8)
        keep = (torch.arange(block, device=DEV) < held[:, None])[:, :, None, None] & (start < lens)[:, None, None, None]
        bytes_[old_page[:, None], :, at] = torch.where(keep, val, old)
        bytes_[s["page_table"][seq, pos // page].long(), :, pos % page] = _quantise(x, new[where][:, :, None], c)
        touched = torch.zeros(flat.shape[0], dtype=torch.bool, device=DEV)
        touched[where] = True
        flat = torch.where(touched[:, None], new, flat)
        scales.copy_(flat.view(-1, page // block, c["kv_heads"]).permute(0, 2, 1))
    return s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]


def _gathered(s, codes, scales):
    """A cache's values in f32, [batch, kv_heads, positions, head]."""
    c = s["case"]
    tab = s["page_table"][:, :-(-s["max_ctx"] // c["page"])].long().clamp(min=0)
    x = codes.view(torch.int8)[tab]
    x = x.float() if c["dtype"] == "s8" else x.view(torch.float8_e4m3fn).float()
    x = x * scales[tab].repeat_interleave(c["block"], -1)[..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(c["batch"], c["kv_heads"], -1, c["head"])


def _attend(s):
    c = s["case"]
    batch, kv, group, head = c["batch"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["head"]
    seq, i, valid = _owner(s)
    off, lens = s["q_offsets"].long(), s["kv_lens"].long()
    n = off[1:] - off[:-1]
    rows = torch.arange(s["max_new"], device=DEV)
    q = s["q"][(off[:-1, None] + rows).clamp(max=s["tokens"] - 1)].float()  # [batch, new, q_heads, head]
    q = q.view(batch, -1, kv, group, head).permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, head)
    k = _gathered(s, s["k_cache"], s["k_scales"])
    j = torch.arange(k.shape[2], device=DEV)
    p = (lens - n)[:, None] + rows  # positions of the rows
    seen = (j < lens[:, None, None]).expand(-1, rows.numel(), -1)
    if c["causal"]:
        seen = seen & (j <= p[:, :, None])
    if c["window"]:
        seen = seen & (j > p[:, :, None] - c["window"])
    seen = seen[:, None, :, None, :].expand(-1, kv, -1, group, -1).reshape(batch, kv, -1, j.numel())
    x = q.matmul(k.transpose(2, 3)) * s["scale"]
    del k
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    # rows that see nothing come out as zero
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top.clamp(min=-1e30))
    total = x.sum(-1, keepdim=True)
    out = x.matmul(_gathered(s, s["v_cache"], s["v_scales"])) / total.clamp(min=1e-37)
    out = out.view(batch, kv, -1, group, head).permute(0, 2, 1, 3, 4).reshape(batch, -1, c["q_heads"], head)
    i = i.clamp(max=s["max_new"] - 1)
    zero = torch.zeros((), device=DEV)
    out = torch.where(valid[:, None, None], out[seq, i], zero).to(torch.bfloat16)
    if not c["lse"]:
        return out
    lse = (top + torch.log(total))[..., 0].view(batch, kv, -1, group).permute(0, 2, 1, 3).reshape(batch, -1, c["q_heads"])
    return out, torch.where(valid[:, None], lse[seq, i], zero - math.inf)


def _pages(s):
    c = s["case"]
    batch, pages, page, table = c["batch"], c["pages"], c["page"], c["table"]
    tab, lens, refs, req = s["page_table"], s["kv_lens"], s["ref_counts"], s["request"]
    j = torch.arange(table, device=DEV)
    have = (lens + page - 1) // page
    mine = j < have[:, None]
    none = torch.full((), -1, dtype=torch.int32, device=DEV)
    tab = torch.where(mine, tab, none)
    no_moves = torch.empty((0, 2), dtype=torch.int32, device=DEV)
    free = refs == 0
    rank = torch.cumsum(free, 0)
    slots = torch.full((pages + 1,), -1, dtype=torch.int32, device=DEV)  # the free pages in order
    slots[torch.where(free, rank - 1, pages)] = torch.arange(pages, dtype=torch.int32, device=DEV)
    slots[pages] = -1
    if c["kind"] == "RESERVE":
        want = (req + page - 1) // page
        valid = (req >= lens) & (want <= table)
        need = torch.where(valid, want - have, torch.zeros_like(want))
        upto = torch.cumsum(need, 0)
        granted = valid & ((need == 0) | (upto <= rank[-1]))
        fresh = granted[:, None] & (j >= have[:, None]) & (j < want[:, None])
        at = (upto - need - have)[:, None] + j
        given = slots[torch.where(fresh, at, pages)]
        refs = refs.clone()
        refs[torch.where(fresh, given, none)[fresh].long()] = 1
        return torch.where(fresh, given, tab), torch.where(granted, req, lens), refs, no_moves, granted.to(torch.int32)
    if c["kind"] == "FORK":
        src, dst = req[:, 0].long(), req[:, 1].long()
        valid = (src != dst) & (lens[dst] == 0)
        valid = valid & ~((dst[:, None] == dst[None, :]).tril(-1).any(1))
        need = (valid & (lens[src] % page != 0)).to(torch.int32)
        upto = torch.cumsum(need, 0)
        granted = valid & ((need == 0) | (upto <= rank[-1]))
        copied = granted & (need > 0)
        page_new = slots[torch.where(copied, upto - 1, pages)]
        last = (have[src] - 1).clamp(min=0)
        rows = tab[src]
        page_old = rows.gather(1, last[:, None].long())[:, 0]
        rows = torch.where(copied[:, None] & (j == last[:, None]), page_new[:, None], rows)
        refs = refs.clone()
        shared = rows[granted].reshape(-1)
        refs.index_add_(0, shared[shared >= 0].long(), torch.ones_like(shared[shared >= 0]))
        tab = tab.clone()
        tab[dst[granted]] = rows[granted]
        lens = lens.clone()
        lens[dst[granted]] = lens[src[granted]]
        moves = torch.full((req.shape[0] + 1, 2), -1, dtype=torch.int32, device=DEV)
        moves[torch.where(copied, upto - 1, req.shape[0])] = torch.stack([page_old, page_new], 1)
        return tab, lens, refs, moves[:-1], granted.to(torch.int32)
    if c["kind"] == "FREE":
        seq = req.long()
        status = ~((seq[:, None] == seq[None, :]).tril(-1).any(1))
        gone = torch.zeros(batch, dtype=torch.bool, device=DEV)
        gone[seq] = True
        held = tab[gone].reshape(-1)
        refs = refs.clone()
        refs.index_add_(0, held[held >= 0].long(), -torch.ones_like(held[held >= 0]))
        return torch.where(gone[:, None], none, tab), torch.where(gone, 0, lens), refs, no_moves, status.to(torch.int32)
    used = pages - rank[-1]  # COMPACT
    ids = torch.arange(pages, device=DEV)
    goes = ~free & (ids >= used)
    k = torch.cumsum(goes, 0) - 1
    to = torch.where(goes, slots[torch.where(goes, k, pages)], ids.to(torch.int32))
    moves = torch.full((pages // 2 + 1, 2), -1, dtype=torch.int32, device=DEV)
    moves[torch.where(goes, k, pages // 2)] = torch.stack([ids.to(torch.int32), to], 1)
    new = torch.zeros_like(refs)
    new[to[~free].long()] = refs[~free]
    tab = torch.where(tab >= 0, to[tab.long().clamp(min=0)], tab)
    return tab, lens.clone(), new, moves[:-1], torch.empty((0,), dtype=torch.int32, device=DEV)


def _copy(s):
    live = s["moves"][s["moves"][:, 0] >= 0].long()
    for x in s["buffers"]:
        x = x.view(torch.int8)
        x[live[:, 1]] = x[live[:, 0]]
    return s["buffers"]


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "copy":
        per = 2 * c["kv_heads"] * (c["page"] * c["head"] + c["page"] // c["block"] * 4)
        return {"bytes": 2 * c["moves"] * per + c["slots"] * 8, "flops": 0}
    if c["op"] == "pages":
        state = c["batch"] * c["table"] + c["batch"] + c["pages"]
        return {"bytes": 4 * (2 * state + c["batch"] + (c["pages"] if c["kind"] == "COMPACT" else 0)), "flops": 0}
    ctx, new = _lens(c)
    if c["op"] == "write":
        n = sum(new)
        blocks = sum(-(-l // c["block"]) - (l - m) // c["block"] for l, m in zip(ctx, new))
        return {"bytes": 2 * c["kv_heads"] * (3 * n * c["head"] + 4 * blocks), "flops": 2 * 3 * n * c["kv_heads"] * c["head"]}
    total = pairs = 0
    for l, m in zip(ctx, new):
        low = 0 if not c["window"] else max(0, l - m - c["window"] + 1)
        total += l - low
        for p in range(l - m, l):
            hi = p + 1 if c["causal"] else l
            pairs += hi - (max(0, p - c["window"] + 1) if c["window"] else 0)
    rows = sum(new) * c["q_heads"]
    return {"bytes": 2 * c["kv_heads"] * total * (c["head"] + 4 / c["block"]) + rows * (4 * c["head"] + (4 if c["lse"] else 0)),
            "flops": 4 * pairs * c["q_heads"] * c["head"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------

def _value(codes, c):
    return codes.double() if c["dtype"] == "s8" else codes.float().double()


def _nearest(x, c):
    """The code nearest to the f32 number x, ties to the even code."""
    x = x.clamp(-QMAX[c["dtype"]], QMAX[c["dtype"]])
    if c["dtype"] == "s8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    c = case
    if c["op"] in ("pages", "copy"):
        return None  # whole numbers and moved bytes
    s = _inputs(c, seed)
    ctx, new = _lens(c)
    page, block, heads = c["page"], c["block"], c["kv_heads"]
    table = s["page_table"].tolist()
    if c["op"] == "write":
        done = []
        for x, codes, scales in ((s["k"], s["k_cache"], s["k_scales"]), (s["v"], s["v_cache"], s["v_scales"])):
            codes, scales, row = _value(codes, c), scales.double(), 0
            for b, (l, m) in enumerate(zip(ctx, new)):
                pos = l - m
                while pos < l:  # one block after the other
                    b0 = pos // block * block
                    end = min(l, b0 + block)
                    pg, o = table[b][pos // page], b0 % page
                    t = x[row:row + end - pos].double().transpose(0, 1)  # [heads, tokens, head]
                    scale = (t.abs().amax((1, 2)) / QMAX[c["dtype"]]).float()
                    if pos > b0:
                        was = scales[pg, :, o // block].float()
                        scale = torch.maximum(scale, was)
                        ratio = (was.double() / scale.double()).float().double()[:, None, None]
                        held = codes[pg, :, o:o + pos - b0]
                        codes[pg, :, o:o + pos - b0] = _nearest((held * ratio).float().double(), c)
                    codes[pg, :, pos % page:pos % page + end - pos] = _nearest((t / scale.double()[:, None, None]).float().double(), c)
                    scales[pg, :, o // block] = scale.double()
                    row, pos = row + end - pos, end
            done.append((codes, scales))
        (kc, ks), (vc, vs) = done
        return [kc, vc, ks, vs]
    group = c["q_heads"] // heads
    out = torch.zeros((s["tokens"], c["q_heads"], c["head"]), dtype=torch.float64, device=DEV)
    lse = torch.full((s["tokens"], c["q_heads"]), -math.inf, dtype=torch.float64, device=DEV)
    row = 0
    for b, (l, m) in enumerate(zip(ctx, new)):
        tab = torch.tensor(table[b][:-(-l // page)], device=DEV)
        p = torch.arange(l - m, l, device=DEV)[:, None]
        j = torch.arange(l, device=DEV)[None, :]
        hidden = torch.zeros((m, l), dtype=torch.bool, device=DEV)
        if c["causal"]:
            hidden |= j > p
        if c["window"]:
            hidden |= j <= p - c["window"]
        for h in range(heads):
            k, v = ((_value(x[tab, h], c) * y[tab, h].double().repeat_interleave(block, 1)[..., None]).reshape(-1, c["head"])[:l]
                    for x, y in ((s["k_cache"], s["k_scales"]), (s["v_cache"], s["v_scales"])))
            for q in range(h * group, (h + 1) * group):
                x = s["q"][row:row + m, q].double() @ k.t() * s["scale"]
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                x[hidden] = -math.inf
                lse[row:row + m, q] = torch.logsumexp(x, 1)
                out[row:row + m, q] = torch.softmax(x, 1) @ v
        row += m
    return [out, lse] if c["lse"] else out
