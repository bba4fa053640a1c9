"""The calls over the 8-bit paged key/value cache against their plain restatement: codes, scales and
book-keeping bit for bit, attention within bounds that follow from its roundings (oracle/kv_cache.py)."""
import threading

import numpy as np
import pytest
import torch

from oracle import kv_cache as plain
from xla_amd import dtypes, ffi, hlo_runner, ops

pytestmark = pytest.mark.gpu

KINDS = ("s8", "f8")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def bf16(a):
    """(tensor, the f32 values it holds)"""
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16)
    return t.cuda(), t.float().numpy()


class Pool:
    """A cache of random codes on the host and the device, and a table that scatters its pages."""

    def __init__(self, rng, kind, lens, heads, head, page, block, width=None, spare=3):
        self.kind, self.page, self.block = kind, page, block
        lens = np.asarray(lens, np.int32)
        per = [-(-int(n) // page) for n in lens]
        width = max(per + [1]) if width is None else width
        pages = sum(per) + spare
        order = rng.permutation(pages).astype(np.int32)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lens = lens
        shape = (pages, heads, page, head)
        if kind == "s8":
            draw = lambda: np.clip(np.rint(rng.standard_normal(shape) * 32), -127, 127).astype(np.int8)
        else:
            draw = lambda: dtypes.f32_to_f8e4m3fn(np.clip(rng.standard_normal(shape) * 110, -448, 448).astype(np.float32))
        scale = lambda: (rng.uniform(0.5, 1.5, (pages, heads, page // block)) / (32 if kind == "s8" else 110)).astype(np.float32)
        self.k, self.v, self.ks, self.vs = draw(), draw(), scale(), scale()

    def device(self):
        return [dev(x) for x in (self.k, self.v, self.ks, self.vs, self.table, self.lens)]


def offsets(new, start=0):
    return np.concatenate([[start], start + np.cumsum(new)]).astype(np.int32)


def check_attention(pool, q, q_offsets, *, lse=True, scratch="auto", tiny=0.0, **kw):
    print("attention", pool.kind, q.shape, pool.k.shape, pool.block, pool.lens.tolist()[:8], kw, flush=True)
    qt, qf = bf16(q)
    scale = kw.pop("scale", q.shape[2] ** -0.5)
    out, got_lse = ops.kv_cache_attention(qt, *pool.device(), dev(q_offsets), scale=scale, lse=True, scratch=scratch, **kw)
    torch.cuda.synchronize()
    ref, ref_lse, spread, slack, largest = plain.attention(qf, pool.k, pool.v, pool.ks, pool.vs, pool.kind, pool.table, pool.lens,
                                                  q_offsets, np.float32(scale), **kw)
    tol, tol_lse = plain.attention_tolerance(ref, ref_lse, spread, slack, largest, int(pool.lens.max(initial=0)))
    got = out.float().cpu().numpy().astype(np.float64)
    bad = ~(np.abs(got - ref) <= tol + tiny)
    assert not bad.any(), (int(bad.sum()), bad.size, [(tuple(i), got[tuple(i)], ref[tuple(i)], tol[tuple(i)]) for i in np.argwhere(bad)[:4]])
    g = got_lse.cpu().numpy().astype(np.float64)
    none = np.isneginf(ref_lse)
    assert np.array_equal(np.isneginf(g), none)
    with np.errstate(invalid="ignore"):
        off = np.where(none, 0.0, np.abs(g - ref_lse))
    assert (off <= tol_lse).all(), (off - tol_lse).max()
    return out, got_lse


# ---- attention -------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("head, heads, group, page, block", [
    (128, 2, 4, 64, 16), (64, 1, 1, 16, 16), (80, 2, 3, 32, 4), (96, 1, 16, 16, 1), (256, 2, 8, 128, 128), (16, 3, 2, 16, 2),
    (48, 1, 40, 64, 8), (112, 2, 5, 256, 64), (144, 1, 7, 32, 32), (192, 1, 17, 64, 1), (128, 1, 128, 16, 16)])
def test_single_tokens(kind, head, heads, group, page, block):
    """One row each over lengths around every tile: none, one, 15 to 17, 31 to 33, 63 to 65, 127 to 129, several pages."""
    rng = np.random.default_rng(head * 7 + group)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 191, 257, 511, 1025]
    pool = Pool(rng, kind, lens, heads, head, page, block)
    q = rng.standard_normal((len(lens), heads * group, head))
    check_attention(pool, q, offsets([1] * len(lens)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("causal, window, softcap", [(True, 0, 0.0), (False, 0, 0.0), (True, 1, 0.0), (True, 7, 5.0),
                                                     (True, 100, 0.0), (False, 0, 2.5), (True, 1 << 40, 0.0)])
@pytest.mark.parametrize("head, heads, group, page, block", [(128, 2, 4, 64, 16), (80, 1, 3, 16, 8), (64, 2, 1, 128, 1), (256, 1, 2, 32, 32)])
def test_several_tokens(kind, causal, window, softcap, head, heads, group, page, block):
    """Ragged calls: sequences without rows, with fewer positions than rows (rows that see nothing), drafts, prompts;
    rows in front of the first and behind the last sequence."""
    rng = np.random.default_rng(window % 1000 + head)
    new = [0, 1, 3, 5, 17, 40, 2, 130, 0, 1, 9]
    lens = [33, 1, 3, 2, 17, 300, 1000, 130, 0, 0, 64]
    pool = Pool(rng, kind, lens, heads, head, page, block, width=1000 // page + 3)
    q = rng.standard_normal((sum(new) + 3 + 2, heads * group, head))
    check_attention(pool, q, offsets(new, 3), causal=causal, window=window, softcap=softcap)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("head, group, n", [(128, 4, 300), (64, 8, 200), (96, 1, 513), (256, 2, 150), (208, 3, 129)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(kind, head, group, n, causal):
    """Many rows: a prompt alone, one behind an earlier part, a short one, single tokens between them."""
    rng = np.random.default_rng(n)
    new = [n, 1, n // 2 + 1, 33, 1]
    lens = [n, 200, n + 77, 33, 700]
    pool = Pool(rng, kind, lens, 2, head, 64, 16)
    q = rng.standard_normal((sum(new) + 1, 2 * group, head))
    check_attention(pool, q, offsets(new), causal=causal)
    if causal:
        check_attention(pool, q, offsets(new), window=65, softcap=10.0)


# (head, heads, group, page, block, new, lens): many more packed rows than sequences, so that the kernel of the prompts
# takes part; its tiles are of 128 packed rows, its stages of 64 positions
PROMPTS = [(128, 2, 16, 64, 16, [140, 1, 33, 3], [140, 700, 210, 65]), (64, 1, 32, 16, 1, [70, 9], [70, 333]),
           (80, 1, 40, 32, 2, [55, 2, 0, 5], [120, 64, 9, 3]), (128, 1, 64, 16, 2, [36, 4], [1, 129]),
           (16, 2, 64, 128, 4, [64], [64]), (256, 1, 16, 64, 32, [128, 8, 1], [191, 8, 63]), (208, 1, 24, 16, 1, [87, 5], [900, 5]),
           (96, 3, 24, 256, 256, [100], [257]), (64, 2, 3, 64, 64, [700, 1, 65], [1500, 3, 65])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scratch", ["auto", None])
@pytest.mark.parametrize("head, heads, group, page, block, new, lens", PROMPTS)
def test_prompts_of_many_heads(kind, scratch, head, heads, group, page, block, new, lens):
    """Also sequences with fewer positions than rows, and rows of nobody at both ends."""
    rng = np.random.default_rng(head + group)
    pool = Pool(rng, kind, lens, heads, head, page, block)
    q = rng.standard_normal((sum(new) + 3, heads * group, head))
    for kw in (dict(), dict(causal=False), dict(window=50), dict(window=1), dict(window=130, softcap=3.0), dict(causal=False, softcap=20.0)):
        a = check_attention(pool, q, offsets(new, 1), scratch=scratch, **kw)
        assert ffi.last_kernel().startswith("kv_cache_attention_prompt")
    b = check_attention(pool, q, offsets(new, 1), scratch=scratch, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("new, lens", [([40] * 70, [40 + 3 * i for i in range(70)]), ([1] * 90 + [300], [64 + i for i in range(91)]),
                                       ([8] * 40, [2000] * 40), ([1100], [1100]), ([129, 0, 1, 258, 20], [4100, 0, 3000, 2300, 20])])
def test_tiles_cut_and_whole(new, lens):
    """More tiles than are worth cutting, few among many single rows, pieces of very different lengths."""
    rng = np.random.default_rng(len(new))
    pool = Pool(rng, "f8", lens, 2, 64, 64, 16)
    q = rng.standard_normal((sum(new), 2 * 8, 64))
    check_attention(pool, q, offsets(new))
    assert ffi.last_kernel().startswith("kv_cache_attention_prompt")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("head, group, new", [(128, 4, [1, 2, 20]), (64, 32, [1, 90, 4]), (128, 32, [70, 2, 3]), (256, 16, [150, 1, 3])])
@pytest.mark.parametrize("block", [1, 16])
def test_scales_of_every_size(kind, head, group, new, block):
    """Blocks whose scales are zero, negative, tiny, subnormal or large, in both kernels.  A weight times its value's
    scale that is below 2^-126 may become zero: 2^-126 times a code, for each position; the weights' sum is 1 or more."""
    rng = np.random.default_rng(head + group)
    pool = Pool(rng, kind, [90, 300, 20], 2, head, 16, block)
    shape = pool.ks.shape
    pool.vs *= rng.choice([1.0, 0.0, -1.0, 1e-30, 1e-42, 1e-3, 50.0], shape).astype(np.float32)
    pool.ks *= rng.choice([1.0, 0.0, -1.0, 1e-30, 1e-42, 1e-3, 3.0], shape).astype(np.float32)
    q = rng.standard_normal((sum(new), 2 * group, head))
    check_attention(pool, q, offsets(new), tiny=300 * 448 * 2.0 ** -126)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group", [2, 64])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_value_scale_that_is_no_number(kind, group, bad):
    """It reaches the result and the lse of the rows that see it, and no others, in both kernels."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, kind, [64], 1, 128, 64, 16)
    pool.vs[pool.table[0, 0], 0, 2] = bad          # positions 32 to 47
    q = rng.standard_normal((64, group, 128))
    out, lse = ops.kv_cache_attention(bf16(q)[0], *pool.device(), dev(offsets([64])), lse=True)
    assert ffi.last_kernel().startswith("kv_cache_attention_prompt") == (group == 64)
    assert torch.isnan(out[32:]).all() and torch.isnan(lse[32:]).all()
    assert torch.isfinite(out[:32]).all() and torch.isfinite(lse[:32]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads, new", [(2, 1), (64, 60)])
@pytest.mark.parametrize("scale", [1e-4, 0.01, 300.0])
def test_many_small_weights(kind, heads, new, scale):
    """One position has all but 2% of the weight and values of 0; 20000 with 2^-20 each have the result.  Each of these
    weights is rounded to f16 by at most 2^-25 of the largest one, 2^-5 of itself; they are alike, so it stays that much."""
    n = 20000
    pool = Pool(np.random.default_rng(3), kind, [n + new], 1, 64, 64, 16)
    pool.k[:], pool.v[:] = 0, (64 if kind == "s8" else 0x68)      # 64 in f8e4m3fn
    pool.k[pool.table[0, 0], 0, 7] = 1 if kind == "s8" else 0x38   # 1
    pool.v[pool.table[0, 0], 0, 7] = 0
    pool.ks[:], pool.vs[:] = 1.0, scale
    q = np.zeros((new, heads, 64))
    q[:, :, 0] = 14.0
    out = ops.kv_cache_attention(bf16(q)[0], *pool.device(), dev(offsets([new])), causal=False, scale=20 * np.log(2.0) / 14)
    w = 2.0 ** -20 * (n + new - 1)
    want = 64 * scale * w / (1 + w)
    got = out.float().cpu().numpy()
    assert (np.abs(got / want - 1) <= 2.0 ** -5 + 2.0 ** -8 + 1e-4).all(), (got.min(), got.max(), want)


@pytest.mark.parametrize("kind", KINDS)
def test_maxima_that_grow_along_the_keys(kind):
    """Scores that rise by far more than a weight bears, from stage to stage, half to half and block to block."""
    rng = np.random.default_rng(7)
    pool = Pool(rng, kind, [640], 1, 64, 64, 4)
    pool.k[:] = np.abs(pool.k) if kind == "s8" else pool.k & 0x7f
    pool.ks *= (2.0 ** np.arange(pool.ks.shape[2]) / 64).astype(np.float32)
    order = rng.permutation(pool.ks.shape[2])
    q = np.abs(rng.standard_normal((100, 64, 64)))
    check_attention(pool, q, offsets([100]))
    check_attention(pool, -q, offsets([100]))
    pool.ks = np.ascontiguousarray(pool.ks[:, :, order])
    check_attention(pool, q, offsets([100]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scratch", ["auto", None])
@pytest.mark.parametrize("new, lens", [([1], [9001]), ([1, 1, 1], [5, 12001, 700]), ([4, 2], [6000, 3333]), ([150], [5000]),
                                       ([1] * 40, list(range(60, 1260, 30)))])
def test_long_contexts_with_and_without_scratch(kind, scratch, new, lens):
    """With scratch the keys of a sequence are split over workgroups; without it they are not."""
    rng = np.random.default_rng(len(new) + lens[0])
    pool = Pool(rng, kind, lens, 2, 128, 64, 32, width=max(lens) // 64 + 40)
    q = rng.standard_normal((sum(new), 8, 128))
    a, la = check_attention(pool, q, offsets(new), scratch=scratch)
    b, lb = check_attention(pool, q, offsets(new), scratch=scratch)
    assert torch.equal(a, b) and torch.equal(la, lb)   # one order of the sums


def test_scratch_that_is_too_small_or_holds_anything():
    rng = np.random.default_rng(5)
    pool = Pool(rng, "f8", [4000, 700], 2, 128, 64, 16)
    q = rng.standard_normal((2, 8, 128))
    need = ffi.library().xla_amd_kv_cache_attention_workspace_bytes(2, 2, 8, 2, 128, pool.table.shape[1] * 64)
    want, _ = check_attention(pool, q, offsets([1, 1]))
    for fill in (0x00, 0xff, 0x7f):
        scratch = torch.full((max(need, 16),), fill, dtype=torch.uint8, device="cuda")
        got, _ = check_attention(pool, q, offsets([1, 1]), scratch=scratch)
        assert torch.equal(got, want)
    check_attention(pool, q, offsets([1, 1]), scratch=torch.full((48,), 0x7f, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("batch", [65, 300, 1100])
def test_many_sequences(batch):
    """More sequences than the lanes of a wave and the threads of a workgroup look at together."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 90, batch)
    new = rng.integers(0, 3, batch)
    pool = Pool(rng, "s8", lens, 1, 64, 16, 8)
    q = rng.standard_normal((int(new.sum()), 4, 64))
    check_attention(pool, q, offsets(new))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 60, 200]])
def test_positions_that_nobody_sees_may_hold_anything(kind, new):
    """NaN codes and NaN or infinite scales behind a sequence's length, in free pages, and before a window."""
    rng = np.random.default_rng(11)
    lens = [40, 65, 333]
    pool = Pool(rng, kind, lens, 2, 128, 16, 8, width=40)
    used = np.zeros(pool.k.shape[0], bool)
    for b, n in enumerate(lens):
        pages = pool.table[b, :-(-n // 16)]
        used[pages] = True
        last, o = pages[-1], n % 16
        if o:
            for codes, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
                codes[last, :, o:] = 0x7f if kind == "f8" else -128
                scales[last, :, -(-o // 8):] = np.nan
    for codes, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
        codes[~used] = 0xff if kind == "f8" else -128
        scales[~used] = np.inf
    q = rng.standard_normal((sum(new), 4, 128))
    check_attention(pool, q, offsets(new))
    # with a window of 33 the first blocks of the longest sequence are out of every row's sight
    hidden = (lens[2] - new[2] - 33 + 1) // 8
    for i in range(max(0, hidden)):
        page, o = pool.table[2, i * 8 // 16], i * 8 % 16 // 8
        for scales in (pool.ks, pool.vs):
            scales[page, :, o] = np.nan
    check_attention(pool, q, offsets(new), window=33)


@pytest.mark.parametrize("kind", KINDS)
def test_a_block_that_is_no_number_reaches_only_the_rows_that_see_it(kind):
    rng = np.random.default_rng(3)
    pool = Pool(rng, kind, [64], 1, 128, 64, 16)
    pool.vs[pool.table[0, 0], 0, 3] = np.nan       # positions 48 to 63
    pool.ks[pool.table[0, 0], 0, 2] = np.nan       # positions 32 to 47
    q = rng.standard_normal((64, 2, 128))
    qt, qf = bf16(q)
    out = ops.kv_cache_attention(qt, *pool.device(), dev(offsets([64]))).float().cpu().numpy()
    assert np.isnan(out[32:]).all() and np.isfinite(out[:32]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [4, 100, 30, 7]])
def test_pages_outside_the_pool_are_not_read(kind, new):
    rng = np.random.default_rng(17)
    lens = [200, 333, 90, 64]
    pool = Pool(rng, kind, lens, 2, 64, 32, 8)
    pages = pool.k.shape[0]
    pool.table[0, 2], pool.table[1, 0], pool.table[1, 7], pool.table[2, 1] = pages, -5, 2 ** 31 - 1, -2 ** 31
    pool.table[3, :] = -1                      # nothing at all is left of this one
    q = rng.standard_normal((sum(new), 4, 64))
    check_attention(pool, q, offsets(new))


def test_lengths_and_offsets_out_of_range_stay_inside():
    """Lengths beyond the table or negative, offsets beyond the rows or falling: clamped."""
    rng = np.random.default_rng(23)
    pool = Pool(rng, "s8", [64, 64, 64, 64], 1, 64, 16, 16)
    pool.lens = np.array([1000, -7, 64, 2 ** 31 - 1], np.int32)
    q = rng.standard_normal((9, 2, 64))
    check_attention(pool, q, np.array([0, 2, 4, 6, 100], np.int32))
    check_attention(pool, q, np.array([-3, 2, 4, 6, 9], np.int32))


def test_empty_calls():
    rng = np.random.default_rng(29)
    pool = Pool(rng, "f8", [20], 1, 64, 16, 16)
    check_attention(pool, np.zeros((0, 2, 64)), offsets([0]))
    pool.table, pool.lens = pool.table[:0], pool.lens[:0]
    check_attention(pool, rng.standard_normal((3, 2, 64)), offsets([]))      # rows of nobody
    pool = Pool(rng, "f8", [20], 1, 64, 16, 16)
    pool.table = pool.table[:, :0]
    check_attention(pool, rng.standard_normal((3, 2, 64)), offsets([3]))     # a table of no width
    pool = Pool(rng, "f8", [0], 1, 64, 16, 16, spare=0)
    check_attention(pool, rng.standard_normal((3, 2, 64)), offsets([3]))     # no pages


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 30.0])
def test_scales_of_the_softmax(scale):
    """Also a negative one, zero (a plain mean), and one that leaves a single weight."""
    rng = np.random.default_rng(31)
    pool = Pool(rng, "s8", [150, 70], 2, 64, 16, 4)
    check_attention(pool, rng.standard_normal((12, 4, 64)), offsets([1, 11]), scale=scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 2], [130, 40]])
def test_a_cache_beyond_32_bits(kind, new):
    """Pages whose first byte lies past 2^32: the offsets are 64 bits wide, reading and writing."""
    rng = np.random.default_rng(37)
    heads, head, page, block = 8, 128, 256, 64
    pages = (1 << 32) // (heads * head * page) + 40
    small = Pool(rng, kind, [300, 200], heads, head, page, block, width=2, spare=0)
    far = np.array([pages - 1 - 7 * i for i in range(small.k.shape[0])], np.int32)
    dt = torch.int8 if kind == "s8" else torch.uint8
    k, v = (torch.empty((pages, heads, page, head), dtype=dt, device="cuda") for _ in range(2))
    ks, vs = (torch.empty((pages, heads, page // block), device="cuda") for _ in range(2))
    table = np.where(small.table >= 0, far[small.table], -1).astype(np.int32)
    at = dev(far.astype(np.int64))
    for big, x in ((k, small.k), (v, small.v), (ks, small.ks), (vs, small.vs)):
        big[at] = dev(x)
    new_k, new_kf = bf16(rng.standard_normal((sum(new), heads, head)))
    off = offsets(new)
    ops.kv_cache_write(new_k, new_k, k, v, ks, vs, dev(table), dev(small.lens), dev(off))
    small.k, small.ks = plain.write(new_kf, small.k, small.ks, kind, small.table, small.lens, off)
    small.v, small.vs = plain.write(new_kf, small.v, small.vs, kind, small.table, small.lens, off)
    for big, x in ((k, small.k), (v, small.v), (ks, small.ks), (vs, small.vs)):
        assert np.array_equal(big[at].cpu().numpy(), x)
    q = rng.standard_normal((sum(new), 16, head))
    want, want_lse = check_attention(small, q, off)
    got, got_lse = ops.kv_cache_attention(bf16(q)[0], k, v, ks, vs, dev(table), dev(small.lens), dev(off), lse=True)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    near = torch.arange(at.numel(), dtype=torch.int32, device="cuda")
    ops.kv_cache_copy_pages(torch.stack([at.to(torch.int32), near], 1).contiguous(), [k, v, ks, vs])
    for big, x in ((k, small.k), (v, small.v), (ks, small.ks), (vs, small.vs)):
        assert np.array_equal(big[:at.numel()].cpu().numpy(), x)


# ---- write -----------------------------------------------------------------------------------------

def check_write(pool, k, v, q_offsets):
    print("write", pool.kind, k.shape, pool.k.shape, pool.block, pool.lens.tolist()[:8], flush=True)
    kt, kf = bf16(k)
    vt, vf = bf16(v)
    got = ops.kv_cache_write(kt, vt, *pool.device(), dev(q_offsets))
    torch.cuda.synchronize()
    want_k = plain.write(kf, pool.k, pool.ks, pool.kind, pool.table, pool.lens, q_offsets)
    want_v = plain.write(vf, pool.v, pool.vs, pool.kind, pool.table, pool.lens, q_offsets)
    for g, w, what in zip(got, (want_k[0], want_v[0], want_k[1], want_v[1]), ("k", "v", "k_scales", "v_scales")):
        g = g.cpu().numpy()
        same = np.array_equal(g.view(np.uint32), w.view(np.uint32)) if g.dtype == np.float32 and not np.isnan(w).any() else \
            np.array_equal(g, w, equal_nan=g.dtype == np.float32)
        assert same, (what, np.argwhere(g != w)[:5].tolist(), int((g != w).sum()))
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads, head, page, block", [(2, 128, 64, 16), (1, 64, 16, 1), (3, 80, 16, 16), (8, 256, 32, 4), (5, 16, 128, 128),
                                                      (1, 48, 1024, 512), (4, 208, 64, 2), (2, 128, 1024, 1024)])
def test_write(kind, heads, head, page, block):
    """Tokens that start, continue and end blocks and pages, sequences without new rows, with fewer positions than
    rows, rows of nobody; pages and codes that the call does not name stay as they were."""
    rng = np.random.default_rng(head + page + block)
    new = [1, 1, 0, 5, 17, 64, 130, 3, 1, 7, 0, 33]
    lens = [1, 40, 50, 5, 20, 64, 200, 2, 0, 23, 0, page + 33]
    pool = Pool(rng, kind, lens, heads, head, page, block, width=max(lens) // page + 2)
    pool.ks *= rng.choice([0.05, 1.0, 3.0], pool.ks.shape).astype(np.float32)
    shape = (sum(new) + 2 + 3, heads, head)
    k = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:2] + (1,)))
    v = rng.standard_normal(shape)
    check_write(pool, k, v, offsets(new, 2))


@pytest.mark.parametrize("kind", KINDS)
def test_write_of_special_values(kind):
    """Zeros, a NaN, infinities, the smallest and largest numbers of bf16, into fresh and held blocks."""
    rng = np.random.default_rng(41)
    for case in range(7):
        for lens in ([4], [12], [16]):
            pool = Pool(rng, kind, lens, 2, 32, 16, 8)
            k = rng.standard_normal((4, 2, 32)).astype(np.float32)
            if case == 0:
                k[:] = 0.0
            elif case == 1:
                k[1, 0, 3] = np.nan
            elif case == 2:
                k[2, 1, 5], k[3, 0, 0] = np.inf, -np.inf
            elif case == 3:
                k *= np.float32(1e-38)
            elif case == 4:
                k = np.sign(k) * np.float32(2.0 ** -133)     # bf16's smallest: the scale rounds in f32's denormals
            elif case == 5:
                k = np.sign(k) * np.float32(3.3e38)
            else:
                k[:, :, ::2] = -0.0
                pool.ks[:] = 0.0
                pool.vs[:] = np.nan
            check_write(pool, k, rng.standard_normal((4, 2, 32)) if case != 6 else k, offsets([4]))


@pytest.mark.parametrize("kind", KINDS)
def test_write_one_token_at_a_time_and_bad_pages(kind):
    rng = np.random.default_rng(43)
    pool = Pool(rng, kind, [90, 90], 2, 64, 16, 8)
    pool.table[1, 1], pool.table[1, 3] = pool.k.shape[0], -1
    tensors = pool.device()
    for t in range(1, 40):
        pool.lens = np.array([t, t + 50], np.int32)
        tensors[5] = dev(pool.lens)
        kt, kf = bf16(rng.standard_normal((2, 2, 64)) * np.exp(rng.standard_normal()))
        ops.kv_cache_write(kt, kt, *tensors, dev(offsets([1, 1])))
        pool.k, pool.ks = plain.write(kf, pool.k, pool.ks, kind, pool.table, pool.lens, offsets([1, 1]))
        pool.v, pool.vs = plain.write(kf, pool.v, pool.vs, kind, pool.table, pool.lens, offsets([1, 1]))
    for g, w in zip(tensors, (pool.k, pool.v, pool.ks, pool.vs)):
        assert np.array_equal(g.cpu().numpy(), w)


def test_write_random_calls():
    rng = np.random.default_rng(47)
    for trial in range(30):
        kind = KINDS[trial % 2]
        page = int(rng.choice([16, 32, 64, 128]))
        block = int(rng.choice([b for b in (1, 2, 4, 8, 16, 32, 64, 128) if b <= page]))
        batch, heads, head = int(rng.integers(1, 90)), int(rng.integers(1, 5)), 16 * int(rng.integers(1, 17))
        new = rng.integers(0, int(rng.choice([2, 6, 60])), batch)
        lens = rng.integers(0, 200, batch)
        pool = Pool(rng, kind, lens, heads, head, page, block, width=200 // page + 2)
        shape = (int(new.sum()), heads, head)
        check_write(pool, rng.standard_normal(shape), rng.standard_normal(shape) * 3, offsets(new))


# ---- pages and copies ------------------------------------------------------------------------------

def random_book(rng, batch, width, pages, page, fill):
    table = rng.integers(-3, pages + 3, (batch, width)).astype(np.int32)   # also entries outside the pool
    lens = np.zeros(batch, np.int32)
    refs = np.zeros(pages, np.int32)
    order, at = rng.permutation(pages), 0
    for b in range(batch):
        n = int(rng.integers(0, width + 1))
        n = min(n, int(pages * fill) - at)
        if n <= 0 or rng.random() < 0.2:
            continue
        table[b, :n] = order[at:at + n]
        refs[order[at:at + n]] = rng.integers(1, 3, n)
        lens[b] = (n - 1) * page + rng.integers(1, page + 1)
        at += n
    return table, lens, refs


@pytest.mark.parametrize("op", ["RESERVE", "FORK", "FREE", "COMPACT"])
@pytest.mark.parametrize("batch, width, pages, page, fill", [(1, 1, 1, 16, 1.0), (5, 7, 40, 16, 0.6), (70, 33, 2500, 64, 0.7), (300, 9, 900, 1, 0.95),
                                                             (1500, 5, 6001, 32, 0.6), (40, 300, 9000, 16, 0.99), (3, 4, 12, 16, 0.0)])
def test_pages(op, batch, width, pages, page, fill):
    rng = np.random.default_rng(batch + width + ord(op[1]))
    for trial in range(3):
        table, lens, refs = random_book(rng, batch, width, pages, page, fill)
        if trial == 2 and batch > 2:
            lens[1], lens[2] = -4, width * page + 99        # what no table can hold
        request = None
        if op == "RESERVE":
            request = (lens + rng.integers(-2, page * 3, batch)).astype(np.int32)
            if batch > 3:
                request[3] = 2 ** 31 - 1
        elif op == "FORK":
            request = rng.integers(-1, batch + 1, (max(1, batch // 2) * (trial + 1), 2)).astype(np.int32)
        elif op == "FREE":
            request = rng.integers(-1, batch + 1, max(1, batch // 2)).astype(np.int32)
        print("pages", op, batch, width, pages, trial, flush=True)
        got = ops.kv_cache_pages(op, dev(table), dev(lens), dev(refs), None if request is None else dev(request), page_size=page)
        want = plain.pages(op, table, lens, refs, request, page)
        for g, w, what in zip(got, want, ("page_table", "kv_lens", "ref_counts", "moves", "status")):
            assert np.array_equal(g.cpu().numpy(), w), (what, np.argwhere(g.cpu().numpy() != w)[:4].tolist())


def test_pages_of_empty_states():
    none = lambda *d: torch.zeros(d, dtype=torch.int32, device="cuda")
    for op, request in (("RESERVE", none(0)), ("FORK", none(0, 2)), ("FREE", none(0)), ("COMPACT", None)):
        for pages in (0, 4):
            t, n, r, m, s = ops.kv_cache_pages(op, none(0, 3), none(0), none(pages), request, page_size=16)
            assert t.shape == (0, 3) and not r.any()
    t, n, r, m, s = ops.kv_cache_pages("RESERVE", none(2, 3), none(2), none(0), torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                                       page_size=16)
    assert s.tolist() == [1, 0] and t.tolist() == [[-1] * 3] * 2


def test_copy_pages_of_every_type_and_size():
    """Pages of 16-byte, 4-byte and odd sizes, several buffers at once, skipped pairs, parts beyond one workgroup."""
    rng = np.random.default_rng(53)
    pages = 37
    shapes = [((3, 16, 48), torch.int8), ((5,), torch.float32), ((7,), torch.uint8), ((3,), torch.bfloat16), ((2, 11), torch.int32),
              ((100001,), torch.uint8), ((4, 64, 256), torch.float8_e4m3fn), ((), torch.float32)]
    host = [rng.integers(0, 255, (pages, int(np.prod(s)) * torch.empty((), dtype=dt).element_size())).astype(np.uint8) for s, dt in shapes]
    buffers = [dev(h).view(dt).view((pages,) + s) for h, (s, dt) in zip(host, shapes)]
    order = rng.permutation(pages)
    moves = np.array([(order[2 * i], order[2 * i + 1]) for i in range(12)] + [(-1, -1), (3, pages), (pages, 3), (-1, 2), (5, -2 ** 31), (9, 9)],
                     np.int32)
    rng.shuffle(moves)
    ops.kv_cache_copy_pages(dev(moves), buffers)
    for h, b in zip(host, buffers):
        for src, dst in moves:
            if 0 <= src < pages and 0 <= dst < pages:
                h[dst] = h[src]
        assert np.array_equal(b.contiguous().view(torch.uint8).cpu().numpy().reshape(pages, -1), h)
    # no pairs, and an offset view that is only aligned to 4 bytes
    ops.kv_cache_copy_pages(torch.zeros((0, 2), dtype=torch.int32, device="cuda"), buffers)
    whole = torch.arange(1 + 6 * 8, dtype=torch.int32, device="cuda")
    part = whole[1:].view(6, 8)
    ops.kv_cache_copy_pages(dev(np.array([[0, 5]], np.int32)), [part])
    assert torch.equal(part[5], part[0]) and whole[0] == 0 and whole[40].item() == 40


# ---- as a program uses them ------------------------------------------------------------------------

def test_copy_pages_unaligned_and_large():
    """Pages of sizes and at addresses that no wide access fits, larger and smaller than a workgroup's part."""
    rng = np.random.default_rng(89)
    buffers, want = [], []
    for size, shift in ((1, 0), (4095, 1), (4097, 3), (16385, 0), (40000, 4), (33000, 1), (20004, 0), (65536, 16)):
        flat = torch.from_numpy(rng.integers(0, 256, 9 * size + shift, dtype=np.uint8)).cuda()
        buffers.append(flat[shift:].view(9, size))
        want.append(buffers[-1].clone())
    moves = [[3, 0], [-1, -1], [8, 5], [2, 9], [4, 4], [7, 1]]
    ops.kv_cache_copy_pages(torch.tensor(moves, dtype=torch.int32, device="cuda"), buffers)
    for got, w in zip(buffers, want):
        for a, b in ((3, 0), (8, 5), (7, 1)):
            w[b] = w[a]
        assert torch.equal(got, w), got.shape


def test_copy_pages_of_more_moves_than_workgroups():
    moves = torch.full((3 << 20, 2), -1, dtype=torch.int32, device="cuda")
    for at, pair in ((0, [1, 2]), ((1 << 21) + 3, [5, 0]), ((3 << 20) - 1, [4, 3])):
        moves[at] = torch.tensor(pair, dtype=torch.int32)
    large = torch.arange(6 * 5000, dtype=torch.int32, device="cuda").view(6, 5000)
    small = torch.arange(6 * 8, dtype=torch.int32, device="cuda").view(6, 8)
    want = [t[[5, 1, 1, 4, 4, 5]].clone() for t in (large, small)]
    ops.kv_cache_copy_pages(moves, [large, small])
    assert torch.equal(large, want[0]) and torch.equal(small, want[1])


@pytest.mark.parametrize("kind", KINDS)
def test_a_generation(kind):
    """Reserve, write, attend, fork, copy, diverge, free, compact, copy, attend again: against the plain calls at every
    step, and the attention over moved pages is bit for bit the one before."""
    rng = np.random.default_rng(59)
    batch, width, pages, heads, head, page, block = 5, 9, 30, 2, 64, 16, 8
    dt = torch.int8 if kind == "s8" else torch.uint8
    i32 = lambda *d, fill=0: torch.full(d, fill, dtype=torch.int32, device="cuda")
    table, lens, refs = i32(batch, width, fill=-1), i32(batch), i32(pages)
    cache = [torch.zeros((pages, heads, page, head), dtype=dt, device="cuda") for _ in range(2)] + \
            [torch.zeros((pages, heads, page // block), device="cuda") for _ in range(2)]

    def book(op, request=None):
        nonlocal table, lens, refs
        host = [t.cpu().numpy() for t in (table, lens, refs)]
        req = None if request is None else np.asarray(request, np.int32)
        got = ops.kv_cache_pages(op, table, lens, refs, None if req is None else dev(req), page_size=page)
        for g, w in zip(got, plain.pages(op, *host, req, page)):
            assert np.array_equal(g.cpu().numpy(), w), op
        table, lens, refs = got[:3]
        if got[3].numel():
            ops.kv_cache_copy_pages(got[3], cache)
        return got[4]

    def step(new):
        off = offsets(new)
        kt, kf = bf16(rng.standard_normal((sum(new), heads, head)))
        vt, vf = bf16(rng.standard_normal((sum(new), heads, head)))
        host = [c.cpu().numpy() for c in cache]
        where = (table.cpu().numpy(), lens.cpu().numpy(), off)
        ops.kv_cache_write(kt, vt, *cache, table, lens, dev(off))
        k, ks = plain.write(kf, host[0], host[2], kind, *where)
        v, vs = plain.write(vf, host[1], host[3], kind, *where)
        for g, w in zip(cache, (k, v, ks, vs)):
            assert np.array_equal(g.cpu().numpy(), w)
        return attend(new)

    def attend(new):
        q = np.random.default_rng(sum(new)).standard_normal((sum(new), 3 * heads, head))
        pool = Pool.__new__(Pool)
        pool.kind, pool.page, pool.block, pool.table, pool.lens = kind, page, block, table.cpu().numpy(), lens.cpu().numpy()
        pool.k, pool.v, pool.ks, pool.vs = (c.cpu().numpy() for c in cache)
        return check_attention(pool, q, offsets(new))[0]

    grow = lambda new: book("RESERVE", lens.cpu().numpy() + np.array(new))
    new = [37, 0, 16, 50, 0]
    assert grow(new).all()
    step(new)
    assert book("FORK", [[0, 1], [2, 4], [3, 3]]).tolist() == [1, 1, 0]
    for _ in range(20):
        new = [1, 1, 1, 0, 1]
        assert grow(new).all()
        out = step(new)
    assert not torch.equal(out[0], out[1])
    book("FREE", [0, 3, 3])
    before = attend([0, 1, 1, 0, 1])
    book("COMPACT")
    used = int((refs > 0).sum())
    assert (refs[:used] > 0).all()
    assert torch.equal(before, attend([0, 1, 1, 0, 1]))
    assert not grow([200, 0, 0, 0, 0])[0]       # more than the table holds
    book("FREE", [1, 2, 4, 0])
    assert not refs.any() and not lens.any()


def test_a_decoder_layer():
    """The cache between the framework's dots: RMSNorm and quantise, f8 dot to q, k, v, write, attend, weight-only dot."""
    rng = np.random.default_rng(61)
    batch, hidden, q_heads, heads, head, page, block = 6, 512, 8, 2, 64, 16, 16
    x = torch.randn((batch, hidden), device="cuda").to(torch.bfloat16)
    gamma = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    a, a_scale = ops.rowwise_quantize_fp8(x, gamma)
    n = (q_heads + 2 * heads) * head
    w = (torch.randn((hidden, n), device="cuda") * 30).clamp(-448, 448).to(torch.float8_e4m3fn)
    qkv = ops.fp8_scaled_dot(a, w.view(torch.uint8), a_scale, torch.full((), 1 / 600, device="cuda"))
    q, k, v = (t.contiguous().view(batch, -1, head) for t in qkv.split([q_heads * head, heads * head, heads * head], 1))
    lens = rng.integers(1, 100, batch)
    pool = Pool(rng, "f8", lens, heads, head, page, block)
    tensors = pool.device()
    off = offsets([1] * batch)
    ops.kv_cache_write(k, v, *tensors, dev(off))
    o = ops.kv_cache_attention(q, *tensors, dev(off))
    pool.k, pool.ks = plain.write(k.float().cpu().numpy(), pool.k, pool.ks, "f8", pool.table, pool.lens, off)
    pool.v, pool.vs = plain.write(v.float().cpu().numpy(), pool.v, pool.vs, "f8", pool.table, pool.lens, off)
    want, _ = check_attention(pool, q.float().cpu().numpy(), off)
    assert torch.equal(o, want)
    wo = torch.randint(-127, 128, (q_heads * head, hidden), dtype=torch.int8, device="cuda")
    y = ops.dequant_dot(o.view(batch, -1), wo, torch.full((hidden,), 1e-3, device="cuda"))
    ref = o.view(batch, -1).double() @ (wo.double() * float(np.float32(1e-3)))
    size = o.view(batch, -1).double().abs() @ (wo.double().abs() * 1e-3)
    # f32 sums of 512 products and one rounding to bf16
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 512 * 2.0 ** -24 * size).all()


def test_calls_replay_from_a_graph():
    """Write, attend and book-keeping captured on a side stream; every replay works on what the buffers hold then, with
    eager work and synchronisation in between, and is bit for bit the eager result."""
    rng = np.random.default_rng(67)
    pool = Pool(rng, "f8", [200, 3000, 31], 2, 128, 64, 16)
    tensors = pool.device()
    new = [1, 2, 1]
    k, _ = bf16(rng.standard_normal((4, 2, 128)))
    q, _ = bf16(rng.standard_normal((4, 8, 128)))
    off = dev(offsets(new))
    refs = torch.zeros(pool.k.shape[0], dtype=torch.int32, device="cuda")
    used = tensors[4][tensors[4] >= 0].long()
    refs[used] = 1
    request = dev(pool.lens)
    calls = [ops.kv_cache_write(k, k, *tensors, off, build_only=True),
             ops.kv_cache_attention(q, *tensors, off, lse=True, build_only=True),
             ops.kv_cache_pages("RESERVE", tensors[4], tensors[5], refs, request, page_size=64, build_only=True),
             ops.kv_cache_pages("COMPACT", tensors[4], tensors[5], refs, page_size=64, build_only=True)]
    copy = ops.kv_cache_copy_pages(calls[3].result[3], [torch.arange(refs.numel() * 8, device="cuda", dtype=torch.int32).view(-1, 8)],
                                   build_only=True)
    for c in calls + [copy]:
        c.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            for c in calls:
                c.run()
    torch.cuda.current_stream().wait_stream(side)
    start = [t.clone() for t in tensors[:4]]
    for turn in range(4):
        k.copy_(torch.randn_like(k.float()).to(torch.bfloat16) * (turn + 1))
        q.copy_(torch.randn_like(q.float()).to(torch.bfloat16))
        lens = torch.tensor([150 + turn * 13, 2900 - 500 * turn, 4 + turn], dtype=torch.int32)
        tensors[5].copy_(lens)
        request.copy_(lens + turn)
        for t, s in zip(tensors, start):
            t.copy_(s)
        for c in calls:
            c.run()
        torch.cuda.synchronize()
        want = [t.clone() for t in tensors[:4]] + [t.clone() for c in calls[1:] for t in c.result]
        for t, s in zip(tensors, start):
            t.copy_(s)
        for c in calls[1:]:
            for t in c.result:
                t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = list(tensors[:4]) + [t for c in calls[1:] for t in c.result]
        for i, (g, w) in enumerate(zip(got, want)):
            assert torch.equal(g, w), (turn, i)


@pytest.mark.parametrize("new", [[1, 2, 1], [80, 1, 3]])
def test_graphs_that_share_scratch(new):
    """Two graphs whose calls have one scratch between them, replayed in turn."""
    rng = np.random.default_rng(79)
    scratch = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    calls = []
    for lens in ([500, 3000, 31], [90, 700, 2000]):
        pool = Pool(rng, "s8", lens, 2, 64, 64, 16, width=50)
        q, _ = bf16(rng.standard_normal((sum(new), 2 * 32, 64)))
        calls.append(ops.kv_cache_attention(q, *pool.device(), dev(offsets(new)), lse=True, scratch=scratch, build_only=True))
    want = []
    for c in calls:
        c.run()
        want.append([t.clone() for t in c.result])
    torch.cuda.synchronize()
    graphs = []
    side = torch.cuda.Stream()
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            c.run()
    for turn in range(4):
        for c in calls:
            for t in c.result:
                t.fill_(3)
        scratch.fill_(0xff if turn % 2 else 0)
        for g in graphs[::1 if turn % 2 else -1]:
            g.replay()
        torch.cuda.synchronize()
        for c, w in zip(calls, want):
            assert all(torch.equal(a, b) for a, b in zip(c.result, w))


def test_calls_from_two_threads():
    """Each thread with calls and a stream of its own."""
    rng = np.random.default_rng(83)
    work = []
    for new, lens in (([1, 1], [900, 4000]), ([50, 1], [300, 1000])):
        pool = Pool(rng, "f8", lens, 2, 64, 32, 8)
        q, _ = bf16(rng.standard_normal((sum(new), 2 * 64, 64)))
        call = ops.kv_cache_attention(q, *pool.device(), dev(offsets(new)), build_only=True)
        want = call.run().clone()
        work.append((call, want, []))
    torch.cuda.synchronize()

    def go(call, want, wrong):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                call.result.fill_(5)
                call.run()
                if not torch.equal(call.result, want):
                    wrong.append(1)
    threads = [threading.Thread(target=go, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not any(w[2] for w in work)


def test_calls_on_another_stream():
    rng = np.random.default_rng(71)
    pool = Pool(rng, "s8", [500, 40], 2, 64, 16, 4)
    q, _ = bf16(rng.standard_normal((2, 4, 64)))
    tensors, off = pool.device(), dev(offsets([1, 1]))
    want = ops.kv_cache_attention(q, *tensors, off)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.kv_cache_attention(q, *tensors, off)
    side.synchronize()
    assert torch.equal(got, want)


def test_a_module_that_names_the_calls():
    """The custom calls of an HLO module, the cache aliased with the results."""
    rng = np.random.default_rng(73)
    pool = Pool(rng, "s8", [50, 21], 2, 64, 16, 8)
    pages, width = pool.k.shape[0], pool.table.shape[1]
    text = """HloModule decode_step, entry_computation_layout={()->()}
ENTRY main {
  q = bf16[2,4,64] parameter(0)
  k = bf16[2,2,64] parameter(1)
  v = bf16[2,2,64] parameter(2)
  kc = s8[P,2,16,64] parameter(3)
  vc = s8[P,2,16,64] parameter(4)
  ks = f32[P,2,2] parameter(5)
  vs = f32[P,2,2] parameter(6)
  table = s32[2,W] parameter(7)
  lens = s32[2] parameter(8)
  off = s32[3] parameter(9)
  cache = (s8[P,2,16,64], s8[P,2,16,64], f32[P,2,2], f32[P,2,2]) custom-call(k, v, kc, vc, ks, vs, table, lens, off), custom_call_target="xla_amd.kv_cache_write", output_to_operand_aliasing={{0}: (2, {}), {1}: (3, {}), {2}: (4, {}), {3}: (5, {})}, api_version=API_VERSION_TYPED_FFI
  kc2 = s8[P,2,16,64] get-tuple-element(cache), index=0
  vc2 = s8[P,2,16,64] get-tuple-element(cache), index=1
  ks2 = f32[P,2,2] get-tuple-element(cache), index=2
  vs2 = f32[P,2,2] get-tuple-element(cache), index=3
  att = (bf16[2,4,64], f32[2,4], u8[65536]) custom-call(q, kc2, vc2, ks2, vs2, table, lens, off), custom_call_target="xla_amd.kv_cache_attention", api_version=API_VERSION_TYPED_FFI, backend_config="{causal = true, softmax_scale = 0.125 : f32, window = 30 : i64}"
  out = bf16[2,4,64] get-tuple-element(att), index=0
  lse = f32[2,4] get-tuple-element(att), index=1
  ROOT r = (bf16[2,4,64], f32[2,4], s8[P,2,16,64]) tuple(out, lse, kc2)
}
""".replace("P,", "%d," % pages).replace(",W]", ",%d]" % width)
    q, qf = bf16(rng.standard_normal((2, 4, 64)))
    k, kf = bf16(rng.standard_normal((2, 2, 64)))
    v, vf = bf16(rng.standard_normal((2, 2, 64)))
    tensors = pool.device()
    off = offsets([1, 1])
    (out, lse, kc), rewrites, _ = hlo_runner.compile_and_run(text, [q, k, v] + tensors + [dev(off)])
    assert not rewrites and kc.data_ptr() == tensors[0].data_ptr()
    pool.k, pool.ks = plain.write(kf, pool.k, pool.ks, "s8", pool.table, pool.lens, off)
    pool.v, pool.vs = plain.write(vf, pool.v, pool.vs, "s8", pool.table, pool.lens, off)
    assert np.array_equal(kc.cpu().numpy(), pool.k)
    want, want_lse = check_attention(pool, qf, off, scale=0.125, window=30)
    tol, tol_lse = plain.attention_tolerance(*plain.attention(qf, pool.k, pool.v, pool.ks, pool.vs, "s8", pool.table, pool.lens, off, 0.125,
                                                              window=30), 50)
    assert ((out - want).abs().double().cpu().numpy() <= 2 * tol).all()      # another scratch may split elsewhere
    assert ((lse - want_lse).abs().double().cpu().numpy() <= 2 * tol_lse).all()
