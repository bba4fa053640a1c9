"""The calls over the 8-bit paged key/value cache at the ends of what their definition takes: caps of every size, scales
and scores far from 1, windows and tables of 2^31 positions."""
import numpy as np
import pytest
import torch

from oracle import kv_cache as plain
from tests.test_gpu_kv_cache import KINDS, Pool, bf16, dev, offsets
from xla_amd import ffi, ops

pytestmark = pytest.mark.gpu

# one row and a few heads: the streaming kernel; 64 rows of 64 heads: the prompts' kernel
BOTH = [(1, 3), (64, 64)]


def own_position(kind, new, group, **kw):
    """Rows that see their own position alone (a window of 1): (got, scores, their sizes), where the log-sum-exp is the
    row's score itself and the result the position's value.  Scores of 1e-3 to 1e3 times the usual."""
    rng = np.random.default_rng(new + group)
    pool = Pool(rng, kind, [new + 40], 2, 128, 64, 16)
    pool.ks *= np.exp(rng.uniform(np.log(1e-3), np.log(1e3), pool.ks.shape)).astype(np.float32)
    q = rng.standard_normal((new, 2 * group, 128)) * np.exp(rng.uniform(-3, 1, (new, 2 * group, 1)))
    q[:, 0] = 0.0
    q, qf = bf16(q)
    scale = np.float32(kw.pop("scale", 128 ** -0.5))
    out, lse = ops.kv_cache_attention(q, *pool.device(), dev(offsets([new])), scale=float(scale), window=1, lse=True, **kw)
    assert ffi.last_kernel().startswith("kv_cache_attention_prompt") == (new > 1)
    j = 40 + np.arange(new)
    page, row = pool.table[0, j // 64], j % 64
    k, v = (plain.values(c[page, :, row], kind).astype(np.float64) * s[page, :, row // 16].astype(np.float64)[:, :, None]
            for c, s in ((pool.k, pool.ks), (pool.v, pool.vs)))
    k, v = (x.repeat(group, 1) for x in (k, v))
    got = out.float().cpu().numpy().astype(np.float64)
    # the weight is 1, its value's scale rounded to f16 (2^-11), the result to bf16 (2^-8)
    fine = np.abs(got - v) <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -20) * 1.01 * np.abs(v) + 1e-37
    x = (qf.astype(np.float64) * k).sum(-1) * float(scale)
    # a score whose multiple by log2 e = 1.4427 passes f32's largest number, 3.4028e38, is infinite, and the row no number
    held = np.abs(x) < 3.4e38 / 1.4427
    assert fine[held].all(), (int((~fine[held]).sum()), int((~held).sum()))
    return lse.cpu().numpy().astype(np.float64)[held], x[held], (np.abs(qf) * np.abs(k)).sum(-1)[held] * abs(float(scale))


CAPS = [1e-40, 1e-6, 0.3, 3.0, 50.0, 1e3, 1e4, 1e5, 1e6, 1e7, 1e8, 1e9, 1e20, 3.3e38]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, group", BOTH)
@pytest.mark.parametrize("cap", CAPS)
def test_caps_of_every_size(kind, new, group, cap):
    """A capped score is off by its product's f32 sum (136 roundings of its size; tanh is no steeper than 1) and, relative to
    itself, by: the argument's three roundings, 3 * 2^-24 at most, the exponential, the sum and the reciprocal,
    2.5 * 2^-23 of 1 - tanh, which is 1.16 tanh at most where they are used (from cap / 2 on), the polynomial below 2^-24, the
    factors cap, log2 e and log 2 and their products 5 * 2^-24: less than 2^-20 together."""
    got, x, size = own_position(kind, new, group, softcap=cap)
    c = float(np.float32(cap))
    want = c * np.tanh(x / c)
    tol = (128 + 8) * 2.0 ** -24 * size + 2.0 ** -20 * np.abs(want) + 1e-37
    off = np.abs(got - want)
    assert (off <= tol).all(), ((off / tol).max(), off.max(), want.flat[(off / tol).argmax()])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, group", [(3, 4), (130, 32)])
@pytest.mark.parametrize("cap", [0.5, 8.0, 1e3, 1e4, 1e6, 1e8])
def test_attention_under_caps_of_every_size(kind, new, group, cap):
    """Against the formula; the room that the uncapped scores have, (head + 8) 2^-24 of the product's size and more, is above
    4 * 2^-20 of a score, so a quarter more covers the cap's 2^-20."""
    rng = np.random.default_rng(new)
    pool = Pool(rng, kind, [new + 300, 70], 2, 64, 32, 8)
    q, qf = bf16(rng.standard_normal((new + 1, 2 * group, 64)) * 4)
    off, scale = offsets([new, 1]), np.float32(64 ** -0.5)
    out, lse = ops.kv_cache_attention(q, *pool.device(), dev(off), softcap=cap, lse=True)
    assert ffi.last_kernel().startswith("kv_cache_attention_prompt") == (new == 130)
    args = (qf, pool.k, pool.v, pool.ks, pool.vs, kind, pool.table, pool.lens, off, scale)
    ref, ref_lse, spread, _, largest = plain.attention(*args, softcap=float(np.float32(cap)))
    slack = plain.attention(*args)[3]
    tol, tol_lse = plain.attention_tolerance(ref, ref_lse, spread, 1.25 * slack, largest, int(pool.lens.max()))
    assert (np.abs(out.float().cpu().numpy() - ref) <= tol).all()
    assert (np.abs(lse.cpu().numpy() - ref_lse) <= tol_lse).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group", [2, 64])
@pytest.mark.parametrize("block", [16, 1])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_key_scale_that_is_no_number(kind, group, block, cap, bad):
    """It reaches the result and the lse of the rows that see it, whatever the sign of their products, and no others."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, kind, [64], 1, 128, 64, block)
    pool.ks[pool.table[0, 0], 0, 32 // block] = bad    # positions from 32 on
    q = rng.standard_normal((64, group, 128))
    out, lse = ops.kv_cache_attention(bf16(q)[0], *pool.device(), dev(offsets([64])), lse=True, softcap=cap)
    assert ffi.last_kernel().startswith("kv_cache_attention_prompt") == (group == 64)
    assert torch.isnan(out[32:]).all() and torch.isnan(lse[32:]).all()
    assert torch.isfinite(out[:32]).all() and torch.isfinite(lse[:32]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, group", BOTH)
@pytest.mark.parametrize("scale", [-1e32, 1e30, 1e34])
def test_scores_of_every_size(kind, new, group, scale):
    """Scores far below -1e30 are scores: the row's sum is 1 and its lse the score, off by the product's f32 sum and, relative
    to itself, the scale, log2 e, log 2 and their products."""
    got, x, size = own_position(kind, new, group, scale=scale)
    assert (x < -1e31).any()
    tol = (128 + 8) * 2.0 ** -24 * size + 6 * 2.0 ** -24 * np.abs(x)
    assert (np.abs(got - x) <= tol).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new, group", BOTH)
@pytest.mark.parametrize("scale", [1.0, 1e6, 1e9, 1e12, 1e30])
def test_one_score_far_above_the_others(kind, new, group, scale):
    """Position 77's product is 2 q . 112 / 3 and the others' are below q . 112 / 3 at most, q being 1 or more: all
    weights but one are below e^-37, however large the scores are, and the result is that position's value."""
    rng = np.random.default_rng(9)
    pool = Pool(rng, kind, [400 + new], 2, 64, 64, 16)
    pool.k[:] = 0
    pool.ks[:] = 1 / 3
    pool.k[..., 0] = rng.integers(-112, 113, pool.k.shape[:3]) if kind == "s8" else rng.integers(0, 0x6e, pool.k.shape[:3])
    pool.k[pool.table[0, 1], :, 13, :2] = 112 if kind == "s8" else 0x6e    # 77; 112 either way
    q = np.zeros((new, 2 * group, 64))
    q[..., :2] = np.abs(rng.standard_normal((new, 2 * group, 1))) + 1
    q, qf = bf16(q)
    out, lse = ops.kv_cache_attention(q, *pool.device(), dev(offsets([new])), scale=scale, lse=True)
    assert ffi.last_kernel().startswith("kv_cache_attention_prompt") == (new > 1)
    v = plain.values(pool.v[pool.table[0, 1], :, 13], kind) * pool.vs[pool.table[0, 1], :, 0][:, None]
    v = v.repeat(group, 0)[None].astype(np.float64)
    got = out.float().cpu().numpy()
    # an f16 weight, a bf16 result, 464 weights of e^-37 times values up to 1.5 * 448 / 110
    assert (np.abs(got - v) <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -20) * 1.01 * np.abs(v) + 1e-12).all()
    x = 2 * qf[..., 0].astype(np.float64) * 112 * float(np.float32(1 / 3)) * float(np.float32(scale))
    assert (np.abs(lse.cpu().numpy() - x) <= 8 * 2.0 ** -24 * x).all()


@pytest.mark.parametrize("group", [1, 4])
def test_a_window_of_nearly_all_positions(group):
    """A table of 2^31 - 1040 positions and a window just below, more rows than positions: the first rows stand 5000 before
    the sequence, and such a position less the window does not fit 32 bits."""
    rng = np.random.default_rng(13)
    new, length, window = 6000, 1000, 2 ** 31 - 1045
    pool = Pool(rng, "s8", [length], 1, 16, 16, 16)
    tensors = pool.device()
    tensors[4] = torch.full((1, 2 ** 27 - 65), -1, dtype=torch.int32, device="cuda")
    tensors[4][:, :pool.table.shape[1]] = dev(pool.table)
    q, qf = bf16(rng.standard_normal((new, group, 16)))
    for scratch in ("auto", None):
        out, lse = ops.kv_cache_attention(q, *tensors, dev(offsets([new])), window=window, lse=True, scratch=scratch)
        assert ffi.last_kernel().startswith("kv_cache_attention_prompt")
        ref, ref_lse, spread, slack, largest = plain.attention(qf, pool.k, pool.v, pool.ks, pool.vs, "s8", pool.table, pool.lens,
                                                               offsets([new]), np.float32(0.25), window=window)
        tol, tol_lse = plain.attention_tolerance(ref, ref_lse, spread, slack, largest, length)
        assert (np.abs(out.float().cpu().numpy() - ref) <= tol).all()
        got = lse.cpu().numpy()
        assert np.isneginf(got[:5000]).all() and (np.abs(got[5000:] - ref_lse[5000:]) <= tol_lse[5000:]).all()
    # few rows for the streaming kernel, 1490 of them in front of the sequence
    out = ops.kv_cache_attention(q[:1500, :1].contiguous(), *tensors[:5], dev(np.array([10], np.int32)), dev(offsets([1500])), window=window)
    assert not ffi.last_kernel().startswith("kv_cache_attention_prompt")
    ref, ref_lse, spread, slack, largest = plain.attention(qf[:1500, :1], pool.k, pool.v, pool.ks, pool.vs, "s8", pool.table, [10],
                                                           offsets([1500]), np.float32(0.25), window=window)
    tol, _ = plain.attention_tolerance(ref, ref_lse, spread, slack, largest, 10)
    assert (np.abs(out.float().cpu().numpy() - ref) <= tol).all() and ref[-10:].all()
