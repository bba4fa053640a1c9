"""The calls over the 8-bit paged cache without a GPU: what they refuse, before any launch, and the plain
restatement that the GPU tests compare with, on cases worked out by hand."""
import numpy as np
import pytest
import torch

from oracle import kv_cache as plain
from xla_amd import dtypes, ffi, ops

FAKE = 0x1000
S8, F8, F32, S32, BF16, U8 = dtypes.S8, dtypes.F8E4M3FN, dtypes.F32, dtypes.S32, dtypes.BF16, dtypes.U8


def cache(pages=4, heads=2, page=16, head=32, block=8, batch=3, width=5, dt=S8, ptr=FAKE):
    codes, scales = (dt, ptr, (pages, heads, page, head)), (F32, ptr, (pages, heads, page // block))
    return [codes, codes, scales, scales, (S32, ptr, (batch, width)), (S32, ptr, (batch,)), (S32, ptr, (batch + 1,))]


def write_frame(c, k=None, rets=None):
    k = k or (BF16, FAKE, (7, c[0][2][1], c[0][2][3]))
    return ffi.Frame(ffi.Host(), [k, k] + c, c[:4] if rets is None else rets)


def refused(target, frame, match):
    with pytest.raises(ffi.FfiError, match=match) as e:
        ffi.invoke(target, frame)
    assert e.value.code == 3


@pytest.mark.parametrize("change, match", [
    (dict(page=8), "page size must be a power of two from 16 to 1024"),
    (dict(page=48, block=16), "page size must be a power of two"),
    (dict(page=2048, block=16), "page size must be a power of two"),
    (dict(page=64, block=12), r"scales must be \[pages,kv_heads,page/block\]"),
    (dict(head=24), "head size must be a multiple of 16 from 16 to 256"),
    (dict(head=272), "head size must be a multiple of 16 from 16 to 256"),
    (dict(dt=U8), "Wrong buffer dtype: expected S8|F8E4M3FN but got U8"),
    (dict(batch=(1 << 20) + 1), "at most"),
    (dict(width=1 << 28), "2\\^31 positions"),
    (dict(ptr=FAKE + 8), "caches must be aligned to 16 bytes"),
    (dict(ptr=None), "null"),
])
def test_sizes_that_a_cache_cannot_have(change, match):
    refused("xla_amd.kv_cache_write", write_frame(cache(**change)), match)


def test_write_refuses_other_operands():
    c = cache()
    refused("xla_amd.kv_cache_write", write_frame(c, k=(BF16, FAKE, (7, 2, 48))), r"k and v must be \[rows,kv_heads,head\]")
    refused("xla_amd.kv_cache_write", write_frame(c, k=(BF16, FAKE, (7, 3, 32))), r"k and v must be \[rows,kv_heads,head\]")
    refused("xla_amd.kv_cache_write", write_frame(c, k=(F32, FAKE, (7, 2, 32))), "Wrong buffer dtype: expected BF16 but got F32")
    refused("xla_amd.kv_cache_write", write_frame(c, k=(BF16, FAKE + 2, (7, 2, 32))), "k and v must be aligned")
    refused("xla_amd.kv_cache_write", write_frame(c, k=(BF16, None, (7, 2, 32))), "null k or v")
    refused("xla_amd.kv_cache_write", write_frame(c, k=(BF16, FAKE, ((1 << 24) + 1, 2, 32))), "2\\^24 rows")
    other = [(dt, FAKE + 16, dims) for dt, _, dims in c[:4]]
    refused("xla_amd.kv_cache_write", write_frame(c, rets=other), "own buffers")
    refused("xla_amd.kv_cache_write", write_frame(c, rets=c[:3]), "Wrong number of results")
    bad = list(c)
    bad[1] = (S8, FAKE, (5, 2, 16, 32))
    refused("xla_amd.kv_cache_write", write_frame(bad), "k_cache and v_cache must have one shape and type")
    bad = list(c)
    bad[5] = (S32, FAKE, (2,))
    refused("xla_amd.kv_cache_write", write_frame(bad), "kv_lens must have one entry per row of page_table")
    bad = list(c)
    bad[6] = (S32, FAKE, (3,))
    refused("xla_amd.kv_cache_write", write_frame(bad), "q_offsets must have one entry more")


def test_attention_refuses():
    c = cache()
    t = "xla_amd.kv_cache_attention"

    def frame(q=(BF16, FAKE, (7, 6, 32)), rets=None, attrs=None, c=c):
        return ffi.Frame(ffi.Host(), [q] + c, [q] if rets is None else rets, attrs or {})
    refused(t, frame(q=(BF16, FAKE, (7, 5, 32))), "q_heads a multiple of kv_heads")
    refused(t, frame(q=(BF16, FAKE, (7, 6, 48))), "q must be")
    refused(t, frame(rets=[(BF16, FAKE, (7, 6, 48))]), "out must have the shape of q")
    refused(t, frame(rets=[(BF16, FAKE, (7, 6, 32)), (F32, FAKE, (7, 5))]), r"lse must be \[rows,q_heads\]")
    refused(t, frame(rets=[(BF16, FAKE, (7, 6, 32)), (U8, FAKE, (64,)), (F32, FAKE, (7, 6))]), r"results are out\[, lse\]\[, scratch\]")
    refused(t, frame(attrs={"window": ffi.Attr.i64(-1)}), "window must not be negative")
    refused(t, frame(attrs={"window": ffi.Attr.i64(4), "causal": ffi.Attr.pred(False)}), "a window needs causal")
    refused(t, frame(attrs={"softcap": ffi.Attr.f32(-1.0)}), "softcap must be")
    refused(t, frame(attrs={"softcap": ffi.Attr.f32(float("nan"))}), "softcap must be")
    refused(t, frame(attrs={"softmax_scale": ffi.Attr.f32(float("inf"))}), "softmax_scale must be a number")
    refused(t, frame(attrs={"causal": ffi.Attr.i64(1)}), "Wrong scalar data type: expected PRED")
    refused(t, frame(q=(BF16, FAKE + 8, (7, 6, 32))), "aligned to 16 bytes")
    refused(t, frame(q=(BF16, None, (7, 6, 32))), "null q or out")


def test_keys_and_values_in_one_buffer():
    refused("xla_amd.kv_cache_write", write_frame(cache()), "buffers of their own")


def test_sizes_that_a_grid_cannot_hold():
    c = cache()
    q = (BF16, FAKE, ((1 << 22) + 1, 128, 32))
    refused("xla_amd.kv_cache_attention", ffi.Frame(ffi.Host(), [q] + c, [q], {}), "2\\^29 rows times heads")
    refused("xla_amd.kv_cache_write", write_frame(c, k=(BF16, FAKE, (1 << 24, 2, 32))), "fewer than 2\\^24 rows")


def pages_frame(op="FREE", batch=3, width=5, pages=8, request=(S32, FAKE, (2,)), moves=0, status=2, page=16, scratch=1 << 20,
                new=2 * FAKE, shapes=None):
    state = [(S32, FAKE, (batch, width)), (S32, FAKE, (batch,)), (S32, FAKE, (pages,))]
    rets = [(S32, new, d) for _, _, d in state] if shapes is None else shapes
    rets = rets + [(S32, 3 * FAKE, (moves, 2)), (S32, 4 * FAKE, (status,)), (U8, 5 * FAKE, (scratch,))]
    return ffi.Frame(ffi.Host(), state + ([request] if request else []), rets,
                     {"op": ffi.Attr.str(op), "page_size": ffi.Attr.i64(page)})


@pytest.mark.parametrize("change, match", [
    (dict(op="GROW"), "Unknown op `GROW`"),
    (dict(op="COMPACT", moves=4, status=0), "a request goes with RESERVE, FORK and FREE"),
    (dict(request=None, status=0), "a request goes with"),
    (dict(op="RESERVE"), r"the request of RESERVE must be \[batch\]"),
    (dict(op="FORK"), r"the request of FORK must be \[n,2\]"),
    (dict(op="FORK", request=(S32, FAKE, (2, 2)), moves=1), "moves must be"),
    (dict(op="COMPACT", request=None, moves=8, status=0), "moves must be"),
    (dict(status=3), "status must have one entry per request"),
    (dict(page=0), "page_size must be"),
    (dict(scratch=16), "scratch must hold"),
    (dict(new=FAKE), "buffers other than the old one's"),
    (dict(shapes=[(S32, FAKE, (3, 4)), (S32, FAKE, (3,)), (S32, FAKE, (8,))]), "the old ones' shapes"),
    (dict(request=(dtypes.S64, FAKE, (2,))), "Wrong buffer dtype: expected S32 but got S64"),
])
def test_pages_refuses(change, match):
    refused("xla_amd.kv_cache_pages", pages_frame(**change), match)


def test_copy_pages_refuses():
    t = "xla_amd.kv_cache_copy_pages"
    a, b, moves = (S8, FAKE, (4, 16)), (F32, FAKE, (5, 3)), (S32, FAKE, (2, 2))
    run = lambda args, rets: ffi.Frame(ffi.Host(), args, rets)
    refused(t, run([moves, a, b], [a, b]), "same number of pages")
    refused(t, run([moves, a], [a, a]), "one result per buffer")
    refused(t, run([moves, a], [(S8, FAKE + 16, (4, 16))]), "own buffers")
    refused(t, run([(S32, FAKE, (2, 3)), a], [a]), r"moves must be \[m,2\]")
    refused(t, run([moves, (dtypes.S4, FAKE, (4, 16))], [(dtypes.S4, FAKE, (4, 16))]), "Wrong buffer dtype")
    refused(t, run([moves] + [a] * 65, [a] * 64), "Wrong number of arguments")


def test_python_wrappers_refuse_what_a_frame_cannot_say():
    t = torch.zeros((4, 2, 16, 32), dtype=torch.int8)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.kv_cache_copy_pages(torch.zeros((1, 2), dtype=torch.int32), [t])
    with pytest.raises(ValueError, match="must be contiguous"):
        ops._operand(t.transpose(1, 2), "k_cache", ops._CACHE, 4)
    with pytest.raises(ValueError, match="must have 4 dimensions"):
        ops._operand(t[0], "k_cache", ops._CACHE, 4)
    with pytest.raises(TypeError, match="element type torch.int16"):
        ops._operand(t.to(torch.int16), "k_cache", ops._CACHE, 4)
    with pytest.raises(TypeError, match="scratch: element type torch.float32"):
        ops._operand(torch.zeros(4), "scratch", {torch.uint8: U8, torch.int8: S8}, 1)
    with pytest.raises(ValueError, match="op must be RESERVE"):
        ops.kv_cache_pages("reserve", None, None, None, page_size=16)


# ---- the restatement itself ------------------------------------------------------------------------

def test_plain_write_by_hand():
    codes, scales = np.zeros((2, 1, 16, 16), np.int8), np.zeros((2, 1, 2), np.float32)
    x = np.zeros((1, 1, 16), np.float32)
    x[0, 0, 0], x[0, 0, 1] = 254.0, -1.0
    table = np.array([[1]], np.int32)
    codes, scales = plain.write(x, codes, scales, "s8", table, [1], [0, 1])
    assert scales[1, 0, 0] == 2.0 and codes[1, 0, 0, 0] == 127
    assert codes[1, 0, 0, 1] == 0   # -0.5 goes to the even code
    # a larger row in the same block doubles the scale: 127 * 0.5 = 63.5 goes to 64
    x[0, 0, 0], x[0, 0, 1] = 508.0, 0.0
    codes, scales = plain.write(x, codes, scales, "s8", table, [2], [0, 1])
    assert scales[1, 0, 0] == 4.0 and codes[1, 0, 0, 0] == 64 and codes[1, 0, 1, 0] == 127
    # a smaller one keeps it
    x[0, 0, 0] = 4.0
    codes, scales = plain.write(x, codes, scales, "s8", table, [3], [0, 1])
    assert scales[1, 0, 0] == 4.0 and codes[1, 0, 2, 0] == 1 and not scales[0].any()


def test_plain_attention_by_hand():
    k = np.zeros((1, 1, 16, 16), np.int8)
    v = np.zeros_like(k)
    k[0, 0, 0, 0], v[0, 0, 0, 0], v[0, 0, 1, 0] = 1, 10, 20
    one = np.ones((1, 1, 16), np.float32)
    q = np.zeros((2, 1, 16), np.float32)
    q[:, 0, 0] = np.log(3.0)
    out, lse = plain.attention(q, k, v, one, one, "s8", np.array([[0]]), [2], [0, 2], 1.0)[:2]
    assert np.allclose(out[:, 0, 0], [10.0, 12.5])      # weights 1, then 3/4 and 1/4
    assert np.allclose(lse[:, 0], [np.log(3.0), np.log(4.0)])
    out, lse = plain.attention(q, k, v, one, one, "s8", np.array([[0]]), [2], [0, 2], 1.0, window=1)[:2]
    assert np.allclose(out[:, 0, 0], [10.0, 20.0])
    out, lse = plain.attention(q, k, v, one, one, "s8", np.array([[-1]]), [2], [0, 2], 1.0)[:2]
    assert not out.any() and np.isneginf(lse).all()


def test_plain_pages_by_hand():
    table = np.array([[3, 5, -1], [-1, -1, -1], [1, -1, -1]], np.int32)
    lens, refs = np.array([20, 0, 16], np.int32), np.array([0, 1, 0, 1, 0, 1], np.int32)
    t, n, r, m, s = plain.pages("RESERVE", table, lens, refs, np.array([33, 5, 15], np.int32), 16)
    assert t.tolist() == [[3, 5, 0], [2, -1, -1], [1, -1, -1]] and n.tolist() == [33, 5, 16]
    assert r.tolist() == [1, 1, 1, 1, 0, 1] and s.tolist() == [1, 1, 0]
    t, n, r, m, s = plain.pages("FORK", table, lens, refs, np.array([[0, 1], [2, 1]], np.int32), 16)
    assert t[1].tolist() == [3, 0, -1] and r.tolist() == [1, 1, 0, 2, 0, 1] and m.tolist() == [[5, 0], [-1, -1]]
    assert s.tolist() == [1, 0] and n.tolist() == [20, 20, 16]
    t, n, r, m, s = plain.pages("FREE", table, lens, refs, np.array([0, 0, 7], np.int32), 16)
    assert t[0].tolist() == [-1, -1, -1] and r.tolist() == [0, 1, 0, 0, 0, 0] and s.tolist() == [1, 0, 0]
    t, n, r, m, s = plain.pages("COMPACT", table, lens, refs, None, 16)
    assert t.tolist() == [[0, 2, -1], [-1, -1, -1], [1, -1, -1]] and m.tolist() == [[3, 0], [5, 2], [-1, -1]]
    assert r.tolist() == [1, 1, 1, 0, 0, 0]


def test_scratch_sizes():
    L = ffi.library()
    assert L.xla_amd_kv_cache_pages_workspace_bytes(3, 8, 2) >= 3 * 8 * 4
    assert L.xla_amd_kv_cache_pages_workspace_bytes(-1, 8, 2) == 0
    size = L.xla_amd_kv_cache_attention_workspace_bytes
    assert size(0, 0, 8, 8, 128, 0) == 0
    # the pieces are as many as the device takes at a time, however long the cache or the prompt
    assert size(1, 1, 64, 8, 128, 1 << 24) <= 512 * 2 * 16 * (130 * 4 + 1)
    assert size(1 << 16, 4, 64, 8, 128, 1 << 24) <= 512 * 2 * 32 * (130 * 4 + 1) + 1024 * 128 * (130 * 4 + 1)
