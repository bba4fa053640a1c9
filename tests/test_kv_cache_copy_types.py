"""Page copies of every element type whose values fill whole bytes."""
import numpy as np
import pytest
import torch

from xla_amd import dtypes, ffi, ops

BYTES = {dtypes.PRED: 1, dtypes.S8: 1, dtypes.U8: 1, dtypes.F8E5M2: 1, dtypes.F8E4M3FN: 1, dtypes.F8E4M3B11FNUZ: 1,
         dtypes.F8E5M2FNUZ: 1, dtypes.F8E4M3FNUZ: 1, dtypes.F8E4M3: 1, dtypes.F8E3M4: 1, dtypes.F8E8M0FNU: 1, dtypes.S16: 2,
         dtypes.U16: 2, dtypes.F16: 2, dtypes.BF16: 2, dtypes.S32: 4, dtypes.U32: 4, dtypes.F32: 4, dtypes.S64: 8, dtypes.U64: 8,
         dtypes.F64: 8, dtypes.C64: 8, dtypes.C128: 16}


@pytest.mark.parametrize("dt", BYTES)
def test_every_type_is_taken(dt):
    """A call without moves ends before any launch."""
    buf = (dt, 0x1000, (4, 16))
    ffi.invoke("xla_amd.kv_cache_copy_pages", ffi.Frame(ffi.Host(), [(dtypes.S32, 0x1000, (0, 2)), buf], [buf]))


@pytest.mark.parametrize("dt", [dtypes.S4, dtypes.U4, 17, 26, 30, 32])
def test_types_of_part_of_a_byte_are_refused(dt):
    buf = (dt, 0x1000, (4, 16))
    with pytest.raises(ffi.FfiError, match="Wrong buffer dtype"):
        ffi.invoke("xla_amd.kv_cache_copy_pages", ffi.Frame(ffi.Host(), [(dtypes.S32, 0x1000, (0, 2)), buf], [buf]))


@pytest.mark.gpu
def test_pages_of_every_type():
    """Seven values a page, so that no page but C128's has a size that a wide access fits."""
    rng = np.random.default_rng(97)
    moves = torch.tensor([[0, 3], [4, 1]], dtype=torch.int32, device="cuda")
    host = [rng.integers(0, 2, (5, 7 * BYTES[k])).astype(np.uint8) for k in ops._ANY.values()]
    buffers = [torch.from_numpy(h).cuda().view(t) for h, t in zip(host, ops._ANY)]
    ops.kv_cache_copy_pages(moves, buffers)
    for h, b, t in zip(host, buffers, ops._ANY):
        h[3], h[1] = h[0], h[4]
        assert np.array_equal(b.view(torch.uint8).cpu().numpy(), h), t
