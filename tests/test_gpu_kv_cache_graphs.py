"""Book-keeping and the copies that it asks for, captured into one graph."""
import numpy as np
import pytest
import torch

from oracle import kv_cache as plain
from tests.test_gpu_kv_cache import dev, random_book
from xla_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["COMPACT", "FORK"])
def test_moves_and_their_copies_replay_from_one_graph(op):
    """Every replay has other books, so other moves, and pages of its own content; its results are the eager ones, with eager
    work and a synchronisation between the replays."""
    rng = np.random.default_rng(101)
    batch, width, pages, page = 40, 12, 500, 16
    books = []
    for _ in range(5):
        table, lens, refs = random_book(rng, batch, width, pages, page, 0.6)
        request = np.stack([rng.integers(0, batch, 30), rng.permutation(batch)[:30]], 1).astype(np.int32)
        books.append((table, lens, refs, request))
    state = [dev(x) for x in books[0]]
    buffers = [torch.empty((pages, 2, 1000), dtype=torch.int32, device="cuda"), torch.empty((pages, 33), dtype=torch.uint8, device="cuda")]
    book = ops.kv_cache_pages(op, *state[:3], state[3] if op == "FORK" else None, page_size=page, build_only=True)
    copy = ops.kv_cache_copy_pages(book.result[3], buffers, build_only=True)

    def fill(turn):
        for t, x in zip(state, books[turn]):
            t.copy_(torch.from_numpy(x))
        for i, b in enumerate(buffers):
            n = b.numel()
            b.copy_(((torch.arange(n, device="cuda") * (7 + turn) + i) % 251).to(b.dtype).view(b.shape))
    fill(0)
    book.run()
    copy.run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        book.run()
        copy.run()
    lists = set()
    for turn in (0, 1, 2, 3, 4, 1):
        fill(turn)
        book.run()
        copy.run()
        torch.cuda.synchronize()
        want = [t.clone() for t in list(book.result) + buffers]
        for got, w in zip(want, plain.pages(op, *books[turn][:3], books[turn][3], page)):
            assert np.array_equal(got.cpu().numpy(), w)
        fill(turn)
        for t in book.result:
            t.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        for i, (got, w) in enumerate(zip(list(book.result) + buffers, want)):
            assert torch.equal(got, w), (turn, i)
        moved = want[3][want[3][:, 0] >= 0].long()
        assert len(moved) > 3
        fill(turn)
        for got, b in zip(want[5:], buffers):
            b[moved[:, 1]] = b[moved[:, 0]]
            assert torch.equal(got, b)
        lists.add(tuple(moved.flatten().tolist()))
    assert len(lists) == 5
