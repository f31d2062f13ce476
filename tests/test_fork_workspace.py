"""The workspace of ``BatchedPagedKVCache.fork``: a captured fork keeps its address, so it must not move."""
import pytest
import torch

from metagross_b200 import batched


class Recorder:
    """Stands in for the compiled calls: notes the workspace that each fork was given."""

    def __init__(self):
        self.seen = []

    def fork_workspace_bytes(self, n):
        return 4 * (2 + n)

    def fork_sequences(self, *args):
        self.seen.append(args[-2])


@pytest.fixture
def cache(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(batched, "_get_C", lambda: rec)

    class Allocator:
        def __init__(self, n, device):
            self.free_stack = self.n_free = self.in_use = torch.zeros(n, dtype=torch.int32)

    monkeypatch.setattr(batched, "DeviceBlockAllocator", Allocator)
    return batched.BatchedPagedKVCache(1, 9, 2, 64, num_pages=8, max_blocks=4, device="cpu"), rec.seen


def test_it_stays_where_it_is(cache):
    c, seen = cache
    first = None
    for dst in ([1], [1, 2, 3], list(range(1, 9)), [4]):
        c.fork([0] * len(dst), dst)
        first = first or seen[0].data_ptr()
        assert seen[-1].data_ptr() == first and seen[-1].numel() >= 2 + len(dst)


def test_more_pairs_than_sequences_have_one_of_their_own(cache):
    """Some of them are skipped, but the call is valid; it must not take the fixed one's place."""
    c, seen = cache
    c.fork([0], [1])
    c._fork([0] * 30, [1] * 30, None)
    assert seen[1].numel() >= 32 and not seen[1].any() and seen[1].data_ptr() != seen[0].data_ptr()
    c.fork([0], [1])
    assert seen[2].data_ptr() == seen[0].data_ptr()


@pytest.mark.gpu
def test_a_captured_fork_replays_after_larger_ones():
    from test_gpu_fork import Model, make

    c = make([100, 40, 20, 64, 0, 33])
    m = Model(c)
    src, dst = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.fork(src, dst)
    m.check()
    for s, d in (([0, 0, 1], [3, 4, 5]), ([3] * 5, [0, 1, 2, 4, 5])):
        c.fork(s, d)
        m.fork(s, d)
        m.check()
        other = torch.full((64,), 7, dtype=torch.int32, device="cuda")  # takes what the allocator has free
        graph.replay()
        m.fork([0], [2])
        m.check()
        assert (other == 7).all()
    c.fork(torch.zeros(20, dtype=torch.int32, device="cuda"), torch.full((20,), 1, dtype=torch.int32, device="cuda"))
    m.fork([0], [1])
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0x80  # the 19 that name the same target again
    c.status.zero_()
    m.check()
    graph.replay()
    m.fork([0], [2])
    m.check()
