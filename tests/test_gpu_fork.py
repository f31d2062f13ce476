"""Sequences that become copies of others (``BatchedPagedKVCache.fork``), and what
shared pages mean for free and truncate, against a replay on the host: a LIFO
free list, a count of holders per page, and the staging rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(lens, layers=3, hkv=2, d=64, page=16, kv="int8", scales="page", staging=torch.float16, seed=0, extra=8):
    from metagross_b200.batched import BatchedPagedKVCache

    g = torch.Generator(device="cuda").manual_seed(seed)
    c = BatchedPagedKVCache(layers, len(lens), hkv, d, page_size=page, num_pages=sum(n // page for n in lens) + extra,
                            max_blocks=max(lens) // page + 4, kv_dtype=kv, scale_granularity=scales,
                            staging_dtype=staging)
    c.begin_step(torch.tensor(lens, dtype=torch.int32))
    T = max(max(lens), 1)
    for layer in range(layers):
        k, v = (torch.randn(len(lens), T, hkv, d, generator=g, device="cuda").to(staging) for _ in range(2))
        c.append(layer, k, v)
    c.check()
    return c


class Model:
    """The cache's tables, free list, holders and staging rows, on the host."""

    def __init__(self, c):
        self.c, self.P = c, c.page_size
        self.free = c.allocator.free_list()
        self.held = c.allocator.in_use.tolist()
        self.bt = c.block_tables.tolist()
        self.lens = c.seq_lens.tolist()
        self.st = {x: getattr(c, "staging_" + x).clone() for x in ("k", "v")}

    def release(self, s, keep=0):
        for j in range(keep, self.lens[s] // self.P):
            page = self.bt[s][j]
            self.held[page] -= 1
            if self.held[page] == 0:
                self.free.append(page)

    def fork(self, src, dst, lens=None):
        c, P = self.c, self.P
        want = [self.lens[s] if lens is None else lens[i] for i, s in enumerate(src)]
        for d in dst:
            self.release(d)
        for s, d, n in zip(src, dst, want):
            m, r = n // P, n % P
            for j in range(m):
                self.bt[d][j] = self.bt[s][j]
                self.held[self.bt[s][j]] += 1
            cut = m < self.lens[s] // P
            for x, st in self.st.items():
                if not cut:
                    st[:, d, :r] = st[:, s, :r]
                    continue
                page = self.bt[s][m]
                codes = getattr(c, x + "_pool")[:, page]
                if c.kv_dtype == "int4":
                    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int16)
                    codes = torch.where(codes > 7, codes - 16, codes)
                sc = getattr(c, x + "_scales")[:, page]
                sc = sc[..., None] if sc.dim() == 3 else sc[:, None, None, None]
                st[:, d, :r] = (codes.float() * sc).to(st.dtype)[:, :r]
            self.lens[d] = n

    def check(self):
        c = self.c
        torch.cuda.synchronize()
        c.check()
        assert c.seq_lens.tolist() == self.lens
        assert c.block_tables.tolist() == self.bt
        assert c.allocator.in_use.tolist() == self.held
        assert c.allocator.free_list() == self.free
        assert torch.equal(c.staging_k, self.st["k"]) and torch.equal(c.staging_v, self.st["v"])


CASES = [dict(kv="int8"), dict(kv="int4"), dict(kv="int8", d=128, hkv=3, page=24), dict(kv="int4", scales="token_head"),
         dict(kv="int8", scales="token_head", page=8), dict(kv="int8", staging=torch.float32),
         dict(kv="int4", staging=torch.float32, page=1), dict(kv="int8", page=64, layers=1)]


@pytest.mark.parametrize("case", CASES)
def test_whole_sequences_and_prefixes(case):
    lens = [100, 37, 0, 64, 16, 250, 3, 0]
    c = make(lens, **case)
    m = Model(c)
    for src, dst, cut in (([0], [2], None), ([5, 5, 0], [7, 3, 6], None), ([5, 0, 5], [7, 3, 2], [129, 95, 250]),
                          ([5, 5, 3], [6, 1, 7], [0, 15, 17]), ([4], [0], None), ([1, 3], [5, 2], [1, 16])):
        c.fork(src, dst, cut)
        m.fork(src, dst, cut)
        m.check()


def test_again_is_the_same_and_many_targets_on_device():
    lens = [333, 20, 150] + [40, 0, 17, 90] * 20
    c = make(lens, hkv=4)
    m = Model(c)
    dst = torch.arange(3, len(lens), dtype=torch.int32, device="cuda")
    src = (dst * 7 % 3).to(torch.int32)
    cut = torch.tensor([1 + (i * 37) % lens[s] for i, s in enumerate(src.tolist())], dtype=torch.int32, device="cuda")
    for lens_ in (None, cut, cut, None):
        c.fork(src, dst, lens_)
        m.fork(src.tolist(), dst.tolist(), None if lens_ is None else lens_.tolist())
        m.check()


def test_copies_attend_like_their_source_and_then_diverge():
    c = make([100, 0, 31, 0], layers=1, hkv=4, extra=24)
    c.fork([0, 2], [1, 3])
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(4, 8, 64, generator=g, device="cuda").half()
    q[1], q[3] = q[0], q[2]
    out = c.attend(0, q)
    assert torch.allclose(out[0], out[1], atol=1e-3) and torch.allclose(out[2], out[3], atol=1e-3)
    before = c.k_pool.clone()
    shared = c.block_tables[0, :6].tolist()
    for _ in range(20):  # both fill pages of their own
        c.begin_step(1)
        kv = torch.randn(2, 4, 4, 64, generator=g, device="cuda").half()
        c.append(0, kv[0], kv[1])
    torch.cuda.synchronize()
    c.check()
    assert c.block_tables[0, :6].tolist() == c.block_tables[1, :6].tolist() == shared
    assert torch.equal(c.k_pool[0, shared], before[0, shared])
    assert c.block_tables[0, 6] != c.block_tables[1, 6]
    assert not torch.equal(c.attend(0, q)[0], c.attend(0, q)[1])


@pytest.mark.parametrize("ids", [[0, 1, 2], [2, 0], [1, 1, 0, 2], [4, 3, 2, 1, 0]])
def test_free_returns_a_page_with_its_last_holder(ids):
    c = make([100, 0, 0, 64, 0])
    c.fork([0, 0, 3], [1, 2, 4])
    m = Model(c)
    c.free(ids)
    for s in ids:
        m.release(s)
        m.lens[s] = 0
    m.check()
    rest = [s for s in range(5) if s not in ids]
    c.free(rest)
    torch.cuda.synchronize()
    c.check()
    assert c.allocator.num_free == c.num_pages and not c.allocator.in_use.any()


def test_free_of_many_copies_is_in_list_order():
    """More pages than one round of the freeing kernel, held by many sequences."""
    n = 40
    c = make([1600] + [0] * n + [320], extra=4, layers=1)
    c.fork([0] * n, list(range(1, n + 1)))
    m = Model(c)
    ids = list(range(n + 1, -1, -1))
    c.free(ids)
    for s in ids:
        m.release(s)
        m.lens[s] = 0
    m.check()


def test_truncate_of_a_copy():
    c = make([100, 0])
    c.fork([0], [1])
    m = Model(c)
    c.truncate([32], [1])
    m.release(1, keep=2)
    m.lens[1] = 32
    m.check()
    c.truncate([32], [0])
    m.release(0, keep=2)
    m.lens[0] = 32
    m.check()


def test_bad_pairs_are_skipped_and_flagged():
    c = make([100, 40, 20, 0])
    m = Model(c)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for src, dst, lens, good in (([0, 9], [3, 2], None, [0]), ([0, 1], [-1, 3], None, [1]), ([0, 0], [1, 1], None, [0]),
                                 ([0, 2], [2, 3], None, [1]), ([0, 1], [2, 3], [101, 7], [1]),
                                 ([0, 1], [2, 3], [-1, 7], [1]), ([1, 0], [1, 3], None, [1])):
        c.fork(dev(src), dev(dst), None if lens is None else dev(lens))
        torch.cuda.synchronize()
        assert int(c.status.item()) == 0x80
        c.status.zero_()
        m.fork([src[i] for i in good], [dst[i] for i in good], None if lens is None else [lens[i] for i in good])
        m.check()


def test_a_page_that_is_already_free_is_flagged_and_stays_free_once():
    c = make([100, 40, 40])
    c.allocator.in_use[c.block_tables[1, 0].long()] = 0  # as if its holder had let it go
    page = int(c.block_tables[1, 0])
    c.fork([0], [1])
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0x4
    assert page not in c.allocator.free_list() and int(c.allocator.in_use[page]) == 0


def test_refusals():
    c = make([100, 40, 20, 0])
    with pytest.raises(ValueError, match="same length"):
        c.fork([0, 1], [3])
    with pytest.raises(ValueError, match=r"\[0, 4\)"):
        c.fork([0], [4])
    with pytest.raises(ValueError, match="target"):
        c.fork([0, 1], [3, 3])
    with pytest.raises(ValueError, match="target"):
        c.fork([0, 3], [3, 2])
    with pytest.raises(RuntimeError, match="one entry per pair"):
        c.fork([0, 1], [2, 3], [5])
    c.fork([], [])
    Model(c).check()
