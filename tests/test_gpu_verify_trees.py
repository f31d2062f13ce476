"""What ``LlamaDecoder.verify`` and ``LlamaDecoder.fork`` refuse, skip and report, and verified steps that
cross pages against a plain torch form of the same step."""
import pytest
import torch

from test_gpu_verify import B, SHAPE, decoder, prompt

pytestmark = pytest.mark.gpu


def test_a_second_root_is_refused():
    """A token without a parent would have nothing to be checked against: only column 0 is one."""
    d = decoder()
    d.prefill(prompt())
    ids, lens = d.ids.clone(), d.cache.seq_lens.clone()
    tree = torch.zeros(B, 3, dtype=torch.long, device="cuda")
    tree[:, 0] = d.ids
    for parents in ([-1, -1, 1], [-1, 0, -5], [[-1, 0, 1], [-1, 0, 0], [-1, -1, 0]]):
        for p in (parents, torch.tensor(parents), torch.tensor(parents, device="cuda")):
            with pytest.raises(ValueError, match="column 0"):
                d.verify(tree, p)
    assert torch.equal(d.ids, ids) and torch.equal(d.cache.seq_lens, lens)


def test_parents_of_another_shape_are_refused():
    d = decoder()
    d.prefill(prompt())
    tree = torch.zeros(B, 3, dtype=torch.long, device="cuda")
    for parents in ([-1], [-1, 0], [-1, 0, 1, 2], [[-1, 0, 1]] * (B + 1), [[-1]] * B, [[[-1, 0, 1]] * B]):
        with pytest.raises(ValueError, match="parents must be"):
            d.verify(tree, parents)
    assert d.cache.seq_lens.tolist() == [21] * B
    for parents in ([-1, 0, 1], [[-1, 0, 1]], [[-1, 0, 1]] * B):
        d.verify(tree, parents)
    d.cache.check()


@pytest.mark.parametrize("captured", [False, True])
def test_a_normed_decoder_past_its_tables_is_reported(captured):
    d = decoder(qk_norm=True)  # up to 96 tokens
    d.prefill(prompt(n=90))
    if captured:
        d.capture()
    d.decode(7)  # six steps: positions 90 .. 95
    d.cache.check()
    d.decode(2)
    with pytest.raises(RuntimeError, match="argument"):
        d.cache.check()


def four():
    """Four sequences of different lengths and pending tokens."""
    d = decoder(batch=4)
    d.prefill(prompt(4, n=40))
    d.cache.truncate([32, 16], [1, 2])
    d.pos.copy_(d.cache.seq_lens)
    d.ids.copy_(torch.tensor([11, 12, 13, 14], device="cuda"))
    return d


def same(d, ids, lens):
    assert d.ids.tolist() == ids and d.pos.tolist() == lens and d.cache.seq_lens.tolist() == lens


def test_fork_copies_what_the_cache_copies():
    """Device ids: a pair that the cache skips moves neither the position nor the pending token."""
    dev = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    d = four()
    d.fork(dev(0, 2), dev(2, 3))  # 2 is a source: only the second pair
    same(d, [11, 12, 13, 13], [40, 32, 16, 16])
    d = four()
    d.fork(dev(0, 1), dev(3, 3))  # 3 twice: the first pair
    same(d, [11, 12, 13, 11], [40, 32, 16, 40])
    d = four()
    d.cache.status.fill_(0x1)  # a refused step: nothing is done
    d.fork(dev(0), dev(1))
    same(d, [11, 12, 13, 14], [40, 32, 16, 40])


def test_fork_skips_ids_out_of_range():
    dev = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    d = four()
    d.fork(dev(9, 0, -1, 1, 0), dev(2, 3, 3, 70000, -2))
    same(d, [11, 12, 13, 11], [40, 32, 16, 40])
    with pytest.raises(RuntimeError, match="argument"):
        d.cache.check()


def test_drafts_may_be_a_view_of_the_pending_tokens():
    d = decoder()
    d.prefill(prompt())
    for _ in range(4):
        pending = d.ids.clone()
        tokens, n = d.verify(d.ids[:, None], [-1])
        assert torch.equal(tokens[:, 0], pending) and (n == 1).all()
        assert not torch.equal(d.ids, pending)
