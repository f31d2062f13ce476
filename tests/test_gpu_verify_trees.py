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
