"""Drafted tokens through the model (``LlamaDecoder.verify``), forked samples
(``LlamaDecoder.fork``) and models that normalise q and k per head, on a small
random-init shape."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = dict(vocab=64, hidden=512, layers=2, heads=8, kv_heads=2, ffn=512)  # head_dim 64
B = 3


def decoder(qk_norm=False, kv="int8", batch=B, keep=False):
    from metagross_b200.llama import LlamaDecoder, LlamaShape

    return LlamaDecoder(LlamaShape(qk_norm=qk_norm, **SHAPE), batch=batch, max_len=96, kv_dtype=kv, seed=5,
                        keep_logits=keep)


def prompt(batch=B, n=21):
    return torch.randint(0, SHAPE["vocab"], (batch, n), generator=torch.Generator().manual_seed(9)).cuda()


@pytest.mark.parametrize("qk_norm", [False, True])
def test_right_guesses_are_accepted_and_wrong_ones_are_not(qk_norm):
    """Guesses taken from plain greedy decoding, on one branch of a tree whose other
    branches are wrong: the path is accepted as far as it goes inside one page (the two
    ways see the same exact rows there), and the cache ends as the plain one."""
    plain, d = decoder(qk_norm), decoder(qk_norm)
    plain.prefill(prompt())
    d.prefill(prompt())
    want = plain.decode(7)  # the pending token and six more: positions 21 .. 26, inside page 1
    #          0 pending; 1 wrong, 2 right; 3 under 1, 4 right under 2, 5 wrong under 2; 6 right under 4
    parents = [-1, 0, 0, 1, 2, 2, 4]
    tree = torch.empty(B, 7, dtype=torch.long, device="cuda")
    wrong = lambda t: (want[:, t] + 1) % SHAPE["vocab"]  # noqa: E731
    for i, col in enumerate([want[:, 0], wrong(1), want[:, 1], want[:, 2], want[:, 2], wrong(2), want[:, 3]]):
        tree[:, i] = col
    tokens, n = d.verify(tree, parents)
    d.cache.check()
    assert n.tolist() == [4] * B
    assert torch.equal(tokens[:, :4], want[:, :4])
    assert torch.equal(d.ids, want[:, 4]) and d.pos.tolist() == [25] * B
    assert d.cache.seq_lens.tolist() == [25] * B
    # nothing right: only the pending token is appended
    tree = torch.stack([want[:, 4], wrong(5), wrong(5)], 1)
    tokens, n = d.verify(tree, [-1, 0, 1])
    assert n.tolist() == [1] * B and torch.equal(d.ids, want[:, 5])
    for x in ("staging_k", "staging_v"):
        a, b = getattr(d.cache, x)[:, :, 5:10].float(), getattr(plain.cache, x)[:, :, 5:10].float()
        assert (a - b).abs().max() <= 2e-2 * b.abs().max()


def test_each_sequence_accepts_its_own_length():
    plain, d = decoder(), decoder()
    plain.prefill(prompt())
    d.prefill(prompt())
    want = plain.decode(6)
    tree = want[:, :5].clone()
    tree[1, 2] = (tree[1, 2] + 1) % SHAPE["vocab"]  # wrong from the second guess on
    tree[2, 1] = (tree[2, 1] + 1) % SHAPE["vocab"]
    tokens, n = d.verify(tree, [-1, 0, 1, 2, 3])
    d.cache.check()
    assert n.tolist() == [5, 2, 1]
    assert d.ids.tolist() == [int(want[0, 5]), int(want[1, 2]), int(want[2, 1])]
    assert d.cache.seq_lens.tolist() == [26, 23, 22] == d.pos.tolist()


def test_a_long_run_of_verified_steps():
    """Steps that cross pages: every appended token is the greedy continuation of what
    is in the cache (checked by the next step's own prediction)."""
    d = decoder(kv="int4")
    d.prefill(prompt())
    g = torch.Generator(device="cuda").manual_seed(1)
    total = torch.full((B,), 21, device="cuda")
    for _ in range(20):
        tree = torch.randint(0, SHAPE["vocab"], (B, 6), generator=g, device="cuda")
        tree[:, 0] = d.ids
        _, n = d.verify(tree, [-1, 0, 0, 1, 1, 2])
        total += n
    d.cache.check()
    assert torch.equal(d.cache.seq_lens.long(), total) and torch.equal(d.pos, total)


def test_qk_norm_step_matches_dense_attention_over_the_cache():
    from test_gpu_llama import _reference_logits

    d = decoder(qk_norm=True, keep=True)
    d.prefill(prompt())
    for _ in range(3):
        ids, pos = d.ids.clone(), d.pos.clone()
        d._step()
        d.cache.check()
        ref = _reference_logits(d, ids, pos)
        err = (d.logits.float() - ref).abs().max().item()
        assert err <= 2e-2 * ref.abs().max().item() + 1e-3, err


def test_forked_samples_continue_as_their_source():
    d = decoder(batch=4)
    d.prefill(prompt(4))
    used = d.cache.allocator.num_used
    d.fork([0, 0], [2, 3])
    assert d.cache.allocator.num_used == used - 2  # one page each before, now shared
    d.capture()
    out = d.decode(30)
    d.cache.check()
    assert torch.equal(out[0], out[2]) and torch.equal(out[0], out[3])
    d.cache.free([0, 1, 2, 3])
    assert d.cache.allocator.num_free == d.cache.num_pages
