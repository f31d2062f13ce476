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


def dense_step(d, drafts, mask, depth):
    """The verified step in plain torch, fp16 storage and fp32 attention over ``cache.gather``: the logits of every
    drafted token [B, T, vocab] and their K and V [layers, B, T, heads, D]."""
    s, c = d.s, d.cache
    T, rep = drafts.shape[1], s.heads // s.kv_heads
    pos = d.pos[:, None] + depth
    x = d.w["embed"][drafts]
    ks, vs = [], []
    for i in range(s.layers):
        q, k, v = d._qkv(i, d._rms(x, d.w[f"{i}.n1"]))
        q, k = d._rope(q, pos), d._rope(k, pos)
        ks.append(k)
        vs.append(v)
        kc, vc, cu = c.gather(i, dtype=torch.float32)
        o = torch.empty(q.shape, dtype=torch.float32, device=q.device)
        for b in range(c.batch):
            at = slice(int(cu[b]), int(cu[b + 1]))
            K, V = (torch.cat([y[at], z[b].float()]).repeat_interleave(rep, 1) for y, z in ((kc, k), (vc, v)))
            a = torch.einsum("thd,nhd->htn", q[b].float(), K) / s.head_dim ** 0.5
            a[:, :, K.shape[0] - T:].masked_fill_(~mask[b], float("-inf"))
            o[b] = torch.einsum("htn,nhd->thd", torch.softmax(a, -1), V)
        x = x + o.to(x.dtype).flatten(2) @ d.w[f"{i}.wo"]
        x = d._mlp(i, x)
    return d._logits(x).float(), torch.stack(ks), torch.stack(vs)


def walk(guess, right, parents, b):
    """The accepted path of sequence b: from column 0 along children that are their parent's prediction,
    the first of the deepest."""
    T = len(parents)
    best = [0]
    for t in range(T):
        path, u = [], t
        while u >= 0:
            path.append(u)
            u = parents[u]
        path = path[::-1]
        if all(guess[b][w] == right[b][v] for v, w in zip(path, path[1:])) and len(path) > len(best):
            best = path
    return best


@pytest.mark.parametrize("kv,qk_norm", [("int8", False), ("int4", True)])
def test_verified_steps_across_pages_follow_the_dense_step(kv, qk_norm):
    """Trees whose branches hold the dense step's own predictions: paths of several tokens are accepted, pages
    fill in the middle of a path, and what the step appends, predicts and returns is what the dense step says.
    Bar for K and V: 2e-2 of their largest, as for a decode step over the same cache (test_gpu_llama.py). A
    sequence sits a step out where a prediction on its way leads the next by less than 1e-2 of the largest
    logit (some twenty roundings to fp16 lie between the two), which a fifth of the way's five may do."""
    from metagross_b200.tree import tree_depths, tree_mask

    d = decoder(qk_norm, kv=kv)
    d.prefill(prompt())
    #          0; 1 wrong under it; 2 right; 3, 4 under 2, 4 right; 5 under 4 right; 6 under 5 right but for sequence 1
    parents = [-1, 0, 0, 2, 2, 4, 5]
    mask = tree_mask(parents).cuda().expand(B, 7, 7)
    depth = tree_depths(mask)
    vocab, longest, crossed, checked = SHAPE["vocab"], 0, 0, 0
    for step in range(9):
        tree = torch.zeros(B, 7, dtype=torch.long, device="cuda")
        tree[:, 0] = d.ids
        for t in (2, 4, 5, 6):  # the right children, one level after the other
            logits = dense_step(d, tree, mask, depth)[0]
            tree[:, t] = logits[:, parents[t]].argmax(-1)
        tree[:, 1], tree[:, 3] = (tree[:, 2] + 1) % vocab, (tree[:, 4] + 1) % vocab
        tree[1, 6] = (tree[1, 6] + 1) % vocab
        tree[2, 4 if step % 2 else 5] += 1  # sequence 2: two or three tokens
        tree[2] %= vocab
        logits, k, v = dense_step(d, tree, mask, depth)
        lens = d.cache.seq_lens.tolist()
        tokens, n = d.verify(tree, parents)
        d.cache.check()
        right, guess = logits.argmax(-1).tolist(), tree.tolist()
        top = logits.topk(2).values
        clear = (top[..., 0] - top[..., 1] > 1e-2 * logits.abs().max())[:, [0, 2, 4, 5, 6]].all(1).tolist()
        for b in range(B):
            assert d.pos[b] == d.cache.seq_lens[b] == lens[b] + int(n[b])
            if not clear[b]:
                continue
            checked += 1
            path = walk(guess, right, parents, b)
            assert n[b] == len(path) and tokens[b, :len(path)].tolist() == [guess[b][t] for t in path]
            assert d.ids[b] == right[b][path[-1]]
            longest, crossed = max(longest, len(path)), crossed + (lens[b] // 16 < (lens[b] + len(path) - 1) // 16)
            for i in range(d.s.layers):
                kc, vc, cu = d.cache.gather(i, dtype=torch.float32)
                for got, want, scales in ((kc, k, d.cache.k_scales), (vc, v, d.cache.v_scales)):
                    got = got[int(cu[b]) + lens[b]:int(cu[b + 1])]
                    want = want[i, b, path].float()
                    # half a code's step where the token's page is full
                    page = (lens[b] + torch.arange(len(path), device="cuda")) // 16
                    full = page < d.cache.seq_lens[b] // 16
                    step_of = scales[i, d.cache.block_tables[b, page.clamp(max=d.cache.max_blocks - 1)].long()] * full
                    bar = 2e-2 * want.abs().max() + 0.5 * step_of
                    assert ((got - want).abs().amax((1, 2)) <= bar).all()
        # the next step's logits, from what is in the cache now
        twin = dense_step(d, d.ids[:, None], torch.ones(B, 1, 1, dtype=torch.bool, device="cuda"),
                          torch.zeros(B, 1, dtype=torch.long, device="cuda"))[0][:, 0]
        seen = d.ids.clone(), d.pos.clone(), d.cache.seq_lens.clone()
        one, count = d.verify(d.ids[:, None], [-1])
        top = twin.topk(2).values
        clear = top[:, 0] - top[:, 1] > 1e-2 * twin.abs().max()
        assert torch.equal(one[:, 0], seen[0]) and (count == 1).all()
        assert torch.equal(d.ids[clear], twin.argmax(-1)[clear])
        assert torch.equal(d.pos, seen[1] + 1) and torch.equal(d.cache.seq_lens, seen[2] + 1)
    assert longest == 5 and crossed >= 1 and checked >= 9
