"""Attention of drafted tokens over the paged cache (``BatchedPagedKVCache.attend_tree``)
against the definition in 64 bits over the cache's own codes, scales and exact rows.

The bar, for each output element with A = sum_j p_j |v_j|:
  2^-11 (A + |ref|)            probabilities and the output are rounded to fp16 once each
  + 4 (D + 4) 2^-24 smax A     fp32 accumulation of a score (|error| <= D 2^-24 sum |q_i k_i| scale, smax the
                               largest of these sums) moves each probability by twice that, numerator and sum
  + 2^-24                      half a unit of the smallest fp16
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make_cache(lens, hkv, d, kv="int8", page=16, scales="page", layers=1, seed=0, gain=1.0, spare=0):
    from metagross_b200.batched import BatchedPagedKVCache

    B, top = len(lens), max(max(lens), 1)
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = top // page + 4
    c = BatchedPagedKVCache(layers, B + spare, hkv, d, page_size=page, num_pages=sum(n // page for n in lens) + 64,
                            max_blocks=width, kv_dtype=kv, scale_granularity=scales)
    n = torch.tensor(lens + [0] * spare, dtype=torch.int32)
    # scatter the pages: allocate and free once in another order
    perm = torch.randperm(c.num_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    c.allocator.free_stack.copy_(perm)
    c.begin_step(n)
    for layer in range(layers):
        k, v = (gain * torch.randn(B + spare, top, hkv, d, generator=g, device="cuda") for _ in range(2))
        c.append(layer, k.half(), v.half())
    c.check()
    return c


def context(c, layer, b):
    """K and V [n, Hkv, D] in 64 bits."""
    n, P, D = int(c.seq_lens[b]), c.page_size, c.head_dim
    out = []
    for pool, sc, st in ((c.k_pool, c.k_scales, c.staging_k), (c.v_pool, c.v_scales, c.staging_v)):
        ids = c.block_tables[b, :n // P].long()
        x = pool[layer, ids]
        if c.kv_dtype == "int4":
            x = torch.stack([x & 15, x >> 4], -1).flatten(-2).to(torch.int16)
            x = torch.where(x > 7, x - 16, x)
        s = sc[layer, ids].double()
        x = x.double() * (s[..., None] if s.dim() == 3 else s[:, None, None, None])
        out.append(torch.cat([x.reshape(-1, c.num_kv_heads, D), st[layer, b, :n % P].double()]))
    return out


def reference(c, layer, q, k, v, mask=None, n_draft=None, scale=None):
    """(ref, bar) in 64 bits."""
    B, T, hq, D = q.shape
    G = hq // c.num_kv_heads
    scale = D ** -0.5 if scale is None else scale
    ref = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bar = torch.full_like(ref, 2.0 ** -24)
    for b in range(B):
        t = T if n_draft is None else int(n_draft[b])
        if t == 0:
            continue
        kc, vc = context(c, layer, b)
        n = kc.shape[0]
        K, V = torch.cat([kc, k[b, :t].double()]), torch.cat([vc, v[b, :t].double()])
        m = torch.ones(T, T, device=q.device).tril().bool() if mask is None else (mask if mask.dim() == 2 else mask[b])
        seen = torch.cat([torch.ones(t, n, dtype=torch.bool, device=q.device), m[:t, :t].bool()], 1)
        for h in range(hq):
            qq, kk, vv = q[b, :t, h].double(), K[:, h // G], V[:, h // G]
            s = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, 1), nan=0.0)
            # masked keys take no part, whatever they hold
            vz = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
            ref[b, :t, h] = p @ vz
            a = p @ vz.abs()
            fin = torch.where(torch.isfinite(kk), kk, torch.zeros_like(kk))
            smax = ((qq.abs() @ fin.abs().T) * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True) if seen.any() else 0.0
            bar[b, :t, h] += 2.0 ** -11 * (a + ref[b, :t, h].abs()) + 4 * (D + 4) * 2.0 ** -24 * smax * a
    return ref, bar


def drafts(c, T, hq, seed=1, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, D = c.batch, c.num_kv_heads, c.head_dim
    return ((torch.randn(B, T, hq, D, generator=g, device="cuda") * 1.5).half(),
            (gain * torch.randn(B, T, H, D, generator=g, device="cuda")).half(),
            (gain * torch.randn(B, T, H, D, generator=g, device="cuda")).half())


def random_tree(B, T, seed=2):
    from metagross_b200.tree import tree_mask

    g = torch.Generator().manual_seed(seed)
    par = (torch.arange(T) - torch.randint(1, 6, (B, T), generator=g)).clamp(min=-1)
    return tree_mask(par).cuda()


def compare(c, q, k, v, layer=0, **kw):
    out = c.attend_tree(layer, q, k, v, **kw)
    torch.cuda.synchronize()
    c.check()
    kw.pop("plan", None)
    kw.pop("out", None)
    ref, bar = reference(c, layer, q, k, v, **kw)
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    worst = (err / bar).max().item()
    assert worst <= 1.0, worst
    return out


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 777]


@pytest.mark.parametrize("T", [1, 2, 5, 16, 33, 70])
@pytest.mark.parametrize("kv,hq,hkv,d", [("int8", 12, 12, 64), ("int4", 32, 4, 64), ("int8", 8, 2, 128),
                                         ("int4", 4, 1, 128), ("int8", 6, 2, 64)])
def test_matches_the_definition(kv, hq, hkv, d, T):
    c = make_cache(LENS, hkv, d, kv)
    q, k, v = drafts(c, T, hq)
    compare(c, q, k, v, mask=random_tree(c.batch, T))
    compare(c, q, k, v)  # a chain


@pytest.mark.parametrize("page", [1, 3, 8, 24, 32, 64])
@pytest.mark.parametrize("scales", ["page", "token_head"])
@pytest.mark.parametrize("kv,d", [("int8", 64), ("int4", 128)])
def test_page_sizes_and_scale_layouts(page, scales, kv, d):
    c = make_cache([0, 1, 70, 333, 64, 200], 2, d, kv, page=page, scales=scales)
    for T in (3, 40):
        q, k, v = drafts(c, T, 8)
        compare(c, q, k, v, mask=random_tree(c.batch, T))


@pytest.mark.parametrize("hq,hkv,d,T", [(12, 12, 64, 8), (32, 4, 64, 5), (32, 4, 64, 24), (16, 2, 128, 9),
                                        (16, 2, 128, 40)])
def test_long_contexts_are_split_and_joined(hq, hkv, d, T):
    c = make_cache([9001, 3, 4100], hkv, d, "int8")
    q, k, v = drafts(c, T, hq)
    a = compare(c, q, k, v, mask=random_tree(c.batch, T))
    b = c.attend_tree(0, q, k, v, mask=random_tree(c.batch, T))
    assert torch.equal(a, b)  # the join does not depend on which CTA ended first


def test_many_sequences_take_several_waves():
    r = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 900, (300,), generator=r).tolist() + [12000]
    c = make_cache(lens, 4, 64, "int4")
    q, k, v = drafts(c, 6, 32)
    n = torch.randint(0, 7, (c.batch,), generator=r, dtype=torch.int32).cuda()
    compare(c, q, k, v, mask=random_tree(c.batch, 6), n_draft=n)


@pytest.mark.parametrize("kv,hq,hkv,d", [("int8", 32, 4, 64), ("int4", 16, 4, 128)])
def test_a_chunk_of_a_prompt(kv, hq, hkv, d):
    c = make_cache([500, 0, 1999], hkv, d, kv)
    q, k, v = drafts(c, 301, hq)
    compare(c, q, k, v)


def test_ragged_drafts_leave_zeros():
    c = make_cache([40, 0, 100, 7], 2, 64)
    q, k, v = drafts(c, 9, 8)
    n = torch.tensor([9, 0, 3, 1], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    compare(c, q, k, v, mask=random_tree(4, 9), n_draft=n, out=out)
    for b, t in enumerate(n.tolist()):
        assert (out[b, t:] == 0).all()


@pytest.mark.parametrize("T,d", [(6, 64), (40, 64), (40, 128)])
def test_rows_that_see_nothing_are_zero(T, d):
    c = make_cache([0, 33], 2, d)
    q, k, v = drafts(c, T, 8)
    mask = torch.eye(T, dtype=torch.bool, device="cuda")
    mask[2] = False
    out = compare(c, q, k, v, mask=mask)
    assert (out[0, 2] == 0).all() and (out[1, 2] != 0).any()
    mask[:] = False
    out = compare(c, q, k, v, mask=mask)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("T,hq,d", [(5, 8, 64), (40, 8, 64), (40, 16, 128)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_masked_infinities_and_nan_take_no_part(T, hq, d, value):
    c = make_cache([50, 0, 3000], 2, d)
    q, k, v = drafts(c, T, hq)
    mask = torch.eye(T, dtype=torch.bool, device="cuda")
    mask[:, 0] = True
    mask[2:, 1] = False  # token 1 is seen by itself only
    n = torch.tensor([T, T - 1, T], dtype=torch.int32, device="cuda")
    clean = c.attend_tree(0, q, k, v, mask=mask, n_draft=n)
    k[:, 1], v[:, 1] = value, value
    k[1, T - 1:], v[1, T - 1:] = value, value  # past n_draft: not read at all
    out = c.attend_tree(0, q, k, v, mask=mask, n_draft=n)
    torch.cuda.synchronize()
    c.check()
    rows = [t for t in range(T) if t != 1]
    assert torch.equal(out[:, rows], clean[:, rows])


@pytest.mark.parametrize("T,hq,d", [(5, 8, 64), (40, 16, 128)])
def test_seen_infinities_come_out(T, hq, d):
    c = make_cache([50, 2000], 2, d)
    q, k, v = drafts(c, T, hq)
    clean = c.attend_tree(0, q, k, v)
    v[:, 2, :, 5], v[:, 2, :, 6], v[:, 2, :, 7] = math.inf, -math.inf, math.nan
    out = c.attend_tree(0, q, k, v)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :2], clean[:, :2])
    assert (out[:, 2:, :, 5] == math.inf).all() and (out[:, 2:, :, 6] == -math.inf).all()
    assert out[:, 2:, :, 7].isnan().all()
    keep = [i for i in range(d) if i not in (5, 6, 7)]
    assert torch.equal(out[..., keep], clean[..., keep])


@pytest.mark.parametrize("gain", [1e-5, 1e-3, 300.0])
@pytest.mark.parametrize("kv", ["int8", "int4"])
@pytest.mark.parametrize("T", [4, 40])
def test_very_small_and_large_values(gain, kv, T):
    c = make_cache([100, 16, 400], 2, 64, kv, gain=gain)
    q, k, v = drafts(c, T, 8, gain=gain)
    q = (q.float() / max(gain, 0.02) / 4).half() if gain > 1 else q
    compare(c, q, k, v)


def test_strided_inputs_and_a_shared_mask():
    c = make_cache([100, 5, 260], 4, 64)
    B, T, hq, H, D = 3, 7, 8, 4, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(B, T, (hq + 2 * H) * D, generator=g, device="cuda").half()
    q = qkv[..., :hq * D].unflatten(-1, (hq, D))
    k = qkv[..., hq * D:(hq + H) * D].unflatten(-1, (H, D))
    v = qkv[..., (hq + H) * D:].unflatten(-1, (H, D))
    heads_first = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v)]
    mask = random_tree(1, T)[0]
    a = compare(c, q, k, v, mask=mask)
    b = compare(c, *heads_first, mask=mask)
    assert torch.equal(a, b)
    wide = random_tree(1, T).expand(B, T, T)
    assert torch.equal(a, c.attend_tree(0, q, k, v, mask=wide))


def test_a_given_scale_and_one_plan_for_all_layers():
    c = make_cache([100, 5, 700], 4, 64, layers=3)
    plan = c.plan_tree(6, 8)
    mask = random_tree(3, 6)
    for layer in range(3):
        q, k, v = drafts(c, 6, 8, seed=layer)
        compare(c, q, k, v, layer=layer, mask=mask, plan=plan, scale=0.3)


def test_one_drafted_token_equals_decode_attention():
    c = make_cache([100, 5, 700, 33], 4, 64)
    q, k, v = drafts(c, 1, 8)
    out = c.attend_tree(0, q, k, v)[:, 0]
    c.begin_step(1)
    c.append(0, k, v)  # no length above fills a page with this token
    dec = c.attend(0, q[:, 0].contiguous())
    torch.cuda.synchronize()
    c.check()
    assert (out.float() - dec.float()).abs().max().item() <= 2e-3


def test_another_stream_and_a_captured_step():
    c = make_cache([100, 5, 700], 4, 64, layers=2)
    q, k, v = drafts(c, 6, 8)
    mask = random_tree(3, 6)
    want = [c.attend_tree(layer, q, k, v, mask=mask) for layer in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.attend_tree(1, q, k, v, mask=mask)
    side.synchronize()
    assert torch.equal(got, want[1])
    out = torch.zeros(2, *q.shape, device="cuda").half()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = c.plan_tree(6, 8)
        for layer in range(2):
            c.attend_tree(layer, q, k, v, mask=mask, plan=plan, out=out[layer])
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    from metagross_b200.batched import BatchedPagedKVCache

    c = make_cache([20, 5], 2, 64)
    q, k, v = drafts(c, 4, 8)
    with pytest.raises(ValueError, match="q must be"):
        c.attend_tree(0, q[0], k, v)
    with pytest.raises(ValueError, match="divisible"):
        c.attend_tree(0, q[:, :, :7], k, v)
    with pytest.raises(RuntimeError, match="float16"):
        c.attend_tree(0, q.float(), k, v)
    with pytest.raises(RuntimeError, match="k_draft"):
        c.attend_tree(0, q, k[:, :3], v)
    with pytest.raises(RuntimeError, match="mask"):
        c.attend_tree(0, q, k, v, mask=torch.ones(4, 3, dtype=torch.bool, device="cuda"))
    with pytest.raises(RuntimeError, match="mask"):
        c.attend_tree(0, q, k, v, mask=torch.ones(4, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="layer 1"):
        c.attend_tree(1, q, k, v)
    with pytest.raises(ValueError, match="scale"):
        c.attend_tree(0, q, k, v, scale=float("nan"))
    with pytest.raises(ValueError, match="one entry per sequence"):
        c.plan_tree(4, 8, torch.tensor([1, 2, 3]))
    plan = c.plan_tree(4, 8)
    with pytest.raises(ValueError, match="another"):
        c.attend_tree(0, q[:, :3], k[:, :3], v[:, :3], plan=plan)
    with pytest.raises(ValueError, match="plan_tree"):
        c.attend_tree(0, q, k, v, plan=plan, n_draft=torch.tensor([1, 2]))
    c.begin_step(1)
    with pytest.raises(ValueError, match="stale"):
        c.attend_tree(0, q, k, v, plan=plan)
    c32 = BatchedPagedKVCache(1, 2, 2, 64, num_pages=8, max_blocks=4, staging_dtype=torch.float32)
    with pytest.raises(ValueError, match="float16 staging"):
        c32.attend_tree(0, q, k, v)
    c96 = BatchedPagedKVCache(1, 2, 2, 96, num_pages=8, max_blocks=4)
    with pytest.raises(RuntimeError, match="head_dim 64 or 128"):
        c96.plan_tree(4, 8)


def test_bad_lengths_counts_and_pages_are_flagged():
    c = make_cache([40, 40], 2, 64)
    q, k, v = drafts(c, 4, 8)
    out = c.attend_tree(0, q, k, v, n_draft=torch.tensor([5, 4], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0x80
    assert (out[0] == 0).all() and (out[1] != 0).any()
    c.status.zero_()
    c.seq_lens[0] = -3
    c.invalidate_plan()
    out = c.attend_tree(0, q, k, v)
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0x80 and (out[0] == 0).all()
    c.status.zero_()
    c.seq_lens[0] = 40
    c.block_tables[0, 1] = c.num_pages
    c.invalidate_plan()
    c.attend_tree(0, q, k, v)
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0x2


def test_nothing_to_do():
    c = make_cache([40, 0], 2, 64)
    q, k, v = drafts(c, 0, 8)
    assert c.attend_tree(0, q, k, v).shape == (2, 0, 8, 64)
    q, k, v = drafts(c, 4, 8)
    out = c.attend_tree(0, q, k, v, n_draft=torch.zeros(2, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    c.check()
    assert (out == 0).all()
