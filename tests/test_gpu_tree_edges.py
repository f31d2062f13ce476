"""Drafted-token attention where its two kernels (up to 48 query rows a kv head, and more) can go
wrong: repeated runs, V scales at the ends of the range, long tails of small probabilities, random
shapes and masks, plans of other shapes.  Definition and bar: test_gpu_tree.py."""
import dataclasses
import random

import pytest
import torch

from test_gpu_tree import compare, drafts, make_cache, random_tree, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,hq,hkv,d,T", [("int8", 32, 4, 64, 301), ("int4", 16, 4, 128, 130), ("int8", 12, 12, 64, 49),
                                           ("int8", 32, 4, 64, 6), ("int4", 8, 8, 128, 7)])
def test_repeated_runs_agree(kv, hq, hkv, d, T):
    """Nothing depends on which warp comes first: the same bits every time, and right."""
    c = make_cache([497, 498, 499, 500], hkv, d, kv)
    q, k, v = drafts(c, T, hq)
    first = compare(c, q, k, v).clone()
    for _ in range(30):
        assert torch.equal(c.attend_tree(0, q, k, v), first)


def value_cache(gain, kv, hkv, d, scales, n, page=16):
    """Keys of unit size, values of `gain` times that."""
    from metagross_b200.batched import BatchedPagedKVCache

    g = torch.Generator(device="cuda").manual_seed(5)
    c = BatchedPagedKVCache(1, len(n), hkv, d, page_size=page, num_pages=sum(x // page for x in n) + 8,
                            max_blocks=max(n) // page + 2, kv_dtype=kv, scale_granularity=scales)
    c.begin_step(torch.tensor(n, dtype=torch.int32))
    k, v = (torch.randn(len(n), max(n), hkv, d, generator=g, device="cuda") for _ in range(2))
    c.append(0, k.half(), (gain * v).half())
    c.check()
    return c


# INT8 scales: 8000 * 4 / 127 = 250; INT4: 4500.  1e-6 rounds to fp16 subnormals and scales near 2^-27.
@pytest.mark.parametrize("gain", [8000.0, 2000.0, 1e-4, 1e-6])
@pytest.mark.parametrize("kv,d,scales", [("int8", 64, "page"), ("int4", 64, "token_head"), ("int4", 128, "page")])
@pytest.mark.parametrize("T", [3, 30])
def test_values_at_the_ends_of_the_range(gain, kv, d, scales, T):
    c = value_cache(gain, kv, 2, d, scales, [200, 31, 70])
    q, k, v = drafts(c, T, 8)
    compare(c, q, k, (v.float() * gain).half())


@pytest.mark.parametrize("T", [3, 30])
@pytest.mark.parametrize("scales", ["page", "token_head"])
def test_pages_of_mixed_scales(T, scales):
    """Pages whose V scales differ by 2^20, and pages of zeros, side by side."""
    from metagross_b200.batched import BatchedPagedKVCache

    g = torch.Generator(device="cuda").manual_seed(6)
    c = BatchedPagedKVCache(1, 2, 2, 64, num_pages=40, max_blocks=20, kv_dtype="int8", scale_granularity=scales)
    c.begin_step(torch.tensor([205, 180], dtype=torch.int32))
    k, v = (torch.randn(2, 205, 2, 64, generator=g, device="cuda") for _ in range(2))
    factor = torch.tensor([1.0, 1e-3, 1e4, 0.0, 30.0], device="cuda")[torch.arange(205, device="cuda") // 16 % 5]
    c.append(0, k.half(), (v * factor[None, :, None, None]).half())
    q, kd, vd = drafts(c, T, 8)
    compare(c, q, kd, vd)


@pytest.mark.parametrize("T,hq", [(2, 4), (60, 4)])
@pytest.mark.parametrize("drop", [10.0, 14.0])
def test_a_long_tail_under_one_dominating_key(T, hq, drop):
    """One key with probability near 1 and value 0, thousands of e^-drop with value 1: the output is the
    tail's mass.  fp16 keeps a probability to half of 2^-24 of a reference below twice the largest, so
    each key adds at most 2^-24 |v| to the bar."""
    from metagross_b200.batched import BatchedPagedKVCache

    n, d = 6000, 64
    c = BatchedPagedKVCache(1, 1, hq, d, num_pages=400, max_blocks=400, kv_dtype="int8")
    c.begin_step(torch.tensor([n], dtype=torch.int32))
    k = torch.zeros(1, n, hq, d, device="cuda")
    v = torch.ones(1, n, hq, d, device="cuda")
    k[:, :, :, 0] = -drop
    k[:, :16, :, 0] = 0.0  # its own page: the scale of the others does not matter
    k[:, 1:16, :, 0] = -drop
    v[:, 0] = 0.0
    c.append(0, k.half(), v.half())
    q = torch.zeros(1, T, hq, d, device="cuda")
    q[..., 0] = 1.0
    kd = torch.zeros(1, T, hq, d, device="cuda")
    kd[..., 0] = -drop
    vd = torch.ones(1, T, hq, d, device="cuda")
    q, kd, vd = q.half(), kd.half(), vd.half()
    out = c.attend_tree(0, q, kd, vd, scale=1.0)
    ref, bar = reference(c, 0, q, kd, vd, scale=1.0)
    assert ((out.double() - ref).abs() <= bar + (n + T) * 2.0 ** -24).all()


def configurations():
    r = random.Random(11)
    for i in range(24):
        hkv, g = r.choice((1, 2, 3, 8)), r.choice((1, 2, 3, 5, 8))
        yield (r.choice(("int8", "int4")), hkv * g, hkv, r.choice((64, 128)), r.choice((1, 5, 8, 16, 24, 48)),
               r.choice(("page", "token_head")), r.choice((1, 3, 9, 17, 40, 90, 150)),
               [r.choice((0, 1, r.randint(2, 200), r.randint(200, 1500))) for _ in range(r.randint(1, 6))], i)


@pytest.mark.parametrize("kv,hq,hkv,d,page,scales,T,lens,seed", list(configurations()))
def test_random_shapes_with_random_masks(kv, hq, hkv, d, page, scales, T, lens, seed):
    c = make_cache(lens, hkv, d, kv, page=page, scales=scales, seed=seed)
    q, k, v = drafts(c, T, hq, seed=seed)
    g = torch.Generator().manual_seed(seed)
    # any mask: tokens that see later ones, not themselves, or nothing
    mask = (torch.rand(c.batch, T, T, generator=g) < 0.4).cuda()
    mask[:, T // 2] = False
    n = torch.randint(0, T + 1, (c.batch,), generator=g).to(torch.int32).cuda()
    compare(c, q, k, v, mask=mask, n_draft=n)
    compare(c, q, k, v, mask=random_tree(c.batch, T))


@pytest.mark.parametrize("T", [4, 40])
def test_a_plan_of_other_shapes_is_flagged(T):
    """Below the Python checks: the kernels compare the plan's shapes with their own and write nothing."""
    c = make_cache([100, 40], 2, 64)
    other = make_cache([100, 40, 7], 2, 64)
    q, k, v = drafts(c, T, 8)
    plan, wrong = c.plan_tree(T, 8), other.plan_tree(T, 8)
    assert wrong.buf.numel() >= plan.buf.numel()
    plan = dataclasses.replace(plan, buf=wrong.buf, nbytes=wrong.nbytes)
    out = torch.full((2, T, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    c.attend_tree(0, q, k, v, plan=plan, out=out)
    torch.cuda.synchronize()
    assert int(c.status.item()) == 0x80
    assert (out == 7.0).all()


def test_verify_refuses_what_would_leave_its_tables():
    from test_gpu_verify import B, decoder, prompt

    d = decoder()  # up to 96 tokens
    d.prefill(prompt(n=90))  # positions 90 .. 95 are left
    ids = torch.zeros(B, 7, dtype=torch.long, device="cuda")
    chain = list(range(-1, 6))
    with pytest.raises(ValueError, match="max_len"):
        d.verify(ids, chain)
    with pytest.raises(ValueError, match="parent"):
        d.verify(ids, torch.tensor([-1, 0, 9, 0, 0, 0, 0], device="cuda"))
    for bad in (-1, 64):
        with pytest.raises(ValueError, match="token ids"):
            d.verify(torch.full_like(ids, bad), [-1, 0, 0, 0, 0, 0, 0])
    tokens, n = d.verify(ids, [-1, 0, 0, 0, 0, 0, 0])  # wide, but short
    d.cache.check()
    assert (n >= 1).all()
