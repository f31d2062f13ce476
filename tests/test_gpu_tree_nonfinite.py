"""Drafted-token attention with queries, values and scales at the ends of their range: what comes out
does not depend on how the plan cuts a sequence, nor on which of the two kernels takes it.
Definition and bar: test_gpu_tree.py."""
import math

import pytest
import torch

from test_gpu_tree import compare, context, drafts, make_cache, reference

pytestmark = pytest.mark.gpu


def is_cut(plan):
    """Whether a plan of full drafts cuts some sequence into pieces (the join has work)."""
    return bool(plan.buf[:16].view(torch.int32)[1])


@pytest.mark.parametrize("kv,d", [("int8", 64), ("int4", 128)])
@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite(kv, d, T, value):
    """NaN where a seen score is NaN or +inf, zeros where all are -inf, as the definition has it, in a
    sequence that is cut, in one of drafted tokens only, and in one of a tail."""
    c = make_cache([3000, 0, 40, 5], 2, d, kv)
    q, k, v = drafts(c, T, 8)
    ref, bar = reference(c, 0, q, k, v)
    q[:, 1, 5, 3] = value
    assert is_cut(c.plan_tree(T, 8))
    out = c.attend_tree(0, q, k, v)
    torch.cuda.synchronize()
    c.check()
    for b in range(c.batch):
        keys = torch.cat([context(c, 0, b)[0], k[b, :2].double()])[:, 1]
        s = (q[b, 1, 5].double() * keys).sum(-1)
        if (s == -math.inf).all():
            assert (out[b, 1, 5] == 0).all(), b
        else:
            assert (s.isnan() | (s == math.inf)).any()
            assert out[b, 1, 5].isnan().all(), b
    other = torch.ones(out.shape[:3], dtype=torch.bool, device="cuda")
    other[:, 1, 5] = False
    assert ((out.double() - ref).abs() <= bar)[other].all()


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("lens,cut", [([3000], True), ([20] * 700, False), ([0] * 700, False)])
def test_an_infinity_in_a_value_of_vanishing_weight(T, lens, cut):
    """The drafted keys score e^-300 of the cached ones, less than fp32 can hold: the row that sees an infinity
    gets it all the same, whether the drafted tokens are a piece of their own or not."""
    c = make_cache(lens, 2, 64)
    c.k_pool.zero_()  # every cached score is 0
    c.staging_k.zero_()
    q, k, v = drafts(c, T, 8)
    q.zero_()
    k.zero_()
    q[..., 0], k[..., 0] = 1.0, -300.0
    assert is_cut(c.plan_tree(T, 8)) == cut
    clean = c.attend_tree(0, q, k, v, scale=1.0)
    v[:, 1, :, 5], v[:, 1, :, 6], v[:, 1, :, 7] = math.inf, -math.inf, math.nan
    out = c.attend_tree(0, q, k, v, scale=1.0)
    torch.cuda.synchronize()
    c.check()
    assert torch.equal(out[:, :1], clean[:, :1])
    assert (out[:, 1:, :, 5] == math.inf).all() and (out[:, 1:, :, 6] == -math.inf).all()
    assert out[:, 1:, :, 7].isnan().all()
    keep = [i for i in range(64) if i not in (5, 6, 7)]
    assert torch.equal(out[..., keep], clean[..., keep])


@pytest.mark.parametrize("T", [3, 40])
def test_an_infinity_in_a_staged_value_of_vanishing_weight(T):
    """The same where the staged rows fill the last piece of the context."""
    c = make_cache([47 * 64 - 1], 2, 64, page=64)
    c.k_pool.zero_()
    c.staging_k.zero_()
    c.staging_k[..., 0] = -300.0
    q, k, v = drafts(c, T, 8)
    q.zero_()
    k.zero_()
    q[..., 0] = 1.0
    clean = c.attend_tree(0, q, k, v, scale=1.0)
    c.staging_v[:, :, 9, :, 5], c.staging_v[:, :, 9, :, 6] = math.inf, -math.inf
    out = c.attend_tree(0, q, k, v, scale=1.0)
    torch.cuda.synchronize()
    c.check()
    assert (out[..., 5] == math.inf).all() and (out[..., 6] == -math.inf).all()
    keep = [i for i in range(64) if i not in (5, 6)]
    assert torch.equal(out[..., keep], clean[..., keep])


@pytest.mark.parametrize("T", [1, 3, 6, 30])
@pytest.mark.parametrize("scales,page", [("page", 16), ("token_head", 16), ("page", 24)])
@pytest.mark.parametrize("mixed", [False, True])
def test_values_of_a_few_of_the_smallest_halves(T, scales, page, mixed):
    """V rows of 0 to 15 times 2^-24, whose scales lie below 2^-27: such keys count like any other, alone and
    beside pages of ordinary values."""
    from metagross_b200.batched import BatchedPagedKVCache

    g = torch.Generator(device="cuda").manual_seed(7)
    n = [200, 31, 70]
    c = BatchedPagedKVCache(1, 3, 2, 64, page_size=page, num_pages=40, max_blocks=16, kv_dtype="int8",
                            scale_granularity=scales)
    c.begin_step(torch.tensor(n, dtype=torch.int32))
    k = torch.randn(3, 200, 2, 64, generator=g, device="cuda")
    v = torch.randint(0, 16, (3, 200, 2, 64), generator=g, device="cuda") * 2.0 ** -24
    if mixed:
        v[:, page:2 * page] = torch.randn(3, page, 2, 64, generator=g, device="cuda")
    c.append(0, k.half(), v.half())
    c.check()
    assert 0 < c.v_scales[0, c.block_tables[0, 0].long()].min() < 2.0 ** -27
    q, kd, _ = drafts(c, T, 8)
    vd = (torch.randint(0, 16, kd.shape, generator=g, device="cuda") * 2.0 ** -24).half()
    out = compare(c, q, kd, vd)
    assert mixed or (out.amax((2, 3)) >= 4 * 2.0 ** -24).all()  # the mean of the values is 7.5 units
