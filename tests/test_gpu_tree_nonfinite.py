"""Drafted-token attention with queries, values and scales at the ends of their range: what comes out
does not depend on how the plan cuts a sequence, nor on which of the two kernels takes it.
Definition and bar: test_gpu_tree.py."""
import math

import pytest
import torch

from test_gpu_tree import context, drafts, make_cache, reference

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
