"""q / k head norms with the rotary embedding (``_C.qk_norm_rope``) against 64 bits.

The bar: 2^-11 |ref| for the one rounding to fp16, 2^-18 (|y_d| + |y_{d + D/2}|)
for the fp32 chain before it (sum of squares, reciprocal root and four products:
under 40 units of 2^-24 of the rotated pair), half a unit of the smallest fp16."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5


def inputs(rows, hq, hkv, d, positions=97, seed=0, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (gain * torch.randn(rows, (hq + 2 * hkv) * d, generator=g, device="cuda")).half()
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).half() for _ in range(2))
    pos = torch.randint(0, positions, (rows,), generator=g, device="cuda")
    a = torch.outer(torch.arange(positions, device="cuda").float(),
                    10000.0 ** (-torch.arange(0, d, 2, device="cuda").float() / d))
    return qkv, wq, wk, pos, a.cos().contiguous(), a.sin().contiguous()


def call(qkv, wq, wk, pos, cos, sin, hq, hkv, d, with_v=True, status=None, eps=EPS):
    from metagross_b200 import _C

    n = qkv.shape[0]
    q = torch.full((n, hq, d), 9.0, device="cuda").half()
    k = torch.full((n, hkv, d), 9.0, device="cuda").half()
    v = torch.full((n, hkv, d), 9.0, device="cuda").half() if with_v else None
    _C.qk_norm_rope(qkv, wq, wk, pos, cos, sin, eps, q, k, v, status)
    torch.cuda.synchronize()
    return q, k, v


def reference(x, w, pos, cos, sin, eps=EPS):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    a, b = y.chunk(2, -1)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    ref = torch.cat([a * c - b * s, b * c + a * s], -1)
    pair = (a.abs() + b.abs()).repeat(1, 1, 2)
    return ref, 2.0 ** -11 * ref.abs() + 2.0 ** -18 * pair + 2.0 ** -24


def check(out, x, w, pos, cos, sin, eps=EPS):
    ref, bar = reference(x, w, pos, cos, sin, eps)
    assert ((out.double() - ref).abs() <= bar).all()


@pytest.mark.parametrize("rows", [1, 3, 64, 2500])
@pytest.mark.parametrize("hq,hkv,d", [(32, 4, 64), (12, 12, 64), (32, 8, 128), (4, 2, 96), (2, 1, 80), (3, 1, 256),
                                      (4, 4, 16), (2, 1, 512), (5, 3, 50), (2, 2, 640), (1, 1, 2)])
def test_matches_the_definition(rows, hq, hkv, d):
    qkv, wq, wk, pos, cos, sin = inputs(rows, hq, hkv, d)
    xq, xk, xv = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    for with_v in (True, False):
        q, k, v = call(qkv, wq, wk, pos, cos, sin, hq, hkv, d, with_v)
        check(q, xq, wq, pos, cos, sin)
        check(k, xk, wk, pos, cos, sin)
        if with_v:
            assert torch.equal(v, xv)


def test_strided_and_unaligned_rows():
    hq, hkv, d = 4, 2, 64
    qkv, wq, wk, pos, cos, sin = inputs(33, hq, hkv, d)
    want = call(qkv, wq, wk, pos, cos, sin, hq, hkv, d)
    wide = torch.zeros(33, qkv.shape[1] + 24, device="cuda").half()
    wide[:, 8:8 + qkv.shape[1]] = qkv  # 16-byte aligned rows
    odd = torch.zeros(33, qkv.shape[1] + 3, device="cuda").half()
    odd[:, 1:1 + qkv.shape[1]] = qkv  # odd offsets: the scalar kernel
    got = call(wide[:, 8:8 + qkv.shape[1]], wq, wk, pos, cos, sin, hq, hkv, d)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    q, k, v = call(odd[:, 1:1 + qkv.shape[1]], wq, wk, pos, cos, sin, hq, hkv, d)
    xq, xk, xv = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    check(q, xq, wq, pos, cos, sin)
    check(k, xk, wk, pos, cos, sin)
    assert torch.equal(v, xv)


@pytest.mark.parametrize("gain", [1e-4, 500.0])
def test_small_and_large_heads(gain):
    qkv, wq, wk, pos, cos, sin = inputs(40, 4, 2, 64, gain=gain)
    qkv[3] = 0  # a head of zeros stays zero
    q, k, _ = call(qkv, wq, wk, pos, cos, sin, 4, 2, 64)
    check(q, qkv[:, :256].unflatten(1, (4, 64)), wq, pos, cos, sin)
    check(k, qkv[:, 256:384].unflatten(1, (2, 64)), wk, pos, cos, sin)
    assert (q[3] == 0).all()


@pytest.mark.parametrize("d", [64, 50])
def test_positions_outside_the_tables(d):
    qkv, wq, wk, pos, cos, sin = inputs(6, 4, 2, d)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q0, k0, v0 = call(qkv, wq, wk, pos, cos, sin, 4, 2, d, status=status)
    assert int(status.item()) == 0
    pos[1], pos[4] = cos.shape[0], -1
    q, k, v = call(qkv, wq, wk, pos, cos, sin, 4, 2, d, status=status)
    assert int(status.item()) == 0x80
    for r in range(6):
        if r in (1, 4):
            assert (q[r] == 0).all() and (k[r] == 0).all()
        else:
            assert torch.equal(q[r], q0[r]) and torch.equal(k[r], k0[r])
    assert torch.equal(v, v0)


def test_nothing_to_do_and_refusals():
    from metagross_b200 import _C

    hq, hkv, d = 4, 2, 64
    qkv, wq, wk, pos, cos, sin = inputs(5, hq, hkv, d)
    call(qkv[:0], wq, wk, pos[:0], cos, sin, hq, hkv, d)
    q, k = torch.empty(5, hq, d, device="cuda").half(), torch.empty(5, hkv, d, device="cuda").half()

    def refused(match, **kw):
        a = dict(qkv=qkv, q_weight=wq, k_weight=wk, pos=pos, cos=cos, sin=sin, eps=EPS, q=q, k=k)
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            _C.qk_norm_rope(**a)

    refused("float16", qkv=qkv.float())
    refused("qkv must be", qkv=qkv[:, :-1])
    refused("contiguous rows", qkv=qkv.t().contiguous().t())
    refused(r"must be \[D\]", q_weight=wq[:32].contiguous())
    refused("int64", pos=pos.int())
    refused("int64", pos=pos[:4])
    refused("tables", cos=cos[:, :16].contiguous())
    refused("tables", sin=sin[:5])
    refused("eps", eps=-1.0)
    refused("v must be", v=torch.empty(5, hkv, d, device="cuda"))
    refused("k ", k=k[:, :, :32].contiguous())
