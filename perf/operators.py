"""Workloads of the operators for drafted and forked sequences over the paged cache.

Three operators, each with a plain form (elementary torch operations in 32 bits) and the package's own call:

  tree   attention of the drafted tokens of every sequence over its quantized cached context and, through a mask,
         over each other (``BatchedPagedKVCache.attend_tree``), for all layers of one step
  norm   RMS norm of every q and k head and its rotation, from a fused q|k|v projection (``_C.qk_norm_rope``)
  fork   sequences that become copies of others: shared pages, copied tails (``BatchedPagedKVCache.fork``)
"""
import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5


def listed():
    return [
        # one user's short chat, a draft of four tokens in a chain: the latency of a small call
        dict(name="tree_small", op="tree", layers=2, batch=1, hq=12, hkv=12, d=64, kv="int8", page=16, scales="page",
             ctx="uniform", lo=90, hi=110, draft=4, shape="chain"),
        # GPT-2-small decode batch with eight drafted tokens a sequence: eight rows share each key
        dict(name="tree_gpt2", op="tree", layers=12, batch=32, hq=12, hkv=12, d=64, kv="int8", page=16, scales="page",
             ctx="uniform", lo=1000, hi=1024, draft=8, shape="tree"),
        # TinyLlama attention shape, trees of 16: 128 rows share each key
        dict(name="tree_tinyllama", op="tree", layers=4, batch=64, hq=32, hkv=4, d=64, kv="int4", page=16,
             scales="page", ctx="uniform", lo=128, hi=2048, draft=16, shape="tree"),
        # heavy-tailed contexts with short ragged drafts: 40 rows a key, the balance over sequences
        dict(name="tree_lognormal", op="tree", layers=2, batch=200, hq=32, hkv=4, d=64, kv="int4", page=16,
             scales="page", ctx="lognormal", lo=1, hi=32768, draft=5, shape="ragged"),
        # head_dim 128, a scale per token and head, pages of 24, a wide tree of odd size
        dict(name="tree_d128", op="tree", layers=2, batch=12, hq=32, hkv=8, d=128, kv="int8", page=24,
             scales="token_head", ctx="uniform", lo=1500, hi=6000, draft=61, shape="tree"),
        # a chunk of 512 prompt tokens over a long quantized prefix (chain mask)
        dict(name="tree_chunk", op="tree", layers=2, batch=8, hq=32, hkv=4, d=64, kv="int8", page=16, scales="page",
             ctx="uniform", lo=3000, hi=5000, draft=512, shape="chain"),
        # the projection of one decode step: 64 rows, 32 q and 4 kv heads
        dict(name="norm_decode", op="norm", rows=64, hq=32, hkv=4, d=64, positions=2048, with_v=True),
        # the rows of a verified step: 64 sequences x 16 drafts; the attention reads v where it is
        dict(name="norm_tree", op="norm", rows=1024, hq=32, hkv=4, d=64, positions=2064, with_v=False),
        # a prompt batch of odd length, head_dim 128
        dict(name="norm_prompt", op="norm", rows=9 * 2047, hq=32, hkv=8, d=128, positions=4096, with_v=True),
        # two samples of one prompt
        dict(name="fork_small", op="fork", layers=12, src=1, dst=2, hkv=12, d=64, kv="int8", page=16, ctx=300,
             cut=False),
        # beams that continue from other beams: 16 prompts, 64 sequences, 22 layers
        dict(name="fork_beams", op="fork", layers=22, src=16, dst=64, hkv=4, d=64, kv="int4", page=16, ctx=1500,
             cut=False),
        # many samples from prefixes of a few prompts: the page that a prefix cuts is dequantized
        dict(name="fork_prefix", op="fork", layers=12, src=4, dst=256, hkv=12, d=64, kv="int8", page=16, ctx=1024,
             cut=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


#: head layouts (q heads, kv heads, head_dim): GPT-2 small, TinyLlama, grouped heads of 128
HEADS = ((12, 12, 64), (32, 4, 64), (32, 8, 128))


def draw(rng):
    op = rng.choice(("tree", "tree", "norm", "fork"))
    hq, hkv, d = rng.choice(HEADS)
    kv = rng.choice(("int8", "int4"))
    page = rng.choice((16, 16, 8, 24, 32))
    if op == "norm":
        return dict(op=op, rows=_log_int(rng, 1, 9 * 2047), hq=hq, hkv=hkv, d=d, positions=_log_int(rng, 512, 4096),
                    with_v=rng.random() < 0.5)
    if op == "fork":
        return dict(op=op, layers=rng.randint(2, 12), src=_log_int(rng, 1, 16), dst=_log_int(rng, 1, 200), hkv=hkv,
                    d=d, kv=kv, page=page, ctx=_log_int(rng, 64, 1024), cut=rng.random() < 0.5)
    draft = _log_int(rng, 1, 300)
    shape = rng.choice(("chain", "tree", "ragged"))
    hi = _log_int(rng, 64, 8192)
    ctx = rng.choice(("uniform", "uniform", "lognormal"))
    # the batch that keeps the pass under the largest listed one's products and the padded plain form in bounds
    most = min(4e11 / (4.0 * draft * hq * d * (hi + draft)), 1.5e9 / (hi * hkv * d), 1.5e9 / (hq * draft * (hi + draft)))
    return dict(op=op, layers=1, batch=_log_int(rng, 1, max(1, min(128, int(most)))), hq=hq, hkv=hkv, d=d, kv=kv,
                page=page, scales=rng.choice(("page", "page", "token_head")), ctx=ctx, lo=max(1, hi // 8), hi=hi,
                draft=draft, shape=shape)


# ------------------------------------------------------------------ what a case fixes
def lengths(case):
    """Cached tokens of every sequence of a tree case."""
    r = random.Random(7919 * case["batch"] + case["hi"])
    if case["ctx"] == "lognormal":  # median a sixteenth of the largest, as served contexts are
        draw_one = lambda: math.exp(r.gauss(math.log(case["hi"] / 16.0), 1.0))  # noqa: E731
        return [max(case["lo"], min(case["hi"], int(draw_one()))) for _ in range(case["batch"])]
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def drafts(case):
    """Drafted tokens of every sequence of a tree case."""
    r = random.Random(104729 * case["batch"] + case["draft"])
    if case["shape"] != "ragged":
        return [case["draft"]] * case["batch"]
    return [r.randint(0, case["draft"]) for _ in range(case["batch"])]


def fork_lengths(case):
    """(lengths of the sources, of the old contents of the targets, source of each target, its new length)."""
    r = random.Random(31 * case["src"] + 17 * case["dst"] + case["ctx"])
    src = [r.randint(max(1, case["ctx"] // 2), case["ctx"]) for _ in range(case["src"])]
    old = [r.randint(0, case["ctx"] // 4) for _ in range(case["dst"])]
    parent = [r.randrange(case["src"]) for _ in range(case["dst"])]
    new = [r.randint(1, src[p]) if case["cut"] else src[p] for p in parent]
    return src, old, parent, new


# ------------------------------------------------------------------ inputs
def _tokens(g, *shape):
    """K / V values: unit normal with one in a hundred eight times as large."""
    x = torch.randn(*shape, generator=g, device=DEV)
    return torch.where(torch.rand(*shape, generator=g, device=DEV) < 0.01, x * 8, x)


def _quantized(g, layers, pages, case):
    """Codes [L, N, P, Hkv, D] int8 (int4 values in [-7, 7]) of random tokens and their scales."""
    top = 127.0 if case["kv"] == "int8" else 7.0
    th = case.get("scales") == "token_head"
    codes = torch.empty(layers, pages, case["page"], case["hkv"], case["d"], dtype=torch.int8, device=DEV)
    scales = torch.empty(layers, pages, case["page"] if th else 1, case["hkv"] if th else 1, 1, device=DEV)
    step = max(1, (1 << 27) // (case["page"] * case["hkv"] * case["d"]))
    for layer in range(layers):
        for a in range(0, pages, step):
            x = _tokens(g, min(step, pages - a), case["page"], case["hkv"], case["d"])
            s = x.abs().amax(-1 if th else (1, 2, 3), keepdim=True) / top
            codes[layer, a:a + step] = torch.round(x / s).clamp(-top, top).to(torch.int8)
            scales[layer, a:a + step] = s
    if case["kv"] == "int4":
        codes = (codes[..., 0::2] & 15 | codes[..., 1::2] << 4).view(torch.uint8)
    return codes, (scales[..., 0] if th else scales.flatten(1))


def _tables(g, lens, page, pages, width, perm):
    """Block tables with the pages of every sequence taken off `perm` in order, and how many were taken."""
    full = torch.tensor([n // page for n in lens], device=DEV)
    first = torch.cumsum(full, 0) - full
    j = torch.arange(width, device=DEV)
    at = (first[:, None] + j).clamp(max=pages - 1)
    return torch.where(j < full[:, None], perm[at], 0).to(torch.int32), int(full.sum())


def _cache(case, layers, batch, pages, width):
    from metagross_b200.batched import BatchedPagedKVCache

    return BatchedPagedKVCache(layers, batch, case["hkv"], case["d"], page_size=case["page"], num_pages=pages,
                               max_blocks=width, kv_dtype=case["kv"], scale_granularity=case.get("scales", "page"),
                               device=DEV)


def _fill(cache, s):
    """The package's cache in the state that the tensors of `s` describe."""
    for name in ("k_pool", "v_pool", "k_scales", "v_scales", "staging_k", "staging_v", "block_tables", "seq_lens"):
        getattr(cache, name).copy_(s[name])
        s[name] = getattr(cache, name)
    for name in ("free_stack", "n_free", "in_use"):
        if name in s:
            getattr(cache.allocator, name).copy_(s[name])
            s[name] = getattr(cache.allocator, name)
    cache.invalidate_plan()
    s["cache"] = cache


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"tree": _prepare_tree, "norm": _prepare_norm, "fork": _prepare_fork}[case["op"]](case, g)


def _prepare_tree(case, g):
    L, B, T, P = case["layers"], case["batch"], case["draft"], case["page"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = lengths(case)
    pages = max(1, sum(n // P for n in lens))
    width = max(lens) // P + 1
    s = {}
    s["k_pool"], s["k_scales"] = _quantized(g, L, pages, case)
    s["v_pool"], s["v_scales"] = _quantized(g, L, pages, case)
    s["block_tables"], _ = _tables(g, lens, P, pages, width, torch.randperm(pages, generator=g, device=DEV))
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["staging_k"], s["staging_v"] = (_tokens(g, L, B, P, hkv, d).half() for _ in range(2))
    # the projection that the drafted tokens come from: q and k rotated out of it, v read in place
    qkv = _tokens(g, L, B, T, (hq + 2 * hkv) * d).half()
    s["q"] = qkv[..., :hq * d].unflatten(-1, (hq, d)).contiguous()
    s["k"] = qkv[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d)).contiguous()
    s["v"] = qkv[..., (hq + hkv) * d:].unflatten(-1, (hkv, d))
    n = torch.tensor(drafts(case), dtype=torch.int32, device=DEV)
    s["n_draft"] = n if case["shape"] == "ragged" else None
    s["mask"] = None
    if case["shape"] != "chain":
        # every token's parent is one of the eight before it: the ancestors are the closure of that relation
        i = torch.arange(T, device=DEV)
        back = torch.randint(1, 9, (B, T), generator=g, device=DEV)
        link = torch.zeros(B, T, T, device=DEV)
        link.scatter_(2, (i - back).clamp(min=0)[..., None], 1.0)
        link = torch.maximum(link * (i[:, None] > 0), torch.eye(T, device=DEV))
        for _ in range(max(1, T).bit_length()):
            link = (link @ link > 0).float()
        s["mask"] = link.bool()
    s["out"] = torch.empty_like(s["q"])
    if own:
        _fill(_cache(case, L, B, pages, width), s)
    return s


def _prepare_norm(case, g):
    hq, hkv, d, rows = case["hq"], case["hkv"], case["d"], case["rows"]
    s = {"qkv": torch.randn(rows, (hq + 2 * hkv) * d, generator=g, device=DEV).half(),
         "wq": (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).half(),
         "wk": (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).half(),
         "pos": torch.randint(0, case["positions"], (rows,), generator=g, device=DEV)}
    angle = torch.outer(torch.arange(case["positions"], device=DEV).float(),
                        10000.0 ** (-torch.arange(0, d, 2, device=DEV).float() / d))
    s["cos"], s["sin"] = angle.cos(), angle.sin()
    s["q"] = torch.empty(rows, hq, d, dtype=torch.float16, device=DEV)
    s["k"] = torch.empty(rows, hkv, d, dtype=torch.float16, device=DEV)
    s["v"] = torch.empty_like(s["k"]) if case["with_v"] else None
    if own:
        from metagross_b200 import _C

        s["C"] = _C
    return s


def _prepare_fork(case, g):
    L, P, hkv, d = case["layers"], case["page"], case["hkv"], case["d"]
    src, old, parent, new = fork_lengths(case)
    lens = src + old
    B, width = len(lens), case["ctx"] // P + 1
    pages = sum(n // P for n in lens) + 7
    s = {}
    s["k_pool"], s["k_scales"] = _quantized(g, L, pages, case)
    s["v_pool"], s["v_scales"] = _quantized(g, L, pages, case)
    perm = torch.randperm(pages, generator=g, device=DEV)
    s["block_tables"], used = _tables(g, lens, P, pages, width, perm)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["staging_k"], s["staging_v"] = (_tokens(g, L, B, P, hkv, d).half() for _ in range(2))
    s["in_use"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
    s["in_use"][perm[:used]] = 1
    s["free_stack"] = torch.cat([perm[used:], perm[:used]]).to(torch.int32)
    s["n_free"] = torch.tensor([pages - used], dtype=torch.int32, device=DEV)
    s["src"] = torch.tensor(parent, dtype=torch.int32, device=DEV)
    s["dst"] = torch.arange(len(src), B, dtype=torch.int32, device=DEV)
    s["lens"] = torch.tensor(new, dtype=torch.int32, device=DEV) if case["cut"] else None
    s["page"], s["kv"] = P, case["kv"]
    if own:
        _fill(_cache(case, L, B, pages, width), s)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    if "qkv" in state:
        return _run_norm(state)
    if "dst" in state:
        return _run_fork(state)
    return _run_tree(state)


def _unpacked(codes):
    """Codes as 32-bit floats; packed bytes hold the even element in the low nibble."""
    if codes.dtype == torch.int8:
        return codes.float()
    low, high = (codes & 15).to(torch.int8), (codes >> 4).to(torch.int8)
    both = torch.stack([low, high], -1).flatten(-2)
    return torch.where(both > 7, both - 16, both).float()


def _plain_context(s, name, layer):
    """Cached values [B, pages * P, Hkv, D] of one layer in 32 bits, by the block tables."""
    bt = s["block_tables"].long()
    x = _unpacked(s[name + "_pool"][layer][bt])
    sc = s[name + "_scales"][layer][bt]
    x *= sc[..., None] if sc.dim() == 4 else sc[..., None, None, None]
    return x.flatten(1, 2)


def _run_tree(s):
    if own:
        cache = s["cache"]
        # a step has new lengths: its plan is made once, for all layers
        plan = cache.plan_tree(s["q"].shape[2], s["q"].shape[3], s["n_draft"])
        for layer in range(s["q"].shape[0]):
            cache.attend_tree(layer, s["q"][layer], s["k"][layer], s["v"][layer], mask=s["mask"], plan=plan,
                              out=s["out"][layer])
        return s["out"]
    L, B, T, hq, d = s["q"].shape
    P, hkv = s["staging_k"].shape[2:4]
    dev = s["q"].device
    # which keys each drafted token sees: whole pages, the tail, the drafted tokens of the mask
    lens = s["seq_lens"][:, None]
    whole = lens // P * P
    paged = torch.arange(s["block_tables"].shape[1] * P, device=dev) < whole
    tail = torch.arange(P, device=dev) < lens - whole
    i = torch.arange(T, device=dev)
    tree = s["mask"] if s["mask"] is not None else (i[:, None] >= i).expand(B, T, T)
    seen = torch.cat([torch.cat([paged, tail], 1)[:, None].expand(B, T, -1), tree], 2)
    if s["n_draft"] is not None:
        live = i < s["n_draft"][:, None]
        drafted = torch.cat([torch.ones_like(seen[:, 0, :-T]), live], 1)
        seen = seen & drafted[:, None] & live[..., None]
    seen = seen[:, None, :, None]  # [B, 1, T, 1, keys]
    for layer in range(L):
        k = torch.cat([_plain_context(s, "k", layer), s["staging_k"][layer].float(), s["k"][layer].float()], 1)
        q = s["q"][layer].float().view(B, T, hkv, hq // hkv, d)
        a = torch.einsum("bthgd,bnhd->bhtgn", q, k) / math.sqrt(d)
        del k
        a = a.masked_fill(~seen, -math.inf)
        top = a.amax(-1, keepdim=True)
        a = torch.exp(a - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = a.sum(-1, keepdim=True)
        v = torch.cat([_plain_context(s, "v", layer), s["staging_v"][layer].float(), s["v"][layer].float()], 1)
        o = torch.einsum("bhtgn,bnhd->bhtgd", a, v) / torch.where(total > 0, total, torch.ones_like(total))
        s["out"][layer] = o.permute(0, 2, 1, 3, 4).reshape(B, T, hq, d)
    return s["out"]


def _run_norm(s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        s["C"].qk_norm_rope(s["qkv"], s["wq"], s["wk"], s["pos"], s["cos"], s["sin"], EPS, q, k, v)
    else:
        hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
        xq, xk, xv = s["qkv"].split([hq * d, hkv * d, hkv * d], 1)
        q.copy_(_plain_norm(xq.view(-1, hq, d), s["wq"], s))
        k.copy_(_plain_norm(xk.view(-1, hkv, d), s["wk"], s))
        if v is not None:
            v.copy_(xv.view(-1, hkv, d))
    return [q, k] if v is None else [q, k, v]


def _plain_norm(x, w, s):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    c, n = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * n, b * c + a * n], -1)


def _run_fork(s):
    if own:
        s["cache"].fork(s["src"], s["dst"], s["lens"])
    else:
        _plain_fork(s)
    return [s[n] for n in ("block_tables", "seq_lens", "in_use", "free_stack", "n_free", "staging_k", "staging_v")]


def _plain_fork(s):
    P, bt, sl, count = s["page"], s["block_tables"], s["seq_lens"], s["in_use"]
    src, dst = s["src"].long(), s["dst"].long()
    j = torch.arange(bt.shape[1], device=bt.device)
    # the targets give up their pages; one that nobody holds any more goes back, in the order of its last holder
    held = bt[dst][j < (sl[dst] // P)[:, None]].long()
    count.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    last = torch.full_like(count, -1).scatter_reduce_(0, held, torch.arange(held.numel(), device=bt.device,
                                                                          dtype=torch.int32), "amax")
    back = torch.nonzero((count == 0) & (last >= 0)).flatten()
    back = back[last[back].argsort()]
    s["free_stack"].index_copy_(0, s["n_free"].long() + torch.arange(back.numel(), device=bt.device), back.int())
    s["n_free"] += back.numel()
    # they take the sources' pages and the exact rows after them
    length = sl[src] if s["lens"] is None else s["lens"]
    shared = j < (length // P)[:, None]
    pages = bt[src][shared].long()
    count.index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
    bt[dst] = torch.where(shared, bt[src], bt[dst])
    cut = length // P < sl[src] // P
    page = bt[src].gather(1, (length // P).long().clamp(max=bt.shape[1] - 1)[:, None])[:, 0]
    page = torch.where(cut, page, torch.zeros_like(page)).long()
    rows = (torch.arange(P, device=bt.device) < (length % P)[:, None])[None, :, :, None, None]
    for name in ("k", "v"):
        st = s["staging_" + name]
        exact_rows = _unpacked(s[name + "_pool"][:, page]) * s[name + "_scales"][:, page, None, None, None]
        new = torch.where(cut[:, None, None, None], exact_rows, st[:, src].float())
        st[:, dst] = torch.where(rows, new, st[:, dst].float()).to(st.dtype)
    sl[dst] = length.int()


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    d = case["d"]
    if case["op"] == "norm":
        moved = case["rows"] * (case["hq"] + case["hkv"] * (2 if case["with_v"] else 1)) * d
        return {"bytes": 2 * 2 * moved + 8 * case["rows"], "flops": 8 * moved}
    hkv, P = case["hkv"], case["page"]
    bits = 8 if case["kv"] == "int8" else 4
    if case["op"] == "fork":
        src, old, parent, new = fork_lengths(case)
        row = hkv * d
        b = f = 0
        for p, n in zip(parent, new):
            r = n % P
            read = bits / 8.0 if n // P < src[p] // P else 2
            b += case["layers"] * 2 * r * row * (read + 2) + 12 * (n // P)
            f += case["layers"] * 2 * r * row if n // P < src[p] // P else 0
        return {"bytes": int(b), "flops": int(f)}
    hq, T = case["hq"], case["draft"]
    b = f = 0
    for n, t in zip(lengths(case), drafts(case)):
        whole = n // P * P
        per_scale = 8 * whole * hkv if case["scales"] == "token_head" else 8 * (whole // P)
        b += 2 * whole * hkv * d * bits // 8 + per_scale + 4 * (whole // P) + 4 * (n - whole) * hkv * d
        b += 4 * t * hq * d + 4 * t * hkv * d + (0 if case["shape"] == "chain" else t * t)
        f += 4 * hq * d * (t * n + t * (t + 1) // 2)
    return {"bytes": int(b * case["layers"]), "flops": int(f * case["layers"])}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "norm": _exact_norm, "fork": _exact_fork}[case["op"]](case, s)


def _exact_values(pool, scale):
    """One page's values [P, Hkv, D] in 64 bits."""
    if pool.dtype == torch.uint8:
        byte = pool.to(torch.int64)
        low, high = byte % 16, byte // 16
        value = torch.empty(*pool.shape[:-1], 2 * pool.shape[-1], dtype=torch.float64, device=pool.device)
        value[..., 0::2] = low - 16 * (low >= 8)
        value[..., 1::2] = high - 16 * (high >= 8)
    else:
        value = pool.double()
    scale = scale.double()
    while scale.dim() < value.dim():
        scale = scale.unsqueeze(-1)
    return value * scale


def _exact_tree(case, s):
    d, P, G = case["d"], case["page"], case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for layer in range(case["layers"]):
        for b, (n, t) in enumerate(zip(lengths(case), drafts(case))):
            if t == 0:
                continue
            ids = s["block_tables"][b, :n // P].long()
            keys, values = (torch.cat([_exact_values(s[x + "_pool"][layer, ids], s[x + "_scales"][layer, ids])
                                       .reshape(-1, case["hkv"], d),
                                       s["staging_" + x][layer, b, :n % P].double(), s[x][layer, b, :t].double()])
                            for x in ("k", "v"))
            tree = torch.ones(t, t, device=DEV).tril().bool() if s["mask"] is None else s["mask"][b, :t, :t]
            for h in range(case["hq"]):
                a = s["q"][layer, b, :t, h].double() @ keys[:, h // G].T * d ** -0.5
                a[:, n:][~tree] = -math.inf
                out[layer, b, :t, h] = torch.softmax(a, 1) @ values[:, h // G]
    return out


def _exact_norm(case, s):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = s["qkv"].view(case["rows"], hq + 2 * hkv, d)
    cos, sin = s["cos"].double()[s["pos"]].unsqueeze(1), s["sin"].double()[s["pos"]].unsqueeze(1)

    def heads(part, w):
        part = part.double()
        part = part / torch.sqrt(part.square().sum(-1, keepdim=True) / d + EPS) * w.double()
        turned = torch.empty_like(part)
        turned[..., :d // 2] = part[..., :d // 2] * cos - part[..., d // 2:] * sin
        turned[..., d // 2:] = part[..., d // 2:] * cos + part[..., :d // 2] * sin
        return turned

    out = [heads(x[:, :hq], s["wq"]), heads(x[:, hq:hq + hkv], s["wk"])]
    return out + [x[:, hq + hkv:].double()] if case["with_v"] else out


def _exact_fork(case, s):
    src, old, parent, new = fork_lengths(case)
    P = case["page"]
    staged = [s["staging_k"].double(), s["staging_v"].double()]
    for i, (p, n) in enumerate(zip(parent, new)):
        to, r, j = len(src) + i, n % P, n // P
        for x, st in zip(("k", "v"), staged):
            if j < src[p] // P:
                at = s["block_tables"][p, j].long()
                st[:, to, :r] = _exact_values(s[x + "_pool"][:, at], s[x + "_scales"][:, at])[:, :r]
            else:
                st[:, to, :r] = s["staging_" + x][:, p, :r].double()
    return [None] * 5 + staged
