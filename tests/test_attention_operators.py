"""Operators of the attention sublayer (ops.qk_norm_rotary, ops.biased_attention) against their definitions in 64 bits.

Tolerances are bounds from the arithmetic, element by element.  With u = 2^-8 for a value that is rounded to bf16 (half a
step, relative) and e = 2^-24 for fp32:

  out      the probabilities are rounded once to the operands' type, the output once: |err| <= (u + w) A + u |out| with
           A = sum_j p_j |v_j| and w the fp32 part: an error h in the exponent moves p and its normaliser by h each, and a sum of n
           terms is off by n e of its absolute sum
  dq, dk   ds = p (dp - delta) inherits w from p, d e sum |do| |v| from dp, the error of delta, and one rounding
  dv       as out;   dtable: the fp32 part alone, delta being summed in fp32

h counts d + 8 steps of the score's absolute products, 8 of its value (scaling, cap, bias, exponent) and, for the cap of bf16
operands, 4 steps of the cap itself (as 1 - 2 / (1 + e^2x), or a polynomial of that error where the score is small)."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
E = 2.0 ** -24


def dev():
    return torch.device("cuda")


# ------------------------------------------------------------------------------------------------ attention: definition
def definition(q, k, v, heads, kv, mask=None, causal=False, prefix=None, documents=None, q_start=None, softcap=None,
               slopes=None, table=None, buckets=None, scale=None, dout=None, pairs=None):
    """64-bit values and bounds: {"out": (value, bound), ...}; operands (B, S, heads, d)"""
    dt = q.dtype
    u = U[dt]
    B, Sq, H, d = q.shape
    Sk = k.size(1)
    G = H // kv
    q, k, v = (t.detach().double().transpose(1, 2) for t in (q, k, v))              # (B, heads, S, d)
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    scale = d ** -0.5 if scale is None else scale
    if mask is not None:                        # what a hidden key holds does not count
        keep = mask.ne(0)[:, None, :, None]
        k, v = (torch.where(keep, t, torch.zeros_like(t)) for t in (k, v))
    if documents is not None:
        keep = documents.ge(0)[:, None, :, None]
        k, v = (torch.where(keep, t, torch.zeros_like(t)) for t in (k, v))
    raw = q @ k.transpose(2, 3) * scale
    mag = q.abs() @ k.abs().transpose(2, 3) * abs(scale)
    x, slope = raw, torch.ones_like(raw)
    if softcap:
        t = torch.tanh(raw / softcap)
        x, slope = softcap * t, 1 - t * t
    start = torch.full((B,), Sk - Sq, device=q.device) if q_start is None else torch.as_tensor(q_start, device=q.device).expand(B).long()
    i = start[:, None] + torch.arange(Sq, device=q.device)
    j = torch.arange(Sk, device=q.device)
    rel = j[None, None, :] - i[:, :, None]
    if slopes is not None:
        x = x - slopes.double()[None, :, None, None] * rel[:, None].abs()
    if table is not None:
        R = buckets.numel() // 2
        which = buckets.long()[rel.clamp(-R, R) + R]
        x = x + table.detach().double()[which].permute(0, 3, 1, 2)
    see = torch.ones(B, Sq, Sk, dtype=torch.bool, device=q.device)
    if causal:
        see &= rel <= 0
        if prefix is not None:
            see |= j[None, None, :] < prefix.long()[:, None, None]
    if mask is not None:
        see &= mask.ne(0)[:, None, :]
    if documents is not None:
        mine = documents.long().gather(1, i.clamp(0, Sk - 1))
        see &= (documents.long()[:, None, :] == mine[:, :, None]) & (mine >= 0)[:, :, None]
    if pairs is not None:
        see &= pairs
    see = see[:, None]
    h = E * ((d + 8) * mag + 8 * x.abs() + (4 * softcap if softcap and dt == torch.bfloat16 else 0.0) + 8)
    h = torch.where(see, h, torch.zeros_like(h)).amax(-1, keepdim=True)
    x = x.masked_fill(~see, -math.inf)
    p = torch.softmax(x, -1).nan_to_num(0.0).masked_fill(~see, 0.0)
    out = p @ v
    w = 2 * h + (Sk + 16) * E
    A = p @ v.abs()
    eo = (u + w) * A + max(u, 2 * E) * out.abs()
    back = lambda t: t.transpose(1, 2)
    res = {"out": (back(out), back(eo))}
    if dout is None:
        return res
    do = dout.double().transpose(1, 2)
    dp = do @ v.transpose(2, 3)
    adp = do.abs() @ v.abs().transpose(2, 3)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    wide = w * (do.abs() * A).sum(-1, keepdim=True) + (d + 4) * E * (do.abs() * A).sum(-1, keepdim=True)
    edelta = (do.abs() * eo).sum(-1, keepdim=True) + (d + 4) * E * (do.abs() * A).sum(-1, keepdim=True)
    exact_delta = table is not None and table.requires_grad
    base = p * (w * (dp - delta).abs() + (d + 4) * E * (adp + delta.abs()))
    eds = base + p * (wide if exact_delta else edelta)
    if table is not None:
        dtable, etable = (torch.zeros(table.shape, dtype=torch.float64, device=q.device) for _ in range(2))
        et = base + p * wide
        n = B * Sq * Sk
        for hh in range(H):
            dtable[:, hh] = torch.bincount(which.flatten(), ds[:, hh].flatten(), table.size(0))
            etable[:, hh] = torch.bincount(which.flatten(), (et[:, hh] + min(n, 1 << 14) * E * ds[:, hh].abs()).flatten(), table.size(0))
        res["dtable"] = (dtable, etable)
    dx = ds * slope * scale
    edx = (eds * slope.abs() + ds.abs() * (8 * E * (1 + (softcap or 0))) + (u + 4 * E) * (ds * slope).abs()) * abs(scale)
    share = lambda t: t.view(B, kv, G, Sk, -1).sum(2)
    r = max(u, 2 * E)
    dq = dx @ k
    res["dq"] = (back(dq), back(edx @ k.abs() + Sk * E * (dx.abs() @ k.abs()) + r * dq.abs()))
    T = lambda t: t.transpose(2, 3)
    dk, dv = share(T(dx) @ q), share(T(p) @ do)
    res["dk"] = (back(dk), back(share(T(edx) @ q.abs() + Sq * E * (T(dx).abs() @ q.abs())) + r * dk.abs()))
    res["dv"] = (back(dv), back(share((T(p * (u + w)) @ do.abs()) + Sq * E * (T(p) @ do.abs())) + r * dv.abs()))
    return res


def check(name, got, value, bound, floor=1e-30):
    err = (got.double() - value.reshape(got.shape)).abs()
    over = err > bound.reshape(got.shape) + floor
    assert not got.isnan().any(), f"{name}: NaN"
    assert not over.any(), (f"{name}: {int(over.sum())} of {over.numel()} values beyond their bound, "
                            f"worst {float((err / (bound.reshape(got.shape) + floor)).max()):.2f} times")


def inputs(B, Sq, Sk, heads, kv, d, dtype, seed=0, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k, v = (1.2 * n(B, Sq, heads, d)).to(dtype), (1.2 * n(B, Sk, kv, d)).to(dtype), n(B, Sk, kv, d).to(dtype)
    dout = n(B, Sq, heads, d).to(dtype)
    if grad:
        q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    return g, q, k, v, dout


def attention_case(B, Sq, Sk, heads, kv, d, dtype, seed=0, grad=True, flat=False, **opt):
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(B, Sq, Sk, heads, kv, d, dtype, seed, grad)
    args = [t.flatten(2) for t in (q, k, v)] if flat else [q, k, v]
    out = ops.biased_attention(*args, heads, kv, **opt)
    assert out.shape == args[0].shape and out.dtype == dtype and out.is_contiguous()
    ref = definition(q, k, v, heads, kv, dout=dout if grad else None, **opt)
    check("out", out, *ref["out"])
    if grad:
        table = opt.get("table")
        leaves = [q, k, v] + ([table] if table is not None and table.requires_grad else [])
        grads = torch.autograd.grad(out, leaves, dout.flatten(2) if flat else dout)
        for n, t in zip(("dq", "dk", "dv", "dtable"), grads):
            check(n, t, *ref[n])
    return out


TYPES = [torch.float32, torch.bfloat16]


def padded(B, S, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(1, S + 1, (B, 1), generator=g)
    n[0] = S
    return (torch.arange(S)[None, :] < n).long().cuda()


def slopes_of(heads):
    return (2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32) / heads)).cuda()


def table_of(n, heads, R, both, seed=0, grad=True):
    from nonauto_lm_amd import ops
    t = 0.5 * torch.randn(n, heads, generator=torch.Generator().manual_seed(seed))
    return dict(table=t.cuda().requires_grad_(grad), buckets=ops.relative_buckets(n, R, both, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
def test_attention_head_sizes(d, dtype):
    attention_case(2, 70, 70, 4, 2, d, dtype, seed=d, causal=True, softcap=5.0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257])
def test_attention_lengths(S, dtype):
    attention_case(2, S, S, 2, 1, 32, dtype, seed=S)
    attention_case(1, S, S, 2, 2, 64, dtype, seed=S, causal=True, mask=padded(1, S, S), flat=True)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 300), (3, 129), (40, 41), (130, 260), (5, 700), (33, 64)])
def test_attention_new_tokens_over_longer_keys(Sq, Sk, dtype):
    attention_case(3, Sq, Sk, 6, 3, 48, dtype, seed=Sq + Sk, causal=True, slopes=slopes_of(6))
    # sequences of unequal length, and queries that are not the last positions
    start = torch.tensor([Sk - Sq, 0, (Sk - Sq) // 2], dtype=torch.int32, device="cuda")
    attention_case(3, Sq, Sk, 6, 2, 48, dtype, seed=Sq, causal=True, q_start=start, softcap=20.0)
    attention_case(3, Sq, Sk, 6, 6, 48, dtype, seed=Sq, causal=True, q_start=(Sk - Sq) // 3, **table_of(8, 6, 20, False))
    attention_case(3, Sq, Sk, 6, 6, 48, dtype, seed=Sq, causal=True, q_start=Sk + 7, slopes=slopes_of(6))      # all behind the last key


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_key_mask_with_holes_and_empty_rows(causal, dtype):
    g = torch.Generator().manual_seed(3)
    mask = (torch.rand(4, 150, generator=g) < 0.5).long()
    mask[1] = 0                                   # no key at all: zeros, no gradient
    mask[2, :70] = 0                              # causal: the first 70 rows see nothing
    mask = mask.cuda()
    out = attention_case(4, 150, 150, 2, 2, 32, dtype, mask=mask, causal=causal, softcap=10.0)
    assert out[1].eq(0).all()
    if causal:
        assert out[2, :70].eq(0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_hidden_keys_may_hold_anything(dtype):
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(2, 100, 100, 4, 2, 32, dtype, seed=1, grad=False)
    mask = padded(2, 100, 7)
    mask[1, 40:] = 0
    docs = torch.zeros(2, 100, dtype=torch.int32, device="cuda")
    docs[:, 90:] = -1
    results = []
    for junk in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kk, vv = k.clone(), v.clone()
        kk[mask == 0], vv[mask == 0] = junk, junk
        kk[:, 90:], vv[:, 90:] = junk, junk
        leaves = [t.requires_grad_(True) for t in (q.clone(), kk, vv)]
        out = ops.biased_attention(*leaves, 4, 2, mask=mask, documents=docs)
        results.append([out] + list(torch.autograd.grad(out, leaves, dout)))
    for r in results[1:]:
        for a, b in zip(results[0], r):
            assert torch.equal(a, b)
    assert results[0][2][mask == 0].eq(0).all() and results[0][3][mask == 0].eq(0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_documents(causal, dtype):
    g = torch.Generator().manual_seed(5)
    S = 300
    docs = torch.randint(0, 2, (3, S), generator=g).cumsum(1).to(torch.int32) // 9      # runs of about 18 tokens
    docs[1] = torch.randint(-2, 4, (S,), generator=g).to(torch.int32)                   # any order, some of none
    docs[2, :128], docs[2, 128:256], docs[2, 256:] = 7, 2 ** 31 - 1, -5                 # whole tiles
    docs = docs.cuda()
    out = attention_case(3, S, S, 2, 1, 40, dtype, documents=docs, causal=causal, seed=2, softcap=8.0)
    assert out[docs < 0].eq(0).all()
    attention_case(3, S, S, 2, 2, 64, dtype, documents=docs, causal=causal, mask=padded(3, S, 2), seed=3, slopes=slopes_of(2))
    # the last 50 positions of the same rows, and a start of its own for each
    attention_case(3, 50, S, 2, 2, 64, dtype, documents=docs, causal=causal, seed=4)
    start = torch.tensor([0, 100, 250], dtype=torch.int32, device="cuda")
    attention_case(3, 50, S, 2, 2, 64, dtype, documents=docs, causal=causal, seed=4, q_start=start)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_prefix(dtype):
    S = 200
    prefix = torch.tensor([0, 1, 77, 200, 999, -3], dtype=torch.int32, device="cuda")
    attention_case(6, S, S, 2, 2, 32, dtype, causal=True, prefix=prefix, seed=1)
    attention_case(6, S, S, 2, 1, 64, dtype, causal=True, prefix=prefix, seed=2, mask=padded(6, S, 4), softcap=15.0,
                   **table_of(16, 2, 40, True))
    attention_case(6, 20, S, 2, 1, 64, dtype, causal=True, prefix=prefix, seed=3, q_start=50, slopes=slopes_of(2))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("buckets,R,both", [(2, 1, False), (4, 3, False), (8, 24, True), (32, 128, True), (32, 64, False), (256, 1024, True)])
def test_attention_bucket_bias_and_its_gradient(buckets, R, both, dtype):
    if buckets == 2:
        opt = table_of(2, 4, 2, False)
        opt["buckets"] = torch.tensor([1, 0, 0], dtype=torch.int32, device="cuda")       # a map of one's own
    else:
        opt = table_of(buckets, 4, R, both, seed=R)
    attention_case(3, 180, 180, 4, 2, 32, dtype, seed=R, causal=not both, **opt)
    attention_case(2, 90, 90, 4, 4, 64, dtype, seed=R + 1, mask=padded(2, 90, 1), softcap=6.0, **opt)


@gpu
def test_bucket_values_out_of_range_are_clamped():
    from nonauto_lm_amd import ops
    _, q, k, v, _ = inputs(1, 40, 40, 2, 2, 32, torch.float32, grad=False)
    table = torch.randn(4, 2, device="cuda")
    wild = torch.tensor([-7, 0, 1, 2, 3, 9, 2 ** 30], dtype=torch.int32, device="cuda")
    tame = wild.clamp(0, 3)
    assert torch.equal(ops.biased_attention(q, k, v, 2, table=table, buckets=wild),
                       ops.biased_attention(q, k, v, 2, table=table, buckets=tame))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides_and_layouts(dtype):
    from nonauto_lm_amd import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    B, S, H, G, d = 2, 77, 4, 2, 32
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    q, k, v = n(B, S, H, d), n(B, S, G, d), n(B, S, G, d)
    want = ops.biased_attention(q, k, v, H, G, causal=True)
    packed = torch.cat([t.flatten(2) for t in (q, k, v)], -1)                              # column blocks of one projection
    W = H * d
    got = ops.biased_attention(packed[..., :W], packed[..., W:W + G * d], packed[..., W + G * d:], H, G, causal=True)
    assert torch.equal(got, want.flatten(2))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]      # (B, heads, S, d) in memory
    assert torch.equal(ops.biased_attention(*heads_first, H, G, causal=True), want)
    odd = [torch.empty(t.numel() + 1, device="cuda", dtype=dtype)[1:].view(t.shape).copy_(t) for t in (q, k, v)]     # misaligned
    assert torch.equal(ops.biased_attention(*odd, H, G, causal=True), want)
    long = [torch.cat([t, n(B, 19, t.size(2), d)], 1)[:, :S] for t in (k, v)]              # the filled part of a longer cache
    assert torch.equal(ops.biased_attention(q, *long, H, G, causal=True), want)
    feature = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]          # features not adjacent
    assert torch.equal(ops.biased_attention(*feature, H, G, causal=True), want)
    one = ops.biased_attention(q, k[:1].expand(B, S, G, d), v[:1].expand(B, S, G, d), H, G, causal=True)     # one cache for all rows
    assert torch.equal(one, ops.biased_attention(q, k[:1].repeat(B, 1, 1, 1), v[:1].repeat(B, 1, 1, 1), H, G, causal=True))
    # a gradient that comes broadcast (out.sum())
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    ops.biased_attention(*leaves, H, G, causal=True).float().sum().backward()
    ref = definition(*leaves, H, G, causal=True, dout=torch.ones(B, S, H, d, device="cuda"))
    for name, t in zip(("dq", "dk", "dv"), leaves):
        check(name, t.grad, *ref[name])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(dtype):
    """rows whose scores span hundreds: the running maximum has to follow; and scores that are all alike"""
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(1, 160, 160, 2, 2, 32, dtype, seed=4, grad=False)
    q, k = q * 6, k * 6
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = ops.biased_attention(*leaves, 2, scale=1.0)
    ref = definition(*leaves, 2, 2, scale=1.0, dout=dout)
    check("out", out, *ref["out"])
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)):
        check(n, t, *ref[n])
    out = ops.biased_attention(torch.zeros_like(q), k, v, 2)
    check("out", out, *definition(torch.zeros_like(q), k, v, 2, 2)["out"])


@gpu
def test_attention_partial_gradients_and_repeats():
    """only some inputs learn; the same call twice gives the same bits"""
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(2, 140, 140, 4, 2, 64, torch.bfloat16, seed=9)
    opt = table_of(32, 4, 64, True)
    full = torch.autograd.grad(ops.biased_attention(q, k, v, 4, 2, **opt), [q, k, v, opt["table"]], dout)
    again = torch.autograd.grad(ops.biased_attention(q, k, v, 4, 2, **opt), [q, k, v, opt["table"]], dout)
    assert all(torch.equal(a, b) for a, b in zip(full, again))
    det = lambda t: t.detach()
    out = ops.biased_attention(det(q), det(k), det(v), 4, 2, **opt)
    assert torch.equal(torch.autograd.grad(out, opt["table"], dout)[0], full[3])
    fixed = {n: t.detach() for n, t in opt.items()}
    out = ops.biased_attention(det(q), k, det(v), 4, 2, **fixed)
    dk = torch.autograd.grad(out, k, dout)[0]
    check("dk", dk, *definition(q, k, v, 4, 2, dout=dout, **fixed)["dk"])
    out = ops.biased_attention(q, det(k), det(v), 4, 2, **fixed)
    check("dq", torch.autograd.grad(out, q, dout)[0], *definition(q, k, v, 4, 2, dout=dout, **fixed)["dq"])


@gpu
def test_attention_gradients_against_differences():
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(1, 24, 24, 2, 1, 16, torch.float32, seed=11)
    opt = table_of(8, 2, 12, False)
    loss = lambda *a: (ops.biased_attention(*a[:3], 2, 1, causal=True, softcap=4.0, table=a[3], buckets=opt["buckets"]).double()
                       * dout.double()).sum()
    leaves = [q, k, v, opt["table"]]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    g = torch.Generator(device="cuda").manual_seed(1)
    for n, t in enumerate(leaves):
        step = torch.randn(t.shape, device="cuda", generator=g)
        moved = [[x + s * 2.0 ** -6 * step if m == n else x for m, x in enumerate(leaves)] for s in (1, -1)]
        with torch.no_grad():
            diff = float(loss(*moved[0]) - loss(*moved[1])) * 2.0 ** 5
        want = float((grads[n].double() * step.double()).sum())
        # a central difference is off by h^2 / 6 of a third derivative (h = 2^-6), and its fp32 values by 1e-6 / h
        assert abs(diff - want) <= 2e-3 * (abs(want) + float(grads[n].double().norm() * step.double().norm()))


@gpu
def test_attention_captured_and_replayed():
    from nonauto_lm_amd import ops
    g, q, k, v, _ = inputs(2, 130, 130, 4, 2, 64, torch.bfloat16, seed=3, grad=False)
    opt = table_of(32, 4, 64, True, grad=False)
    mask = padded(2, 130, 3)
    docs = (torch.arange(130, device="cuda") // 50).to(torch.int32).expand(2, 130).contiguous()
    call = lambda: ops.biased_attention(q, k, v, 4, 2, mask=mask, documents=docs, **opt)
    tok = lambda: ops.biased_attention(q[:, -1:], k, v, 4, 2, causal=True, slopes=slopes)
    slopes = slopes_of(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(), tok()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, one = call(), tok()
    for _ in range(3):
        q.normal_(generator=g)
        k.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()) and torch.equal(one, tok())


@gpu
def test_attention_on_a_side_stream():
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(2, 200, 200, 4, 4, 64, torch.bfloat16, seed=5)
    want = ops.biased_attention(q, k, v, 4, causal=True)
    grads = torch.autograd.grad(want, [q, k, v], dout)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = ops.biased_attention(q, k, v, 4, causal=True)
        got = torch.autograd.grad(out, [q, k, v], dout)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, grads))


@gpu
def test_attention_offsets_beyond_32_bits():
    """keys whose batch rows lie more than 2^32 elements apart"""
    from nonauto_lm_amd import ops
    S, G, d = 64, 1, 32
    room = torch.empty(2 ** 32 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    k = torch.as_strided(room, (2, S, G, d), (2 ** 32, G * d, d, 1))
    v = torch.as_strided(room, (2, S, G, d), (2 ** 32, G * d, d, 1), S * G * d)
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in (k, v):
        for b in range(2):
            t[b] = torch.randn(S, G, d, device="cuda", generator=g).to(torch.bfloat16)
    q = torch.randn(2, 40, 2, d, device="cuda", generator=g).to(torch.bfloat16)
    assert torch.equal(ops.biased_attention(q, k, v, 2, 1), ops.biased_attention(q, k.clone(), v.clone(), 2, 1))
    assert torch.equal(ops.biased_attention(q[:, :1], k, v, 2, 1), ops.biased_attention(q[:, :1], k.clone(), v.clone(), 2, 1))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq,heads,kv,d", [(1, 4, 4, 64), (1, 32, 1, 128), (4, 12, 3, 80), (16, 4, 1, 32), (7, 33, 11, 16)])
def test_few_queries_with_masks_documents_prefix_and_bias(Sq, heads, kv, d, dtype):
    """the split form: packed rows of several tiles, key splits that end inside a tile, rows and splits that see nothing"""
    B, Sk = 3, 333
    g = torch.Generator().manual_seed(Sq)
    mask = (torch.rand(B, Sk, generator=g) < 0.6).long().cuda()
    mask[1] = 0
    docs = torch.randint(-1, 3, (B, Sk), generator=g).sort(1)[0].to(torch.int32).cuda()
    start = torch.tensor([Sk - Sq, 3, 100], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([0, 50, 400], dtype=torch.int32, device="cuda")
    grad = dtype == torch.float32 or Sq != 7
    attention_case(B, Sq, Sk, heads, kv, d, dtype, seed=1, grad=grad, mask=mask, causal=True, q_start=start, softcap=9.0)
    attention_case(B, Sq, Sk, heads, kv, d, dtype, seed=2, grad=grad, documents=docs, q_start=start, slopes=slopes_of(heads))
    attention_case(B, Sq, Sk, heads, kv, d, dtype, seed=3, grad=grad, documents=docs, mask=mask, causal=True, prefix=prefix,
                   q_start=start, **table_of(16, heads, 40, True))
    attention_case(B, Sq, Sk, heads, kv, d, dtype, seed=4, grad=False, **table_of(256, heads, 1024, True, grad=False))


@gpu
@pytest.mark.parametrize("dtype,d,causal", [(torch.bfloat16, 128, True), (torch.bfloat16, 64, False), (torch.float32, 96, True)])
def test_attention_longer_rows(dtype, d, causal):
    """many chunks, several parts of a walk, several document tiles beyond the first 64"""
    S = 4500 if dtype == torch.bfloat16 else 1500
    docs = (torch.arange(S, device="cuda") // 700).to(torch.int32)[None]
    attention_case(1, S, S, 2, 1, d, dtype, seed=1, causal=causal, softcap=30.0, documents=docs)
    attention_case(1, S, S, 2, 1, d, dtype, seed=2, causal=causal, **table_of(32, 2, 300, not causal))


@gpu
def test_attention_many_rows_of_one_length():
    """the block order over XCDs: pairs that divide by 8 and that do not, with and without a causal mask"""
    for B, heads, kv in ((9, 4, 4), (8, 4, 2), (33, 1, 1), (16, 2, 1)):
        for causal in (False, True):
            attention_case(B, 140, 140, heads, kv, 16, torch.bfloat16, seed=B, causal=causal, mask=padded(B, 140, B))


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_forward_and_backward_captured(dtype, d):
    """a whole pass of both operators in one graph, replayed on new values with eager work in between"""
    from nonauto_lm_amd import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    B, S, H, G = 2, 150, 4, 2
    n = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
    static = [n(B, S, H, d), n(B, S, G, d), n(B, S, G, d), n(B, S, H, d)]
    const = dict(frequencies=ops.rotary_frequencies(d, device="cuda"))
    opt = table_of(32, H, 64, False)
    qw = torch.ones(d, device="cuda")
    mask = padded(B, S, 1)

    def passes():
        q, k, v = (t.detach().requires_grad_(True) for t in static[:3])          # leaves of this pass alone
        w, table = qw.detach().requires_grad_(True), opt["table"].detach().requires_grad_(True)
        rq, rk = ops.qk_norm_rotary(q, k, H, G, q_weight=w, k_weight=w, **const)
        out = ops.biased_attention(rq, rk, v, H, G, mask=mask, causal=True, softcap=20.0, table=table, buckets=opt["buckets"])
        return [out.detach()] + list(torch.autograd.grad(out, [q, k, v, w, table], static[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = passes()
    for _ in range(3):
        for t in static:
            t.copy_(n(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, passes()):
            assert torch.equal(a, b)


@gpu
def test_attention_saved_state():
    """one graph walked twice, operands that are one tensor, a constant that changed between the passes"""
    from nonauto_lm_amd import ops
    x = torch.randn(2, 50, 2, 32, device="cuda").requires_grad_(True)
    dout = torch.randn(2, 50, 2, 32, device="cuda")
    out = ops.biased_attention(x, x, x, 2, causal=True, slopes=slopes_of(2))
    a = torch.autograd.grad(out, x, dout, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(out, x, dout)[0])
    leaves = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    parts = torch.autograd.grad(ops.biased_attention(*leaves, 2, causal=True, slopes=slopes_of(2)), leaves, dout)
    torch.testing.assert_close(a, parts[0] + parts[1] + parts[2], rtol=0, atol=8 * E * float(a.abs().max() + 1))
    prefix = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    out = ops.biased_attention(x, x, x, 2, causal=True, prefix=prefix)
    prefix.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, x, dout)
    with pytest.raises(RuntimeError):                                            # no second derivative
        y = ops.biased_attention(x, x, x, 2)
        torch.autograd.grad(torch.autograd.grad(y.sum(), x, create_graph=True)[0].sum(), x)


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.float32, 32), (torch.bfloat16, 32), (torch.bfloat16, 128)])
def test_queries_that_see_nothing_may_hold_anything(dtype, d):
    """causal rows before the first visible key, rows before the keys, padded documents: their q and dout meet no product"""
    from nonauto_lm_amd import ops
    B, S = 2, 170
    for case in range(4):
        mask = torch.ones(B, S, dtype=torch.long, device="cuda")
        docs = start = None
        blind = torch.zeros(B, S, dtype=torch.bool, device="cuda")
        rows = S
        if case == 0:                                # left padding
            mask[0, :75] = 0
            mask[1] = 0
            blind = mask == 0
        elif case == 1:
            docs = (torch.arange(S, device="cuda") // 50).to(torch.int32).repeat(B, 1)
            docs[:, 100:135] = -1
            blind = docs < 0
        elif case == 2:
            start = torch.tensor([-40, -500], dtype=torch.int32, device="cuda")
            blind = torch.arange(S, device="cuda")[None] + start[:, None] < 0
        else:                                        # few queries
            rows = 9
            start = torch.tensor([-4, 100], dtype=torch.int32, device="cuda")
            blind = torch.arange(rows, device="cuda")[None] + start[:, None] < 0
        _, q, k, v, dout = inputs(B, rows, S, 4, 2, d, dtype, seed=case, grad=False)
        opt = dict(mask=mask, causal=True, documents=docs, q_start=start)
        for bias in ({}, table_of(8, 4, 20, True)):
            zero = blind[..., None, None]
            ref = definition(q.masked_fill(zero, 0), k, v, 4, 2, softcap=20.0, dout=dout.masked_fill(zero, 0), **opt, **bias)
            for junk in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
                leaves = [t.clone().requires_grad_(True) for t in (q.masked_fill(zero, junk), k, v)] + [t for n, t in bias.items() if n == "table"]
                out = ops.biased_attention(*leaves[:3], 4, 2, softcap=20.0, **opt, **bias)
                grads = torch.autograd.grad(out, leaves, dout.masked_fill(zero, junk))
                # (a tile's scores take one of two forms of the cap together, so rows next to junk may round otherwise: bounds, not bits)
                for n, t in zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)):
                    check(n, t, *ref[n])
                assert out[blind].eq(0).all() and grads[0][blind].eq(0).all()


@gpu
@pytest.mark.parametrize("dtype,d", [(torch.float32, 48), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("Sq", [1, 7, 16, 40, 150])
def test_unwritten_end_of_a_cache(Sq, dtype, d):
    """keys behind the last query's limit hold NaN: same bits as zeros, no gradient; with and without a mask, documents, a prefix"""
    from nonauto_lm_amd import ops
    B, Sk = 3, 500
    _, q, k, v, dout = inputs(B, Sq, Sk, 4, 2, d, dtype, seed=Sq, grad=False)
    start = torch.tensor([0, 33, 250], dtype=torch.int32, device="cuda")
    prefix = torch.tensor([0, 60, 0], dtype=torch.int32, device="cuda")
    for opt in (dict(), dict(mask=(torch.arange(Sk, device="cuda") % 3 > 0).long().expand(B, Sk)), dict(prefix=prefix),
                dict(documents=(torch.arange(Sk, device="cuda") // 120).to(torch.int32).repeat(B, 1)), dict(slopes=slopes_of(4))):
        limit = start + Sq
        if "prefix" in opt:
            limit = torch.maximum(limit, prefix)
        behind = torch.arange(Sk, device="cuda")[None] >= limit[:, None]
        results = []
        for junk in (0.0, float("nan"), float("inf")):
            fill = lambda t: t.masked_fill(behind[..., None, None], junk)
            leaves = [q.clone().requires_grad_(True), fill(k).requires_grad_(True), fill(v).requires_grad_(True)]
            out = ops.biased_attention(*leaves, 4, 2, causal=True, q_start=start, **opt)
            with torch.no_grad():
                assert torch.isfinite(ops.biased_attention(*leaves, 4, 2, causal=True, q_start=start, **opt)).all()
            results.append([out] + list(torch.autograd.grad(out, leaves, dout)))
        for r in results:
            for a, b in zip(results[0], r):
                assert torch.equal(a, b)
            assert r[2][behind].eq(0).all() and r[3][behind].eq(0).all()


@gpu
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("dtype", TYPES)
def test_table_entries_that_hide(dtype, low):
    """-inf or a lowest value in the table: those distances are out, as with a mask of that shape; a row with nothing left is zero"""
    from nonauto_lm_amd import ops
    S, R, H = 200, 40, 2
    _, q, k, v, dout = inputs(2, S, S, H, H, 32, dtype, seed=5)
    opt = table_of(4, H, R, False)
    buckets = torch.arange(-R, R + 1, device="cuda").abs()
    for seen in (buckets < 16, buckets == R, buckets == R + 1):               # near, far, none
        table = opt["table"].detach().clone()
        table[3] = low
        ids = torch.where(seen, torch.randint(0, 3, seen.shape, device="cuda"), 3).to(torch.int32)
        table.requires_grad_(True)
        out = ops.biased_attention(q, k, v, H, table=table, buckets=ids)
        grads = torch.autograd.grad(out, [q, k, v, table], dout)
        rel = torch.arange(S, device="cuda")[None] - torch.arange(S, device="cuda")[:, None]
        finite = table.detach().clone()
        finite[3] = 0
        ref = definition(q, k, v, H, H, dout=dout, table=finite.requires_grad_(True), buckets=ids, pairs=seen[rel.clamp(-R, R) + R])
        for n, t in zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)):
            check(n, t, *ref[n])
        assert grads[3][3].eq(0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_widest_heads_with_the_longest_table(dtype):
    """the largest LDS blocks: heads of 128, 2049 distances and their gradient"""
    attention_case(1, 150, 150, 2, 1, 128, dtype, seed=1, softcap=25.0, **table_of(256, 2, 1024, True))
    attention_case(1, 1500, 1500, 1, 1, 128, dtype, seed=2, causal=True, **table_of(64, 1, 1024, False))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_two_calls_in_flight(dtype):
    """forward and backward on two streams at once: every call has workspaces of its own"""
    from nonauto_lm_amd import ops
    mask = padded(2, 400, 3)
    sets = [inputs(2, 400, 400, 4, 2, 64, dtype, seed=s)[1:] for s in (1, 2)]
    tables = [table_of(16, 4, 50, True, seed=s) for s in (1, 2)]

    def passes(i):
        q, k, v, dout = sets[i]
        out = ops.biased_attention(q, k, v, 4, 2, mask=mask, causal=True, **tables[i])
        return [out.detach()] + list(torch.autograd.grad(out, [q, k, v, tables[i]["table"]], dout))

    want = [passes(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(passes(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def refusals(fn, bad):
    for opt, match in bad:
        with pytest.raises(ValueError, match=match):
            fn(**opt)


def test_attention_refusals(monkeypatch):
    """every refusal is the host's, before anything touches a GPU"""
    from nonauto_lm_amd import _lib, ops
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.biased_attention(*[torch.zeros(1, 4, 32)] * 3, 2)
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    z = torch.zeros
    base = dict(q=z(2, 6, 64), k=z(2, 9, 32), v=z(2, 9, 32), heads=4, kv_heads=2)
    i32 = lambda *s: z(*s, dtype=torch.int32)
    tab = dict(table=z(8, 4), buckets=i32(5))
    refusals(lambda **o: ops.biased_attention(**{**base, **o}), [
        (dict(q=z(2, 6, 64).half(), k=z(2, 9, 32).half(), v=z(2, 9, 32).half()), "float32 or bfloat16"),
        (dict(k=z(2, 9, 32).bfloat16()), "float32 or bfloat16"),
        (dict(heads=3), "heads over"), (dict(kv_heads=0), "heads over"), (dict(heads=5, kv_heads=1), "neither"),
        (dict(v=z(2, 8, 32)), "do not match"), (dict(k=z(1, 9, 32), v=z(1, 9, 32)), "do not match"),
        (dict(q=z(2, 6, 48), k=z(2, 9, 24), v=z(2, 9, 24)), "head size 12"),
        (dict(q=z(2, 6, 4 * 136), k=z(2, 9, 2 * 136), v=z(2, 9, 2 * 136)), "head size 136"),
        (dict(q=z(0, 6, 64), k=z(0, 9, 32), v=z(0, 9, 32)), "batch 0"), (dict(k=z(2, 0, 32), v=z(2, 0, 32)), "lengths 6 and 0"),
        (dict(mask=torch.ones(2, 6)), "mask"), (dict(prefix=i32(2)), "needs causal"),
        (dict(prefix=i32(3), causal=True), "prefix must be"), (dict(prefix=z(2), causal=True), "prefix must be"),
        (dict(documents=z(2, 9, dtype=torch.int64)), "documents must be"), (dict(documents=i32(2, 6)), "documents must be"),
        (dict(slopes=z(2)), "slopes must be"), (dict(slopes=z(4, requires_grad=True)), "no gradient"),
        (dict(table=z(8, 4)), "come together"), (dict(buckets=i32(5)), "come together"), (dict(slopes=z(4), **tab), "come together"),
        (dict(table=z(8, 2), buckets=i32(5)), "table must be"), (dict(table=z(257, 4), buckets=i32(5)), "table must be"),
        (dict(table=z(8, 4).bfloat16(), buckets=i32(5)), "table must be"),
        (dict(table=z(8, 4), buckets=i32(4)), "odd length"), (dict(table=z(8, 4), buckets=i32(2051)), "odd length"),
        (dict(table=z(8, 4), buckets=z(5)), "odd length"),
        (dict(softcap=0.0), "softcap"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
        (dict(softcap=float("inf")), "softcap"), (dict(softcap=1e-31), "too small"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=-0.5), "scale"),
        (dict(q=z(2, 10, 64)), "start at position -1"), (dict(q_start=-1), "start at position"),
        (dict(q_start=4, documents=i32(2, 9)), "documents reach"), (dict(q_start=z(2)), "q_start must be"),
        (dict(q_start=i32(3)), "q_start must be"),
    ])
    for bad in ((7, 16, True), (2, 16, True), (8, 2, True), (1, 16, False)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*bad)


def test_relative_buckets_values():
    from nonauto_lm_amd import ops
    both = ops.relative_buckets(8, 16, True).tolist()
    assert both[16] == 0 and both[15] == 1 and both[17] == 5 and both[14] == 2 and both[0] == 3 and both[-1] == 7
    past = ops.relative_buckets(8, 16, False).tolist()
    assert past[16:] == [0] * 17 and past[12:16] == [4, 3, 2, 1] and past[0] == 7 and sorted(past, reverse=True) == past
    assert ops.relative_buckets(32, 128).dtype == torch.int32 and int(ops.relative_buckets(32, 128).max()) == 31


# ------------------------------------------------------------------------------------------------ norm and rotation
def rotary_definition(x, w, freqs, pos, eps, norm, interleaved, dy):
    """64-bit values and bounds of y, dx, dw for x, dy (B, S, heads, d)"""
    u = max(U[x.dtype], 2 * E)
    x, dy = x.detach().double(), dy.double()
    d = x.size(-1)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    n = x * r * w
    m = 0 if freqs is None else freqs.numel()
    first = torch.arange(m, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else m)

    def turn(t, sign):
        if not m:
            return t
        turns = pos.double()[..., None] * freqs
        a = 2 * math.pi * (turns - turns.round())[:, :, None, :] * sign
        t = t.clone()
        ta, tb = t[..., first], t[..., second]
        t[..., first], t[..., second] = ta * a.cos() - tb * a.sin(), ta * a.sin() + tb * a.cos()
        return t

    def size(t):            # |a| + |b| of a pair bounds every term of its rotation
        t = t.abs().clone()
        if m:
            s = t[..., first] + t[..., second]
            t[..., first] = t[..., second] = s
        return t

    # steps: the row's sum (d), its root and reciprocal, scales, angle (2 pi 2^-25, i.e. 4 steps), products
    f = (d + 24) * E
    y = turn(n, 1)
    g = turn(dy, -1)
    gw = g * w
    xr = x * r
    mean = (gw * xr).mean(-1, keepdim=True)
    dx = r * (gw - xr * mean) if norm else g
    amean = (size(dy) * w.abs() * xr.abs()).mean(-1, keepdim=True)
    edx = f * r * (size(dy) * w.abs() + 2 * xr.abs() * amean)
    dw = (g * xr).sum((0, 1, 2))
    rows = x.numel() // d
    edw = (f + min(rows, 4096) * E) * (size(dy) * xr.abs()).sum((0, 1, 2))
    return (y, f * size(n) + u * y.abs()), (dx, edx + u * dx.abs()), (dw, edw)


def rotary_case(B, S, heads, kv, d, dtype, rot=None, norm=True, weights=True, interleaved=False, far=0, eps=1e-6, seed=0, pos="row"):
    from nonauto_lm_amd import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k = (1.5 * n(B, S, heads, d)).to(dtype).requires_grad_(True), (1.5 * n(B, S, kv, d)).to(dtype).requires_grad_(True)
    qw, kw = ((1 + 0.2 * n(d)).requires_grad_(True) for _ in range(2)) if norm and weights else (None, None)
    freqs = ops.rotary_frequencies(rot, device="cuda") if rot else None
    where = {"row": None, "int": far, "s": torch.arange(S, device="cuda") + far,
             "bs": far + torch.randint(0, far + 7, (B, S), device="cuda", generator=g)}[pos]
    p = torch.arange(S, device="cuda").expand(B, S) + (far if pos == "int" else 0) if not torch.is_tensor(where) else where.expand(B, S)
    yq, yk = ops.qk_norm_rotary(q, k, heads, kv, q_weight=qw, k_weight=kw, eps=eps, frequencies=freqs, positions=where,
                                norm=norm, interleaved=interleaved)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.dtype == dtype
    dyq, dyk = n(B, S, heads, d).to(dtype), n(B, S, kv, d).to(dtype)
    leaves = [q, k] + ([qw, kw] if qw is not None else [])
    grads = torch.autograd.grad((yq, yk), leaves, (dyq, dyk))
    for i, (x, w, y, dy) in enumerate(((q, qw, yq, dyq), (k, kw, yk, dyk))):
        ry, rdx, rdw = rotary_definition(x, w, freqs, p, eps, norm, interleaved, dy)
        check("qk"[i], y, *ry)
        check("dqk"[i + 1], grads[i], *rdx)
        if w is not None:
            check("weight", grads[2 + i], *rdw)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(2, 2), (6, 4), (16, 16), (32, 16), (34, 34), (64, 64), (64, 32), (80, 80), (96, 48), (100, 20),
                                   (128, 128), (130, 2), (254, 254), (256, 256), (256, 128), (64, None), (50, None)])
def test_rotary_head_sizes(d, rot, interleaved, dtype):
    rotary_case(2, 9, 3, 1, d, dtype, rot, interleaved=interleaved, seed=d)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,heads,kv", [(1, 1, 1, 1), (8, 1, 8, 2), (1, 700, 2, 2), (3, 333, 12, 3), (40, 17, 32, 1)])
def test_rotary_shapes(B, S, heads, kv, dtype):
    rotary_case(B, S, heads, kv, 64, dtype, 64, far=50000, pos="bs", seed=S)
    rotary_case(B, S, heads, kv, 48, dtype, 20, far=3, pos="int", weights=False, seed=S)
    rotary_case(B, S, heads, kv, 32, dtype, 32, far=2 ** 31 + 12345, pos="s", norm=False, seed=S)


@gpu
def test_rotary_zero_rows_and_layouts():
    from nonauto_lm_amd import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2, 5, 3 * 64, device="cuda", generator=g).to(torch.bfloat16)
    f = ops.rotary_frequencies(32, device="cuda")
    q, k = x[..., :128], x[..., 128:]                               # blocks of one projection, no copy
    want = ops.qk_norm_rotary(q.contiguous(), k.contiguous(), 4, 2, frequencies=f)
    for a, b in zip(ops.qk_norm_rotary(q, k, 4, 2, frequencies=f), want):
        assert torch.equal(a, b)
    hf = lambda t, h: t.unflatten(2, (h, 32)).transpose(1, 2).contiguous().transpose(1, 2)
    for a, b in zip(ops.qk_norm_rotary(hf(q, 4), hf(k, 2), 4, 2, frequencies=f), want):
        assert torch.equal(a.flatten(2), b)
    zero = torch.zeros(1, 3, 64, device="cuda", requires_grad=True)
    a, b = ops.qk_norm_rotary(zero, zero, 2, frequencies=f)
    assert a.eq(0).all() and torch.autograd.grad(a.sum() + b.sum(), zero)[0].isfinite().all()
    empty = torch.zeros(0, 3, 64, device="cuda")
    assert ops.qk_norm_rotary(empty, empty, 2, frequencies=f)[0].shape == (0, 3, 64)


@gpu
def test_rotary_captured_and_replayed():
    from nonauto_lm_amd import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k = torch.randn(2, 6, 4, 64, device="cuda", generator=g), torch.randn(2, 6, 2, 64, device="cuda", generator=g)
    f, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(6, device="cuda")
    call = lambda: ops.qk_norm_rotary(q, k, 4, 2, frequencies=f, positions=pos)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        q.normal_(generator=g)
        pos.add_(11)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call()))


def test_rotary_refusals(monkeypatch):
    from nonauto_lm_amd import _lib, ops
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.qk_norm_rotary(torch.zeros(1, 2, 8), torch.zeros(1, 2, 8), 2)
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    z = torch.zeros
    base = dict(q=z(2, 5, 64), k=z(2, 5, 32), heads=4, kv_heads=2)
    f64 = lambda n: z(n, dtype=torch.float64)
    refusals(lambda **o: ops.qk_norm_rotary(**{**base, **o}), [
        (dict(q=z(2, 5, 64).half(), k=z(2, 5, 32).half()), "float32 or bfloat16"), (dict(k=z(2, 5, 32).bfloat16()), "float32 or bfloat16"),
        (dict(k=z(2, 4, 32)), "does not match"), (dict(k=z(2, 5, 48), kv_heads=2), "does not match"), (dict(heads=5), "neither"),
        (dict(q=z(2, 5, 36), k=z(2, 5, 18)), "head size 9"), (dict(q=z(2, 5, 4 * 258), k=z(2, 5, 2 * 258)), "head size 258"),
        (dict(q_weight=z(8)), "q_weight must be"), (dict(k_weight=z(16).bfloat16()), "k_weight must be"),
        (dict(norm=False), "neither"), (dict(norm=False, frequencies=f64(4), q_weight=z(16)), "q_weight must be"),
        (dict(frequencies=z(4)), "frequencies must be"), (dict(frequencies=f64(9)), "frequencies must be"),
        (dict(frequencies=f64(0)), "frequencies must be"), (dict(frequencies=f64(4).requires_grad_(True)), "no gradient"),
        (dict(frequencies=f64(4), positions=z(5)), "positions must be"), (dict(frequencies=f64(4), positions=z(2, dtype=torch.int64)), "positions must be"),
        (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    ])
    for bad in ((0, 10.0), (3, 10.0), (4, 0.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(*bad)


def test_entry_points_refuse_without_a_launch():
    """the C entry points check their argument structs themselves: a status and a text, nothing enqueued"""
    import ctypes
    from nonauto_lm_amd import _lib as L
    lib = L.lib()
    p = 1 << 20                                       # never read: every call below is refused
    base = dict(q=p, k=p, v=p, out=p, batch=2, q_len=40, k_len=40, heads=4, kv_heads=2, head_size=32, q_stride=(5120, 128, 32),
                k_stride=(2560, 64, 32), v_stride=(2560, 64, 32), scale=0.2, dtype=1)
    for bad, text in ((dict(dtype=2), "dtype"), (dict(kv_heads=3), "heads"), (dict(head_size=20), "head size"), (dict(head_size=136), "head size"),
                      (dict(q_len=0), "lengths"), (dict(k_len=1 << 25), "lengths"), (dict(q=p + 8), "aligned"), (dict(v=None), "null"),
                      (dict(q_stride=(5120, 127, 32)), "stride"), (dict(k_stride=(-64, 64, 32)), "stride"), (dict(prefix=p), "causal"),
                      (dict(softcap=-1.0), "softcap"), (dict(softcap=1e-31), "too small"), (dict(scale=float("nan")), "scale"), (dict(slopes=p, table=p, buckets=p), "alternatives"),
                      (dict(table=p, num_buckets=4, distance=4), "buckets"), (dict(table=p, buckets=p, num_buckets=300, distance=4), "buckets"),
                      (dict(table=p, buckets=p, num_buckets=4, distance=2000), "distance"), (dict(mask=p), "codes"),
                      (dict(q_start=-1), "q_start"), (dict(out=None), "out"), (dict(out_lo=p), "out_lo"), (dict(q_len=1, k_len=4000), "scratch"),
                      (dict(batch=1 << 26), "many")):
        rc = lib.mivae_biased_attention_fwd(ctypes.byref(L.AttentionArgs(**{**base, **bad})), None)
        assert rc == -1 and text in lib.mivae_last_error().decode(), (bad, lib.mivae_last_error())
    back = dict(base, lse=p, dout=p, scratch=p, dq=p)
    for bad, text in ((dict(lse=None), "null"), (dict(dk=p), "together"), (dict(dtable=p), "table"), (dict(scratch=p + 4), "scratch"), (dict(dq=p + 2), "aligned")):
        rc = lib.mivae_biased_attention_bwd(ctypes.byref(L.AttentionArgs(**{**back, **bad})), None)
        assert rc == -1 and text in lib.mivae_last_error().decode(), (bad, lib.mivae_last_error())
    rot = dict(q=p, k=p, q_out=p, k_out=p, batch=2, len=3, heads=4, kv_heads=2, head_size=32, q_stride=(384, 128, 32), k_stride=(192, 64, 32),
               eps=1e-6, norm=1, dtype=0)
    for bad, text in ((dict(dtype=5), "dtype"), (dict(head_size=31), "head size"), (dict(head_size=258), "head size"), (dict(batch=0), "batch"),
                      (dict(heads=4095), "heads"), (dict(batch=1 << 20, len=1 << 12), "batch"), (dict(freq=p, rotary_dim=34), "rotary"),
                      (dict(freq=p, rotary_dim=3), "rotary"), (dict(norm=0), "neither"), (dict(norm=0, freq=p, rotary_dim=4, q_weight=p), "weights"),
                      (dict(eps=-1.0), "eps"), (dict(q_out=None), "output"), (dict(k=None), "operand"), (dict(dq_weight=p), "weight gradients")):
        rc = lib.mivae_qk_norm_rotary_fwd(ctypes.byref(L.RotaryArgs(**{**rot, **bad})), None)
        assert rc == -1 and text in lib.mivae_last_error().decode(), (bad, lib.mivae_last_error())
    assert lib.mivae_qk_norm_rotary_bwd(ctypes.byref(L.RotaryArgs(**rot)), None) == -1 and "gradient" in lib.mivae_last_error().decode()
    assert lib.mivae_biased_attention_fwd(None, None) == -1 and lib.mivae_qk_norm_rotary_fwd(None, None) == -1
