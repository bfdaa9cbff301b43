"""Workloads of the attention sublayer's operators: what is measured, and the plain form each kernel is held to.

Three operators sit between the q / k / v projections and the output projection of a transformer layer:

  rotary     `ops.qk_norm_rotary`: root-mean-square norm of every query and key head, learned scale, position rotation
  attention  `ops.biased_attention`: scores capped by a tanh, distance slopes, key / document / prefix masks, shared
             key heads, and its form for a few new tokens over a long run of keys
  bias       `ops.biased_attention` with a learned relative position bias by buckets, and the table's gradient

`listed()` holds the fixed cases, `draw(rng)` gives more of the same ranges, `prepare` makes the inputs, `run` is one
pass (plain torch where `own` is False, the package's kernels where it is True), `work` counts bytes and operations and
`exact` restates the operators in 64 bits.
"""
import math

import torch

own = False

if torch.cuda.is_available():
    DEV = torch.device("cuda")
else:
    DEV = torch.device("cpu")

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
BASE = 10000.0


# ------------------------------------------------------------------------------------------------- cases
def _rotary(name, B, S, heads, kv, d, dtype, grad, far, rot=None, interleaved=False):
    return dict(name=name, op="rotary", B=B, S=S, heads=heads, kv=kv, d=d, rot=d if rot is None else rot, dtype=dtype,
                grad=grad, far=far, interleaved=interleaved)


def _attention(name, B, Sq, Sk, heads, kv, d, dtype, grad, causal=False, mask=False, prefix=False, docs=0, cap=0.0,
               slopes=False, buckets=0, distance=0, ragged=False):
    return dict(name=name, op="bias" if buckets else "attention", B=B, Sq=Sq, Sk=Sk, heads=heads, kv=kv, d=d, dtype=dtype,
                grad=grad, causal=causal, mask=mask, prefix=prefix, docs=docs, cap=cap, slopes=slopes, buckets=buckets,
                distance=distance, ragged=ragged)


def listed():
    return [
        # one new token per sequence on its way into the attention of a generating model: launch latency counts
        _rotary("rotary-token", 8, 1, 8, 2, 64, "bf16", False, 100000),
        # the layer of the widest training configuration (64 x 512 tokens, 4 heads of 128), forward + backward
        _rotary("rotary-train", 64, 512, 4, 4, 128, "bf16", True, 0),
        # long documents in fp32, a head size that is no power of two, half of it rotated
        _rotary("rotary-long-fp32", 2, 8191, 16, 4, 96, "fp32", True, 30000, rot=48),
        # the encoder layer of the 128-token training configuration: padded sentences, capped scores
        _attention("train-sentences", 256, 128, 128, 4, 4, 64, "bf16", True, mask=True, cap=30.0),
        # sentences packed behind one another into rows of 4096, each seeing only itself
        _attention("train-documents", 4, 4096, 4096, 16, 16, 64, "bf16", True, causal=True, docs=600, cap=50.0),
        # a given beginning that is seen from everywhere, distance slopes, shared key heads, fp32, odd length
        _attention("train-prefix-fp32", 4, 1001, 1001, 8, 2, 80, "fp32", True, causal=True, prefix=True, slopes=True),
        # a long prompt read in one pass, no gradient
        _attention("read-prompt", 1, 8191, 8191, 16, 4, 128, "bf16", False, causal=True, cap=30.0),
        # the layer of the widest training configuration with learned relative positions and padded rows
        _attention("bias-train", 64, 512, 512, 4, 4, 128, "bf16", True, mask=True, buckets=32, distance=128),
        # a small fp32 model's layer of odd length: latency
        _attention("bias-small-fp32", 8, 33, 33, 4, 4, 16, "fp32", True, mask=True, buckets=16, distance=24),
        # long causal rows with learned relative positions
        _attention("bias-long", 4, 4096, 4096, 16, 4, 64, "bf16", True, causal=True, buckets=32, distance=256),
        # one new token for each of 32 sequences of unequal length over long key / value rows
        _attention("token-long", 32, 1, 8192, 32, 8, 128, "bf16", False, causal=True, ragged=True, cap=30.0),
        # one new token of a single sequence, learned relative positions: latency
        _attention("token-single", 1, 1, 4001, 16, 4, 64, "bf16", False, causal=True, buckets=32, distance=128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case of the listed ranges: sizes spread over their logarithm, odd ones among them."""
    kind = rng.choice(["rotary", "attention", "attention", "bias", "token"])
    heads = rng.choice([1, 2, 4, 6, 8, 12, 16, 32])
    kv = rng.choice([k for k in (1, 2, 3, 4, 6, 8, 12, 16, 32) if heads % k == 0])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "rotary":
        d = rng.choice([16, 32, 64, 96, 128, 256, 2 * rng.randint(2, 128)])
        S = _log(rng, 1, 8192)
        B = max(1, min(_log(rng, 1, 256), (1 << 24) // (S * (heads + kv) * d)))
        rot = rng.choice([d, d, 2 * max(1, d // 4)])
        return {k: v for k, v in _rotary("", B, S, heads, kv, d, dtype, rng.random() < 0.6, rng.choice([0, 0, 100000]), rot,
                                         rng.random() < 0.3).items() if k != "name"}
    d = rng.choice([16, 32, 64, 64, 80, 96, 128, 128, 8 * rng.randint(1, 16)])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if kind == "token":
        heads, kv = rng.choice([(8, 8), (16, 4), (16, 1), (32, 8), (12, 3)])
        Sq = rng.choice([1, 1, 1, 2, 5])
        Sk = _log(rng, 16, 8192)
        B = max(1, min(_log(rng, 1, 32), (1 << 26) // (Sk * kv * d)))
        how = rng.choice(["none", "slopes", "buckets"])
        c = _attention("", B, Sq, max(Sk, Sq), heads, kv, d, dtype, False, causal=True, ragged=True, cap=cap,
                       slopes=how == "slopes", buckets=32 if how == "buckets" else 0, distance=128 if how == "buckets" else 0)
        return {k: v for k, v in c.items() if k != "name"}
    # fp32 products cost sixteen times the bf16 ones: fewer of them
    pairs = 1 << 28 if dtype == "bf16" else 1 << 25
    grad = rng.random() < 0.7
    S = _log(rng, 4 if grad else 1, 4096)      # a row's only key has no gradient through the softmax
    while heads * S * S > pairs:
        S = (2 * S) // 3
    B = max(1, min(_log(rng, 1, 64), pairs // (heads * S * S)))
    causal = rng.random() < 0.6
    docs = _log(rng, 8, 1000) if rng.random() < 0.35 else 0
    c = _attention("", B, S, S, heads, kv, d, dtype, grad, causal=causal, mask=S >= 8 and rng.random() < 0.4,
                   prefix=causal and rng.random() < 0.3, docs=docs, cap=cap,
                   slopes=kind == "attention" and rng.random() < 0.5, buckets=rng.choice([8, 32, 64]) if kind == "bias" else 0,
                   distance=rng.choice([48, 128, 256]) if kind == "bias" else 0)
    return {k: v for k, v in c.items() if k != "name"}


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B, heads, kv, d = case["B"], case["heads"], case["kv"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    st = {"case": case}
    if case["op"] == "rotary":
        S, rot = case["S"], case["rot"]
        st["q"] = normal(B, S, heads * d).mul_(1.5).to(dt)
        st["k"] = normal(B, S, kv * d).mul_(1.5).to(dt)
        st["qw"] = 1.0 + 0.2 * normal(d)
        st["kw"] = 1.0 + 0.2 * normal(d)
        # turns per position of every pair: what a model keeps beside its weights
        st["frequencies"] = BASE ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot) / (2 * math.pi)
        start = torch.randint(0, case["far"] + 1, (B, 1), device=DEV, generator=g)
        st["positions"] = start + torch.arange(S, device=DEV)[None, :]
        if case["grad"]:
            for n in ("q", "k", "qw", "kw"):
                st[n].requires_grad_(True)
            st["dq"] = normal(B, S, heads * d).to(dt)
            st["dk"] = normal(B, S, kv * d).to(dt)
        return st
    Sq, Sk = case["Sq"], case["Sk"]
    st["q"] = normal(B, Sq, heads * d).mul_(1.2).to(dt)
    st["k"] = normal(B, Sk, kv * d).mul_(1.2).to(dt)
    st["v"] = normal(B, Sk, kv * d).to(dt)
    st["mask"] = st["prefix"] = st["documents"] = st["q_start"] = st["slopes"] = st["table"] = st["buckets"] = None
    where = torch.arange(Sk, device=DEV)
    if case["mask"]:           # padded sentences, a quarter to the whole of the row
        n = torch.randint(max(1, Sk // 4), Sk + 1, (B, 1), device=DEV, generator=g)
        st["mask"] = (where[None, :] < n).to(torch.int64)
    if case["prefix"]:
        st["prefix"] = torch.randint(0, Sk // 2 + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    if case["docs"]:           # documents of about `docs` tokens behind one another
        ends = torch.randint(max(1, case["docs"] // 2), 3 * case["docs"] // 2 + 1, (B, 2 * Sk // max(1, case["docs"] // 2) + 2),
                             device=DEV, generator=g).cumsum(1)
        st["documents"] = torch.searchsorted(ends, where[None, :].expand(B, Sk).contiguous(), right=True).to(torch.int32)
    if case["ragged"]:         # sequences of unequal length: the new tokens stand behind the last key of each
        n = torch.randint(max(Sq, Sk // 2), Sk + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
        n[0] = Sk
        st["q_start"] = n - Sq
    if case["slopes"]:
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV, dtype=torch.float32) / heads)
    if case["buckets"]:
        st["table"] = 0.5 * normal(case["buckets"], heads)
        st["buckets"] = _bucket_map(case["buckets"], case["distance"], not case["causal"]).to(DEV)
    if case["grad"]:
        for n in ("q", "k", "v", "table"):
            if st[n] is not None:
                st[n].requires_grad_(True)
        st["dout"] = normal(B, Sq, heads * d).to(dt)
    return st


def _bucket_map(count, distance, both):
    """bucket of every relative distance key - query in [-distance, distance]: the near half of the buckets hold one
    distance each, the far half widths that grow geometrically up to `distance`; with `both`, keys behind and before the
    query have halves of their own, else keys behind the query share bucket 0"""
    rel = torch.arange(-distance, distance + 1, dtype=torch.float64)
    n = count // 2 if both else count
    first = torch.where(rel > 0, n, 0) if both else torch.zeros_like(rel)
    away = rel.abs() if both else (-rel).clamp(min=0)
    near = n // 2
    far = near + (away.clamp(min=near) / near).log() / math.log(distance / near) * (n - near)
    return (first + torch.where(away < near, away, far.floor().clamp(max=n - 1))).to(torch.int32)


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        q, k = _own_rotary(state) if own else _plain_rotary(state)
        if not case["grad"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad((q, k), [state[n] for n in ("q", "k", "qw", "kw")], (state["dq"], state["dk"]))
        return {"q": q, "k": k, **dict(zip(("dq", "dk", "dqw", "dkw"), grads))}
    out = _own_attention(state) if own else _plain_attention(state)
    if not case["grad"]:
        return {"out": out}
    names = [n for n in ("q", "k", "v", "table") if state[n] is not None]
    grads = torch.autograd.grad(out, [state[n] for n in names], state["dout"])
    return {"out": out, **{"d" + n: t for n, t in zip(names, grads)}}


def _own_rotary(s):
    from nonauto_lm_amd import ops
    c = s["case"]
    return ops.qk_norm_rotary(s["q"], s["k"], c["heads"], c["kv"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                              frequencies=s["frequencies"], positions=s["positions"], interleaved=c["interleaved"])


def _own_attention(s):
    from nonauto_lm_amd import ops
    c = s["case"]
    return ops.biased_attention(s["q"], s["k"], s["v"], c["heads"], c["kv"], mask=s["mask"], causal=c["causal"],
                                prefix=s["prefix"], documents=s["documents"], q_start=s["q_start"],
                                softcap=c["cap"] or None, slopes=s["slopes"], table=s["table"], buckets=s["buckets"])


def _plain_rotary(s):
    c = s["case"]
    turns = s["positions"].to(torch.float64)[..., None] * s["frequencies"]
    angle = (turns - turns.round()) * (2 * math.pi)
    cos, sin = angle.cos().float()[:, :, None, :], angle.sin().float()[:, :, None, :]
    return (_plain_heads(s["q"], c["heads"], s["qw"], cos, sin, c), _plain_heads(s["k"], c["kv"], s["kw"], cos, sin, c))


def _plain_heads(x, heads, weight, cos, sin, c):
    h = x.float().view(c["B"], c["S"], heads, c["d"])
    n = h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
    r, rest = n[..., :c["rot"]], n[..., c["rot"]:]
    if c["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = r[..., :c["rot"] // 2], r[..., c["rot"] // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1).reshape(x.shape).to(x.dtype)


def _visible(s):
    """(B, 1, Sq, Sk) truth values of what a query sees, and (B, Sq, Sk) distances key - query"""
    c = s["case"]
    B, Sq, Sk = c["B"], c["Sq"], c["Sk"]
    kpos = torch.arange(Sk, device=DEV)
    start = torch.full((B,), Sk - Sq, device=DEV) if s["q_start"] is None else s["q_start"].long()
    qpos = start[:, None] + torch.arange(Sq, device=DEV)
    rel = kpos[None, None, :] - qpos[:, :, None]
    see = torch.ones(B, Sq, Sk, dtype=torch.bool, device=DEV)
    if c["causal"]:
        see = rel <= 0
        if s["prefix"] is not None:
            see = see | (kpos[None, None, :] < s["prefix"].long()[:, None, None])
    if s["mask"] is not None:
        see = see & s["mask"].ne(0)[:, None, :]
    if s["documents"] is not None:
        mine = s["documents"].gather(1, qpos)
        see = see & (s["documents"][:, None, :] == mine[:, :, None])
    return see[:, None], rel


def _plain_attention(s):
    c = s["case"]
    B, Sq, Sk, H, G, d = c["B"], c["Sq"], c["Sk"], c["heads"], c["kv"], c["d"]
    see, rel = _visible(s)
    q = s["q"].float().view(B, Sq, G, H // G, d).permute(0, 2, 3, 1, 4)
    k = s["k"].float().view(B, Sk, G, 1, d).permute(0, 2, 3, 1, 4)
    v = s["v"].float().view(B, Sk, G, 1, d).permute(0, 2, 3, 1, 4)
    score = (torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5).view(B, H, Sq, Sk)
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    if s["slopes"] is not None:
        score = score - s["slopes"][None, :, None, None] * rel[:, None].abs()
    if s["table"] is not None:
        R = c["distance"]
        if s["q_start"] is None:
            # row i of the bias is a window of the values by distance, from -(Sk - 1) to Sq - 1, that moves with i; in 64
            # bits because the table's gradient is a sum of B Sq Sk values of either sign
            by_distance = s["table"].double()[s["buckets"].long()[torch.arange(1 - Sk, Sq, device=DEV).clamp(-R, R) + R]]
            score = score + by_distance.t().unfold(-1, Sk, 1).flip(1).float()
        else:
            score = score + s["table"][s["buckets"].long()[rel.clamp(-R, R) + R]].permute(0, 3, 1, 2)
    score = score.masked_fill(~see, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), torch.zeros_like(top), top).detach()
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.view(B, G, H // G, Sq, Sk), v)
    return out.permute(0, 3, 1, 2, 4).reshape(B, Sq, H * d).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    B, H, G, d = case["B"], case["heads"], case["kv"], case["d"]
    if case["op"] == "rotary":
        n = B * case["S"] * (H + G) * d
        return {"bytes": n * es * (5 if case["grad"] else 2) + B * case["S"] * 8, "flops": n * (20 if case["grad"] else 8)}
    Sq, Sk = case["Sq"], case["Sk"]
    # pairs that are seen, as the inputs' distributions give them on average
    keys = 0.75 * Sk if case["ragged"] else Sk
    pairs = Sq * keys
    if case["causal"] and Sq == Sk:
        pairs = Sq * (Sk + 1) / 2
        if case["prefix"]:     # a beginning of length P, uniform up to half a row, adds P (P - 1) / 2
            pairs += Sk * Sk / 24
    if case["docs"] and case["docs"] < Sk:
        seen = 13 / 12 * case["docs"]
        pairs = min(pairs, Sq * (seen / 2 if case["causal"] else seen))
    if case["mask"]:
        pairs *= 0.75 if case["causal"] else 0.625
    q, kv = B * Sq * H * d * es, B * keys * G * d * es
    bytes_ = 2 * q + 2 * kv + (3 * q + 2 * kv if case["grad"] else 0)
    return {"bytes": bytes_, "flops": B * H * pairs * d * (14 if case["grad"] else 4)}


# ------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    B, H, G, d = case["B"], case["heads"], case["kv"], case["d"]
    D = {n: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for n, t in s.items()}
    if case["op"] == "rotary":
        S, half = case["S"], case["rot"] // 2
        theta = 2 * math.pi * torch.remainder(D["positions"].double()[..., None] * D["frequencies"], 1.0)
        turn = torch.polar(torch.ones_like(theta), theta)[:, :, None, :]            # unit complex numbers
        first = torch.arange(half, device=DEV) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        out = {}
        for x, w, heads in (("q", "qw", H), ("k", "kw", G)):
            h = D[x].view(B, S, heads, d)
            inv = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS)
            n = h * inv * D[w]
            z = torch.complex(n[..., first], n[..., second]) * turn
            y = n.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[x] = y.view_as(D[x])
            if case["grad"]:
                dy = D["d" + x].view(B, S, heads, d)
                z = torch.complex(dy[..., first], dy[..., second]) * turn.conj()
                dn = dy.clone()
                dn[..., first], dn[..., second] = z.real, z.imag
                out["d" + w] = (dn * h * inv).sum((0, 1, 2))
                dh = dn * D[w]
                out["d" + x] = (inv * dh - inv ** 3 * h * (dh * h).sum(-1, keepdim=True) / d).view_as(D[x])
        return out
    Sq, Sk, R = case["Sq"], case["Sk"], case["distance"]
    j = torch.arange(Sk, device=DEV)
    out = {"out": torch.zeros(B, Sq, H, d, dtype=torch.float64, device=DEV)}
    if case["grad"]:
        out["dq"] = torch.zeros_like(out["out"])
        out["dk"], out["dv"] = (torch.zeros(B, Sk, G, d, dtype=torch.float64, device=DEV) for _ in range(2))
        if D["table"] is not None:
            out["dtable"] = torch.zeros_like(D["table"])
    group = H // G
    for b in range(B):
        i = (Sk - Sq if D["q_start"] is None else int(D["q_start"][b])) + torch.arange(Sq, device=DEV)
        hidden = torch.zeros(Sq, Sk, dtype=torch.bool, device=DEV)
        if case["causal"]:
            hidden |= j[None, :] > i[:, None]
            if D["prefix"] is not None:
                hidden &= (j >= int(D["prefix"][b]))[None, :]
        if D["mask"] is not None:
            hidden |= (D["mask"][b] == 0)[None, :]
        if D["documents"] is not None:
            hidden |= D["documents"][b][None, :] != D["documents"][b][i][:, None]
        away = j[None, :] - i[:, None]
        # as many heads at once as fit a few GiB
        step = max(1, min(group, (1 << 28) // (Sq * Sk)))
        for h0 in [h for g0 in range(G) for h in range(g0 * group, (g0 + 1) * group, step)]:
            hs = torch.arange(h0, min(h0 + step, (h0 // group + 1) * group), device=DEV)
            kvh = h0 // group
            q = D["q"][b].view(Sq, H, d)[:, hs].transpose(0, 1)
            k, v = D["k"][b].view(Sk, G, d)[:, kvh], D["v"][b].view(Sk, G, d)[:, kvh]
            raw = q @ k.t() / math.sqrt(d)
            x, slope = raw, None
            if case["cap"]:
                t = torch.tanh(raw / case["cap"])
                x, slope = case["cap"] * t, 1 - t * t
            if D["slopes"] is not None:
                x = x - D["slopes"][hs][:, None, None] * away.abs()
            if D["table"] is not None:
                which = D["buckets"].long()[away.clamp(-R, R) + R]
                x = x + D["table"][:, hs].t()[:, which]
            x = x.masked_fill(hidden, -math.inf)
            p = torch.softmax(x, -1).masked_fill(hidden.all(-1)[None, :, None], 0.0)
            o = p @ v
            out["out"][b].index_copy_(1, hs, o.transpose(0, 1))
            if case["grad"]:
                do = D["dout"][b].view(Sq, H, d)[:, hs].transpose(0, 1)
                out["dv"][b, :, kvh] += (p.transpose(1, 2) @ do).sum(0)
                ds = p * (do @ v.t() - (do * o).sum(-1, keepdim=True))
                if D["table"] is not None:
                    for n, h in enumerate(hs.tolist()):
                        out["dtable"][:, h] += torch.bincount(which.reshape(-1), ds[n].reshape(-1), case["buckets"])
                if slope is not None:
                    ds = ds * slope
                ds = ds / math.sqrt(d)
                out["dq"][b].index_copy_(1, hs, (ds @ k).transpose(0, 1))
                out["dk"][b, :, kvh] += (ds.transpose(1, 2) @ q).sum(0)
    return {n: t if n == "dtable" else t.flatten(-2) for n, t in out.items()}
