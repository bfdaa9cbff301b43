"""The transformer bracket on the attention sublayer's operators: MultiHeadAttention's score options, alone and inside encoder,
decoder and a whole training step, against the same layer written out in 64 bits.

Tolerance of the fp32 comparisons: every stage (projection, norm, rotation, scores, softmax, values, output projection and
their backward) sums at most 64 terms, an error of at most 64 * 2^-24 = 4e-6 of the largest value; twelve stages in
series, and a factor 2 where an error passes through the exponential: 1e-4 of the largest value of a tensor.  bf16: twelve
roundings of at most 2^-8 in series, 5e-2 of the largest value."""
import math

import pytest
import torch

gpu = pytest.mark.gpu


def written_out(mha, x, keys, mask, documents=None, prefix=None):
    """MultiHeadAttention.forward(x, keys, keys, ...) in 64 bits from the module's own parameters"""
    P = {n: p.double() for n, p in mha.named_parameters()}
    H, G, d = mha._num_heads, mha._kv_heads, mha._attn_size
    lin = lambda t, n: t @ P[n + ".weight"].t() + P[n + ".bias"]
    B, Sq, Sk = x.size(0), x.size(1), keys.size(1)
    q = lin(x, "_projections.query").view(B, Sq, H, d)
    k = lin(keys, "_projections.key").view(B, Sk, G, d)
    v = lin(keys, "_projections.value").view(B, Sk, G, d)
    at = torch.arange(Sk, device=x.device)
    if mha._qk_norm:
        norm = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        q, k = norm(q, P["_query_norm"]), norm(k, P["_key_norm"])
    if mha._rotary:
        m = mha._rotary // 2
        angle = at.double()[:, None] * 10000.0 ** (-torch.arange(m, device=x.device).double() / m)

        def turn(t, a):
            a = a[None, :, None, :]
            u, w, rest = t[..., :m], t[..., m:2 * m], t[..., 2 * m:]
            return torch.cat((u * a.cos() - w * a.sin(), u * a.sin() + w * a.cos(), rest), -1)

        q, k = turn(q, angle[Sk - Sq:]), turn(k, angle)
    k, v = (t.repeat_interleave(H // G, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(d)
    if mha._softcap:
        s = mha._softcap * torch.tanh(s / mha._softcap)
    rel = at[None, :] - at[Sk - Sq:, None]
    if mha._slopes:
        s = s - (2.0 ** (-8.0 * torch.arange(1, H + 1, device=x.device).double() / H))[None, :, None, None] * rel.abs()
    if mha._relative_bias is not None:
        R = mha._buckets.numel() // 2
        s = s + P["_relative_bias"][mha._buckets.long()[rel.clamp(-R, R) + R]].permute(2, 0, 1)
    see = torch.ones(B, Sq, Sk, dtype=torch.bool, device=x.device)
    if mha._mask_tril:
        see &= rel <= 0
        if prefix is not None:
            see |= at[None, None, :] < prefix.long()[:, None, None]
    if mask is not None:
        see &= mask.ne(0)[:, None, :]
    if documents is not None:
        see &= documents[:, None, :] == documents[:, Sk - Sq:, None]
    p = torch.softmax(s.masked_fill(~see[:, None], -1e300), -1) * see[:, None]
    return lin(torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, Sq, H * d), "_output")


def close(name, got, want, tol):
    got, want = got.detach(), want.detach()
    err, scale = float((got.double() - want.double()).abs().max()), float(want.double().abs().max())
    assert err <= tol * max(scale, 1e-3), f"{name}: off by {err} of {scale}"


OPTIONS = [dict(softcap=5.0), dict(relative_bias=dict(num_buckets=8, max_distance=20)), dict(distance_slopes=True, kv_heads=2),
           dict(qk_norm=True), dict(rotary=True), dict(rotary=8, kv_heads=1),
           dict(kv_heads=2, qk_norm=True, rotary=True, softcap=20.0, relative_bias=dict(num_buckets=16, max_distance=30))]


def make(options, causal=False, D=64, heads=4, seed=0):
    from nonauto_lm_amd import nn_bracket as nb
    torch.manual_seed(seed)
    mha = nb.MultiHeadAttention(heads, D, dropout=0.0, mask_tril=causal, **options).cuda()
    with torch.no_grad():
        for n, p in mha.named_parameters():
            if n.startswith(("_relative", "_query", "_key")):
                p.add_(0.3 * torch.randn_like(p))
    return mha


def compare(mha, x, keys, mask, tol, bf16=False, **more):
    params = [p for p in mha.parameters()]
    got = []
    for wide in (False, True):
        leaves = [t.double() if wide else t.clone() for t in ((x, keys) if keys is not None else (x,))]
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        kk = leaves[-1]
        if wide:
            y = written_out(mha, leaves[0], kk, mask, **more)
        else:
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=bf16):
                y = mha(leaves[0], kk, kk, mask, **more)
        weight = torch.sin(torch.arange(y.numel(), device="cuda", dtype=torch.float64)).view(y.shape)
        got.append([y] + list(torch.autograd.grad((y.double() * weight).sum(), leaves + params)))
    names = ["out", "dx", "dkeys"][:1 + len(leaves)] + [n for n, _ in mha.named_parameters()]
    for n, a, b in zip(names, *got):
        if n == "_projections.key.bias" and not mha._qk_norm and not mha._rotary and not mha._softcap:
            continue                   # a shift of all keys cancels in the softmax: the gradient is 0 but for rounding
        close(n, a, b, tol)


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("options", OPTIONS)
def test_layer_matches_written_out_form(options, causal):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 45, 64, device="cuda", generator=g)
    mask = (torch.arange(45, device="cuda")[None, :] < torch.tensor([[45], [20], [1]], device="cuda")).long()
    mha = make(options, causal)
    compare(mha, x, None, mask, 1e-4)
    compare(mha, x, None, None, 1e-4)


@gpu
@pytest.mark.parametrize("options", [OPTIONS[0], OPTIONS[2], OPTIONS[6]])
def test_layer_documents_prefix_and_longer_keys(options):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, keys = torch.randn(2, 40, 64, device="cuda", generator=g), torch.randn(2, 70, 64, device="cuda", generator=g)
    docs = (torch.arange(40, device="cuda") // 15).to(torch.int32).expand(2, 40).contiguous()
    prefix = torch.tensor([0, 25], dtype=torch.int32, device="cuda")
    mha = make(options, causal=True)
    compare(mha, x, None, None, 1e-4, documents=docs)
    compare(mha, x, None, None, 1e-4, prefix=prefix)
    compare(mha, x, keys, None, 1e-4)
    compare(mha, x[:, :1], keys, None, 1e-4)
    step = mha(x[:, -1:], x, x)                                     # the last position alone, as a generating loop computes it
    close("step", step, mha(x, x, x)[:, -1:], 1e-4)


@gpu
def test_layer_under_autocast():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 100, 64, device="cuda", generator=g)
    mask = (torch.arange(100, device="cuda")[None, :] < torch.tensor([[100], [37]], device="cuda")).long()
    for options in (OPTIONS[1], OPTIONS[6]):
        compare(make(options), x, None, mask, 5e-2, bf16=True)


@gpu
def test_layer_first_called_in_inference_mode_or_a_capture():
    """the layer's constants outlive the mode, stream and graph of the call that made them"""
    x = torch.randn(2, 30, 64, device="cuda")
    want = None
    for first in ("inference", "side stream", "capture"):
        torch.manual_seed(1)
        mha = make(dict(rotary=True, distance_slopes=True))
        if first == "inference":
            with torch.inference_mode():
                mha(x, x, x)
        elif first == "side stream":
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                mha(x, x, x)
        else:
            with torch.no_grad():
                mha(x, x, x)
                mha._constants.clear()
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    mha(x, x, x)
            assert not mha._constants
        out = mha(x, x, x)
        want = out if want is None else want
        assert torch.equal(out, want)
        out.sum().backward()


def test_layer_refusals_and_state_dict():
    from nonauto_lm_amd import nn_bracket as nb
    plain = nb.MultiHeadAttention(4, 64)
    assert set(plain.state_dict()) == {f"_projections.{n}.{w}" for n in ("query", "key", "value") for w in ("weight", "bias")} | {
        "_output.weight", "_output.bias"}
    full = nb.MultiHeadAttention(4, 64, dropout=0.0, **OPTIONS[6])
    assert set(full.state_dict()) - set(plain.state_dict()) == {"_relative_bias", "_query_norm", "_key_norm"}
    assert full._projections["key"].weight.shape == (32, 64) and full._relative_bias.shape == (16, 4)
    for bad in (dict(softcap=5.0), dict(softcap=5.0, dropout=0.1), dict(kv_heads=3, dropout=0.0),
                dict(relative_bias={}, distance_slopes=True, dropout=0.0)):
        with pytest.raises(ValueError):
            nb.MultiHeadAttention(4, 64, **bad)
    x = torch.zeros(1, 3, 64)
    with pytest.raises(ValueError, match="score options"):
        plain(x, x, x, documents=torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        full(x, x, x)
    layer = nb.TransformerEncoderLayer(64, 128, 4, dropout=0.1, attention=dict(dropout=0.0, softcap=5.0))
    assert layer._attn._scored and isinstance(layer._pos_ffn._dropout, torch.nn.Dropout)


def config(attention, D=64):
    import bench
    c = bench.model_config(D, 32, 2)
    for part in ("encoder", "decoder"):
        c[part] = dict(c[part], attention=attention)
    return c


@gpu
def test_packed_documents_equal_separate_sentences():
    """an encoder's output for sentences behind one another in a row is that of the sentences by themselves: with relative
    positions alone (the sinusoid differs, so its table is zeroed)"""
    from nonauto_lm_amd import nn_bracket as nb
    torch.manual_seed(0)
    enc = nb.TransformerEncoder(64, 128, 2, 4, attention=dict(relative_bias=dict(num_buckets=8, max_distance=16), rotary=True)).cuda()
    with torch.no_grad():
        enc._pos_enc._pos_enc.zero_()
        for p in enc.parameters():
            p.add_(0.05 * torch.randn_like(p) if p.requires_grad else 0.0)
    lengths = [7, 30, 1, 26]
    x = torch.randn(1, sum(lengths), 64, device="cuda")
    docs = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lengths)])[None].cuda()
    ones = torch.ones(1, sum(lengths), dtype=torch.int64, device="cuda")
    with torch.no_grad():
        packed = enc.encoder(x, ones, documents=docs)
        at = 0
        for n in lengths:
            alone = enc.encoder(x[:, at:at + n].contiguous(), ones[:, :n].contiguous())
            close(f"sentence of {n}", packed[:, at:at + n], alone, 1e-4)
            at += n


@gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_model_trains_with_score_options(bf16):
    """a whole model from its configuration trains, eagerly and captured, and its new parameters learn"""
    import bench
    import nonauto_lm_amd as M
    from nonauto_lm_amd import dp
    from nonauto_lm_amd.step import TrainStep
    attention = dict(kv_heads=2, qk_norm=True, rotary=True, softcap=30.0, relative_bias=dict(num_buckets=8, max_distance=16))
    after = {}
    for graph in (False, True):
        torch.manual_seed(13)
        model = M.VAELmModel.from_params(vocab=M.SimpleVocab(200), **config(attention)).cuda().train()
        model.training_outputs_only = True
        tokens = bench.synthetic_tokens(16, 24, True, 7)
        tokens = torch.where(tokens > 0, tokens % 196 + 4, tokens).cuda()
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        reducer = dp.GradReducer(model.parameters(), flatten_params=True)
        opt = dp.FusedAdam(reducer, lr=1e-3)
        step = TrainStep(model, reducer, opt, tokens, torch.bfloat16 if bf16 else None, 5.0, 2.0, graph=graph, warmup=1)
        losses = [float(step()["batch-loss"].detach()) for _ in range(5)]
        assert all(math.isfinite(v) for v in losses)
        moved = [n for n, p in model.named_parameters() if p.requires_grad and not torch.equal(p, before[n])]
        for n in before:
            if "_relative_bias" in n or "_query_norm" in n or "_key_norm" in n:
                assert n in moved, n
        after[graph] = losses
    # other draws of the posterior's noise, the same batch: the first losses lie within the noise's reach of one another
    assert abs(after[True][0] - after[False][0]) < 0.25 * abs(after[False][0])
