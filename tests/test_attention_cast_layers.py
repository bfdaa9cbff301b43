"""MultiHeadAttention with score options after .bfloat16(): its norm scales and bias table are bf16 parameters then, which the
operators read as fp32 and whose gradients come back in bf16.

The output is held to 5e-2 of its largest value, as for the layer under autocast: twelve roundings of at most 2^-8 in series.
Gradients of parameters are sums over all rows whose terms partly cancel, so they are held to something exact instead: those of
the same layer with the three kept as fp32 parameters of the same values, bit for bit, the three's rounded to bf16."""
import copy

import pytest
import torch

from test_attention_layers import OPTIONS, close, make, written_out
from test_attention_saved_tensors import Recorder

gpu = pytest.mark.gpu


@pytest.mark.parametrize("options", OPTIONS)
def test_cast_layer_reaches_the_operators(monkeypatch, options):
    from nonauto_lm_amd import nn_bracket as nb
    lib = Recorder(monkeypatch)
    mha = nb.MultiHeadAttention(4, 64, dropout=0.0, **options).bfloat16()
    x = torch.randn(2, 9, 64, dtype=torch.bfloat16)
    y = mha(x, x, x)
    assert y.dtype == torch.bfloat16 and lib.calls["mivae_biased_attention_fwd"].dtype == 1
    assert bool(lib.calls["mivae_biased_attention_fwd"].table) == ("relative_bias" in options)
    if options.get("qk_norm"):
        assert lib.calls["mivae_qk_norm_rotary_fwd"].q_weight and lib.calls["mivae_qk_norm_rotary_fwd"].k_weight
    y.sum().backward()
    for n, p in mha.named_parameters():
        assert p.grad is not None and p.grad.dtype == torch.bfloat16, n


@gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("options", OPTIONS)
def test_cast_layer_matches_written_out_form(options, causal):
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(3, 45, 64, device="cuda", generator=g).bfloat16()
    mask = (torch.arange(45, device="cuda")[None, :] < torch.tensor([[45], [20], [1]], device="cuda")).long()
    cast = make(options, causal).bfloat16()
    kept = copy.deepcopy(cast)
    for n in ("_query_norm", "_key_norm", "_relative_bias"):
        if getattr(kept, n) is not None:
            setattr(kept, n, torch.nn.Parameter(getattr(cast, n).detach().float()))
    got = []
    for mha in (cast, kept):
        leaf = x.clone().requires_grad_(True)
        y = mha(leaf, leaf, leaf, mask)
        params = dict(mha.named_parameters())
        weight = torch.sin(torch.arange(y.numel(), device="cuda").float()).view(y.shape)
        got.append(dict(zip(["out", "dx", *params], [y, *torch.autograd.grad((y.float() * weight).sum(), [leaf, *params.values()])])))
    assert all(t.dtype == torch.bfloat16 for t in got[0].values())
    for n, t in got[0].items():
        assert torch.equal(t, got[1][n].bfloat16()), n
    close("out", got[0]["out"], written_out(cast, x.double(), x.double(), mask), 5e-2)
