"""Caps far above the scores: cap * tanh(s / cap) is s itself, to s^2 / (3 cap^2) of it, so outputs and gradients are held to the
definition without a cap and to its bounds, which know nothing of the cap.  (A tanh that is off by 1e-7 absolutely would move
a score by 1e-2 at a cap of 1e5 and be noise at 1e7.)"""
import pytest
import torch

from test_attention_operators import TYPES, check, definition, inputs, padded

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [1e5, 1e7, 1e20])
@pytest.mark.parametrize("Sq,Sk", [(1, 300), (9, 200), (40, 200), (150, 150)])
def test_caps_far_above_the_scores(Sq, Sk, cap, dtype):
    from nonauto_lm_amd import ops
    _, q, k, v, dout = inputs(2, Sq, Sk, 4, 2, 64, dtype, seed=Sq, grad=False)
    q = q * 2                                                  # scores of a standard deviation of 3
    opt = dict(mask=padded(2, Sk, 3), causal=True)
    with torch.no_grad():
        out = ops.biased_attention(q, k, v, 4, 2, softcap=cap, **opt)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    trained = ops.biased_attention(*leaves, 4, 2, softcap=cap, **opt)
    ref = definition(q, k, v, 4, 2, dout=dout, **opt)
    check("out", out, *ref["out"])
    check("out (training)", trained, *ref["out"])
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(trained, leaves, dout)):
        check(n, t, *ref[n])


@gpu
@pytest.mark.parametrize("cap", [100.0, 512.0, 513.0])
@pytest.mark.parametrize("Sq", [1, 9, 60, 150])
def test_both_sides_of_the_short_form(Sq, cap):
    """bf16 without gradients: the largest cap whose tanh takes two instructions, and the smallest beyond"""
    from nonauto_lm_amd import ops
    _, q, k, v, _ = inputs(2, Sq, 200, 4, 2, 64, torch.bfloat16, seed=Sq, grad=False)
    for loud in (2, 200):                                      # scores far below the cap and around it
        out = ops.biased_attention(q * loud, k, v, 4, 2, softcap=cap, causal=True)
        check("out", out, *definition(q * loud, k, v, 4, 2, softcap=cap, causal=True)["out"])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [2, 16, 33, 150])
def test_scores_next_to_ones_near_the_cap(Sq, dtype):
    """every other query's scores reach the cap; its neighbours in the tile are no less exact for it"""
    from nonauto_lm_amd import ops
    cap, Sk, d = 1e5, 170, 64
    _, q, k, v, dout = inputs(2, Sq, Sk, 4, 2, d, dtype, seed=Sq, grad=False)
    dout[:, ::2] = 0                                           # the loud queries pass no gradient to keys and values
    loud = q.clone()
    loud[:, ::2] *= 2 * cap
    for grad in (False, True):
        leaves = [t.clone().requires_grad_(grad) for t in (loud, k, v)]
        out = ops.biased_attention(*leaves, 4, 2, softcap=cap)
        assert torch.isfinite(out).all()
        score = (loud[0, :, 0].double() @ k[0, :, 0].double().t()) * d ** -0.5
        assert bool((score[::2].abs().amax(1) > 0.75 * cap).all())
        ref = definition(q, k, v, 4, 2, dout=dout)
        check("out", out[:, 1::2], *(t[:, 1::2] for t in ref["out"]))
        if grad:
            dq, dk, dv = torch.autograd.grad(out, leaves, dout)
            check("dq", dq[:, 1::2], *(t[:, 1::2] for t in ref["dq"]))
            check("dk", dk, *ref["dk"])
            check("dv", dv, *ref["dv"])
