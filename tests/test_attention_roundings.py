"""The second bf16 values that the training pass carries keep dq and dk at the errors that their last roundings leave:

  out_lo  what the rounding of the output leaves, for delta = dout . out
  rest    what the rounding of large probabilities leaves, in the output's product (and so in delta)
  halves  dS as two bf16 values in its products, for heads of at most 16 columns

Limits relative to a gradient's norm.  A rounding to bf16 is off by 1.66e-3 of a tensor's norm (values of all mantissas), two
independent ones by 2.35e-3.  `emulated` computes the pass in 64 bits with exactly these roundings; the limits lie between
its errors with all three and without the one that a case is for, which the first test holds on to."""
import math

import pytest
import torch

gpu = pytest.mark.gpu

# (what the case is for, batch, heads, length, head size, keys per document, limit)
CASES = [("out_lo", 2, 4, 512, 64, 3, 2.8e-3), ("out_lo", 2, 4, 512, 128, 2, 2.8e-3), ("out_lo", 2, 4, 512, 16, 3, 2.1e-3),
         ("rest", 4, 4, 512, 16, 2, 1.78e-3), ("halves", 1, 4, 1500, 16, 1500, 2.1e-3), ("halves", 1, 4, 1500, 8, 1500, 2.1e-3)]


def case_tensors(B, H, S, d, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=device)
    return [t.bfloat16() for t in (1.2 * n(B, S, H, d), 1.2 * n(B, S, H, d), n(B, S, H, d), n(B, S, H, d))]


def one(t):
    return t.float().bfloat16().double()


def two(t):
    a = one(t)
    return a + one(t - a)


def gradients(q, k, v, dout, n, rounded=None):
    """dq, dk (B, H, S, d) in 64 bits; `rounded`: (of P, of out, of dS, of the result)"""
    in_p, in_out, in_ds, in_result = rounded or (lambda t: t,) * 4
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    S, scale = q.size(2), q.size(3) ** -0.5
    docs = torch.arange(S, device=q.device) // n
    x = (q @ k.transpose(2, 3).contiguous() * scale).masked_fill(docs[:, None] != docs[None], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    l = e.sum(-1, keepdim=True)
    delta = (do * in_out(in_p(e) @ v / l)).sum(-1, keepdim=True)
    ds = in_ds(e / l * (do @ v.transpose(2, 3).contiguous() - delta))
    return in_result(ds @ k * scale), in_result(ds.transpose(2, 3).contiguous() @ q * scale)


def emulated(tensors, n, d, without=None):
    return gradients(*tensors, n, (one if without == "rest" else two, one if without == "out_lo" else two,
                                   one if without == "halves" or d > 16 else two, one))


def errors(got, want):
    return [float((a.double() - b).norm() / b.norm()) for a, b in zip(got, want)]


@pytest.mark.parametrize("what,B,H,S,d,n,limit", CASES)
def test_limits_tell_the_paths_apart(what, B, H, S, d, n, limit):
    tensors = case_tensors(B, H, S, d, "cpu")
    want = gradients(*tensors, n)
    assert max(errors(emulated(tensors, n, d), want)) < 0.97 * limit
    assert max(errors(emulated(tensors, n, d, without=what), want)) > 1.03 * limit


@gpu
@pytest.mark.parametrize("what,B,H,S,d,n,limit", CASES)
def test_gradients_keep_to_their_last_roundings(what, B, H, S, d, n, limit):
    from nonauto_lm_amd import ops
    tensors = case_tensors(B, H, S, d, "cuda")
    docs = (torch.arange(S, device="cuda") // n).to(torch.int32).repeat(B, 1)
    leaves = [t.requires_grad_(True) for t in tensors[:3]]
    out = ops.biased_attention(*leaves, H, documents=docs)
    got = torch.autograd.grad(out, leaves[:2], tensors[3])
    # keys alone: delta comes from a kernel of its own
    q, k, v = (t.detach() for t in leaves)
    k.requires_grad_(True)
    dk = torch.autograd.grad(ops.biased_attention(q, k, v, H, documents=docs), k, tensors[3])[0]
    want = gradients(*(t.detach() for t in tensors), n)
    assert errors([dk.transpose(1, 2)], want[1:])[0] < limit
    for name, e in zip(("dq", "dk"), errors([t.transpose(1, 2) for t in got], want)):
        assert e < limit, f"{name}: {e:.3e} of its norm, limit {limit}"
