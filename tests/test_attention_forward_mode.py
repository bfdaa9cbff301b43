"""Forward-mode derivatives are not offered by the attention sublayer's operators: an operand with a tangent is refused, never
answered with an output that has silently lost it."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_attention_saved_tensors import Recorder


def attention_call():
    from nonauto_lm_amd import ops
    x = {n: torch.randn(2, 6, 64) for n in ("q", "k", "v")}
    biased = dict(x, table=torch.randn(8, 2), buckets=torch.zeros(5, dtype=torch.int32))
    return ops.biased_attention, dict(heads=2), (x, biased, dict(x, slopes=torch.ones(2)))


def rotary_call():
    from nonauto_lm_amd import ops
    x = dict(q=torch.randn(2, 6, 64), k=torch.randn(2, 6, 64), q_weight=torch.ones(32), k_weight=torch.ones(32),
             frequencies=ops.rotary_frequencies(32))
    return ops.qk_norm_rotary, dict(heads=2), (x,)


@pytest.mark.parametrize("learns", [False, True])
@pytest.mark.parametrize("make", [attention_call, rotary_call])
def test_a_tangent_is_refused(monkeypatch, make, learns):
    Recorder(monkeypatch)
    fn, fixed, sets = make()
    for operands in sets:
        fn(**operands, **fixed)
        for name, t in operands.items():
            if not t.is_floating_point() or (learns and name in ("slopes", "frequencies")):
                continue
            with fwd.dual_level():
                dual = fwd.make_dual(t.clone().requires_grad_(learns), torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(**dict(operands, **{name: dual}), **fixed)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    fn(**dict(operands, **{name: dual}), **fixed)
                fn(**dict(operands, **{name: fwd.unpack_dual(dual).primal}), **fixed)          # the value alone is fine


@pytest.mark.parametrize("make", [attention_call, rotary_call])
def test_a_tangent_of_the_outgoing_gradient_is_refused(monkeypatch, make):
    Recorder(monkeypatch)
    fn, fixed, sets = make()
    q = sets[0]["q"].requires_grad_(True)
    out = fn(**sets[0], **fixed)
    out = out[0] if isinstance(out, tuple) else out
    with fwd.dual_level():
        dout = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, q, dout)


@pytest.mark.parametrize("make", [attention_call, rotary_call])
def test_function_transforms_end_in_an_error(monkeypatch, make):
    Recorder(monkeypatch)
    fn, fixed, sets = make()
    rest = {n: t for n, t in sets[0].items() if n != "q"}
    one = lambda q: fn(q=q, **rest, **fixed)
    for call in (lambda q: torch.func.jvp(one, (q,), (q,)), torch.func.vmap(lambda q: one(q[None]))):
        with pytest.raises(Exception):
            call(sets[0]["q"])
