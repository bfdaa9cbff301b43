"""The attention sublayer's operators when their saved tensors come back from a hook elsewhere and in another layout (offloading to the
host turns views with gaps, or every tensor, into contiguous ones): the backward reads what it is given, by that one's strides."""
import contextlib
import ctypes

import pytest
import torch

gpu = pytest.mark.gpu


class Recorder:
    """Stands in for the library on the CPU: the structs that the entry points receive, nothing launched"""

    def __init__(self, monkeypatch):
        from nonauto_lm_amd import _lib as L
        self.calls = {}
        monkeypatch.setattr(L, "require_gpu", lambda *t: None)
        monkeypatch.setattr(L, "stream_of", lambda device: 0)
        monkeypatch.setattr(L, "on_device", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(L, "call", self)

    def __call__(self, name, args, stream):
        self.calls[name] = type(args._obj).from_buffer_copy(args._obj)


def Hooks(back):
    """saved-tensor hooks that hand out what `back` makes of a saved tensor"""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, back)


def shifted(t):
    """the same values, rows apart by two more elements and 4 or 2 bytes off any 16-byte boundary"""
    wide = torch.zeros(*t.shape[:-1], t.size(-1) + 2, dtype=t.dtype, device=t.device)
    wide[..., 1:-1].copy_(t)
    return wide[..., 1:-1]


def packed(B, S, H, G, d, dtype, device, seed=0):
    """q, k, v as column blocks of one projection"""
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(B, S, (H + 2 * G) * d, generator=g, device=device).to(dtype).requires_grad_(True)
    return x, x[..., :H * d], x[..., H * d:(H + G) * d], x[..., (H + G) * d:]


LAYOUTS = {"contiguous": lambda t: t.clone(memory_format=torch.contiguous_format), "shifted": shifted}


class Reader(Recorder):
    """reads the operands (and positions) through the struct's addresses and strides, as the library would"""

    def __call__(self, name, args, stream):
        super().__call__(name, args, stream)
        a = args._obj
        rows = (a.q_len, a.k_len, a.k_len) if hasattr(a, "q_len") else (a.len, a.len)
        dtype = (torch.float32, torch.bfloat16)[a.dtype]
        self.read, self.aligned = {}, True
        for n, S, H in zip("qkv", rows, (a.heads, a.kv_heads, a.kv_heads)):
            st, shape = tuple(getattr(a, n + "_stride")), (a.batch, S, H, a.head_size)
            self.read[n] = self.view(getattr(a, n), dtype, shape, (*st, 1)).flatten(2)
            self.aligned &= getattr(a, n) % 16 == 0 and all(s * dtype.itemsize % 16 == 0 for s in st)
        if getattr(a, "positions", None):
            self.read["positions"] = self.view(a.positions, torch.int64, (a.batch, a.len), tuple(a.position_stride))
        for n, elements in (("lse", 2 * a.batch * a.heads * rows[0]), ("out", a.batch * rows[0] * a.heads * a.head_size)):
            if getattr(a, n, None):
                self.aligned &= getattr(a, n) % 16 == 0
                self.read[n] = self.view(getattr(a, n), torch.float32 if n == "lse" else dtype, (elements,), (1,))

    def view(self, address, dtype, shape, strides):
        last = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
        raw = (ctypes.c_char * (last * dtype.itemsize)).from_address(address)
        return torch.frombuffer(raw, dtype=dtype).as_strided(shape, strides).clone()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_reads_what_it_is_given(monkeypatch, dtype, layout):
    from nonauto_lm_amd import ops
    lib = Reader(monkeypatch)
    B, S, H, G, d = 2, 77, 4, 2, 32
    x, q, k, v = packed(B, S, H, G, d, dtype, "cpu")
    where = torch.arange(2 * S).expand(B, 2 * S)[:, ::2]
    with Hooks(LAYOUTS[layout]):
        out = ops.biased_attention(q, k, v, H, G, mask=torch.ones(B, S, dtype=torch.int64))
        forward = lib.read
        rq, rk = ops.qk_norm_rotary(q, k, H, G, frequencies=ops.rotary_frequencies(d), positions=where)
    assert all(torch.equal(forward[n], t) for n, t in (("q", q), ("k", k), ("v", v)))
    torch.autograd.grad(out, x, torch.zeros_like(out))
    assert lib.aligned and all(torch.equal(lib.read[n], t) for n, t in (("q", q), ("k", k), ("v", v)))
    assert all(torch.equal(lib.read[n].view(torch.int32), forward[n].view(torch.int32)) for n in ("lse", "out"))     # (whatever it holds)
    torch.autograd.grad((rq, rk), x, (torch.zeros_like(rq), torch.zeros_like(rk)))
    assert lib.aligned and all(torch.equal(lib.read[n], t) for n, t in (("q", q), ("k", k), ("positions", where)))


def test_a_hook_that_returns_something_else_is_refused(monkeypatch):
    from nonauto_lm_amd import ops
    Recorder(monkeypatch)
    x, q, k, v = packed(2, 20, 2, 2, 32, torch.float32, "cpu")
    for other in (lambda t: t.double() if t.is_floating_point() else t, lambda t: t[..., :-1], lambda t: t.to("meta"),
                  lambda t: t.transpose(0, 1) if t.dim() == 3 else t):
        with Hooks(other):
            out = ops.biased_attention(q, k, v, 2)
            rq, rk = ops.qk_norm_rotary(q, k, 2, frequencies=ops.rotary_frequencies(32))
        with pytest.raises(RuntimeError, match="biased_attention: a saved-tensor hook"):
            torch.autograd.grad(out, x, torch.zeros_like(out))
        with pytest.raises(RuntimeError, match="qk_norm_rotary: a saved-tensor hook"):
            torch.autograd.grad((rq, rk), x, (torch.zeros_like(rq), torch.zeros_like(rk)))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["packed", "heads first"])
def test_saved_on_the_host(layout, dtype):
    """gradients are those without the hooks, bit for bit"""
    from nonauto_lm_amd import ops
    B, S, H, G, d = 2, 77, 4, 2, 32
    g = torch.Generator(device="cuda").manual_seed(1)
    w = (1 + 0.2 * torch.randn(d, device="cuda", generator=g)).requires_grad_(True)
    table = (0.5 * torch.randn(8, H, device="cuda", generator=g)).requires_grad_(True)
    buckets = ops.relative_buckets(8, 24, True, device="cuda")
    mask = (torch.arange(S, device="cuda")[None] < torch.tensor([[S], [40]], device="cuda")).long()
    freqs = ops.rotary_frequencies(d, device="cuda")
    where = torch.arange(2 * S, device="cuda").expand(B, 2 * S)[:, ::2]
    if layout == "packed":
        x, q, k, v = packed(B, S, H, G, d, dtype, "cuda")
        leaves = [x]
    else:
        leaves = [torch.randn(B, h, S, d, device="cuda", generator=g).to(dtype).requires_grad_(True) for h in (H, G, G)]
        q, k, v = (t.transpose(1, 2) for t in leaves)
    results = []
    for how in (contextlib.nullcontext(), torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
                Hooks(shifted)):
        with how:
            plain = ops.biased_attention(q, k, v, H, G, mask=mask, causal=True, softcap=20.0)
            rq, rk = ops.qk_norm_rotary(q, k, H, G, q_weight=w, k_weight=w, frequencies=freqs, positions=where)
            out = ops.biased_attention(rq, rk, v, H, G, mask=mask, table=table, buckets=buckets)
        do = torch.sin(torch.arange(out.numel(), device="cuda").float()).view(out.shape).to(dtype)
        results.append([*torch.autograd.grad(plain, leaves, do), *torch.autograd.grad(out, leaves + [w, table], do)])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))
