"""The Functions inside torch.compile: what they do is opaque to it, the code around them is traced, and results are those of
the same code uncompiled, through the native autograd nodes and through the Python Functions."""
import warnings

import pytest
import torch

from test_block_gpu import DEV, block, functions, inputs, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["native", "python"])
def native(request, monkeypatch):
    from flashy_linear_attention_b200 import _lib

    if not request.param:
        monkeypatch.setattr(_lib, "host", lambda: None)
    torch._dynamo.reset()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # (that a call ends a traced piece)
        yield request.param
    torch._dynamo.reset()


def single():
    """(call, leaves) of each Function, with what the native nodes cover and what they leave to Python."""
    fla = functions()
    gen = torch.Generator(device=DEV).manual_seed(5)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    x, z, g = randn(2, 3, 50, 64), randn(2, 3, 50, 64), -torch.rand(2, 3, 50, 64, device=DEV, generator=gen)
    s, w, b = randn(2, 3, 64), randn(64), randn(64)
    shared = -torch.rand(2, 3, 50, 1, device=DEV, generator=gen)
    wide = randn(2, 2, 3, 4, 64)
    return {
        "recurrence": (lambda x, g, s: fla.GatedLinearRecurrence.apply(x * 2, g, s), (x, g, s)),
        "recurrence, no state": (lambda x, g: fla.GatedLinearRecurrence.apply(x * 2, g), (x, g)),
        "recurrence, a gate of all channels": (lambda x, g, s: fla.GatedLinearRecurrence.apply(x * 2, g.expand(2, 3, 50, 64), s), (x, shared, s)),
        "norm": (lambda x, w, b: (fla.LayerNorm.apply(x * 2, w, b),), (x, w, b)),
        "norm, five dims": (lambda x, w, b: (fla.LayerNorm.apply(x * 2, w, b, 1e-3),), (wide, w, b)),
        "add_norm": (lambda x, z, w, b: fla.AddLayerNorm.apply(x * 2, z, w, b), (x, z, w, b)),
        "add_norm, five dims": (lambda x, w, b: fla.AddLayerNorm.apply(x * 2, x, w, b), (wide, w, b)),
    }


def step(call, leaves):
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    outs = call(*leaves)
    ups = [torch.linspace(-1, 1, o.numel(), device=o.device).view_as(o).to(o.dtype) for o in outs]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, ups))


def attention():
    fla = functions()
    gen = torch.Generator(device=DEV).manual_seed(6)
    rand = lambda *s: torch.rand(*s, device=DEV, generator=gen).to(torch.bfloat16)  # noqa: E731
    t = [rand(2, 3, 128, 64) for _ in range(3)]
    odd = [rand(2, 3, 128, d) for d in (45, 45, 64)]
    wide = [rand(2, 3, 128, d) for d in (273, 273, 16)]
    raw = [rand(2, 3, 128, d) for d in (16, 16, 64)]
    turned = [a.transpose(2, 3).contiguous().transpose(2, 3) for a in t]
    return {
        "attention": (lambda q, k, v: (fla.LinearAttention.apply(q * 2, k, v),), t),
        "attention, columns apart": (lambda q, k, v: (fla.LinearAttention.apply(q * 2, k, v),), turned),
        "attention, odd widths": (lambda q, k, v: (fla.LinearAttention.apply(q * 2, k, v),), odd),
        "attention, wide": (lambda q, k, v: (fla.LinearAttentionSmallVHD.apply(q * 2, k, v),), wide),
        "attention, a state": (lambda q, k, v: fla.LinearAttentionResumable.apply(q * 2, k, v, None), t),
        "attention, normalised": (lambda q, k, v: (fla.LinearAttentionNormalized.apply(q * 2, k, v),), t),
        "attention, normalised, odd widths": (lambda q, k, v: (fla.LinearAttentionNormalized.apply(q * 2, k, v),), odd),
        "attention, Taylor": (lambda q, k, v: (fla.TaylorLinearAttention.apply(q * 2, k, v),), raw),
    }


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_single_functions(native, backend):
    for name, (call, leaves) in {**single(), **attention()}.items():
        torch._dynamo.reset()
        compiled = torch.compile(call, backend=backend)
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(step(compiled, leaves), step(call, leaves))), name
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(compiled(*leaves), call(*leaves))), name


def test_a_block(native):
    tensors = inputs(70)
    w = {name: t.to(torch.bfloat16) for name, t in weights().items()}
    names = list(w)

    def call(branch, residual, *ws):
        return block(dict(zip(names, ws)), branch, residual)[:2]

    leaves = (*tensors[:2], *w.values())
    compiled = torch.compile(call, backend="eager")
    assert all(torch.equal(a, b) for a, b in zip(step(compiled, leaves), step(call, leaves)))


def test_refusals(native):
    fla = functions()
    x = torch.randn(2, 3, 50, 64, device=DEV)
    for call, error in ((lambda t: fla.LayerNorm.apply(t, t[0, 0, 0, :7]), ValueError), (lambda t: fla.LayerNorm.apply(t.double()), TypeError),
                        (lambda t: fla.AddLayerNorm.apply(t, t[..., :8]), ValueError), (lambda t: fla.GatedLinearRecurrence.apply(t, t[:1]), ValueError)):
        with pytest.raises(error, match="flashlinear"):
            call(x)
        with pytest.raises(error, match="flashlinear"):
            torch.compile(call, backend="eager")(x)


def test_what_a_call_makes_lives_until_the_library_has_it(native, monkeypatch):
    """Such as a gate that is written out for all channels. Traced, a tensor is released when its address has been taken; allocations
    before the launch, which this fills with NaN, then get its memory."""
    from flashy_linear_attention_b200 import layer_norm, ops, recurrence

    def spoiling(call):
        def wrapper(*args, **kwargs):
            spoil = [torch.full((2 * 3 * 128 * 64 // part,), torch.nan, device=DEV) for part in (1, 2, 4, 8) for _ in range(4)]
            del spoil
            return call(*args, **kwargs)

        return wrapper

    for module in (layer_norm, ops, recurrence):
        monkeypatch.setattr(module, "_call", spoiling(module._call))
    fla = functions()
    w, b = torch.randn(64, device=DEV), torch.randn(64, device=DEV)
    apart = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    made = {
        "recurrence": lambda t: fla.GatedLinearRecurrence.apply(t * 2, (-t.abs())[..., :1].expand_as(t))[0],
        "recurrence, columns apart": lambda t: fla.GatedLinearRecurrence.apply(apart(t), -t.abs(), t[:, :, 0].half())[0],
        "norm": lambda t: fla.LayerNorm.apply(apart(t), w.repeat(2)[::2], b),
        "add_norm": lambda t: fla.AddLayerNorm.apply(t, apart(t), w, b.repeat(2)[::2])[0],
        "attention": lambda t: fla.LinearAttention.apply(*(apart(a) for a in (t.bfloat16(), t.bfloat16().abs(), t.bfloat16()))),
    }
    for name, call in made.items():
        torch._dynamo.reset()
        compiled = torch.compile(call, backend="eager")
        for n in (128, 64):
            x = torch.randn(2, 3, n, 64, device=DEV)
            grads = []
            for f in (call, compiled):
                leaf = x.clone().requires_grad_(True)
                out = f(leaf)
                out.float().sum().backward()
                grads.append((out.detach(), leaf.grad))
            assert all(torch.equal(a, b) for a, b in zip(*grads)), (name, n)


@pytest.mark.parametrize("dynamic", [None, True])
def test_calls_of_many_lengths(native, dynamic):
    """More of them than are compiled for."""
    fla = functions()
    w, b = torch.randn(64, device=DEV), torch.randn(64, device=DEV)
    made = {
        "recurrence": lambda t: fla.GatedLinearRecurrence.apply(t * 2, (-t.abs())[..., :1].expand_as(t))[0],
        "norm": lambda t: fla.LayerNorm.apply(t * 2, w, b),
    }
    for name, call in made.items():
        torch._dynamo.reset()
        compiled = torch.compile(call, backend="eager", dynamic=dynamic)
        for n in range(1, 300, 23):
            x = torch.randn(2, 3, n, 64, device=DEV)
            grads = []
            for f in (compiled, call):
                leaf = x.clone().requires_grad_(True)
                out = f(leaf)
                out.sum().backward()
                grads.append((out.detach(), leaf.grad))
            assert all(torch.equal(a, b) for a, b in zip(*grads)), (name, n)
