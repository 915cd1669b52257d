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


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_single_functions(native, backend):
    for name, (call, leaves) in single().items():
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
