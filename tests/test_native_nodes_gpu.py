"""The native autograd nodes against the Python Functions on what calls seldom bring: gradients with a lazy sign, weights of no
dimension."""
import pytest
import torch

from test_block_gpu import DEV, calls, functions

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["native", "python"])
def native(request, monkeypatch):
    from flashy_linear_attention_b200 import _lib

    if not request.param:
        monkeypatch.setattr(_lib, "host", lambda: None)


def test_gradients_with_a_lazy_sign(native):
    """As the imaginary part of a conjugate has: the bits in memory are those of the opposite number."""
    for name, call, inputs in calls():
        for layout in (lambda t: t, lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)):
            leaves = [t.detach().requires_grad_(True) for t in inputs]
            outs = call(*leaves)
            ups = [layout(torch.randn_like(o)) for o in outs]
            lazy = [torch._neg_view(-u) for u in ups]
            assert all(t.is_neg() for t in lazy)
            got = torch.autograd.grad(outs, leaves, lazy, retain_graph=True)
            want = torch.autograd.grad(outs, leaves, ups)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_inputs_with_a_lazy_sign(native):
    for name, call, inputs in calls():
        want = call(*inputs)
        got = call(*(torch._neg_view(-t) for t in inputs))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_weights_of_no_dimension_are_refused_like_any_of_a_wrong_shape(native):
    fla = functions()
    x, one = torch.randn(5, 8, device=DEV), torch.ones((), device=DEV)
    for w, b in ((one, None), (None, one), (torch.ones(8, device=DEV), one)):
        with pytest.raises(ValueError, match="must have shape"):
            fla.LayerNorm.apply(x, w, b)
        with pytest.raises(ValueError, match="must have shape"):
            fla.AddLayerNorm.apply(x, x, w, b)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.bool])
def test_autocast_makes_no_call_right_that_is_refused_without_it(native, dtype):
    fla = functions()
    x, g = torch.ones(1, 2, 5, 8, device=DEV), torch.zeros(1, 2, 5, 8, device=DEV)
    for autocast in (False, True):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            for args in ((x.to(dtype), g), (x, g.to(dtype))):
                with pytest.raises(TypeError, match="flashlinear"):
                    fla.GatedLinearRecurrence.apply(*args)
            with pytest.raises(TypeError, match="flashlinear"):
                fla.LayerNorm.apply(x.to(dtype))
