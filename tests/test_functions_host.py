"""The Functions beside an attention without a GPU: what they refuse, also inside torch.compile."""
import warnings

import pytest
import torch

from test_recurrence_host import fake


def calls():
    from flashy_linear_attention_b200 import AddLayerNorm, GatedLinearRecurrence, LayerNorm

    return [lambda t: LayerNorm.apply(t), lambda t: LayerNorm.apply(t, t[0, 0, 0], None, 1e-3), lambda t: AddLayerNorm.apply(t, t),
            lambda t: GatedLinearRecurrence.apply(t, t), lambda t: GatedLinearRecurrence.apply(t, t, t[:, :, 0])]


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("grad", [False, True])
def test_a_compiled_call_is_refused_like_any_other(which, grad):
    call, x = calls()[which], torch.zeros(1, 1, 4, 8, requires_grad=grad)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call(x)
    torch._dynamo.reset()
    with warnings.catch_warnings(), pytest.raises(RuntimeError, match="no CPU fallback"):
        warnings.simplefilter("ignore")
        torch.compile(call, backend="eager")(x)
    torch._dynamo.reset()


def test_a_residual_that_is_not_there_is_refused():
    from flashy_linear_attention_b200 import AddLayerNorm

    for x in (torch.zeros(4, 8), fake(4, 8), fake(4, 8).requires_grad_(True)):
        with pytest.raises(ValueError, match="residual"):
            AddLayerNorm.apply(x, None)
        with pytest.raises(ValueError, match="residual"):
            AddLayerNorm.apply(x, None, fake(8), fake(8), 1e-3)


def test_sizes_past_the_recurrence_are_refused():
    """Sizes of 2^32 and more would otherwise lose their upper bits on the way to the library."""
    from flashy_linear_attention_b200 import recurrence

    for shape in ((1, 1, 2**30, 1), (1, 1, 1, 2**30), (2**15, 2**15, 1, 1)):
        t = fake(1).expand(shape)
        recurrence.check_inputs(t, t)
    for shape in ((1, 1, 2**30 + 1, 1), (1, 1, 2**32 + 5, 1), (1, 1, 1, 2**32 + 5), (2**32 + 5, 1, 1, 1), (1, 2**30 + 1, 1, 1), (2**16, 2**16, 1, 1)):
        t = fake(1).expand(shape)
        with pytest.raises(ValueError, match="2.30"):
            recurrence.check_inputs(t, t)
    empty = fake(0).reshape(2**32, 0, 1, 1)
    recurrence.check_inputs(empty, empty)


def test_what_a_forward_kept_is_checked_before_its_address_is_used(monkeypatch):
    """It may come back from a hook of autograd's: from the host, shortened, of another type."""
    from flashy_linear_attention_b200 import _lib, layer_norm, recurrence

    monkeypatch.setattr(_lib, "host", lambda: None)
    x = fake(2, 3, 40, 8)
    for states in (None, torch.zeros(4096, dtype=torch.uint8), fake(4096, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="states"):
            recurrence.recurrence_bwd(x, x, x, states)
    rows = fake(5, 8)
    for stats in (torch.zeros(5, 2), fake(4, 2), fake(5, 2, dtype=torch.float64), fake(2, 5).t()):
        with pytest.raises(ValueError, match="statistics"):
            layer_norm.layer_norm_bwd(rows, rows, None, None, stats)
