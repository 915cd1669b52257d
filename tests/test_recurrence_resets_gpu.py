"""A gate of minus infinity drops the state whatever it holds, wherever what is not finite came from: rows, gradients, the state
handed in, or other gates. Compared to the bit with the same call without it, on every kind of kernel: sequences of a warp alone,
tiles of 16-byte and of 4-byte copies, direct loads, single CTAs and clusters."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
KINDS = [(64, BF, BF), (64, HF, FP), (64, FP, FP), (30, BF, BF), (83, BF, BF), (83, HF, FP), (83, FP, FP)]


def make(N, D, dtype, gate, heads=2, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    shape = (1, heads, N, D)
    g = -torch.rand(shape, device=DEV, generator=gen)
    return randn(*shape).to(dtype), g.to(gate), randn(1, heads, D), randn(*shape).to(dtype), randn(1, heads, D)


def run(x, g, s, dy, ds):
    from flashy_linear_attention_b200 import GatedLinearRecurrence

    leaves = [t.detach().requires_grad_(True) for t in (x, g, s)]
    out, s_final = GatedLinearRecurrence.apply(*leaves)
    grads = torch.autograd.grad((out, s_final), leaves, (dy, ds))
    return dict(zip(("out", "s_final", "dx", "dg", "ds"), (out.detach(), s_final.detach(), *grads)))


def same(got, want, what):
    assert torch.equal(got, want), f"{what}: {(got != want).sum().item()} of {want.numel()} differ, {got.isnan().sum().item()} NaN"


def after(got, want, at, what):
    """Token `at` is a reset and what is not finite stands before it."""
    for name in ("out", "dx", "dg"):
        same(got[name][:, :, at:], want[name][:, :, at:], f"{what}: {name} from the reset on")
    same(got["s_final"], want["s_final"], f"{what}: s_final")


def before(got, want, at, what):
    """Token `at` is a reset and what is not finite stands at it or behind."""
    for name in ("out", "dx"):
        same(got[name][:, :, :at], want[name][:, :, :at], f"{what}: {name} before the reset")
    same(got["dg"][:, :, :at + 1], want["dg"][:, :, :at + 1], f"{what}: dg up to the reset")
    same(got["ds"], want["ds"], f"{what}: ds")


def others(got, want, channel, what):
    """Channels that nothing happened to."""
    for name in got:
        rest = [c for c in range(want[name].shape[-1]) if c != channel]
        same(got[name][..., rest], want[name][..., rest], f"{what}: {name} of other channels")


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("N,resets", [(20, (1, 9, 19)), (400, (7, 100, 399)), (5000, (513, 2503))])
def test_no_gate_reaches_past_a_reset(kind, N, resets):
    for at in resets:
        x, g, s, dy, ds = make(N, *kind, seed=at)
        g[:, :, at] = -math.inf
        clean = run(x, g, s, dy, ds)
        for poison in (math.nan, math.inf):
            for away in (1, 2, 5, 40, 300):  # in the same run, in others of a CTA, in another CTA
                for at_gate in (at - away, at + away):
                    if not 0 <= at_gate < N:
                        continue
                    what = f"gate {at_gate} {poison}, reset {at}"
                    bad = g.clone()
                    bad[:, :, at_gate] = poison
                    got = run(x, bad, s, dy, ds)
                    (after if at_gate < at else before)(got, clean, at, what)
                    bad = g.clone()
                    bad[..., at_gate, 3] = poison
                    others(run(x, bad, s, dy, ds), clean, 3, what)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("N,resets", [(20, (1, 9, 19)), (400, (7, 100, 399)), (5000, (513, 2503))])
def test_nothing_passes_a_reset_in_any_kernel(kind, N, resets):
    for at in resets:
        x, g, s, dy, ds = make(N, *kind, seed=at)
        g[:, :, at] = -math.inf
        clean = run(x, g, s, dy, ds)
        for poison in (math.nan, math.inf, -math.inf):
            bad = x.clone()
            bad[:, :, at - 1] = poison
            after(run(bad, g, s, dy, ds), clean, at, f"x {poison}")
            bad = dy.clone()
            bad[:, :, at] = poison
            before(run(x, g, s, bad, ds), clean, at, f"dy {poison}")
            after(run(x, g, torch.full_like(s, poison), dy, ds), clean, at, f"s {poison}")
            before(run(x, g, s, dy, torch.full_like(ds, poison)), clean, at, f"ds {poison}")
            bad = x.clone()
            bad[..., at - 1, 3] = poison
            others(run(bad, g, s, dy, ds), clean, 3, f"x {poison}")


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("N", [20, 400, 5000])
def test_a_gate_that_is_no_number_without_a_reset(kind, N):
    """It spoils the tokens from it on, and backward those before it."""
    x, g, s, dy, ds = make(N, *kind)
    clean = run(x, g, s, dy, ds)
    p = N // 2 + 1
    bad = g.clone()
    bad[:, :, p] = math.nan
    got = run(x, bad, s, dy, ds)
    same(got["out"][:, :, :p], clean["out"][:, :, :p], "out before")
    same(got["dx"][:, :, p:], clean["dx"][:, :, p:], "dx behind")
    for t in (got["out"][:, :, p:], got["s_final"], got["dx"][:, :, :p], got["dg"], got["ds"]):
        assert t.isnan().all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("N", [20, 400, 5000])
def test_no_bit_of_a_channel_depends_on_another(kind, N):
    """Runs with unusual gates are walked another way, and a warp does so for all of its channels."""
    x, g, s, dy, ds = make(N, *kind, seed=1)
    clean = run(x, g, s, dy, ds)
    for value in (-math.inf, math.nan, math.inf):
        for at in (0, N // 2, N // 2 + 1, N - 1):
            other = g.clone()
            other[..., at, 3] = value
            others(run(x, other, s, dy, ds), clean, 3, f"gate {at} {value}")
            spoiled, up = x.clone(), dy.clone()
            spoiled[..., at, 3], up[..., at, 3] = value, value
            others(run(spoiled, other, s, up, ds), clean, 3, f"row and gate {at} {value}")


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("drop", [-1e4, "lowest"])
def test_a_gate_whose_decay_underflows_leaves_nothing_of_the_largest_state(kind, drop):
    """Rows of their type's lowest value, as in masked places, before a gate so low that its decay is zero: also where the gate is the
    only low one of its run and the state comes from the run before."""
    N, D, dtype, gate = 400, *kind
    for at in (17, 48, 208, 256):
        x, g, s, dy, ds = make(N, D, dtype, gate)
        g[:, :, at] = torch.finfo(gate).min if drop == "lowest" else drop
        x[:, :, at - 1] = 0
        clean = run(x, g, s, dy, ds)
        x[:, :, at - 1] = torch.finfo(dtype).min
        got = run(x, g, s, dy, ds)
        same(got["out"][:, :, at:], clean["out"][:, :, at:], "out")
        same(got["s_final"], clean["s_final"], "s_final")
        x[:, :, at - 1] = 0
        dy[:, :, at] = 0
        clean = run(x, g, s, dy, ds)
        dy[:, :, at] = torch.finfo(dtype).min
        got = run(x, g, s, dy, ds)
        same(got["dx"][:, :, :at], clean["dx"][:, :, :at], "dx")
        same(got["ds"], clean["ds"], "ds")
