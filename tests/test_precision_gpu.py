"""fp32 results of the gated linear recurrence and of the layer norms, held to fp32. u = 2^-24, half a step, is what one rounding costs.

Recurrence, fp32 rows, against `scale`, the same sums with absolute values. A run has 8 tokens: a step costs a rounding (u) and the
decay's error (expf, two units in the last place: 4 u), so a run 40 u at most. The state before a run comes through one map a run.
Its factor is off by 3 u where it is near 1 (two floats, roundings of the sum of gates), and that over at most 38 runs of 304 tokens:
133 u with the rounding of each; further from 1, with s the sum of its gates, by (6 + 9 s) u, which the next runs' decays bound by
53 u together. A cluster joins its CTAs by up to 8 more: 30 u. 40 + 133 + 40 + 30 < 256 u = 2^-16 if all pointed the same way. On
average over a tensor they do not: each rounding u / sqrt(3), a run's (1 + 4) of them a token, 8 (4 u)^2 far from 1 or 38 near it:
sqrt(13 + 43 + 13) u < 10 u; 2^-20 = 16 u leaves room for a bias of expf. The gradient of a gate is a product of two such sums, whose scale
counts twice.

16-bit rows sum in 32 bits too, with the fast exponential inside a run of 16 tokens (2^-22 = 4 u, and its argument's product): 90 u^2 of
variance if it had no bias, 16 (4 u) if it were all bias; 2^-18 = 64 u.

Layer norm, up to 1024 columns: a sum over a row has 7 additions in a thread, 1, 5 shuffles and 4 warps: 17 u at most, sqrt(17 / 3) u =
2.4 u on average. n = (x - m) r takes half of that again for the variance, 2.5 u for the root and 3 roundings: 35 u at most, 3.4 u on
average; dx two more sums of such products: 104 u at most, and its average 3 times that of n. 2^-17 = 128 u for all, and on average
2^-21 = 8 u for y, 2^-20 = 16 u for gradients. `size` is that of test_layer_norm_gpu.py."""
import math

import pytest
import torch

import test_layer_norm_gpu as ln
import test_recurrence_gpu as rec

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24


def errors(got, want):
    """Largest and root mean square error, relative to the size of what was summed."""
    value, size = want
    off = (got.double() - value).abs() / size.clamp_min(1e-30)
    return off.max().item(), off.square().mean().sqrt().item()


@pytest.mark.parametrize("N", [9, 31, 40, 129, 304])
@pytest.mark.parametrize("D", [64, 83, 130])
def test_recurrence_of_fp32_rows(N, D):
    for heads, rate in ((2, (1e-3, 2.0)), (2, (1e-4, 1e-2)), (200, (1e-3, 2.0))):
        t = rec.make(1, heads, N, D, FP, seed=N, rate=rate)
        got, want = rec.run(*t), rec.reference(*t)
        for name, value in got.items():
            most, mean = errors(value, want[name])
            # (each result is rounded once itself: u of it, inside what is left)
            assert most <= 256 * U and mean <= 16 * U, (name, heads, rate, most / U, mean / U)


@pytest.mark.parametrize("kind", [(64, BF, BF), (64, HF, FP), (30, BF, BF), (83, BF, BF), (83, HF, FP)], ids=str)
def test_fp32_results_of_16_bit_rows(kind):
    D, dtype, gate = kind
    for N in (20, 40, 304):
        t = rec.make(1, 2, N, D, dtype, gate, seed=N)
        got, want = rec.run(*t), rec.reference(*t)
        for name in ("s_final", "ds") + (("dg",) if gate == FP else ()):
            assert got[name].dtype == FP
            assert errors(got[name], want[name])[1] <= 64 * U, (name, N)


@pytest.mark.parametrize("kind", [(8, FP, FP), (83, FP, FP), (64, BF, FP), (83, BF, BF), (83, HF, HF)], ids=str)
def test_long_memories_forward_and_backward(kind):
    """Constant rows and gates: h = (1 - a^t) / (1 - a), and the same from the end for G; 1250 runs of memory with roundings that have no
    direction stay below 2^-20, the fast exponential in a run of 16 (with 7.5 decays a token on average, off by 2^-22) below 2^-19."""
    D, dtype, gate = kind
    N = 16384
    for rate in (1.03e-4, 0.97e-4, 2.9e-5):
        x = torch.ones(1, 1, N, D, device=DEV, dtype=dtype)
        g = torch.full((1, 1, N, D), -rate, device=DEV, dtype=gate)
        zero = torch.zeros(1, 1, D, device=DEV)
        got = rec.run(x, g, zero, x, zero)
        a = math.exp(g[0, 0, 0, 0].item())
        t = torch.arange(1, N + 1, device=DEV, dtype=torch.float64)
        sums = (1 - a**t) / (1 - a)
        for name, want in (("out", sums), ("dx", sums.flip(0))):
            if dtype == FP:
                off = (got[name][0, 0].double() - want[:, None]).abs() / want[:, None]
                assert off.max() < 2.0**-18, (name, rate)
        for name, want in (("s_final", sums[-1]), ("ds", a * sums[-1])):
            assert ((got[name].double() - want).abs() / want).max() < 2.0**-18, (name, rate)


@pytest.mark.parametrize("dtype", [FP, BF])
def test_a_state_through_thousands_of_calls(dtype):
    """One token a call: two roundings each, 4000 of them without a direction, sqrt(8000 / 3) u < 2^-18.3; bound twice that. A decay held in
    one float would be off by up to 2.8e-8 a token, always the same way: 2^-14.2 to 2^-14.8 for these."""
    N = 4000
    for rate in (0.97e-4, 2.9e-5, 1.37e-4):
        x = torch.ones(1, 2, 1, 64, device=DEV, dtype=dtype)
        g = torch.full((1, 2, 1, 64), -rate, device=DEV)
        state = None
        with torch.no_grad():
            for _ in range(N):
                _, state = rec.recurrence().apply(x, g, state)
        a = math.exp(g[0, 0, 0, 0].item())
        want = (1 - a**N) / (1 - a)
        assert ((state.double() - want).abs() / want).max() < 2.0**-17, rate


@pytest.mark.parametrize("D", [8, 40, 83, 128, 512, 1000, 1023, 1024])
def test_layer_norm_of_fp32_rows(D):
    for rows in (7, 700):
        x, z, w, b, dy, ds = ln.make((rows, D), FP, seed=D)
        for add in (False, True):
            got = ln.run(x, z if add else None, w, b, dy, ds)
            want = ln.reference(got["sum"] if add else x, w, b, 1e-5, dy, ds if add else None)
            for name, value in want.items():
                most, mean = errors(got[name], value)
                assert most <= 128 * U and mean <= (8 if name == "y" else 16) * U, (name, rows, add, most / U, mean / U)
